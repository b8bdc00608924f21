"""Random steps through the packed operators: any mix of prompts, chunks, single tokens, idle slots, head counts, page sizes,
windows and types, each against the formulas in 64 bits (bounds and builders of the operators' own tests)."""
import random

import pytest
import torch

import test_gpu_attention_packed as attn
import test_gpu_rope_packed as rp
from g4b_b200.kernels import fa2

pytestmark = pytest.mark.gpu


def some_rows(rng, most):
    n = rng.choice([1, 2, 3, 5, 9, 17, 40])
    pick = lambda: rng.choice([0, 1, 1, 2, rng.randint(1, 20), rng.randint(1, 130), rng.randint(1, most)])  # noqa: E731
    rows = [pick() for _ in range(n)]
    times = [r + rng.choice([0, 0, 0, rng.randint(0, 40), rng.randint(0, 1500)]) for r in rows]
    if rng.random() < 0.2:                       # rows without a place, contexts without rows
        times[rng.randrange(n)] = rng.randint(0, 50)
    return rows, times


@pytest.mark.parametrize("seed", range(40))
def test_attention(cuda, seed):
    rng = random.Random(seed)
    rows, times = some_rows(rng, 700)
    if seed % 4 == 0:
        times[0] = rows[0] + rng.randint(2000, 12000)
    G = rng.choice([1, 2, 3])
    H = G * rng.choice([1, 2, 3, 4, 5, 8, 16])
    dtype = rng.choice([torch.bfloat16, torch.float16])
    c = attn.make(1000 + seed, rows, times, H=H, G=G, D=rng.choice([128, 256]), page=rng.choice([16, 16, 32, 64, 256]), dtype=dtype,
                  out=rng.choice([None, None, torch.float32]), spare=rng.randint(0, 70), amp=rng.choice([0.01, 1.0, 1.0, 8.0]))
    window = rng.choice([0, 0, rng.randint(1, 100), rng.randint(100, 2000)])
    attn.both(c, sliding_window=window, stage=rng.choice([fa2.STAGE_CAUSAL, fa2.STAGE_CAUSAL, fa2.STAGE_FULL]))


@pytest.mark.parametrize("seed", range(30))
def test_rope(cuda, seed):
    rng = random.Random(seed)
    rows, times = some_rows(rng, 900)
    times = [max(r, t) for r, t in zip(rows, times)]
    G = rng.choice([1, 2, 5])
    c = rp.make(2000 + seed, rows, times, H=G * rng.choice([1, 3, 4]), G=G, D=rng.choice([16, 64, 96, 128, 256, 512]),
                page=rng.choice([1, 2, 16, 128]), axes=rng.choice([1, 2, 3, 7]), dtype=rng.choice([torch.float32, torch.bfloat16, torch.float16]),
                cache=rng.choice([torch.float32, torch.bfloat16, torch.float16]), spare=rng.randint(0, 9), max_pos=rng.choice([10, 4000, 10 ** 6]))
    rp.both(c, **rng.choice([{}, {}, dict(weights=False), dict(norm_v=False), dict(positions=False)]))
