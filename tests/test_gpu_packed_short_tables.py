"""Contexts longer than their block table: a row keeps its position and sees the keys that the table reaches."""
import pytest
import torch

import test_gpu_attention_packed as attn
from g4b_b200.kernels import fa2

pytestmark = pytest.mark.gpu


def seen_rows(c, b, reach, window, stage):
    """(row, visible keys) pairs of slot b by the definition."""
    r, t = c["rows"][b], int(c["times"][b])
    for i in range(r):
        pos = t - r + i
        yield i, [j for j in range(min(t, reach)) if (stage == fa2.STAGE_FULL or j <= pos) and (not window or j > pos - window)]


@pytest.mark.parametrize("beyond", [1, 10, 30, 64, 1000, 2 ** 30, 2 ** 31 - 1])
@pytest.mark.parametrize("window,stage", [(0, fa2.STAGE_CAUSAL), (40, fa2.STAGE_CAUSAL), (700, fa2.STAGE_CAUSAL), (0, fa2.STAGE_FULL)])
def test_positions_stay(cuda, beyond, window, stage):
    rows, reach = [60, 200, 5], [160, 608, 2064]
    c = attn.make(3, rows, reach, H=2, G=1, D=128)          # (full pages, so the tables reach exactly this far)
    width = c["table"].shape[1]
    for b in (0, 2):                                        # slot 1 stays as it is; the table's width bounds the others
        c["times"][b] = min(width * 16 + beyond, 2 ** 31 - 1)
    ids = c["table"][2].clone()
    c["table"][0] = ids                                     # (as wide as slot 2's, whose pages are all there)
    q, k, v = c["q"].double().cpu(), c["k"].double().cpu(), c["v"].double().cpu()
    attn.run(c, sliding_window=window, stage=stage)
    assert torch.isfinite(c["o"][:265].float()).all()
    o, table = c["o"].double().cpu(), c["table"].cpu().long()
    u = 2.0 ** -8
    for b, first in ((0, 0), (1, 60), (2, 260)):
        for i, keys in seen_rows(c, b, width * 16, window, stage):
            if i % 13 and i != c["rows"][b] - 1:
                continue
            for h in range(2):
                got = o[first + i, h]
                if not keys:
                    assert bool((got == 0).all())
                    continue
                j = torch.tensor(keys)
                kk, vv = k[table[b, j // 16], 0, j % 16], v[table[b, j // 16], 0, j % 16]
                w = torch.softmax(kk @ q[first + i, h] * c["scale"], 0)
                # weights rounded once to 8 bits, numerator and sum; a score off by 2 D 2^-24 scale |q| |k|, counted twice
                # (|q|, |k| < 16: 512 x 2^-24 x 256 / sqrt(128) < 2^-10); the output rounded once more
                allowed = (2 * u + 2.0 ** -10) * (w @ vv.abs()) + u * (w @ vv).abs()
                assert bool(((got - w @ vv).abs() <= allowed).all()), f"slot {b} row {i} head {h}"
