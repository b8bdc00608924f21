"""Packed calls that the documentation allows and that no other test makes."""
import subprocess
import sys
from pathlib import Path

import pytest
import torch

import test_gpu_attention_packed as attn
import test_gpu_rope_packed as rp
from g4b_b200 import _cabi
from g4b_b200.kernels import fa2, pages

pytestmark = pytest.mark.gpu
HERE = Path(__file__).resolve().parent

FIRST = """
import sys
sys.path[:0] = [{here!r}, {root!r}]
import torch
import test_gpu_attention_packed as attn, test_gpu_rope_packed as rp
from g4b_b200 import _cabi
from g4b_b200.kernels import pages
a = attn.make(1, [70, 1, 5], [70, 3000, 40])
r = rp.make(2, [30, 2], [30, 9], axes=3)
before = {{n: x.clone() for n, x in r.items() if isinstance(x, torch.Tensor)}}
pool = torch.randn(9, 64, device="cuda")
src, dst = attn.i32([1, 2], "cuda"), attn.i32([5, 6], "cuda")
torch.cuda.synchronize()
graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
with torch.cuda.graph(graph, stream=side):
    rp.run(r)
    attn.run(a)
    pages.copy_pages([pool], src, dst)
o = a["o"].clone()
graph.replay()
torch.cuda.synchronize()
attn.check(a, o)
rp.check(r, before)
assert torch.equal(pool[5:7], pool[1:3])
assert _cabi.device_status() == 0
print("fine")
"""


def test_the_first_calls_of_a_process_are_captured(cuda):
    code = FIRST.format(here=str(HERE), root=str(HERE.parent))
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "fine" in done.stdout, done.stderr[-2000:]


@pytest.mark.parametrize("B", [1, 40, 300])
def test_slots_without_rows(cuda, B):
    """A step in which nobody has any: rows that are there stay, tables of any width."""
    c = attn.make(3, [0] * B, [5000] + [3] * (B - 1), H=2, G=1, D=128, spare=9)
    attn.both(c)
    rp.both(rp.make(4, [0] * B, [7] * B, H=2, G=1, D=64))
    c["table"] = c["table"][:, :0]
    attn.both({**c, "t": [0] * B})


def test_a_table_without_columns(cuda):
    c = attn.make(5, [20, 3], H=2, G=1, D=128)
    c["table"] = c["table"][:, :0]
    attn.run(c)
    assert bool((c["o"][:23] == 0).all())
    r = rp.make(6, [20, 3], [20, 3], H=2, G=1, D=64)
    r["table"] = r["table"][:, :0]
    k = r["k_pool"].clone()
    rp.run(r)
    assert _cabi.device_status() == 0x101 and torch.equal(r["k_pool"], k)


def test_many_kv_heads(cuda):
    attn.both(attn.make(7, [40, 1, 200], [40, 2500, 260], H=80, G=40, D=128))
    rp.both(rp.make(8, [40, 3], [40, 90], H=80, G=40, D=128))


def test_one_token_steps_of_many_slots(cuda):
    """Only single tokens, behind contexts of every length: whole items and shares."""
    times = [1 + 37 * i for i in range(120)]
    attn.both(attn.make(9, [1] * 120, times, H=8, G=2, D=128))
    attn.both(attn.make(10, [1] * 120, times, H=4, G=1), sliding_window=300)


def test_two_captured_steps_replayed_side_by_side(cuda):
    """Workspaces of their own, two streams, one set of pools that both read."""
    cs = [attn.make(11, [300, 1], [300, 6000], H=4, G=2), attn.make(12, [17, 64, 900], [3000, 64, 900], H=4, G=2)]
    befores = [c["o"].clone() for c in cs]
    graphs, streams = [], [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for c, s in zip(cs, streams):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=s):
            attn.run(c)
        graphs.append(g)
    for _ in range(10):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for c, b in zip(cs, befores):
        attn.check(c, b)


def test_a_pool_named_twice_and_pairs_named_twice(cuda):
    pool = torch.randn(9, 3, 64, device=cuda)
    want = pool.clone()
    want[4], want[7] = pool[1], pool[2]
    pages.copy_pages([pool, pool], rp.i32([1, 2], cuda), rp.i32([4, 7], cuda))
    assert torch.equal(pool, want)
    want[5] = want[3]
    pages.copy_pages([pool], rp.i32([3, 3], cuda), rp.i32([5, 5], cuda))         # the second is one destination twice
    assert torch.equal(pool, want) and _cabi.device_status() == 0x105


def test_workspace_of_another_type_and_larger_than_needed(cuda):
    c = attn.make(13, [100, 1], [100, 4000], H=2, G=1)
    c["workspace"] = torch.full((fa2.packed_workspace_bytes(5000, 64, 2, 1) // 4 + 1,), float("nan"), device=cuda)
    attn.both(c)
