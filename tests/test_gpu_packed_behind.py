"""Packed attention calls behind one another, nothing waiting between them: each launch is set up while the one before drains,
with one workspace for all.  What a worker does is fixed by the call's lengths, and it carries nothing from call to call, so every
result has the bits of the first."""
import pytest
import torch

import test_gpu_attention_packed as attn
from g4b_b200 import _cabi

pytestmark = pytest.mark.gpu


def cases():
    return [(attn.make(40, [2500, 700, 1]), dict(sliding_window=300)), (attn.make(41, [5, 17]), {}),
            (attn.make(42, [64, 1], [9000, 4000], dtype=attn.F16), {}), (attn.make(43, [900, 333, 41], D=128, page=64), {}),
            (attn.make(44, [1, 1, 1, 30], [12000, 700, 33, 5000]), {}), (attn.make(45, [400, 1], [400, 3000], out=attn.F32), {})]


@pytest.mark.parametrize("captured", [False, True])
def test_every_call_has_the_bits_of_the_first(cuda, captured):
    cs = cases()
    workspace = torch.zeros(max(c["workspace"].numel() for c, _ in cs), dtype=torch.uint8, device=cuda)
    want = []
    for c, kw in cs:
        c["workspace"] = workspace
        attn.both(c, **kw)
        want.append(c["o"].clone())
        workspace.random_()                              # it needs no initial contents, whatever the next case finds
    order = [(i * i + i // 6) % 6 for i in range(120)]
    outs = [(k, torch.full_like(want[k], float("nan"))) for k in order]
    for k, o in outs:                                    # rows behind the last slot's are not written
        o[sum(cs[k][0]["rows"]):] = want[k][sum(cs[k][0]["rows"]):]
    torch.cuda.synchronize()

    def go():
        for k, o in outs:
            attn.run({**cs[k][0], "o": o}, **cs[k][1])

    if captured:
        graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
        with torch.cuda.graph(graph, stream=side):
            go()
        graph.replay()
    else:
        go()
    torch.cuda.synchronize()
    assert _cabi.device_status() == 0
    for n, (k, o) in enumerate(outs):
        assert torch.equal(o, want[k]), f"call {n}, case {k}: {(o != want[k]).sum().item()} elements differ"
