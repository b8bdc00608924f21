"""Packed norm + rotary (several axes) + append against the formulas in 64 bits.

Tolerance.  With u = 2^-24: a normalised element is off by at most 17 u relative (the sum of squares' at most
20 additions count half in the root, 2 ulp for rsqrtf, three products); sine and cosine by 12 u where the outputs have 16 bits
(2^-21.2 for the fast functions on [-pi, pi], and an angle off by 2^-26 turns, by the rounding of 2 pi and of the
product), by 4 u where they have 32; the two products and the sum of the rotation by 3 u: 32 u (|a| + |c|) for the
pair (a, c).  On top of it half a step of the output type."""
import math

import pytest
import torch

from g4b_b200 import _cabi
from g4b_b200.kernels import rope

EPS = 1e-6
U = 2.0 ** -24


def i32(v, device="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def make(seed, rows, times, *, H=8, G=2, D=256, page=16, axes=1, dtype=torch.float32, cache=torch.bfloat16, device="cuda", spare=5,
         max_pos=4000):
    g = torch.Generator().manual_seed(seed)
    N = sum(rows) + spare                                    # `spare` rows behind the last slot's
    need = [-(-t // page) for t in times]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(rows), max(need) if need else 1), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    rnd = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    c = dict(q=rnd(N, H, D).to(dtype), k=rnd(N, G, D).to(dtype), v=rnd(N, G, D).to(dtype),
             freqs=(10000.0 ** (-torch.arange(0, D, 2).double() / D)).float(),
             positions=torch.randint(0, max_pos, (axes, N), generator=g).int(), pair_axis=torch.randint(0, axes, (D // 2,), generator=g).to(torch.uint8),
             q_w=1 + 0.1 * rnd(D), k_w=1 + 0.1 * rnd(D), starts=i32(starts), times=i32(times), table=table,
             k_pool=rnd(pages, G, page, D).to(cache), v_pool=rnd(pages, G, page, D).to(cache), q_out=rnd(N, H, D).to(cache))
    c = {n: x.to(device) for n, x in c.items()}
    c.update(rows=rows, page=page)
    return c


def oracle(c, *, weights=True, norm_qk=True, norm_v=True, positions=True):
    """[(value, scale)] of the rotated q and k and the normalised v rows, in 64 bits, and each row's place."""
    D = c["q"].shape[-1]
    half = D // 2
    out = {}
    place = torch.full((c["q"].shape[0],), -1)
    for b, r in enumerate(c["rows"]):
        first = int(c["starts"][b])
        place[first:first + r] = int(c["times"][b]) - r + torch.arange(r)
    place = place.to(c["q"].device)
    pos = c["positions"].double()[c["pair_axis"].long()].T if positions else place.double()[:, None].expand(-1, half)
    angle = pos * c["freqs"].double()
    sin, cos = angle.sin()[:, None], angle.cos()[:, None]
    for name in "qkv":
        x = c[name].double()
        if norm_v if name == "v" else norm_qk:
            x = x / (x.square().mean(-1, keepdim=True) + EPS).sqrt()
            if weights and name != "v":
                x = x * c[name + "_w"].double()
        a, e = x[..., :half], x[..., half:]
        scale = (a.abs() + e.abs()).repeat(1, 1, 2)
        if name != "v":
            x = torch.cat([a * cos - e * sin, e * cos + a * sin], -1)
        out[name] = (x, scale)
    return out, place


def close(got, want, scale, what):
    half_step = torch.finfo(got.dtype).eps / 2
    if not got.numel():
        return
    err = (got.double() - want).abs()
    allowed = (32 * U * scale + want.abs() * half_step) * (1 + 2.0 ** -8) + 2.0 ** -25 * (got.dtype == torch.float16)
    worst = (err - allowed).max().item()
    assert worst <= 0, f"{what}: off by {err.max().item():.3e}, {worst:.3e} more than allowed"


def run(c, *, weights=True, q_out=True, positions=True, pair_axis=True, **kw):
    rope.rope_norm_append_packed(c["q"], c["k"], c["v"], c["freqs"], c["positions"] if positions else None, c["starts"], c["times"],
                                 c["k_pool"], c["v_pool"], EPS, block_tables=c["table"], page_size=c["page"],
                                 pair_axis=c["pair_axis"] if pair_axis and positions else None, q_out=c["q_out"] if q_out else None,
                                 q_rmsnorm_w=c["q_w"] if weights else None, k_rmsnorm_w=c["k_w"] if weights else None, **kw)


def check(c, before, *, q_out=True, **kw):
    want, place = oracle({**c, **{n: before[n] for n in "qkv"}}, **kw)
    n = int(c["starts"][-1])
    got_q = c["q_out"] if q_out else c["q"]
    close(got_q[:n], want["q"][0][:n], want["q"][1][:n], "q")
    assert torch.equal(got_q[n:], before["q_out" if q_out else "q"][n:]), "rows behind the last slot's were written"
    touched = {x: torch.zeros(c["k_pool"].shape[0], c["page"], dtype=torch.bool, device=got_q.device) for x in "kv"}
    for b, r in enumerate(c["rows"]):
        first = int(c["starts"][b])
        at = place[first:first + r]
        pg, inside = c["table"][b].long()[at // c["page"]], at % c["page"]
        for x in "kv":
            close(c[x + "_pool"][pg, :, inside], want[x][0][first:first + r], want[x][1][first:first + r], f"{x} of slot {b}")
            touched[x][pg, inside] = True
    for x in "kv":
        rest = ~touched[x][:, None].expand(c[x + "_pool"].shape[:3])
        assert torch.equal(c[x + "_pool"][rest], before[x + "_pool"][rest]), f"{x}: rows of other tokens were written"


def both(c, **kw):
    before = {n: x.clone() for n, x in c.items() if isinstance(x, torch.Tensor)}
    oracle_kw = {n: kw[n] for n in ("weights", "norm_qk", "norm_v", "positions") if n in kw}
    run(c, **kw)
    check(c, before, q_out=kw.get("q_out", True), **oracle_kw)


pytestmark = pytest.mark.filterwarnings("ignore")


@pytest.mark.gpu
@pytest.mark.parametrize("axes", [1, 2, 3, 4])
@pytest.mark.parametrize("rows,times", [([1], [1]), ([3, 0, 5], [3, 40, 21]), ([0, 0, 700, 1, 0], [5, 0, 700, 33, 9]), ([1, 1, 1], [17, 16, 500])])
def test_axes_and_slots(cuda, axes, rows, times):
    both(make(axes, rows, times, axes=axes))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [8, 64, 80, 128, 256, 264, 512])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [5, 1700])
def test_head_dims_and_types(cuda, D, dtype, n):
    cache = torch.float16 if dtype == torch.bfloat16 else torch.bfloat16
    both(make(D, [n, 2], [n + 3, 19], D=D, dtype=dtype, cache=cache, axes=3))


@pytest.mark.gpu
@pytest.mark.parametrize("cache", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("H,G", [(1, 1), (7, 7), (12, 4), (16, 1)])
def test_heads_and_pool_types(cuda, cache, H, G):
    both(make(H, [33, 600], [40, 601], H=H, G=G, cache=cache, page=64, D=128))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(weights=False), dict(norm_qk=False), dict(norm_v=False), dict(positions=False), dict(q_out=False)])
@pytest.mark.parametrize("n", [2, 1500])
def test_options(cuda, kw, n):
    both(make(n, [n, 7], [n + 20, 7]), **kw)


@pytest.mark.gpu
def test_far_positions_keep_their_angle(cuda):
    c = make(9, [300], [300], D=128, cache=torch.float32, max_pos=2 ** 31 - 1, axes=2)
    both(c)
    c = make(10, [300], [300], D=128, cache=torch.float32)
    c["positions"] = (torch.randint(0, 2 ** 33, (1, c["q"].shape[0]), generator=torch.Generator().manual_seed(1))).to(cuda)
    both(c)


@pytest.mark.gpu
def test_many_slots(cuda):
    """More slots than one look of a warp finds, some of them without rows."""
    g = torch.Generator().manual_seed(4)
    for B in (31, 32, 33, 1000, 1025, 2500):
        rows = torch.randint(0, 3, (B,), generator=g).tolist()
        both(make(B, rows, [r + 5 for r in rows], H=2, G=1, D=64))


@pytest.mark.gpu
def test_views_with_strides(cuda):
    c = make(12, [40, 9], [40, 30])
    N, H, D = c["q"].shape
    wide = torch.randn(N, H + 4, D + 8, device=cuda)
    c["q"], c["k"], c["v"] = wide[:, :H, :D], wide[:, H:H + 2, :D], wide[:, H + 2:, :D]
    c["q_out"] = torch.randn(H, N, D, device=cuda).to(torch.bfloat16).transpose(0, 1)
    c["positions"] = c["positions"].T.contiguous().T
    c["table"] = c["table"].T.contiguous().T
    both(c)


@pytest.mark.gpu
def test_nan_and_infinity_stay_in_their_row(cuda):
    c = make(13, [20], [20])
    c["q"][3, 1, 5], c["k"][4, 0, 9], c["v"][6, 1, 0] = float("nan"), float("inf"), float("nan")
    clean = {n: (x.clone() if isinstance(x, torch.Tensor) else x) for n, x in c.items()}
    for n in "qkv":
        clean[n] = torch.nan_to_num(clean[n], nan=1.0, posinf=1.0)
    run(c)
    run(clean)
    assert torch.equal(c["q_out"].isnan().any(-1).nonzero(), torch.tensor([[3, 1]], device=cuda))
    keep = torch.ones(c["q_out"].shape[:2], dtype=torch.bool, device=cuda)
    keep[3, 1] = False
    assert torch.equal(c["q_out"][keep], clean["q_out"][keep])
    assert (~torch.isfinite(c["k_pool"])).any(-1).sum() == 1 and (~torch.isfinite(c["v_pool"])).any(-1).sum() == 1


@pytest.mark.gpu
def test_bad_tables_are_recorded_and_not_followed(cuda):
    c = make(14, [20, 20], [20, 20])
    c["table"][1, 1] = 10 ** 6
    before = {n: x.clone() for n, x in c.items() if isinstance(x, torch.Tensor)}
    run(c)
    assert _cabi.device_status() == 0x102
    want, _ = oracle({**c, **{n: before[n] for n in "qkv"}})
    close(c["q_out"][:40], want["q"][0][:40], want["q"][1][:40], "q")
    c["table"][1, 1] = before["table"][1, 0]
    c["times"][1] = 10                                     # more rows than tokens: places below 0
    run(c)
    assert _cabi.device_status() == 0x101
    c["times"][1] = 1000
    run(c)
    assert _cabi.device_status() == 0x101
    c["times"][1] = 20
    c["pair_axis"][0] = 7
    run(c)
    assert _cabi.device_status() == 0x106


@pytest.mark.gpu
def test_starts_that_decrease_read_and_write_in_bounds(cuda):
    c = make(15, [10, 10, 10], [10, 10, 10])
    c["starts"].copy_(i32([0, 25, 5, 30]))
    run(c)                                                  # rows of a slot that the starts contradict have no place
    _cabi.device_status()


@pytest.mark.gpu
def test_captured_with_new_state_on_another_stream(cuda):
    c = make(16, [30, 2], [30, 9], axes=3)
    run(c)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        run(c)
    other = make(17, [30, 2], [30, 9], axes=3)
    for n in ("q", "k", "v", "positions", "table", "k_pool", "v_pool"):
        c[n].copy_(other[n])
    before = {n: x.clone() for n, x in c.items() if isinstance(x, torch.Tensor)}
    graph.replay()
    check(c, before)


@pytest.mark.gpu
def test_equals_the_padded_launch(cuda):
    """One slot, one axis, near positions: the rows of rope_norm_append, within a rounding of the pool's type (its angles
    are 32-bit products)."""
    c = make(18, [64], [64], spare=0, max_pos=1)
    run(c, positions=False)
    kc, vc = torch.zeros(1, 2, 64, 256, dtype=torch.bfloat16, device=cuda), torch.zeros(1, 2, 64, 256, dtype=torch.bfloat16, device=cuda)
    q2 = torch.zeros(1, 8, 64, 256, dtype=torch.bfloat16, device=cuda)
    rope.rope_norm_append(c["q"].transpose(0, 1)[None], c["k"].transpose(0, 1)[None], c["v"].transpose(0, 1)[None], c["freqs"], i32([0], cuda),
                          kc, vc, EPS, q_out=q2, q_rmsnorm_w=c["q_w"], k_rmsnorm_w=c["k_w"])
    a, b = c["q_out"].float(), q2[0].transpose(0, 1).float()
    assert bool(((a - b).abs() <= b.abs() * 2.0 ** -7 + 1e-4).all())
    assert math.isfinite(a.sum().item())


# ------------------------------------------------------------------------------------------ refusals
def cpu_case(**kw):
    return make(1, [3, 2], [3, 9], device="cpu", **kw)


def call(c, **over):
    a = {**c, **over}
    rope.rope_norm_append_packed(a["q"], a["k"], a["v"], a["freqs"], a["positions"], a["starts"], a["times"], a["k_pool"], a["v_pool"],
                                 EPS, block_tables=a["table"], page_size=a["page"], pair_axis=a["pair_axis"], q_out=a["q_out"],
                                 q_rmsnorm_w=a["q_w"], k_rmsnorm_w=a["k_w"], stream=0)


def test_valid_calls_pass_validation():
    c = cpu_case(axes=3)
    call(c)
    call(c, q_out=None, q_w=None, k_w=None)
    call(c, positions=None, pair_axis=None)
    call(c, positions=c["positions"][0].long(), pair_axis=None)
    call(make(1, [], [], spare=0, device="cpu"))
    call(make(1, [0, 0], [0, 4], spare=0, device="cpu", axes=2))


@pytest.mark.parametrize("over,match", [
    (lambda c: dict(k=c["k"][:-1]), "do not agree"),
    (lambda c: dict(v=c["v"].half()), "one dtype"),
    (lambda c: dict(q=c["q"][..., :-1]), "do not agree|multiple"),
    (lambda c: dict(q=c["q"].transpose(1, 2).contiguous().transpose(1, 2)), "innermost"),
    (lambda c: dict(freqs=c["freqs"][:-1]), "D/2"),
    (lambda c: dict(freqs=c["freqs"].double()), "dtype"),
    (lambda c: dict(positions=c["positions"][:, :-1]), "axes, N"),
    (lambda c: dict(positions=c["positions"].float()), "int32 or int64"),
    (lambda c: dict(pair_axis=None), "need pair_axis"),
    (lambda c: dict(pair_axis=c["pair_axis"].int()), "uint8"),
    (lambda c: dict(positions=None), "needs positions"),
    (lambda c: dict(starts=c["starts"][:-1]), "B \\+ 1"),
    (lambda c: dict(times=c["times"].long()), "int32"),
    (lambda c: dict(table=c["table"][:1]), "B rows"),
    (lambda c: dict(q_w=c["q_w"][:8]), "D entries"),
    (lambda c: dict(k_pool=c["k_pool"][:, :, :8]), "num_pages"),
    (lambda c: dict(k_pool=c["k_pool"].half()), "one dtype"),
    (lambda c: dict(v_pool=c["v_pool"][:-1]), "one dtype and shape"),
    (lambda c: dict(q_out=c["q_out"][:, :4]), "do not agree"),
    (lambda c: dict(page=32), "page_size"),
])
def test_refusals(over, match):
    c = cpu_case(axes=3)
    with pytest.raises((ValueError, TypeError), match=match):
        call(c, **over(c))


@pytest.mark.launches_allowed
def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA tensor"):
        call(cpu_case(axes=3))
