"""Attention of packed rows against the formula in 64 bits.

Tolerance for a row, with u = half a step of the 16-bit type (bf16 2^-8, f16 2^-11), p_j the exact weights, A = sum
p_j |v_j| / sum p_j per element, L = sum exp(s_j - max s):
  * probabilities are rounded once to the 16-bit type before the second product, and the sum is taken over rounded
    or unrounded ones: at most 2 u A;
  * f16 probabilities may be subnormal (the reference maximum lies at most 2^4 above the row's): half a step is
    2^-25 there, 2^-21 sum |v_j| / L;
  * a score is an f32 sum of D exact products, truncated or rounded at each step: off by at most 2 D 2^-24 sum_i |q_i k_i|
    scale, which is at most 2 D 2^-24 scale |q| |k|; a weight by that much (twice, numerator and sum), and by 2^-21 for the exponential: times A;
  * the second product and the sum in f32: n 2^-23 A for n keys is its bound; the terms' signs differ, 2^-16 A is allowed
    up to 2^7 tiles (each tile adds to one accumulator once per 16 keys);
  * the result is rounded once: u |o| (f32 outputs: 2^-24 |o|)."""
import math

import pytest
import torch

from g4b_b200 import _cabi
from g4b_b200.kernels import fa2, rope

BF16, F16, F32 = torch.bfloat16, torch.float16, torch.float32


def i32(v, device="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def make(seed, rows, times=None, *, H=8, G=2, D=256, page=16, dtype=BF16, out=None, device="cuda", spare=3, amp=1.0, dirty=True):
    """Packed rows of slots whose pages are shuffled; `spare` rows behind the last slot's; rows past a context and pages
    of nobody hold NaN."""
    g = torch.Generator().manual_seed(seed)
    times = rows if times is None else times
    N = sum(rows) + spare
    need = [-(-t // page) for t in times]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g)
    table = torch.full((len(rows), max(need + [1])), -1, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        at += n
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    rnd = lambda *s: torch.randn(*s, generator=g).to(device)  # noqa: E731
    k, v = rnd(pages, G, page, D).to(dtype), rnd(pages, G, page, D).to(dtype)
    if dirty:
        live = torch.zeros(pages, page, dtype=torch.bool)
        for b, t in enumerate(times):
            j = torch.arange(t)
            live[table[b].long()[j // page], j % page] = True
        dead = ~live.to(device)[:, None, :, None].expand(k.shape)
        k[dead] = float("nan")
        v[dead] = float("nan")
    c = dict(q=(amp * rnd(N, H, D)).to(dtype), k=k, v=v, o=rnd(N, H, D).to(out or dtype), starts=i32(starts, device),
             times=i32(times, device), table=table.to(device),
             workspace=torch.empty(fa2.packed_workspace_bytes(N, len(rows), H, G), dtype=torch.uint8, device=device))
    c.update(rows=list(rows), t=list(times), page=page, scale=1 / math.sqrt(D))
    return c


def run(c, **kw):
    fa2.flash_attention_packed(c["q"], c["k"], c["v"], c["o"], c["starts"], c["times"], block_tables=c["table"], page_size=c["page"],
                               workspace=c["workspace"], scale=c["scale"], **kw)


def check(c, o_before, *, sliding_window=0, stage=fa2.STAGE_CAUSAL, slots=None):
    q, o, page, scale = c["q"], c["o"], c["page"], c["scale"]
    N, H, D = q.shape
    G = c["k"].shape[1]
    rep = H // G
    u = torch.finfo(q.dtype).eps / 2
    u_out = torch.finfo(o.dtype).eps / 2
    at = 0
    for b, (r, t) in enumerate(zip(c["rows"], c["t"])):
        if r and (slots is None or b in slots):
            j = torch.arange(t, device=q.device)
            ids = c["table"][b].long()[j // page]
            pos = torch.arange(r, device=q.device) + (t - r)
            seen = torch.ones(r, t, dtype=torch.bool, device=q.device)
            if stage == fa2.STAGE_CAUSAL:
                seen &= j[None] <= pos[:, None]
            if sliding_window:
                seen &= j[None] > pos[:, None] - sliding_window
            some = seen.any(1)
            for h in range(H):
                k, v = c["k"][ids, h // rep, j % page].double(), c["v"][ids, h // rep, j % page].double()
                x = q[at:at + r, h].double()
                s = (x @ k.T * scale).masked_fill(~seen, -math.inf)
                top = s.max(1, keepdim=True).values.clamp(min=-1e300) if t else torch.zeros(r, 1, device=q.device).double()
                w = torch.exp(s - top)
                total = w.sum(1, keepdim=True).clamp(min=1e-300)
                want = w @ v / total
                A = w @ v.abs() / total
                norm_k = (seen * k.norm(dim=1)[None]).max(1, keepdim=True).values if t else torch.zeros(r, 1, device=q.device)
                score = 2 * D * 2.0 ** -24 * scale * x.norm(dim=1, keepdim=True) * norm_k
                allowed = (2 * u + 2 * score + 2.0 ** -21 + 2.0 ** -16) * A + u_out * want.abs() + 2.0 ** -25 * (o.dtype == F16)
                if q.dtype == F16:
                    allowed = allowed + 2.0 ** -21 * (seen.double() @ v.abs()) / total
                got = o[at:at + r, h].double()
                assert torch.isfinite(got).all(), f"slot {b} head {h}: not finite"
                worst = ((got - want).abs() - allowed * 1.01)[some]
                assert not worst.numel() or worst.max().item() <= 0, f"slot {b} head {h}: {worst.max().item():.3e} more than allowed"
                assert bool((got[~some] == 0).all()), f"slot {b} head {h}: rows without a key are not zero"
        at += r
    if slots is None:
        assert torch.equal(o[at:], o_before[at:]), "rows behind the last slot were written"


def both(c, **kw):
    before = c["o"].clone()
    run(c, **kw)
    check(c, before, **{**kw, "sliding_window": kw.get("sliding_window") or 0})


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [[1], [2], [16], [17], [63], [64], [65], [128, 129], [200], [5, 0, 40, 1], [0, 0, 0, 300], [500, 33, 1, 64, 700]])
@pytest.mark.parametrize("dtype", [BF16, F16])
def test_prompts(cuda, rows, dtype):
    both(make(sum(rows), rows, dtype=dtype))


@pytest.mark.gpu
@pytest.mark.parametrize("D", [128, 256])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256])
def test_pages_and_head_dims(cuda, D, page):
    both(make(page, [300, 1, 77, 513], [300, 130, 600, 513], D=D, page=page, dtype=F16))
    both(make(page + 1, [90, 200], [1000, 256], D=D, page=page))


@pytest.mark.gpu
@pytest.mark.parametrize("H,G", [(1, 1), (4, 4), (2, 1), (3, 1), (6, 2), (5, 1), (7, 1), (8, 1), (9, 3), (16, 1), (48, 1), (64, 1), (128, 1), (65, 1)])
def test_groups(cuda, H, G):
    both(make(H, [150, 3, 270], [150, 70, 300], H=H, G=G, D=128 if H > 16 else 256))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 128, 200, 1000])
def test_sliding_window(cuda, window):
    both(make(window, [400, 1, 130, 64], [400, 900, 700, 64]), sliding_window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("window", [None, 100])
def test_full_stage(cuda, window):
    both(make(3, [130, 1, 40, 300], [130, 200, 40, 777]), stage=fa2.STAGE_FULL, sliding_window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("D,dtype", [(128, BF16), (256, F16), (256, BF16)])
def test_f32_output(cuda, D, dtype):
    both(make(5, [130, 1, 300], [130, 500, 300], D=D, dtype=dtype, out=F32))


@pytest.mark.gpu
def test_long_prompts_and_cached_contexts(cuda):
    both(make(7, [3000, 1, 700], [3000, 9000, 5000], H=4, G=1))
    both(make(8, [64, 1, 1], [20001, 16384, 5000], H=4, G=2, D=128, dtype=F16, page=64))


@pytest.mark.gpu
@pytest.mark.parametrize("rows,times,kw", [
    ([1], [30000], {}), ([1], [1025], {}), ([1, 1, 1], [5000, 1, 9000], dict(H=3, G=1)), ([5, 0, 20, 0], [9000, 0, 4000, 30], dict(D=128)),
    ([70, 10], [3, 20000], dict(dtype=F16)), ([300], [7000], dict(out=F32)), ([200, 1], [2500, 8000], dict(D=128, out=F32, page=128)),
    ([64] * 9, [700 * i + 64 for i in range(9)], dict(H=4, G=4, dtype=F16)), ([40, 1, 1], [6000, 1500, 16], dict(H=48, G=1, D=128)),
    ([1] * 40 + [100], [20] * 40 + [15000], dict(H=2, G=1)), ([1100], [1100], dict(H=1, G=1))])
def test_shares_of_long_contexts(cuda, rows, times, kw):
    """Few items behind long contexts: their keys are cut at the workers' boundaries and the parts joined."""
    both(make(sum(times), rows, times, **kw))


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [dict(sliding_window=3000), dict(stage=fa2.STAGE_FULL), dict(stage=fa2.STAGE_FULL, sliding_window=2500)])
def test_shares_under_other_masks(cuda, kw):
    both(make(31, [30, 1, 64], [7000, 12000, 64], H=4, G=2), **kw)


@pytest.mark.gpu
def test_shares_repeat_and_do_not_touch_other_rows(cuda):
    c = make(32, [20, 1, 0, 7], [9000, 3000, 50, 12000])
    both(c)
    first = c["o"].clone()
    for _ in range(5):
        run(c)
        assert torch.equal(c["o"], first)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [33, 150, 400])
def test_many_slots(cuda, n):
    g = torch.Generator().manual_seed(n)
    rows = torch.randint(0, 40, (n,), generator=g).tolist()
    times = [r + int(x) for r, x in zip(rows, torch.randint(0, 200, (n,), generator=g).tolist())]
    both(make(n, rows, times, H=2, G=1, D=128))


@pytest.mark.gpu
def test_large_scores(cuda):
    """Softmaxes close to one key, and reference maxima that jump between tiles."""
    both(make(11, [600, 300], amp=30.0, H=4, G=2))
    c = make(12, [700], H=2, G=1, dtype=F16)
    ramp = torch.linspace(0.1, 8, 700, device=cuda)
    j = torch.arange(700, device=cuda)
    ids = c["table"][0].long()[j // 16]
    c["k"][ids, 0, j % 16] = (c["k"][ids, 0, j % 16].float() * ramp[:, None]).half()
    both(c)


@pytest.mark.gpu
def test_scores_of_different_magnitude_behind_one_another(cuda):
    """The reference maximum carried from item to item meets rows hundreds of units away."""
    c = make(13, [300, 300, 300, 300, 300], H=2, G=1, dtype=F16)
    for b, amp in enumerate((30.0, 0.01, 20.0, 1.0, 0.0)):
        c["q"][300 * b:300 * (b + 1)] = (c["q"][300 * b:300 * (b + 1)].float() * amp).half()
    both(c)


@pytest.mark.gpu
def test_more_rows_than_tokens_and_no_tokens(cuda):
    """Rows at positions below 0, and slots without a context, see nothing."""
    both(make(14, [100, 20, 300, 5], [60, 0, 300, 5]))


@pytest.mark.gpu
def test_nan_and_infinity_in_one_slot_stay_there(cuda):
    c = make(15, [200, 130, 70], H=4, G=2)
    c["q"][210, 1] = float("nan")
    c["v"][c["table"][1, 0].long(), 0, 3, 5] = float("inf")
    c["k"][c["table"][1, 2].long(), 1, 3, 5] = float("nan")
    before = c["o"].clone()
    run(c)
    check(c, before, slots=(0, 2))
    run(c)                                   # and not in what a second call makes of the first one's maxima
    check(c, before, slots=(0, 2))


@pytest.mark.gpu
def test_views(cuda):
    c = make(16, [130, 70], H=8, G=2)
    N, H, D = c["q"].shape
    wide = torch.randn(N, H + 3, D + 64, device=cuda).to(BF16)
    wide[:, 1:H + 1, 64:] = c["q"]
    c["q"] = wide[:, 1:H + 1, 64:]
    c["o"] = torch.randn(H, N, D, device=cuda).to(BF16).transpose(0, 1)
    c["table"] = c["table"].T.contiguous().T
    both(c)
    c = make(17, [1], [40], H=1, G=1, spare=0)
    both(c)


@pytest.mark.gpu
def test_bad_entries_are_recorded_and_bounded(cuda):
    c = make(18, [200, 100, 50])
    c["table"][1, 2] = 10 ** 6
    before = c["o"].clone()
    run(c)
    assert _cabi.device_status() == 0x309
    check(c, before, slots=(0, 2))
    assert torch.isfinite(c["o"][200:300]).all()
    c = make(19, [40, 30])
    c["times"][1] = 2 ** 30                   # past the table: attended to as far as it reaches
    c["table"][1] = c["table"][0]
    run(c)
    check(c, before, slots=(0,))
    _cabi.device_status()


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 64])
def test_pages_in_front_of_the_window_may_be_gone(cuda, page):
    """Their entries are -1 or name somebody else's pages, full of NaN: nothing is recorded, nothing read."""
    c = make(33, [300, 1, 64], [900, 2000, 1500], page=page, H=4, G=2)
    window = 200
    for b, (r, t) in enumerate(zip(c["rows"], c["t"])):
        first = max(0, t - r - window + 1) // page
        c["table"][b, :first] = -1
    before = c["o"].clone()
    run(c, sliding_window=window)
    assert _cabi.device_status() == 0
    c["table"].clamp_(min=0)
    check(c, before, sliding_window=window)


@pytest.mark.gpu
def test_output_over_the_queries(cuda):
    c = make(34, [300, 1, 64], [300, 9000, 64], H=8, G=2)
    d = {**c, "q": c["q"].clone()}
    c["o"] = c["q"]
    run(c)
    d["o"] = c["o"]
    check(d, d["q"])


@pytest.mark.gpu
@pytest.mark.parametrize("window", [2 ** 30, 2 ** 31 - 1])
def test_windows_longer_than_any_context(cuda, window):
    both(make(35, [100, 70], [60, 300]), sliding_window=window)


@pytest.mark.gpu
@pytest.mark.parametrize("starts", [[0, 50, 20, 90], [-1, 30, 60, 90], [0, 30, 60, 1000], [90, 60, 30, 0]])
def test_starts_that_contradict_themselves(cuda, starts):
    c = make(20, [30, 30, 30])
    c["starts"].copy_(i32(starts))
    before = c["o"].clone()
    run(c)
    assert _cabi.device_status() == 0x107 and torch.equal(c["o"], before)


@pytest.mark.gpu
def test_starts_that_leave_rows_out(cuda):
    """Rows in front of the first slot and behind the last stay as they are."""
    c = make(21, [30, 60], spare=40)
    c["starts"] += 17
    c["q"] = torch.cat([c["q"][-17:], c["q"][:-17]])
    before = c["o"].clone()
    run(c)
    assert torch.equal(c["o"][:17], before[:17])
    c["o"], c["q"] = c["o"][17:], c["q"][17:]
    check(c, before[17:])


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """Pages behind 4 GB of pool, rows behind 4 GB of q and o."""
    page, D = 128, 256
    c = make(22, [100], [300], H=2, G=1, page=page)
    big = torch.empty(70000, 1, page, D, dtype=BF16, device=cuda)
    v = torch.empty_like(big)
    ids = [69999, 1, 66000]
    for i, p in enumerate(ids):
        big[p], v[p] = c["k"][c["table"][0, i].long()], c["v"][c["table"][0, i].long()]
    c["k"], c["v"], c["table"] = big, v, i32([ids], cuda)
    q = torch.empty(9_000_000, 2, D, dtype=BF16, device=cuda)
    o = torch.zeros_like(q)
    at = q.shape[0] - 120
    q[at:at + 103] = c["q"]
    c["starts"] += at
    c["workspace"] = torch.empty(fa2.packed_workspace_bytes(q.shape[0], 1, 2, 1), dtype=torch.uint8, device=cuda)
    small_q = c["q"]
    c["q"], c["o"] = q, o
    run(c)
    c["q"], c["o"] = small_q, o[at:at + 103].clone()
    check(c, torch.zeros_like(c["o"]))


@pytest.mark.gpu
def test_same_input_same_bits(cuda):
    c = make(23, [700, 1, 300, 40], [700, 5000, 1000, 40])
    run(c)
    first = c["o"].clone()
    for _ in range(3):
        run(c)
        assert torch.equal(c["o"], first)


@pytest.mark.gpu
def test_captured_with_other_lengths_on_another_stream(cuda):
    c = make(24, [200, 40, 60], [300, 40, 500], spare=0)
    run(c)
    graph, side = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        run(c)
    d = make(25, [10, 190, 100], [490, 200, 150], spare=0)
    pages = min(c["k"].shape[0], d["k"].shape[0])
    assert int(d["table"].max()) < c["k"].shape[0] or pages == c["k"].shape[0]
    c["q"].copy_(d["q"])
    c["starts"].copy_(d["starts"])
    c["times"].copy_(d["times"])
    width = min(c["table"].shape[1], d["table"].shape[1])
    c["table"].fill_(-1)
    c["table"][:, :width] = d["table"][:, :width]
    n = min(c["k"].shape[0], d["k"].shape[0])
    c["k"][:n], c["v"][:n] = d["k"][:n], d["v"][:n]
    c["rows"], c["t"] = d["rows"], d["t"]
    before = c["o"].clone()
    graph.replay()
    check(c, before)


@pytest.mark.gpu
def test_many_calls_behind_one_another(cuda):
    """Nothing waits between the calls: each launch is set up while the one before drains, with the same workspace."""
    cases = [make(40, [2500, 700, 1], H=8, G=2), make(41, [5, 17], H=8, G=2), make(42, [64, 1], [9000, 4000], H=8, G=2, dtype=F16),
             make(43, [900, 333, 41], H=8, G=2, D=128, page=64)]
    workspace = max((c["workspace"] for c in cases), key=lambda w: w.numel())
    want = []
    for c in cases:
        c["workspace"] = workspace
        run(c, sliding_window=300 if c is cases[0] else None)
        want.append(c["o"].clone())
    for i in range(400):
        c = cases[i * 7 % 4]
        run(c, sliding_window=300 if c is cases[0] else None)
    for c, w in zip(cases, want):
        assert torch.equal(c["o"], w) or bool(((c["o"] - w).abs().float() <= 2e-2 * w.abs().float() + 4e-3).all())
    assert _cabi.device_status() == 0


@pytest.mark.gpu
def test_two_streams_with_their_own_workspaces(cuda):
    cases = [make(26, [900, 300], H=4, G=1), make(27, [64, 700, 1], [64, 700, 2000], H=4, G=1)]
    before = [c["o"].clone() for c in cases]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    for _ in range(5):
        for c, s in zip(cases, streams):
            run(c, stream=s)
    torch.cuda.synchronize()
    for c, b in zip(cases, before):
        check(c, b)


@pytest.mark.gpu
def test_equals_the_padded_call(cuda):
    """Two prompts of one length: what g4b_flash_attention makes of them, within both kernels' rounding."""
    c = make(28, [256, 256], spare=0)
    run(c)
    o = torch.zeros(2, 8, 256, 256, dtype=BF16, device=cuda)
    q = c["q"].view(2, 256, 8, 256).transpose(1, 2)
    fa2.flash_attention(q, c["k"], c["v"], o, c["times"], None, 256, fa2.PHASE_PREFILL, scale=c["scale"], block_tables=c["table"])
    a, b = c["o"].float(), o.transpose(1, 2).reshape(512, 8, 256).float()
    assert bool(((a - b).abs() <= 2e-3 + 1e-2 * b.abs()).all())


@pytest.mark.gpu
def test_a_packed_step_as_it_is_served(cuda):
    """Rotary, append and attention of a step that mixes prompts, a chunk and single tokens, with the page manager's
    tables; then the same tokens decoded by the one-token kernel read the same pages."""
    from g4b_b200.paging import PagedKVManager

    H, G, D = 8, 2, 256
    m = PagedKVManager(num_pages=120, max_batch=4, max_context=1024, page_size=16)
    m.bind_device(cuda)
    g = torch.Generator().manual_seed(5)
    k_pool = torch.full((120, G, 16, D), float("nan"), dtype=BF16, device=cuda)
    v_pool = k_pool.clone()
    w = torch.empty(fa2.packed_workspace_bytes(1200, 4, H, G), dtype=torch.uint8, device=cuda)
    freqs = (10000.0 ** (-torch.arange(0, D, 2).double() / D)).float().to(cuda)
    held = [0, 0, 0, 0]
    for slot in range(4):
        m.place_request([slot * 1000 + i for i in range(10)])
    for rows in ([300, 0, 64, 1], [1, 128, 100, 0], [1, 1, 1, 40], [1, 1, 1, 1]):
        held = [a + b for a, b in zip(held, rows)]
        m.prepare_packed_inputs(rows, held)
        dev = m.upload()
        N = sum(rows)
        q, k, v = (torch.randn(N, h, D, generator=g).to(cuda) for h in (H, G, G))
        q16, o = torch.empty(N, H, D, dtype=BF16, device=cuda), torch.zeros(N, H, D, dtype=BF16, device=cuda)
        rope.rope_norm_append_packed(q, k, v, freqs, None, dev["q_starts"], dev["time_dim_sizes"], k_pool, v_pool, 1e-6,
                                     block_tables=dev["block_tables"], q_out=q16)
        fa2.flash_attention_packed(q16, k_pool, v_pool, o, dev["q_starts"], dev["time_dim_sizes"], block_tables=dev["block_tables"],
                                   workspace=w, scale=1 / 16)
        torch.cuda.synchronize()
        c = dict(q=q16, k=k_pool, v=v_pool, o=o, table=dev["block_tables"], rows=rows, t=[h if r else 0 for h, r in zip(held, rows)],
                 page=16, scale=1 / 16)
        check(c, o)
    o1 = torch.zeros(4, H, 1, D, dtype=BF16, device=cuda)
    fa2.flash_attention(q16[:, :, None], k_pool, v_pool, o1, dev["time_dim_sizes"], None, 1024, fa2.PHASE_DECODE, scale=1 / 16,
                        block_tables=dev["block_tables"])
    check({**c, "o": o1[:, :, 0]}, o1[:, :, 0])


# ------------------------------------------------------------------------------------------ refusals
def call(c, **over):
    a = {**c, "stage": 3, "window": 0, **over}
    fa2.flash_attention_packed(a["q"], a["k"], a["v"], a["o"], a["starts"], a["times"], block_tables=a["table"], page_size=a["page"],
                               workspace=a["workspace"], scale=a["scale"], sliding_window=a["window"], stage=a["stage"], stream=0)


def cpu_case(**kw):
    return make(1, [3, 2], [3, 9], device="cpu", dirty=False, **kw)


def test_valid_calls_pass_validation():
    call(cpu_case())
    call(cpu_case(D=128, page=64, dtype=F16, out=F32))
    call(make(1, [], [], spare=0, device="cpu", dirty=False))
    call(make(1, [0, 0], [5, 0], spare=0, device="cpu", dirty=False))
    assert fa2.packed_workspace_bytes(0, 0, 8, 2) > 0
    with pytest.raises(ValueError, match="multiple"):
        fa2.packed_workspace_bytes(1, 1, 7, 2)


@pytest.mark.parametrize("over,match", [
    (lambda c: dict(o=c["o"][:-1]), "o shape"),
    (lambda c: dict(q=c["q"].float()), "pools' dtype"),
    (lambda c: dict(q=c["q"].half()), "pools' dtype"),
    (lambda c: dict(o=c["o"].half()), "o must have"),
    (lambda c: dict(k=c["k"].half()), "both"),
    (lambda c: dict(k=c["k"].float(), v=c["v"].float()), "both"),
    (lambda c: dict(k=c["k"][:-1]), "shapes differ"),
    (lambda c: dict(k=c["k"][:, :, :, ::2], v=c["v"][:, :, :, ::2]), "contiguous"),
    (lambda c: dict(q=c["q"][..., :64], o=c["o"][..., :64]), "head dim"),
    (lambda c: dict(q=c["q"][:, :7], o=c["o"][:, :7]), "multiple"),
    (lambda c: dict(page=32), "page_size"),
    (lambda c: dict(page=8, k=c["k"][:, :, :8].contiguous(), v=c["v"][:, :, :8].contiguous()), "power of two"),
    (lambda c: dict(starts=c["starts"][:-1]), "B \\+ 1"),
    (lambda c: dict(starts=c["starts"].long()), "int32"),
    (lambda c: dict(table=c["table"][:1]), "B rows"),
    (lambda c: dict(stage=2), "stage"),
    (lambda c: dict(window=-1), "sliding_window"),
    (lambda c: dict(scale=0.0), "scale"),
    (lambda c: dict(scale=float("nan")), "scale"),
    (lambda c: dict(scale=-1.0), "scale"),
    (lambda c: dict(workspace=c["workspace"][:64]), "workspace"),
    (lambda c: dict(workspace=torch.cat([c["workspace"]] * 2)[1:]), "16-byte"),
    (lambda c: dict(q=c["q"].transpose(1, 2).contiguous().transpose(1, 2)), "innermost"),
    (lambda c: dict(q=torch.zeros(8, 8, 260, dtype=BF16)[..., 4:]), "aligned|multiples"),
    (lambda c: dict(q=c["q"][:1].expand(8, 8, 256)), "positive"),
])
def test_refusals(over, match):
    c = cpu_case()
    with pytest.raises((ValueError, TypeError), match=match):
        call(c, **over(c))


def test_head_dim_512_and_wide_groups_are_refused():
    with pytest.raises(ValueError, match="head dim 512"):
        call(cpu_case(D=512))
    c = cpu_case()
    c["workspace"] = torch.zeros(10 ** 6, dtype=torch.uint8)
    with pytest.raises(ValueError, match="at most 128"):
        call(c, q=torch.zeros(8, 129, 256, dtype=BF16), o=torch.zeros(8, 129, 256, dtype=BF16), k=torch.zeros(3, 1, 16, 256, dtype=BF16),
             v=torch.zeros(3, 1, 16, 256, dtype=BF16))


@pytest.mark.launches_allowed
def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA tensor"):
        call(cpu_case())
