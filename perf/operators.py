"""Cases for the operators of a packed prompt step over a paged KV cache, each in a plain form
(elementary torch operations in 32 bits, 64 where 32 lose what matters) and through the
framework's entry points:

  attention  ``fa2.flash_attention_packed``: prompts and chunks of different lengths, packed row
             behind row without padding, attend causally to their slots' pages
  rope       ``rope.rope_norm_append_packed``: per-head RMS norm, rotary embedding over one or
             several position axes (time, height, width), V norm and the paged append of those
             packed rows
  pages      ``pages.copy_pages``: pages of every layer's pools copied in one launch, when a
             sequence is forked and when the pool is compacted

``own`` selects the framework's calls; it is set by whoever runs the cases."""
import math

import torch

own = False

HEADS, KV_HEADS = 8, 2          # the engine's attention geometry
EPS = 1e-6
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # three one-line questions that arrive together: the smallest step, launch latency counts
        {"name": "attn three short prompts", "op": "attention", "rows": "5,17,40", "cached": "0,0,0", "dim": 256, "type": "bf16",
         "page": 16, "window": 0},
        # sixteen prompts of mixed length, from a single token to a document
        {"name": "attn sixteen prompts", "op": "attention",
         "rows": "1,2000,613,64,128,900,33,1500,257,81,1024,511,7,350,1203,60", "cached": ",".join(["0"] * 16), "dim": 256,
         "type": "f16", "page": 16, "window": 0},
        # a few long documents: the global layers, bound by the tensor pipe
        {"name": "attn long prompts", "op": "attention", "rows": "8192,5000,2500,701", "cached": "0,0,0,0", "dim": 256,
         "type": "bf16", "page": 16, "window": 0},
        # the sliding-window layers of the same engine (window 512)
        {"name": "attn window 512", "op": "attention", "rows": "4096,3001,1500,777,4096,350", "cached": "0,0,0,0,0,0", "dim": 256,
         "type": "bf16", "page": 16, "window": 512},
        # chunks and single tokens behind contexts that earlier steps cached
        {"name": "attn chunks behind cached", "op": "attention", "rows": "256,100,1,37,1,512",
         "cached": "20000,9003,30000,4096,777,16384", "dim": 256, "type": "bf16", "page": 16, "window": 0},
        # head dim 128 with larger pages
        {"name": "attn head dim 128", "op": "attention", "rows": "4000,129,2048,1000,3333", "cached": "0,500,0,64,0", "dim": 128,
         "type": "f16", "page": 64, "window": 0},
        # a handful of rows: a step of single tokens
        {"name": "rope eight single tokens", "op": "rope", "rows": "1,1,1,1,1,1,1,1", "cached": "5,1000,131000,77,16,15,4096,40000",
         "dim": 256, "in": "f32", "type": "bf16", "page": 16, "axes": 1},
        # prompts with images: three position axes, text and patches mixed
        {"name": "rope images three axes", "op": "rope", "rows": "1500,300,2600,17", "cached": "0,128,0,4001", "dim": 256, "in": "f32",
         "type": "bf16", "page": 16, "axes": 3},
        # a full prompt step, streaming
        {"name": "rope large step", "op": "rope", "rows": "16384,8192,5000,3191,1", "cached": "0,0,65536,100,9", "dim": 256,
         "in": "f32", "type": "f16", "page": 16, "axes": 1},
        # four sequences forked: one partial page each, in the K and V pools of 24 layers
        {"name": "pages fork", "op": "pages", "pages": 64, "copies": 4, "pools": 48, "dim": 256, "type": "bf16", "page": 16},
        # 8-bit pools with their scales, a wide fork
        {"name": "pages fork 8 bit", "op": "pages", "pages": 700, "copies": 301, "pools": 12, "dim": 256, "type": "e4m3", "page": 16},
        # the pool compacted after many requests ended
        {"name": "pages compaction", "op": "pages", "pages": 5000, "copies": 2100, "pools": 16, "dim": 256, "type": "bf16",
         "page": 16},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    op = rng.choice(["attention", "attention", "rope", "pages"])
    if op == "attention":
        n = _log_int(rng, 1, 16)
        cached = rng.random() < 0.4
        longest = (1024 if n <= 4 else 256) if cached else 6000 if n <= 2 else 3000 if n <= 8 else 1024
        rows = [_log_int(rng, 1, longest) for _ in range(n)]
        before = [_log_int(rng, 1, 10000) if cached and rng.random() < 0.7 else 0 for _ in range(n)]
        return {"op": op, "rows": ",".join(map(str, rows)), "cached": ",".join(map(str, before)), "dim": rng.choice([128, 256, 256]),
                "type": rng.choice(["f16", "bf16"]), "page": rng.choice([16, 16, 32, 64, 128]),
                "window": rng.choice([0, 0, 512, _log_int(rng, 1, 2000)])}
    if op == "rope":
        n, dim = _log_int(rng, 1, 6), rng.choice([128, 256, 256, 512])
        rows = [_log_int(rng, 1, 5000 if dim <= 256 else 2500) for _ in range(n)]
        return {"op": op, "rows": ",".join(map(str, rows)), "cached": ",".join(str(_log_int(rng, 1, 20000) - 1) for _ in range(n)),
                "dim": dim, "in": rng.choice(["f32", "f32", "bf16", "f16"]), "type": rng.choice(["f16", "bf16"]),
                "page": rng.choice([16, 16, 32, 64]), "axes": rng.choice([1, 2, 3, 4])}
    dim, page = rng.choice([128, 256, 512]), rng.choice([16, 16, 32])
    pages = _log_int(rng, 8, 4000 * 16 * 256 // (page * dim) if page * dim > 16 * 256 else 4000)
    return {"op": op, "pages": pages, "copies": _log_int(rng, 1, pages // 2), "pools": rng.choice([2, 4, 7, 12, 16]), "dim": dim,
            "type": rng.choice(["f16", "bf16", "e4m3"]), "page": page}


def _ints(text):
    return [int(x) for x in text.split(",")]


# -------------------------------------------------------------------------------------- states
def _slots(case, gen):
    """Row offsets, context lengths and shuffled block tables of the case's slots."""
    rows, cached = _ints(case["rows"]), _ints(case["cached"])
    times = [r + c for r, c in zip(rows, cached)]
    page = case["page"]
    need = [-(-t // page) for t in times]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((len(rows), max(need)), -1, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    starts = [0]
    for r in rows:
        starts.append(starts[-1] + r)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")  # noqa: E731
    return rows, times, pages, {"q_starts": i32(starts), "time": i32(times), "table": table}


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, generator=gen, device="cuda")  # noqa: E731
    state = dict(case)
    if case["op"] == "pages":
        n, copies, dt = case["pages"], case["copies"], TYPES[case["type"]]
        pools = []
        for i in range(case["pools"]):
            x = randn(n, KV_HEADS, case["page"], case["dim"])
            if case["type"] == "e4m3" and i % 2:      # an 8-bit pool and the scales beside it
                x = (randn(n, KV_HEADS).abs() + 0.01).to(torch.float32)
                pools.append(x)
            else:
                pools.append(x.to(dt))
        order = torch.randperm(n, generator=gen, device="cuda").to(torch.int32)
        state.update(pools=pools, src=order[:copies].contiguous(), dst=order[n - copies:].contiguous())
        return state
    rows, times, pages, slots = _slots(case, gen)
    state.update(slots)
    D, dt, N = case["dim"], TYPES[case["type"]], sum(rows)
    pool = lambda: torch.empty(pages, KV_HEADS, case["page"], D, dtype=dt, device="cuda")  # noqa: E731
    if case["op"] == "attention":
        state["k_pool"], state["v_pool"] = pool().copy_(randn(pages, KV_HEADS, case["page"], D)), pool().copy_(randn(pages, KV_HEADS, case["page"], D))
        state["q"] = randn(N, HEADS, D).to(dt)
        state["o"] = torch.empty(N, HEADS, D, dtype=dt, device="cuda")
        state["scale"] = 1 / math.sqrt(D)
        # memory that a serving program allocates once, at its largest step
        state["workspace"] = torch.empty(256 << 20, dtype=torch.uint8, device="cuda")
        return state
    state["q"], state["k"], state["v"] = (randn(N, h, D).to(TYPES[case["in"]]) for h in (HEADS, KV_HEADS, KV_HEADS))
    state["q_w"], state["k_w"] = 1 + 0.1 * randn(D), 1 + 0.1 * randn(D)
    state["freqs"] = (10000.0 ** (-torch.arange(0, D, 2, device="cuda", dtype=torch.float64) / D)).float()
    state["k_pool"], state["v_pool"] = pool().zero_(), pool().zero_()
    state["q_out"] = torch.zeros(N, HEADS, D, dtype=dt, device="cuda")
    # positions: the place in the sequence along every axis, as for text; a stretch of every
    # longer prompt is an image whose patches differ in height and width instead
    A = case["axes"]
    bounds = torch.tensor([0] + rows, device="cuda").cumsum(0)
    row = torch.arange(N, device="cuda")
    slot = torch.searchsorted(bounds, row, right=True) - 1
    local = row - bounds[slot]
    pos = (local + torch.tensor(times, device="cuda")[slot] - torch.tensor(rows, device="cuda")[slot]).repeat(A, 1)
    if A > 1:
        image = (local >= 16) & (local < 16 + 24 * 32)
        patch = local - 16
        for axis, along in ((A - 1, patch % 32), (A - 2, patch // 32)):
            pos[axis] = torch.where(image, pos[axis] - local + 16 + along, pos[axis])
    state["positions"] = pos.to(torch.int32).contiguous()
    # rotation pairs dealt to the axes in turn
    state["pair_axis"] = (torch.arange(D // 2, device="cuda") % A).to(torch.uint8)
    return state


# ---------------------------------------------------------------------------------------- runs
def _padded_rows(s):
    """[B, longest] indices of the packed rows of every slot, and which of them exist."""
    first, last = s["q_starts"][:-1, None].long(), s["q_starts"][1:, None].long()
    at = first + torch.arange(max(_ints(s["rows"])), device="cuda")[None]
    return at.clamp(max=s["q"].shape[0] - 1), at < last


def _plain_attention(s):
    at, real = _padded_rows(s)
    B, L = at.shape
    D, G, page = s["dim"], KV_HEADS, s["page"]
    rep = HEADS // G
    pages = s["table"].clamp(min=0).long()
    T = pages.shape[1] * page
    k, v = (p[pages].permute(0, 2, 1, 3, 4).reshape(B, G, T, D).float() for p in (s["k_pool"], s["v_pool"]))
    time = s["time"].long()[:, None]
    count = (s["q_starts"][1:] - s["q_starts"][:-1]).long()[:, None]
    q_pos = time - count + torch.arange(L, device="cuda")[None]                       # [B, L]
    key = torch.arange(T, device="cuda")
    seen = (key[None, None] <= q_pos[..., None]) & (key[None, None] < time[..., None])
    if s["window"]:
        seen &= key[None, None] > q_pos[..., None] - s["window"]
    q = s["q"][at].float().reshape(B, L, G, rep, D).permute(0, 2, 3, 1, 4).reshape(B, G, rep * L, D)
    x = (q @ k.transpose(2, 3)).mul_(s["scale"]).reshape(B, G, rep, L, T)
    x = x.masked_fill_(~seen[:, None, None], float("-inf"))
    x = x.sub_(x.amax(-1, keepdim=True).clamp_(min=-1e30)).exp_()
    total = x.sum(-1, keepdim=True)
    out = (x.reshape(B, G, rep * L, T) @ v).reshape(B, G, rep, L, D) / total
    out = out.permute(0, 3, 1, 2, 4).reshape(B, L, HEADS, D)
    s["o"][at[real]] = out[real].to(s["o"].dtype)
    return s["o"]


def _plain_rope(s):
    D, half, dt = s["dim"], s["dim"] // 2, s["k_pool"].dtype
    q, k, v = s["q"].float(), s["k"].float(), s["v"].float()
    q, k, v = (x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) for x in (q, k, v))
    q, k = q * s["q_w"], k * s["k_w"]
    angle = s["positions"].double()[s["pair_axis"].long()].T * s["freqs"].double()     # [N, D/2], far positions need 64 bits
    sin, cos = angle.sin().float()[:, None], angle.cos().float()[:, None]
    turn = lambda x: torch.cat([x[..., :half] * cos - x[..., half:] * sin, x[..., half:] * cos + x[..., :half] * sin], -1)  # noqa: E731
    s["q_out"].copy_(turn(q))
    row = torch.arange(q.shape[0], device="cuda")
    starts = s["q_starts"].long()
    slot = torch.searchsorted(starts, row, right=True) - 1
    place = s["time"].long()[slot] - starts[slot + 1] + row
    pages, inside = s["table"][slot, place // s["page"]].long(), place % s["page"]
    s["k_pool"][pages, :, inside] = turn(k).to(dt)
    s["v_pool"][pages, :, inside] = v.to(dt)
    return s["q_out"], s["k_pool"], s["v_pool"]


def _plain_pages(s):
    src, dst = s["src"].long(), s["dst"].long()
    for p in s["pools"]:
        raw = p.view(torch.uint8) if p.element_size() == 1 else p
        raw[dst] = raw[src]
    return s["pools"]


def run(state):
    s = state
    if own:
        from g4b_b200.kernels import fa2, pages, rope

        if s["op"] == "attention":
            fa2.flash_attention_packed(s["q"], s["k_pool"], s["v_pool"], s["o"], s["q_starts"], s["time"], block_tables=s["table"],
                                       page_size=s["page"], workspace=s["workspace"], scale=s["scale"],
                                       sliding_window=s["window"])
            return s["o"]
        if s["op"] == "rope":
            rope.rope_norm_append_packed(s["q"], s["k"], s["v"], s["freqs"], s["positions"], s["q_starts"], s["time"], s["k_pool"],
                                         s["v_pool"], EPS, block_tables=s["table"], page_size=s["page"], pair_axis=s["pair_axis"],
                                         q_out=s["q_out"], q_rmsnorm_w=s["q_w"], k_rmsnorm_w=s["k_w"])
            return s["q_out"], s["k_pool"], s["v_pool"]
        pages.copy_pages(s["pools"], s["src"], s["dst"])
        return s["pools"]
    return {"attention": _plain_attention, "rope": _plain_rope, "pages": _plain_pages}[s["op"]](s)


# ---------------------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "pages":
        size = 0
        for i in range(case["pools"]):
            if case["type"] == "e4m3":
                size += KV_HEADS * 4 if i % 2 else KV_HEADS * case["page"] * case["dim"]
            else:
                size += KV_HEADS * case["page"] * case["dim"] * 2
        return {"bytes": 2 * case["copies"] * size + 8 * case["copies"], "flops": 0}
    rows, cached, D = _ints(case["rows"]), _ints(case["cached"]), case["dim"]
    N = sum(rows)
    tables = sum(-(-(r + c) // case["page"]) * 4 for r, c in zip(rows, cached))
    if case["op"] == "rope":
        size = 2 if case["in"] != "f32" else 4
        heads = HEADS + 2 * KV_HEADS
        return {"bytes": N * D * heads * (size + 2) + N * 4 * case["axes"] + tables, "flops": N * D * heads * 6}
    pairs = keys = 0
    for r, c in zip(rows, cached):
        reach = case["window"] or r + c
        # query i of the slot sees min(c + i + 1, reach) keys
        full = max(0, min(r, reach - c))
        pairs += sum((c + 1, c + full)) * full // 2 + (r - full) * reach
        keys += min(r + c, reach + r - 1)
    return {"bytes": N * HEADS * D * 4 + keys * KV_HEADS * D * 4 + tables, "flops": 4 * HEADS * D * pairs}


# --------------------------------------------------------------------------------------- exact
def _exact_attention(s):
    rows, cached = _ints(s["rows"]), _ints(s["cached"])
    if sum((r + c) * r for r, c in zip(rows, cached)) > 200e6:
        return None
    out = torch.zeros(s["o"].shape, dtype=torch.float64, device="cuda")
    rep, at = HEADS // KV_HEADS, 0
    for b, (r, c) in enumerate(zip(rows, cached)):
        t = r + c
        ids = s["table"][b, :-(-t // s["page"])].long()
        dist = (torch.arange(r, device="cuda")[:, None] + c) - torch.arange(t, device="cuda")[None]
        hidden = dist < 0
        if s["window"]:
            hidden |= dist >= s["window"]
        for g in range(KV_HEADS):
            k = s["k_pool"][ids, g].reshape(-1, s["dim"])[:t].double()
            v = s["v_pool"][ids, g].reshape(-1, s["dim"])[:t].double()
            for h in range(g * rep, (g + 1) * rep):
                w = s["q"][at:at + r, h].double() @ k.T * s["scale"]
                w[hidden] = -math.inf
                w = torch.exp(w - w.max(1, keepdim=True).values)
                out[at:at + r, h] = (w @ v) / w.sum(1, keepdim=True)
        at += r
    return out


def _exact_rope(s):
    rows, cached, half = _ints(s["rows"]), _ints(s["cached"]), s["dim"] // 2
    norm = lambda x: x / (x.square().sum(-1, keepdim=True) / s["dim"] + EPS).sqrt()  # noqa: E731
    freqs, axis = s["freqs"].double(), s["pair_axis"].long()
    spin = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), freqs[None] * s["positions"].double()[axis, :].T)

    def turned(x, w):
        x = norm(x.double()) * w.double()
        z = torch.complex(x[..., :half], x[..., half:]) * spin[:, None]
        return torch.cat([z.real, z.imag], -1)

    k_pool, v_pool = s["k_pool"].double(), s["v_pool"].double()
    k, v, at = turned(s["k"], s["k_w"]), norm(s["v"].double()), 0
    for b, (r, c) in enumerate(zip(rows, cached)):
        place = torch.arange(c, c + r, device="cuda")
        page = s["table"][b].long()[place // s["page"]]
        k_pool[page, :, place % s["page"]] = k[at:at + r]
        v_pool[page, :, place % s["page"]] = v[at:at + r]
        at += r
    return turned(s["q"], s["q_w"]), k_pool, v_pool


def _exact_pages(s):
    come_from = torch.arange(s["pages"])
    come_from[s["dst"].long().cpu()] = s["src"].long().cpu()
    come_from = come_from.cuda()
    moved = []
    for p in s["pools"]:
        raw = p.view(torch.uint8) if p.element_size() == 1 else p       # bytes move as they are
        moved.append(raw[come_from].view(p.dtype))
    return moved


def exact(case, seed):
    s = prepare(case, seed)
    return {"attention": _exact_attention, "rope": _exact_rope, "pages": _exact_pages}[case["op"]](s)
