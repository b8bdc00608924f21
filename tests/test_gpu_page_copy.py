"""Pages copied on the device, bit for bit, in pools of several types and sizes, and lists that
contradict themselves."""
import numpy as np
import pytest
import torch

from g4b_b200 import _cabi
from g4b_b200.kernels import pages
from g4b_b200.paging import PagedKVManager


def followed(src, dst, num_pages):
    """The entries of a list that are carried out, by the rule in the header, and what is recorded."""
    fine = [0 <= s < num_pages and 0 <= d < num_pages and s != d for s, d in zip(src, dst)]
    out, codes = [], set()
    for i, (s, d) in enumerate(zip(src, dst)):
        if s < 0 or d < 0 or s == d:
            continue
        if not fine[i]:
            codes.add(0x104)
            continue
        others = [j for j in range(len(src)) if j != i and fine[j]]
        if any(dst[j] == s for j in others) or any(dst[j] == d and j < i for j in others):
            codes.add(0x105)
            continue
        out.append((s, d))
    return out, codes


def i32(v, device="cpu"):
    return torch.tensor(v, dtype=torch.int32, device=device)


def make_pools(n, device, seed=0):
    g = torch.Generator().manual_seed(seed)
    shapes = [((n, 2, 16, 256), torch.bfloat16), ((n, 2, 16, 256), torch.float16), ((n, 1, 32, 128), torch.uint8), ((n, 1), torch.float32),
              ((n, 3, 16, 80), torch.float32), ((n, 5), torch.uint8), ((n, 7), torch.float16), ((n, 4, 64, 512), torch.bfloat16)]
    return [torch.randint(0, 120, s, generator=g).to(t).to(device) for s, t in shapes]


def test_the_rule_itself():
    assert followed([0, 1], [1, 0], 4) == ([], {0x105})
    assert followed([0, 2], [1, 1], 4) == ([(0, 1)], {0x105})
    assert followed([0, 1], [1, 2], 4) == ([(0, 1)], {0x105})
    assert followed([0, 0, -1, 3], [1, 2, 3, 3], 4) == ([(0, 1), (0, 2)], set())
    assert followed([9, 0], [1, 9], 4) == ([], {0x104})


def test_refusals():
    a, b = torch.zeros(4, 8), torch.zeros(4, 2, dtype=torch.uint8)
    pages.copy_pages([a, b], i32([0]), i32([1]), stream=0)
    pages.copy_pages([], i32([0]), i32([1]), stream=0)
    pages.copy_pages([a], i32([]), i32([]), stream=0)
    with pytest.raises(ValueError, match="same number of pages"):
        pages.copy_pages([a, torch.zeros(5, 8)], i32([0]), i32([1]), stream=0)
    with pytest.raises(ValueError, match="contiguous"):
        pages.copy_pages([a[:, ::2]], i32([0]), i32([1]), stream=0)
    with pytest.raises(ValueError, match="one length"):
        pages.copy_pages([a], i32([0, 1]), i32([1]), stream=0)
    with pytest.raises(ValueError, match="int32"):
        pages.copy_pages([a], torch.tensor([0]), torch.tensor([1]), stream=0)
    with pytest.raises(ValueError, match="one length"):
        pages.copy_pages([a], i32([[0]]), i32([[1]]), stream=0)
    with pytest.raises(TypeError):
        pages.copy_pages([a], [0], [1], stream=0)
    with pytest.raises(ValueError, match="65536"):
        pages.copy_pages([a], torch.zeros(65537, dtype=torch.int32), torch.zeros(65537, dtype=torch.int32), stream=0)


@pytest.mark.launches_allowed
def test_host_tensors_are_refused():
    with pytest.raises(ValueError, match="CUDA tensor"):
        pages.copy_pages([torch.zeros(4, 8)], i32([0]), i32([1]), stream=0)


@pytest.mark.gpu
@pytest.mark.parametrize("n,copies", [(2, 1), (9, 4), (40, 1), (300, 150), (2000, 700)])
def test_bit_exact_in_every_pool(cuda, n, copies):
    pools = make_pools(n, cuda, seed=n)
    want = [p.clone() for p in pools]
    order = torch.randperm(n, generator=torch.Generator().manual_seed(copies))
    src, dst = order[:copies], order[n - copies:]
    for w in want:
        w[dst.to(cuda)] = w[src.to(cuda)]
    pages.copy_pages(pools, src.to(cuda, torch.int32), dst.to(cuda, torch.int32))
    for p, w in zip(pools, want):
        assert torch.equal(p, w)


@pytest.mark.gpu
def test_unaligned_pools_and_strided_lists(cuda):
    base = torch.arange(4 * 64 + 3, device=cuda, dtype=torch.int32).to(torch.uint8)
    pools = [base[o:o + 256].view(4, 64) for o in (1, 2, 3)][:1]
    want = [p.clone() for p in pools]
    want[0][3] = want[0][0]
    lists = i32([[0, 3], [-1, -1]], cuda)
    pages.copy_pages(pools, lists[:, 0], lists[:, 1])
    assert torch.equal(pools[0], want[0])


@pytest.mark.gpu
def test_one_page_to_many(cuda):
    pool = torch.randn(50, 2, 16, 256, device=cuda)
    pages.copy_pages([pool], i32([7] * 40, cuda), i32([i for i in range(41) if i != 7], cuda))
    assert all(torch.equal(pool[i], pool[7]) for i in range(41))


@pytest.mark.gpu
@pytest.mark.parametrize("seed", range(4))
def test_contradicting_lists_follow_the_rule(cuda, seed):
    rng = np.random.default_rng(seed)
    n, k = 30, [3, 12, 40, 400][seed]
    src, dst = rng.integers(-1, n + 1, k).tolist(), rng.integers(-1, n + 1, k).tolist()
    pools = make_pools(n, cuda, seed)
    want = [p.clone() for p in pools]
    pairs, codes = followed(src, dst, n)
    for w, p in zip(want, pools):
        for s, d in pairs:
            w[d] = p[s]
    pages.copy_pages(pools, i32(src, cuda), i32(dst, cuda))
    for p, w in zip(pools, want):
        assert torch.equal(p, w)
    status = _cabi.device_status()
    assert status in codes if codes else status == 0


@pytest.mark.gpu
def test_more_pools_than_a_launch_takes(cuda):
    pools = [torch.full((3, 16), float(i), device=cuda) for i in range(400)]
    for p in pools:
        p[0] += 0.5
    pages.copy_pages(pools, i32([0], cuda), i32([2], cuda))
    for i, p in enumerate(pools):
        assert p[2, 0].item() == i + 0.5 and p[1, 0].item() == i


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    pool = torch.zeros(70000, 65536, dtype=torch.uint8, device=cuda)      # 4.6 GB
    pool[69999] = 7
    pages.copy_pages([pool], i32([69999], cuda), i32([69998], cuda))
    assert bool((pool[69998] == 7).all()) and not bool(pool[69997].any())


@pytest.mark.gpu
def test_captured_on_another_stream_with_a_list_that_changes(cuda):
    pool = torch.randn(20, 64, device=cuda)
    src, dst = i32([-1] * 6, cuda), i32([-1] * 6, cuda)
    pages.copy_pages([pool], src, dst)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=side):
        pages.copy_pages([pool], src, dst)
    for pairs in ([(0, 1)], [(2, 3), (2, 4), (5, 6)]):
        want = pool.clone()
        src.fill_(-1)
        for i, (s, d) in enumerate(pairs):
            src[i], dst[i] = s, d
            want[d] = pool[s]
        graph.replay()
        assert torch.equal(pool, want)


@pytest.mark.gpu
def test_manager_forks_and_compacts_pools(cuda):
    """What the manager says is copied; the forked and moved sequences read what they read before."""
    m = PagedKVManager(num_pages=24, max_batch=4, max_context=128, page_size=16)
    m.bind_device(cuda)
    pools = [torch.randn(24, 2, 16, 256, device=cuda) for _ in range(3)]
    slots = []
    for n in (40, 70):
        slot, _ = m.place_request(list(range(n * 100, n * 100 + n)))
        m.prepare_prefill_inputs(None, [0] * 4, [n if i == slot else 0 for i in range(4)])
        slots.append((slot, n))
    read = lambda slot, n: [p[torch.as_tensor(m.block_tables[slot, : -(-n // 16)]).long().to(cuda)].transpose(1, 2).reshape(-1, 2, 256)[:n].clone() for p in pools]  # noqa: E731
    before = read(*slots[1])
    new, copies = m.fork(slots[1][0])
    s, d = zip(*copies)
    pages.copy_pages(pools, i32(s, cuda), i32(d, cuda))
    assert all(torch.equal(a, b) for a, b in zip(read(new, 70), before))
    m.free(slots[0][0])
    src, dst = m.compact()
    assert len(src)
    pages.copy_pages(pools, torch.from_numpy(src).to(cuda), torch.from_numpy(dst).to(cuda))
    for slot in (slots[1][0], new):
        assert all(torch.equal(a, b) for a, b in zip(read(slot, 70), before))
    dev = m.upload()
    torch.cuda.synchronize()
    assert torch.equal(dev["block_tables"].cpu(), torch.from_numpy(m.block_tables))
