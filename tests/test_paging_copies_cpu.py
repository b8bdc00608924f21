"""Copies that several forks, frees and compactions hand out, launched together through copy_stages: the lists follow the
page copy's own rule for contradictions, and end where the copies one by one would."""
import random

import numpy as np
import pytest

from g4b_b200.paging import PagedKVManager, copy_stages
from test_gpu_page_copy import followed

PAGE = 16


def one_by_one(content, copies):
    content = list(content)
    for s, d in copies:
        content[d] = content[s]
    return content


def in_stages(content, copies):
    """As copy_pages carries the lists out: an entry that contradicts another would be skipped and recorded."""
    content = list(content)
    for src, dst in copy_stages(copies):
        assert src.dtype == dst.dtype == np.int32
        pairs, codes = followed(src.tolist(), dst.tolist(), len(content))
        assert not codes and len(pairs) == len(src)
        old = list(content)
        for s, d in pairs:
            content[d] = old[s]
    return content


def manager(num_pages=40, B=6):
    return PagedKVManager(num_pages=num_pages, max_batch=B, max_context=256, page_size=PAGE)


def place(m, n, first):
    slot, _ = m.place_request(list(range(first, first + n)))
    rows, times = [0] * m.max_batch, [0] * m.max_batch
    rows[slot] = times[slot] = n
    m.prepare_packed_inputs(rows, times)
    return slot


def test_fork_free_fork():
    """A beam pruned between two forks: the second copies into the page that the first reads."""
    m = manager()
    a, b = place(m, 40, 0), place(m, 40, 1000)
    held = list(range(40))
    want = held[m.slots[a].pages[2]]
    _, first = m.fork(a)
    m.free(a)
    _, second = m.fork(b)
    assert second[0][1] == first[0][0]                      # (else this tests nothing)
    after = in_stages(held, first + second)
    assert after == one_by_one(held, first + second) and after[first[0][1]] == want
    assert len(copy_stages(first + second)) == 2


def test_fork_of_a_fork():
    m = manager()
    a = place(m, 40, 0)
    b, first = m.fork(a)
    c, second = m.fork(b)
    held = list(range(40))
    after = in_stages(held, first + second)
    assert after[m.slots[c].pages[2]] == after[m.slots[b].pages[2]] == m.slots[a].pages[2]
    assert len(copy_stages(first + second)) == 1


def test_fork_and_compact():
    m = manager()
    a, b, c = place(m, 60, 0), place(m, 40, 1000), place(m, 50, 2000)
    held = list(range(40))
    want = [held[p] for p in m.slots[c].pages]
    new, copies = m.fork(c)
    m.free(a)
    copies = list(copies) + list(zip(*m.compact()))
    after = in_stages(held, copies)
    assert [after[p] for p in m.slots[c].pages] == want
    assert [after[p] for p in m.slots[new].pages] == want


def test_forks_of_different_sequences_are_one_list():
    m = manager()
    slots = [place(m, 30, 1000 * i) for i in range(3)]
    copies = sum((m.fork(s)[1] for s in slots), [])
    (src, dst), = copy_stages(copies)
    assert list(zip(src.tolist(), dst.tolist())) == copies


def test_nothing_and_padding():
    assert copy_stages([]) == [] and copy_stages([(-1, 3), (2, -1), (4, 4)]) == []


@pytest.mark.parametrize("seed", range(200))
def test_any_pairs(seed):
    rng = random.Random(seed)
    n = rng.randint(2, 12)
    copies = [(rng.randrange(n), rng.randrange(n)) for _ in range(rng.randint(1, 20))]
    assert in_stages(range(n), copies) == one_by_one(range(n), copies)


@pytest.mark.parametrize("seed", range(20))
def test_what_a_manager_hands_out(seed):
    """Random forks, frees and compactions between two steps: every sequence keeps what it held."""
    rng = random.Random(seed)
    m = manager(num_pages=60)
    for i in range(3):
        place(m, rng.randint(1, 120), 1000 * i)
    for _ in range(6):
        held, copies = list(range(60)), []
        value = {i: [held[p] for p in s.pages] for i, s in enumerate(m.slots) if s.active}
        length = {i: s.length for i, s in enumerate(m.slots) if s.active}
        for _ in range(rng.randint(1, 8)):
            busy = [i for i, s in enumerate(m.slots) if s.active]
            what = rng.choice(["fork", "fork", "free", "compact"])
            if what == "fork" and m.free_slots() and m.alloc.free_pages > 9:
                a = rng.choice(busy)
                b, c = m.fork(a)
                copies += c
                value[b], length[b] = value[a], length[a]
            elif what == "free" and len(busy) > 1:
                m.free(rng.choice(busy))
            elif what == "compact":
                copies += zip(*m.compact())
        after = in_stages(held, copies)
        for i, s in enumerate(m.slots):
            if s.active:
                n = -(-length[i] // PAGE)                   # pages that hold tokens
                assert [after[p] for p in s.pages[:n]] == value[i][:n]


@pytest.mark.gpu
def test_on_the_device(cuda):
    import torch

    from g4b_b200.kernels import pages

    m = manager()
    a, b = place(m, 40, 0), place(m, 40, 1000)
    pools = [torch.randn(40, 2, PAGE, 64, device=cuda) for _ in range(3)]
    read = lambda slot: [p[torch.tensor(m.slots[slot].pages, device=cuda)].clone() for p in pools]  # noqa: E731
    want_a, want_b = read(a), read(b)
    c, copies = m.fork(a)
    d, more = m.fork(c)
    copies += more
    m.free(a)
    e, more = m.fork(b)
    copies += more + list(zip(*m.compact()))
    for src, dst in copy_stages(copies):
        pages.copy_pages(pools, torch.from_numpy(src).to(cuda), torch.from_numpy(dst).to(cuda))
    for slot, want in ((b, want_b), (c, want_a), (d, want_a), (e, want_b)):
        assert all(torch.equal(x, y) for x, y in zip(read(slot), want))
