"""Forking, freeing and compacting on the host page manager, and the inputs of packed steps."""
import numpy as np
import pytest

from g4b_b200.paging import OutOfPages, PagedKVManager

PAGE = 16


def manager(num_pages=40, B=4, max_context=256, **kw):
    return PagedKVManager(num_pages=num_pages, max_batch=B, max_context=max_context, page_size=PAGE, **kw)


def place(m, n, first=0):
    slot, pos = m.place_request(list(range(first, first + n)))
    times = [0] * m.max_batch
    times[slot] = n
    m.prepare_prefill_inputs(None, [0] * m.max_batch, times)
    return slot


def check(m):
    """Reference counts, free list and tables agree."""
    refs = np.zeros(m.alloc.num_pages, dtype=int)
    for s in m.slots:
        for p in s.pages:
            refs[p] += 1
    assert (refs == m.alloc._refs).all()
    assert sorted(m.alloc._free) == list(np.flatnonzero(refs == 0))
    for i, s in enumerate(m.slots):
        assert list(m.block_tables[i, : len(s.pages)]) == s.pages and (m.block_tables[i, len(s.pages):] == -1).all()


@pytest.mark.parametrize("n", [1, 15, 16, 17, 32, 33, 100])
def test_fork_shares_full_pages_and_copies_the_last(n):
    m = manager()
    a = place(m, n)
    b, copies = m.fork(a)
    shared = (n - 1) // PAGE
    pa, pb = m.slots[a].pages, m.slots[b].pages
    assert b != a and m.slots[b].active and len(pb) == len(pa)
    assert pa[:shared] == pb[:shared] and not set(pa[shared:]) & set(pb[shared:])
    assert copies == [(pa[shared], pb[shared])]
    assert m.time_dim_sizes[b] == m.time_dim_sizes[a] and m.user_phase[b] == m.user_phase[a]
    check(m)
    m.retire(a)
    m.free(b)
    check(m)
    assert all(m.alloc.refcount(p) == 1 for p in pa)


def test_a_forked_pair_never_writes_one_row():
    """In decode the state is advanced before the step that writes the new token: the row of that
    token must not lie in a shared page, whatever the length."""
    for n in range(1, 3 * PAGE + 2):
        m = manager()
        a = place(m, n)
        m.prepare_decode_inputs(None, [n] + [0] * 3, [n + 1] + [0] * 3)
        for _ in range(3):
            m.advance_decode()
        t = int(m.time_dim_sizes[a])
        b, _ = m.fork(a)
        row_page = (t - 1) // PAGE
        assert m.slots[a].pages[row_page] != m.slots[b].pages[row_page]
        for _ in range(20):
            m.advance_decode()
            t = int(m.time_dim_sizes[a])
            assert m.slots[a].pages[(t - 1) // PAGE] != m.slots[b].pages[(t - 1) // PAGE]
        check(m)


def test_fork_of_a_fork_and_of_nothing():
    m = manager()
    a = place(m, 40)
    b, _ = m.fork(a)
    c, copies = m.fork(b)
    assert m.alloc.refcount(m.slots[a].pages[0]) == 3 and copies[0][0] == m.slots[b].pages[2]
    d, _ = m.fork(a)
    check(m)
    with pytest.raises(RuntimeError, match="no free slot"):
        m.fork(a)
    m.free(d)
    m.free(c)
    with pytest.raises(ValueError, match="no tokens"):
        m.fork(c)
    m.retire(b)
    with pytest.raises(ValueError, match="no tokens of a running"):
        m.fork(b)


def test_fork_drops_cached_pages_but_not_its_own():
    m = manager(num_pages=9, B=3)
    old = place(m, 64, first=500)             # 4 pages
    m.retire(old)
    a = place(m, 80)                          # 5 pages, the pool is full
    b, copies = m.fork(a)                     # the retired slot's pages make room
    assert len(copies) == 1
    check(m)
    m.free(b)
    m2 = manager(num_pages=5, B=3)
    a = place(m2, 80)
    with pytest.raises(OutOfPages):
        m2.fork(a)
    check(m2)
    assert len(m2.slots[a].pages) == 5 and m2.slots[a].active


def test_free_keeps_shared_pages():
    m = manager()
    a = place(m, 50)
    b, _ = m.fork(a)
    before = list(m.slots[b].pages)
    m.free(a)
    check(m)
    assert m.slots[b].pages == before and m.time_dim_sizes[a] == 0 and m.user_phase[a] == 0
    assert a in m.free_slots()


def test_compact_moves_pages_to_the_front():
    rng = np.random.default_rng(3)
    m = manager(num_pages=60, B=8)
    kept = np.arange(60) * 1000               # what each page holds
    for round_ in range(30):
        free = m.free_slots()
        if free:
            place(m, int(rng.integers(1, 150)), first=int(rng.integers(0, 10**6))) if m.alloc.free_pages > 12 else None
        busy = [i for i, s in enumerate(m.slots) if s.active]
        if len(busy) > 4:
            (m.free if rng.random() < 0.5 else m.retire)(int(rng.choice(busy)))
        elif busy and m.free_slots() and m.alloc.free_pages > 12:
            m.fork(int(rng.choice(busy)))
        held = [[kept[p] for p in s.pages] for s in m.slots]
        src, dst = m.compact()
        assert not set(src) & set(dst) and len(set(dst)) == len(dst) and src.dtype == dst.dtype == np.int32
        kept[dst] = kept[src]
        live = int((m.alloc._refs > 0).sum())
        assert (m.alloc._refs[live:] == 0).all()
        assert [[kept[p] for p in s.pages] for s in m.slots] == held
        check(m)
    assert m.compact()[0].size == 0


def test_packed_inputs():
    m = manager()
    a = place(m, 20)
    m.place_request(list(range(100, 150)))
    starts, tables, times = m.prepare_packed_inputs([1, 50, 0, 0], [21, 50, 0, 0])
    assert list(starts) == [0, 1, 51, 51, 51] and list(times) == [21, 50, 0, 0]
    assert list(m.cache_offsets[:2]) == [20, 0] and list(m.user_phase) == [1, 1, 0, 0]
    assert (tables[1, :4] >= 0).all() and len(m.slots[1].pages) == 4 and a == 0
    check(m)
    with pytest.raises(ValueError, match="entry for every slot"):
        m.prepare_packed_inputs([1], [2])
    with pytest.raises(ValueError, match="new rows"):
        m.prepare_packed_inputs([5, 0, 0, 0], [4, 0, 0, 0])
    with pytest.raises(ValueError, match="new rows"):
        m.prepare_packed_inputs([-1, 0, 0, 0], [4, 0, 0, 0])
