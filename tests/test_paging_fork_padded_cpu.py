"""Forks of slots whose last prefill chunk was padded, or that sat out the last step: no page that either sequence still
writes is shared, and every row that holds a token is in both."""
import numpy as np
import pytest

from g4b_b200.paging import PHASE_DECODE, PHASE_UNALLOCATED, OutOfPages, PagedKVManager

PAGE = 16


def manager(**kw):
    return PagedKVManager(**{"num_pages": 60, "max_batch": 4, "max_context": 512, "page_size": PAGE, **kw})


def prefill(m, n, chunk):
    """A prompt of n tokens in padded chunks, whose time counts the padding."""
    slot, pos = m.place_request(list(range(n)))
    while pos < n:
        off, times = [0] * m.max_batch, [0] * m.max_batch
        off[slot], times[slot] = pos, pos + chunk
        m.prepare_prefill_inputs(None, off, times)
        pos += chunk
    return slot


def decode_at(m, times):
    m.prepare_decode_inputs(None, [max(t - 1, 0) for t in times], times)


def rows_of(m, slot, content, n):
    return [content[m.slots[slot].pages[i // PAGE], i % PAGE] for i in range(n)]


@pytest.mark.parametrize("chunk", [16, 64, 128])
@pytest.mark.parametrize("n", [1, 15, 16, 17, 31, 32, 33, 63, 64, 65, 100])
@pytest.mark.parametrize("when", ["behind the prefill", "decode prepared", "decoding"])
def test_nothing_written_later_is_shared(n, chunk, when):
    m = manager()
    a = prefill(m, n, chunk)
    t = n
    if when != "behind the prefill":
        t += 1
        decode_at(m, [t if b == a else 0 for b in range(4)])
    if when == "decoding":
        for _ in range(5):
            m.advance_decode()
            t += 1
    content = np.full((60, PAGE), -1)
    for i in range(t):
        content[m.slots[a].pages[i // PAGE], i % PAGE] = i
    b, copies = m.fork(a)
    assert len({d for _, d in copies}) == len(copies) and not {s for s, _ in copies} & {d for _, d in copies}
    for s, d in copies:
        content[d] = content[s]
    assert rows_of(m, b, content, t) == rows_of(m, a, content, t) == list(range(t))
    # the row the next step writes, and those behind it that have pages, belong to one slot each
    first = t - 1 if when != "behind the prefill" else t
    for s in (a, b):
        assert all(m.alloc.refcount(p) == 1 for p in m.slots[s].pages[first // PAGE:])
    assert not set(m.slots[a].pages[first // PAGE:]) & set(m.slots[b].pages[first // PAGE:])
    decode_at(m, [t + 1 if s in (a, b) else 0 for s in range(4)])
    for _ in range(70):
        for s in (a, b):
            assert m.alloc.refcount(m.slots[s].pages[(int(m.time_dim_sizes[s]) - 1) // PAGE]) == 1
        m.advance_decode()


def test_only_the_last_token_s_page_is_copied_where_the_length_is_known():
    m = manager()
    a = prefill(m, 17, 64)
    decode_at(m, [18 if b == a else 0 for b in range(4)])
    b, copies = m.fork(a)
    assert copies == [(m.slots[a].pages[1], m.slots[b].pages[1])] and m.slots[a].pages[0] == m.slots[b].pages[0]
    assert m.user_phase[b] == PHASE_DECODE and m.time_dim_sizes[b] == 18 and m.cache_offsets[b] == 17


def test_a_chunk_past_the_prompt_counts_from_its_first_token():
    """A further turn, prefilled behind a prompt that the manager knows: every page that may hold a token is copied."""
    m = manager()
    a = prefill(m, 20, 32)
    m.prepare_prefill_inputs(None, [20 if b == a else 0 for b in range(4)], [52 if b == a else 0 for b in range(4)])
    b, copies = m.fork(a)
    pa, pb = m.slots[a].pages, m.slots[b].pages
    assert pa[0] == pb[0] or (pa[0], pb[0]) in copies
    assert copies == list(zip(pa[1:4], pb[1:4]))


def test_a_slot_that_sat_out_the_last_step_forks_with_all_its_tokens():
    m = manager()
    a = prefill(m, 40, 40)
    other, _ = m.place_request(list(range(1000, 1010)))
    rows, after = [0] * 4, [0] * 4
    rows[other] = after[other] = 10
    m.prepare_packed_inputs(rows, after)
    b, copies = m.fork(a)
    assert copies == [(m.slots[a].pages[2], m.slots[b].pages[2])]
    assert m.time_dim_sizes[b] == 40 and m.cache_offsets[b] == 40 and m.user_phase[b] == PHASE_UNALLOCATED
    rows, after = [0] * 4, [0] * 4
    for s in (a, b):
        rows[s], after[s] = 1, 41
    m.prepare_packed_inputs(rows, after)
    assert all(m.alloc.refcount(m.slots[s].pages[2]) == 1 for s in (a, b))


def test_a_prefix_that_was_just_placed_forks_at_its_own_length():
    """Nothing of the state that the slot's last request left behind is taken over."""
    m = manager(prefill_chunk=16)
    a = prefill(m, 70, 16)
    decode_at(m, [71 if b == a else 0 for b in range(4)])
    m.retire(a)
    slot, pos = m.place_request(list(range(40)) + [7, 8, 9])
    assert slot == a and pos == 32
    b, copies = m.fork(slot)
    assert m.time_dim_sizes[b] == 32 and m.user_phase[b] == PHASE_UNALLOCATED
    assert copies == [(m.slots[a].pages[1], m.slots[b].pages[1])]


def test_a_fork_that_finds_no_pages_leaves_the_prefix_cache():
    m = manager(num_pages=9, max_batch=3)
    old = prefill(m, 32, 16)                              # two pages, cached behind the request
    m.retire(old)
    m.prepare_packed_inputs([0] * 3, [0] * 3)
    a, _ = m.place_request(list(range(500, 510)))
    m.prepare_packed_inputs([10 if b == a else 0 for b in range(3)], [10 if b == a else 0 for b in range(3)])
    m.ensure(a, 7 * PAGE)                                 # seven pages reserved, none of them full
    b, _ = m.place_request([9] * 3)
    free = m.alloc.free_pages
    tables = m.block_tables.copy()
    with pytest.raises(OutOfPages):
        m.fork(a)
    assert len(m.slots[old].pages) == 2 and m.alloc.free_pages == free
    assert (m.block_tables == tables).all()
    slot, pos = (m.retire(b), m.place_request(list(range(32))))[1]
    assert pos == 31 // 16 * 16
