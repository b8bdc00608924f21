"""A step that finds no pages, or is too long for the table, was never announced: lengths, phases and what later requests
may share stay as they were."""
import numpy as np
import pytest

from g4b_b200.paging import OutOfPages, PagedKVManager

STATE = ("cache_offsets", "time_dim_sizes", "user_phase", "q_starts")


@pytest.mark.parametrize("how", ["packed", "prefill", "decode"])
@pytest.mark.parametrize("long,error", [(200, OutOfPages), (400, ValueError)])
def test_state_stays(how, long, error):
    m = PagedKVManager(num_pages=12, max_batch=3, max_context=320, page_size=16, prefill_chunk=16)
    prompt = list(range(64))
    a, _ = m.place_request(prompt)
    b, _ = m.place_request(list(range(1000, 1000 + long)))
    m.prepare_packed_inputs([0, 0, 0], [0, 0, 0])
    before = {n: getattr(m, n).copy() for n in STATE}
    rows = [0] * 3
    rows[a], rows[b] = 64, long
    with pytest.raises(error):
        if how == "packed":
            m.prepare_packed_inputs(rows, rows)
        else:
            (m.prepare_prefill_inputs if how == "prefill" else m.prepare_decode_inputs)(None, [0] * 3, rows)
    for n in STATE:
        assert np.array_equal(getattr(m, n), before[n]), n
    _, pos = m.place_request(prompt)
    assert pos == 0                              # nothing has been written that could be shared
    with pytest.raises(ValueError, match="no tokens"):
        m.fork(a)
    m.free(b)
    rows[b] = 0
    starts, _, times = m.prepare_packed_inputs(rows, rows)      # the step without the request that did not fit
    assert starts[-1] == 64 and times[a] == 64
