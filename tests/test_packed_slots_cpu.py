"""How many slots a packed step may have: more than any program's, and few enough that a look at all starts ends soon."""
import pytest
import torch

import test_gpu_rope_packed as rp


def test_slots_are_bounded():
    c = rp.cpu_case(axes=3)
    one = lambda *shape: torch.zeros([1] * len(shape), dtype=torch.int32).expand(*shape)  # noqa: E731
    for B, fine in ((1 << 24, True), ((1 << 24) + 1, False), (2 ** 31 - 2, False)):
        over = dict(starts=one(B + 1), times=one(B), table=one(B, 1))
        if fine:
            rp.call(c, **over)
        else:
            with pytest.raises(ValueError, match="slots"):
                rp.call(c, **over)
