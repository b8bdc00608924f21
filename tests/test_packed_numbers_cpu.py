"""The plain numbers of the packed calls: what the padded calls take is taken, what does not fit is a ValueError."""
import numpy as np
import pytest

import test_gpu_attention_packed as attn
import test_gpu_rope_packed as rp
from g4b_b200.kernels import rope


def call_rope(c, page_size, eps=1e-6):
    rope.rope_norm_append_packed(c["q"], c["k"], c["v"], c["freqs"], c["positions"], c["starts"], c["times"], c["k_pool"], c["v_pool"], eps,
                                 block_tables=c["table"], page_size=page_size, pair_axis=c["pair_axis"], q_out=c["q_out"], stream=0)


@pytest.mark.parametrize("page", [16, 16.0, np.int64(16), np.float32(16)])
def test_taken(page):
    attn.call(attn.cpu_case(), page=page, window=np.int32(40), scale=np.float64(0.1), stage=np.int8(3))
    attn.call(attn.cpu_case(), page=page, window=40.0, scale=1)
    call_rope(rp.cpu_case(axes=3), page, eps=np.float32(1e-6))


@pytest.mark.parametrize("over", [dict(page=2 ** 40 + 16), dict(window=2 ** 31), dict(stage=2 ** 33 + 3), dict(scale=1e300), dict(scale=float("inf"))])
def test_refused(over):
    with pytest.raises(ValueError):
        attn.call(attn.cpu_case(), **over)


def test_refused_by_the_rotary():
    for page, eps in ((2 ** 40 + 16, 1e-6), (-2 ** 35, 1e-6), (16, 1e300)):
        with pytest.raises(ValueError):
            call_rope(rp.cpu_case(axes=3), page, eps)
