"""The compiled argument packing gives the bytes of the Python one, and leaves to it what it does not take."""
import pytest
import torch

from g4b_b200 import _cabi
from g4b_b200.kernels import fa2, pages


class Like:
    """A tensor-like that is not torch's."""

    def __init__(self, t):
        self.shape, self.dtype, self.t = tuple(t.shape), str(t.dtype).replace("torch.", ""), t
        self.stride = tuple(t.stride())

    def data_ptr(self):
        return self.t.data_ptr()


def python_views(*tensors):
    fast, _cabi._fast = _cabi._fast, None
    try:
        return _cabi.views(*tensors)
    finally:
        _cabi._fast = fast


def some_tensors():
    x = torch.arange(2 * 3 * 4 * 5 * 6, dtype=torch.float32).view(2, 3, 4, 5, 6)
    return [x, x[..., 0], x.permute(4, 2, 0, 1, 3), x[0, 0, 0, 0], x[:, :0], torch.tensor(3.0), x.half()[1:, ::2], x.bfloat16(), x.int(),
            x.long()[:, 1], x.to(torch.uint8), x[0].to(torch.float8_e4m3fn), x.expand(2, 3, 4, 5, 6), torch.empty(0, dtype=torch.int32), None]


def test_the_module_is_built_and_loaded():
    _cabi.load()
    assert _cabi._fast is not None


def test_same_bytes():
    _cabi.load()
    for t in some_tensors():
        assert _cabi._fast.views(False, (t,)) == python_views(t)
    every = tuple(some_tensors())
    assert _cabi.views(*every) == python_views(*every) == b"".join(python_views(t) for t in every)


def test_what_it_does_not_take():
    _cabi.load()
    x = torch.zeros(2, 3)
    for other in (Like(x), [1, 2], x.double(), torch.zeros(1, 1, 1, 1, 1, 1), torch.zeros(3, dtype=torch.bool)):
        assert _cabi._fast.views(False, (x, other)) is None
    assert _cabi._fast.views(True, (x,)) is None                     # host memory
    assert _cabi.views(Like(x)) == _cabi.views(x)
    with pytest.raises(TypeError, match="unsupported dtype"):
        _cabi.views(x.double())
    with pytest.raises(ValueError, match="rank > 5"):
        _cabi.views(torch.zeros(1, 1, 1, 1, 1, 1))
    with pytest.raises(TypeError, match="tensor-like"):
        _cabi.views([1, 2])


def test_calls_with_and_without_it_agree(monkeypatch):
    """Valid and refused calls, torch tensors and other tensor-likes, through either packing."""
    q, pool = torch.zeros(5, 4, 128, dtype=torch.half), torch.zeros(3, 2, 16, 128, dtype=torch.half)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32)  # noqa: E731
    a = [q, pool, pool, q, i32([0, 2, 5]), i32([2, 9])]
    table, w = torch.zeros(2, 1, dtype=torch.int32), torch.empty(fa2.packed_workspace_bytes(5, 2, 4, 2), dtype=torch.uint8)
    for fast in (True, False):
        if not fast:
            monkeypatch.setattr(_cabi, "_fast", None)
        fa2.flash_attention_packed(*a, block_tables=table, workspace=w, stream=0)
        fa2.flash_attention_packed(Like(q), *a[1:], block_tables=table, workspace=w, stream=0)
        with pytest.raises(ValueError, match="scale"):
            fa2.flash_attention_packed(*a, block_tables=table, workspace=w, scale=-1.0, stream=0)
        with pytest.raises(ValueError, match="B rows"):
            fa2.flash_attention_packed(*a, block_tables=table[:1], workspace=w, stream=0)
        pages.copy_pages([pool, pool], i32([0]), i32([1]), stream=0)
        pages.copy_pages([], i32([0]), i32([1]), stream=0)
        with pytest.raises(ValueError, match="same number"):
            pages.copy_pages([pool, torch.zeros(4)], i32([0]), i32([1]), stream=0)
        with pytest.raises(ValueError, match="contiguous"):
            pages.copy_pages([pool, pool[..., ::2]], i32([0]), i32([1]), stream=0)
