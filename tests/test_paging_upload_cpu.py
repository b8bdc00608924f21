"""What an upload copies: a step without packed rows costs what it did before there were any."""
import torch

from g4b_b200.paging import PagedKVManager


def test_starts_go_only_behind_a_packed_step(monkeypatch):
    m = PagedKVManager(num_pages=12, max_batch=3, max_context=64, page_size=16)
    m.bind_device("cpu")
    assert m.upload()["q_starts"].tolist() == [0, 0, 0, 0]
    m.prepare_packed_inputs([2, 0, 5], [2, 0, 9])
    assert m.upload()["q_starts"].tolist() == [0, 2, 2, 7]
    copied = []
    copy = torch.Tensor.copy_
    monkeypatch.setattr(torch.Tensor, "copy_", lambda self, other, **kw: (copied.append(tuple(self.shape)), copy(self, other, **kw))[1])
    m.prepare_decode_inputs(None, [2, 0, 9], [3, 0, 10])
    dev = m.upload()
    assert dev["q_starts"].tolist() == [0, 2, 2, 7] and dev["time_dim_sizes"].tolist() == [3, 0, 10]
    assert (4,) not in copied and copied.count((3,)) == 6
    m.bind_device("cpu")
    assert m.upload()["q_starts"].tolist() == [0, 2, 2, 7]
