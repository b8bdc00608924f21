"""q_starts that contradict themselves: neither q nor a live page is written, and the device status word says so."""
import pytest
import torch

import test_gpu_rope_packed as rp
from g4b_b200 import _cabi

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("starts", [[0, 25, 5, 30], [0, 10, 20, 19], [0, 30, 30, 10], [-1, 10, 20, 30], [0, 10, 20, 1000], [30, 20, 10, 0],
                                    [0, 10, 2 ** 31 - 1, 30], [-2 ** 31, 10, 20, 30]])
@pytest.mark.parametrize("q_out", [True, False])
@pytest.mark.parametrize("D", [128, 256])
def test_nothing_is_appended(cuda, starts, q_out, D):
    c = rp.make(15, [10, 10, 10], [10, 40, 10], D=D)
    c["starts"].copy_(rp.i32(starts))
    before = {n: x.clone() for n, x in c.items() if isinstance(x, torch.Tensor)}
    rp.run(c, q_out=q_out)
    assert _cabi.device_status() == 0x107
    for n in ("k_pool", "v_pool", "q_out", "q", "k", "v"):
        assert torch.equal(c[n], before[n]), n


@pytest.mark.parametrize("B,at", [(40, 35), (200, 150), (200, 199), (1000, 31), (1000, 32), (1000, 999)])
def test_one_start_among_many(cuda, B, at):
    """Wherever it stands, and whichever slot a row belongs to."""
    c = rp.make(B, [2] * B, [20] * B, H=2, G=1, D=64)
    c["starts"][at] += 3                       # past the next one (the last: not the end of the rows that are there)
    before = {n: x.clone() for n, x in c.items() if isinstance(x, torch.Tensor)}
    rp.run(c)
    assert _cabi.device_status() == 0x107
    for n in ("k_pool", "v_pool", "q_out"):
        assert torch.equal(c[n], before[n]), n


@pytest.mark.parametrize("B", [1, 31, 32, 33, 63, 64, 65, 160])
def test_rows_in_front_and_empty_slots(cuda, B):
    """Starts that begin behind row 0, and slots without rows anywhere, are in order."""
    rows = [(i * 7) % 3 for i in range(B)]
    c = rp.make(B, rows, [r + 9 for r in rows], H=2, G=1, D=64, spare=8)
    for n in ("q", "k", "v"):
        c[n] = c[n].roll(4, 0)
    c["positions"] = c["positions"].roll(4, 1)
    c["starts"] += 4
    before = {n: x.clone() for n, x in c.items() if isinstance(x, torch.Tensor)}
    rp.run(c)
    assert torch.equal(c["q_out"][:4], before["q_out"][:4])
    owned = {n: (x[4:] if n in ("q", "k", "v", "q_out") else x) for n, x in c.items()}
    owned["positions"], owned["starts"] = c["positions"][:, 4:], c["starts"] - 4
    rp.check(owned, {n: (x[4:] if n in ("q", "k", "v", "q_out") else x) for n, x in before.items()})


@pytest.mark.parametrize("B", [3, 126, 127, 128, 129, 255, 256, 300])
@pytest.mark.parametrize("layout", ["aligned", "off by one", "strided"])
def test_layouts_of_the_starts(cuda, B, layout):
    rows = [(i * 5) % 4 for i in range(B)]
    c = rp.make(B + 1, rows, [r + 9 for r in rows], H=2, G=1, D=64)
    if layout != "aligned":
        wide = torch.full((2 * B + 4,), -7, dtype=torch.int32, device=cuda)
        view = wide[1:B + 2] if layout == "off by one" else wide[:2 * B + 2:2]
        c["starts"] = view.copy_(c["starts"])
    rp.both(c)
    c["starts"][B] = c["q"].shape[0] + 1
    before = {n: x.clone() for n, x in c.items() if isinstance(x, torch.Tensor)}
    rp.run(c)
    assert _cabi.device_status() == 0x107
    for n in ("k_pool", "v_pool", "q_out"):
        assert torch.equal(c[n], before[n]), n
