"""Rows that the packed operators write must not lie over one another; layouts whose rows interleave are taken."""
import itertools

import pytest
import torch

import test_gpu_attention_packed as attn
import test_gpu_rope_packed as rp

D = 128


def view(n, h, row, head, dtype):
    return torch.zeros((n + 1) * max(row, 1) + (h + 1) * max(head, 1) + D, dtype=dtype).as_strided((n, h, D), (row, head, 1))


def overlap(n, h, row, head):
    """By looking at every element."""
    seen = [i * row + j * head for i in range(n) for j in range(h)]
    return any(abs(x - y) < D for x, y in itertools.combinations(seen, 2))


LAYOUTS = [(a, b) for a in (0, 8, 64, D - 8, D, D + 8, 2 * D, 3 * D, 5 * D, 7 * D, 8 * D, 9 * D + 8, 20 * D) for b in (0, 8, 64, D - 8, D, 2 * D, 3 * D, 4 * D + 8, 8 * D, 40 * D)]


@pytest.mark.parametrize("n,h", [(1, 4), (2, 4), (7, 4), (3, 2), (5, 1), (5, 8)])
def test_every_layout(n, h):
    c = rp.make(1, [n], [n], H=h, G=1, D=D, spare=0, device="cpu", dtype=torch.bfloat16)
    a = attn.make(1, [n], H=h, G=1, D=D, spare=0, device="cpu", dirty=False)
    for row, head in LAYOUTS:
        x = view(n, h, row, head, torch.bfloat16)
        calls = [("q_out", lambda: rp.call(c, q_out=x)), ("q", lambda: rp.call(c, q=x, q_out=None))]
        if (row > 0 or n == 1) and (head > 0 or h == 1):         # (others: "positive multiples")
            calls.append(("o", lambda: attn.call(a, o=x)))
        for name, call in calls:
            if overlap(n, h, row, head):
                with pytest.raises(ValueError, match=f"{name}: rows that are written"):
                    call()
            else:
                call()


def test_rows_that_are_only_read_may_be_one():
    c = rp.make(1, [4], [4], H=4, G=1, D=D, spare=0, device="cpu", dtype=torch.bfloat16)
    rp.call(c, q=torch.zeros(1, 1, D, dtype=torch.bfloat16).expand(4, 4, D), k=torch.zeros(1, 1, D, dtype=torch.bfloat16).expand(4, 1, D))
