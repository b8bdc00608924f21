"""The hand-over of probabilities in the two prompt kernels, followed through every interleaving on a model of their barriers.

In tile j a softmax warp waits for the scores S(j), may wait for P.V(j-1) (a barrier with one phase bit) and hands P(j) to the issuer,
which multiplies once all warps have; behind the last tile it waits for the last product.  Two warps of any speed, the issuer and the
tensor pipe, whose products end in the order they were issued in.  Which steps a path through a tile takes, and in which order, is read from the
kernels' source.  No state may be reached in which nobody can go on before all is done, and no wait may pass before what it waits for."""
import itertools
import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "g4b_b200" / "csrc"
TILES = 4
# the issuer: two tiles of scores ahead, then products and scores in turn
ISSUED = [("S", 0), ("S", 1)] + [x for j in range(TILES) for x in [("PV", j)] + [("S", j + 2)] * (j + 2 < TILES)]


def program(tiles):
    """What a warp does whose tile j takes the path tiles[j], a list of "wait" (where j > 0) and "hand"."""
    out = []
    for j, path in enumerate(tiles):
        out.append(("scores", j))
        for step in path:
            if step == "hand":
                out.append((step, j))
            elif j > 0:
                out.append(("wait", j - 1))
    return out + [("wait", TILES - 1)]


def goes_wrong(first, second):
    """"stuck", "early" or None: two warps with these programs, in every interleaving."""
    programs = (first, second)
    hand_at = [[p.index(("hand", j)) for j in range(TILES)] for p in programs]
    done_pv = [sum(kind == "PV" for kind, _ in ISSUED[:n]) for n in range(len(ISSUED) + 1)]
    done_s = [sum(kind == "S" for kind, _ in ISSUED[:n]) for n in range(len(ISSUED) + 1)]
    start = (0, 0, 0, 0)                                # steps of either warp; products and scores issued, and done
    seen, todo = {start}, [start]
    while todo:
        a, b, issued, done = todo.pop()
        after = []
        for warp, at in enumerate((a, b)):
            if at == len(programs[warp]):
                continue
            step, j = programs[warp][at]
            if step == "scores":
                free = j < done_s[done]
            elif step == "hand":
                free = True
            else:                                       # product j counts as done while the bit of the phase at hand differs from j's
                free = (done_pv[done] & 1) != (j & 1)
                if free and done_pv[done] <= j:
                    return "early"
            if free:
                after.append((a + (warp == 0), b + (warp == 1), issued, done))
        if issued < len(ISSUED):
            kind, j = ISSUED[issued]
            if kind == "S" or all(at > hand_at[w][j] for w, at in enumerate((a, b))):
                after.append((a, b, issued + 1, done))
        if done < issued:
            after.append((a, b, issued, done + 1))
        if not after and (a, b) != (len(first), len(second)):
            return "stuck"
        for s in after:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return None


def any_mixture(paths):
    """The first failure over all ways to send two warps through the paths (warps of other rows choose for themselves)."""
    programs = {tuple(program(tiles)) for tiles in itertools.product(paths, repeat=TILES)}
    return next((wrong for x in programs for y in programs if (wrong := goes_wrong(x, y))), None)


def test_the_model():
    assert any_mixture([["wait", "hand"]]) is None
    assert any_mixture([["hand", "wait"]]) == "stuck"
    assert any_mixture([["hand"]]) == "early"


def paths(name):
    text = (CSRC / name).read_text()
    text = text[text.index("softmax / epilogue"):]
    loop = text[text.index("for (int j = 0; j < n_tiles && ok; ++j) {"):text.index("m_carry = m_used")]
    for part in loop.split("continue;"):
        steps = re.findall(r"mbar_wait\(bar_pv|arrive_issuer\((?:q2 == 0 \? bar_pa : )?bar_pb\)", part)
        yield ["hand" if "bar_pb" in s else "wait" for s in steps]


@pytest.mark.parametrize("name,count", [("prefill_sm100.cu", 3), ("prefill_packed_sm100.cu", 2)])
def test_no_path_goes_wrong(name, count):
    found = list(paths(name))
    assert len(found) == count and all(sorted(p) == ["hand", "wait"] for p in found), found
    assert any_mixture(found) is None
