"""The two warps that share the rows of a query tile in the windowed attention's forward (csrc/window_fwd.cu), in every
order that their steps can come in, without a GPU.

The steps are taken from the source, in its order: each warp puts a value into its stage, meets the other at a barrier and
reads the other's stage (``exchange``); at a unit's end it writes its results over its stage.  A value that is written
over before the other warp has read it is a race."""
from __future__ import annotations

import os
import re

import pytest

SOURCE = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thetascan_b200", "csrc", "window_fwd.cu")
# what each step is made of; "meet" is the barrier of the two warps
STEPS = {
    "exchange": ("put", "meet", "read"),
    "pair_meets": ("meet",),
    "store": ("over",),
}


def _steps():
    """The steps of a unit: of a key tile, and of its end."""
    with open(SOURCE) as f:
        text = f.read()
    text = re.sub(r"//.*", "", text[text.index("// ---- rows: two threads"):])
    text = text[text.index("for (int unit = blockIdx.x"):text.index("window_fwd_launch(")]
    found = [(m.start(), m.group()) for m in re.finditer(r"\bexchange\(|\bpair_meets\(|\bst_shared_v4\(stage", text)]
    names = ["store" if n.startswith("st_") else n[:-1] for _, n in found]
    assert names.count("exchange") == 2 and names.count("store") == 1
    tile = names.index("exchange") + 1
    return names[:tile], names[tile:]


def _program(tiles, units=2):
    """(what, place) of two units; a unit's exchanges use two places of the stage in turn, its results both."""
    tile, end = _steps()
    out, turn = [], 0
    for _ in range(units):
        for name in tile * tiles + end:
            out += [(what, turn & 1) for what in STEPS[name]]
            turn += name == "exchange"
    return out


def _races(program):
    """Whether some order of the two warps' steps writes over a value that the other has still to read."""
    seen, todo = set(), [((0, 0), (frozenset(), frozenset()))]   # next steps; places that hold a value not yet read
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        at, held = state
        what = [program[i][0] if i < len(program) else None for i in at]
        if what[0] == what[1] == "meet":
            todo.append(((at[0] + 1, at[1] + 1), held))
        for w in range(2):
            if what[w] in (None, "meet"):
                continue
            place, now = program[at[w]][1], list(held)
            if what[w] == "put":
                if place in held[w]:
                    return True
                now[w] = held[w] | {place}
            elif what[w] == "read":
                now[1 - w] = held[1 - w] - {place}
            elif held[w]:
                return True
            todo.append((tuple(i + (n == w) for n, i in enumerate(at)), tuple(now)))
    return False


@pytest.mark.parametrize("tiles", [0, 1, 2, 5])   # none: a tile behind its sequence
def test_nothing_is_written_over_before_it_is_read(tiles):
    assert not _races(_program(tiles))


def test_a_missing_barrier_is_found():
    assert _races([("put", 0), ("meet", 0), ("read", 0), ("over", 0)])
    assert _races([("put", 0), ("meet", 0), ("read", 0), ("put", 0)])
    assert not _races([("put", 0), ("meet", 0), ("read", 0), ("meet", 0), ("over", 0)])
    assert not _races([("put", 0), ("meet", 0), ("read", 0), ("put", 1), ("meet", 1), ("read", 1), ("put", 0)])
