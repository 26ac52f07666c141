"""What the warps of the windowed attention wait for (csrc/window_fwd.cu, window_bwd.cu), without a GPU: the two warps that
share the rows of a query tile in the forward, in every order that their steps can come in, and what each kind of warp
does when a wait gives up.

The steps are taken from the source, in its order: each warp puts a value into its stage, meets the other at a barrier and
reads the other's stage (``exchange``); at a unit's end it writes its results over its stage.  A value that is written
over before the other warp has read it is a race.  A wait for the copies or the tensor cores gives up after a while, in
either warp; a warp that meets one that has left waits for ever."""
from __future__ import annotations

import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "thetascan_b200", "csrc")
SOURCE = os.path.join(CSRC, "window_fwd.cu")
# what each step is made of; "meet" is the barrier of the two warps, "agree" one at which either can say that both leave
STEPS = {
    r"\bexchange\(": ("put", "meet", "read"),
    r"\bpair_meets\(": ("meet",),
    r"\bthreads_agree<64>\(": ("agree",),
    r"\bmbar_wait(?:_warp)?\(": ("wait",),
    r"\bif \(!ok\) break": ("leave",),
    r"\bst_shared_v4\(stage": ("over",),
}


def _steps():
    """The steps of a unit: of a key tile, and of its end."""
    with open(SOURCE) as f:
        text = f.read()
    text = re.sub(r"//.*", "", text[text.index("// ---- rows: two threads"):])
    text = text[text.index("for (int unit = blockIdx.x"):text.index("window_fwd_launch(")]
    found = sorted((m.start(), name) for name in STEPS for m in re.finditer(name, text))
    names = [name for _, name in found]
    last_of_tile = text.index("signal(&p_full[x])")
    assert names.count(r"\bexchange\(") == 2 and names.count(r"\bst_shared_v4\(stage") == 1
    return [n for at, n in found if at < last_of_tile], [n for at, n in found if at > last_of_tile]


def _program(tiles, units=2):
    """(what, place) of two units; a unit's exchanges use two places of the stage in turn, its results both."""
    tile, end = _steps()
    out, turn = [], 0
    for _ in range(units):
        for name in tile * tiles + end:
            out += [(what, turn & 1) for what in STEPS[name]]
            turn += name == r"\bexchange\("
    return out


def _faults(program):
    """What some order of the two warps' steps, with waits that give up in either, leads to: "race" where one writes over a
    value that the other has still to read, "hang" where one meets the other after that has left."""
    faults, seen, end = set(), set(), len(program)
    # next steps; places that hold a value not yet read; whether no wait has given up
    todo = [((0, 0), (frozenset(), frozenset()), (True, True))]
    while todo:
        state = todo.pop()
        if state in seen:
            continue
        seen.add(state)
        at, held, ok = state
        what = [program[i][0] if i < end else None for i in at]
        meets = [x in ("meet", "agree") for x in what]
        if all(meets):
            assert what[0] == what[1] and at[0] == at[1]
            both = at[0] + 1 if what[0] == "meet" or all(ok) else end
            todo.append(((both, both), held, ok))
        elif any(meets) and what[meets.index(False)] is None:
            faults.add("hang")
        for w in range(2):
            if what[w] is None or meets[w]:
                continue

            def go(step=at[w] + 1, now=held, fine=ok[w]):
                todo.append((tuple(step if n == w else i for n, i in enumerate(at)), tuple(now),
                             tuple(fine if n == w else o for n, o in enumerate(ok))))

            place, now = program[at[w]][1], list(held)
            if what[w] == "wait":
                go()
                go(fine=False)
            elif what[w] == "leave":
                go(step=at[w] + 1 if ok[w] else end)
            elif what[w] == "put":
                if place in held[w]:
                    faults.add("race")
                now[w] = held[w] | {place}
                go(now=now)
            elif what[w] == "read":
                now[1 - w] = held[1 - w] - {place}
                go(now=now)
            else:
                if held[w]:
                    faults.add("race")
                go()
    return faults


@pytest.mark.parametrize("tiles", [0, 1, 2, 4])   # none: a tile behind its sequence
def test_nothing_is_written_over_before_it_is_read(tiles):
    assert "race" not in _faults(_program(tiles))


@pytest.mark.parametrize("tiles", [0, 1, 2, 4])
def test_a_wait_that_gives_up_ends_both(tiles):
    assert "hang" not in _faults(_program(tiles))


@pytest.mark.parametrize("name,kernels", [("window_fwd.cu", 1), ("window_bwd.cu", 2)])
def test_the_lanes_of_a_warp_leave_together(name, kernels):
    """Each lane has its own outcome of a wait; those that stayed behind would wait for the others at the next instruction
    of the whole warp.  What ends or skips a turn of the row warps' loops is the same in all lanes."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//.*", lambda m: m.group() if "---- rows" in m.group() else "", f.read())
    rows = re.findall(r"// ---- rows:.*?tmem_dealloc", text, re.S)
    assert len(rows) == kernels
    alike = ("!threads_agree<", "!__all_sync(", "!mine.exists)", "!some[c])", "channel >= w.dim)")
    for part in rows:
        for condition in re.findall(r"if \((.*)(?:break|continue);", part):
            assert condition.startswith(alike), condition
        for condition in re.findall(r"for \(int n = 0;([^;]*);", part):
            assert "ok" not in condition


@pytest.mark.parametrize("name,kernels", [("window_fwd.cu", 1), ("window_bwd.cu", 2)])
def test_copies_in_flight_land_before_the_memory_goes(name, kernels):
    """A warp of loads that gives up waits, for a bounded time, on every barrier that a copy of its own may still complete."""
    with open(os.path.join(CSRC, name)) as f:
        parts = re.findall(r"// ---- loads(.*?)(// given up.*?)\} else if", f.read(), re.S)
    assert len(parts) == kernels
    for loads, given_up in parts:
        started = set(re.findall(r"&(\w*full)\b", loads))
        assert started and started == set(re.findall(r"&(\w*full)\b", given_up))


def test_faults_are_found():
    unread = [("put", 0), ("meet", 0), ("read", 0)]
    assert _faults(unread + [("over", 0)]) == {"race"} and _faults(unread + [("put", 0)]) == {"race"}
    assert not _faults(unread + [("meet", 0), ("over", 0)])
    assert not _faults(unread + [("put", 1), ("meet", 1), ("read", 1), ("put", 0)])
    assert _faults([("wait", 0), ("leave", 0), ("meet", 0)]) == {"hang"}
    assert not _faults([("wait", 0), ("agree", 0), ("meet", 0)])
