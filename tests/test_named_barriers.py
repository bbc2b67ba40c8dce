"""A warp whose bounded wait ran out must not leave others behind a barrier.

The product kernel's epilogues may join the four warps of a column half at named
barriers (finish()); a warp that leaves settles them in give_up().  The barriers
count arrivals, not warps.  The sequences are read from the source and run on a
model of the hardware's counters, in every order: on the GPU the case would need
a wait that runs out."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "aethelstream_b200", "csrc")
WARPS, TILES = 4, 2


def body(text, start):
    """The text between the brace that follows `start` and its partner."""
    at = text.index("{", start)
    depth = 0
    for i in range(at, len(text)):
        depth += {"{": 1, "}": -1}.get(text[i], 0)
        if depth == 0:
            return text[at + 1:i]
    raise AssertionError("unbalanced braces")


def epilogues():
    """name -> ([barriers of finish], [barriers of give_up]); a barrier is (waits, its id's expression)."""
    out = {}
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"struct (\w+)(?= \{)", text):
            b = body(text, m.end())
            if "give_up(" not in b:
                continue

            def bars(fn):
                return [(w == "", e) for w, e in re.findall(r"named_bar(_arrive|)\((.*?), 128\)", body(b, b.index(fn)))]

            out[m.group(1)] = (bars("void finish("), bars("void give_up("))
    return out


def stuck(finish, give_up):
    """A reachable state in which warps wait at a barrier and nothing can move, or None.

    A warp's state is (tile, what it does there: None before its accumulator, its
    list of barriers, how many it has passed, whether it waits at the next); a
    barrier's is (arrivals, the warps that wait).  `abort` is set by the first warp
    whose wait runs out; a warp that sees it gives up too."""
    ids = sorted({e for _, e in finish + give_up})
    start = (((0, None, 0, False),) * WARPS, tuple((0, frozenset()) for _ in ids), False)
    seen, todo = {start}, [start]
    while todo:
        warps, bars, abort = todo.pop()
        moves = []
        for i, (tile, act, at, waits) in enumerate(warps):
            def put(w, b=bars, a=abort):
                moves.append((warps[:i] + (w,) + warps[i + 1:], b, a))
            if tile == TILES or waits:
                continue
            if act is None:  # waits for the accumulator, bounded
                put((tile, "give_up", 0, False), a=True)
                if not abort:
                    put((tile, "finish", 0, False))
                continue
            steps = finish if act == "finish" else give_up
            if at == len(steps):
                put((tile + 1 if act == "finish" else TILES, None, 0, False))
                continue
            blocks, e = steps[at]
            k = ids.index(e)
            count, held = bars[k][0] + 1, bars[k][1] | ({i} if blocks else set())
            new = list(warps)
            new[i] = (tile, act, at + 1, blocks)
            if count == WARPS:
                for j in held:
                    new[j] = new[j][:3] + (False,)
                count, held = 0, frozenset()
            moves.append((tuple(new), bars[:k] + ((count, frozenset(held)),) + bars[k + 1:], abort))
        if not moves and any(w[3] for w in warps):
            return warps, bars
        for s in moves:
            if s not in seen:
                seen.add(s)
                todo.append(s)
    return None


def test_the_model():
    """What it must find: one barrier settled twice, or waited for by those who leave."""
    a, b = (True, "1"), (True, "2")
    arrive = lambda x: (False, x[1])  # noqa: E731
    assert stuck([a], [arrive(a)]) is None and stuck([], []) is None
    assert stuck([a, b], [arrive(a), arrive(b)]) is None
    assert stuck([a, a], [arrive(a), arrive(a)])  # both arrivals may fall into the first wait
    assert stuck([a, a], [a, a])  # the warp that left is missing at the next tile
    assert stuck([a, b], [arrive(a)]) and stuck([a], [])


def test_epilogues_with_barriers_are_found():
    assert {n for n, (f, _) in epilogues().items() if f} == {"HeadStatsT"}


@pytest.mark.parametrize("name", sorted(epilogues()))
def test_a_warp_that_gives_up_leaves_nobody_waiting(name):
    finish, give_up = epilogues()[name]
    assert stuck(finish, give_up) is None


def loops():
    """(file, text) of every `for` loop in the kernels that waits at a named barrier."""
    out = []
    for name in sorted(os.listdir(CSRC)):
        with open(os.path.join(CSRC, name)) as f:
            text = re.sub(r"//[^\n]*", "", f.read())
        for m in re.finditer(r"\bfor \(", text):
            depth, i = 1, m.end()
            while depth:
                depth += {"(": 1, ")": -1}.get(text[i], 0)
                i += 1
            if not text[i:].lstrip().startswith("{"):
                continue
            b = body(text, i)
            if re.search(r"named_bar\(", b):
                out.append((name, b))
    return out


def test_no_warp_leaves_such_a_loop_by_itself():
    """After a bounded wait the warps vote, or the one that leaves settles the barrier."""
    waits = 0
    for name, b in loops():
        for m in re.finditer(r"mbar_wait\(", b):
            waits += 1
            leave = b.find("break;", m.end())
            assert leave < 0 or re.search(r"named_bar_and\(|named_bar_arrive\(", b[m.end():leave]), (name, b[m.start():leave + 6])
    assert waits >= 4  # both projections, the weight write's, the ring's
