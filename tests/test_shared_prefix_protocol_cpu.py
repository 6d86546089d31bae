"""CPU models of what the shared-prefix kernels (csrc/shared_prefix.cu) leave behind when a wait runs out:
no copy into shared memory may be in flight when a CTA ends, and every partial that was not computed has
to be marked.  Each model walks the kernel's own steps and slot arithmetic and stops at every wait in turn.
And a model of the plan's counts for lists that name more pieces than there can be."""
import random

import pytest

RING = 4  # pieces_kernel: 16-key tiles of a warp's ring


def pieces_warp(tiles, stop, drain=True):
    """One piece of `tiles` tiles whose waits run out at step `stop` (of two tiles), behind a ring that has
    taken any number of tiles before.  Returns the copies in flight at the end, by tile."""
    asked = set(range(min(RING, tiles)))  # the first RING tiles
    taken = set()
    k = 0
    while k < tiles:
        if k == stop:
            break
        taken |= {t for t in (k, k + 1) if t < tiles}
        asked |= {t for t in (k + RING, k + RING + 1) if t < tiles and k + RING < tiles}
        k += 2
    else:
        return asked - taken
    waited = set(range(k, min(tiles, k + RING))) if drain else set()
    assert waited <= asked, "a wait for a tile that was never asked for would only end by its limit"
    for uses in range(2 * RING):  # the slots' phases: each slot is waited for once, one phase past the last taken
        slots = [(uses + t) % RING for t in waited]
        assert len(slots) == len(set(slots))
        for t in waited:
            before = [u for u in taken if (uses + u) % RING == (uses + t) % RING]
            assert all((uses + u) // RING < (uses + t) // RING for u in before)
            assert t < RING or (uses + t) // RING - 1 in [(uses + u) // RING for u in before]
    return asked - taken - waited


@pytest.mark.parametrize("tiles", range(1, 40))
def test_pieces_leave_no_copy_in_flight(tiles):
    for stop in range(0, tiles, 2):
        assert not pieces_warp(tiles, stop)
        assert pieces_warp(tiles, stop, drain=False)  # what the model is there to see


def loader(blocks, stop, k_slots, v_slots, counts=2):
    """prefix_kernel's loads of K and V blocks, stopped at wait number `stop` (None: never).  Returns the
    copies in flight after the drain: ('k' or 'v', block).  counts=1: K drained by the count of V blocks."""
    flight, keys, j, waits = set(), 0, 0, 0
    while j < blocks:
        if waits == stop:  # the K slot is not free
            break
        waits += 1
        flight.add(("k", j))
        keys = j + 1
        if waits == stop:  # the V slot is not free
            break
        waits += 1
        flight.add(("v", j))
        j += 1
    for i in range(k_slots + v_slots):
        kind, n, slot = ("k", k_slots, i) if i < k_slots else ("v", v_slots, i - k_slots)
        asked = keys if kind == "k" and counts == 2 else j
        if asked <= slot:
            continue
        use = (asked - 1 - slot) // n
        last = use * n + slot
        assert last < asked <= last + n, "the last use of the slot"
        flight -= {(kind, b) for b in range(slot, last + 1, n)}  # the phase before is complete, too
    return flight


@pytest.mark.parametrize("k_slots", [2, 3])
@pytest.mark.parametrize("blocks", [1, 2, 3, 4, 7, 12])
def test_the_loader_leaves_no_copy_in_flight(blocks, k_slots):
    for stop in [None] + list(range(2 * blocks)):
        assert not loader(blocks, stop, k_slots, 2)
    assert any(loader(blocks, stop, k_slots, 2, counts=1) for stop in range(2 * blocks))


@pytest.mark.parametrize("pieces,warps", [(1, 4), (7, 4), (50, 12), (12, 12)])
def test_every_piece_of_a_warp_that_stops_is_marked(pieces, warps):
    """Pieces go round the warps; one that stops marks the piece it is at and all that it had left."""
    for who in range(warps):
        mine = list(range(who, pieces, warps))
        for at in range(len(mine)):
            written = set(mine[:at])
            marked = {mine[at]}
            piece = mine[at] + warps
            while piece < pieces:
                marked.add(piece)
                piece += warps
            others = {p for p in range(pieces) if p % warps != who}
            assert written | marked | others == set(range(pieces)) and not written & marked


def plan(work, cap=(1 << 26) - 1):
    """pieces_kernel's scan: `work` is (splits, row blocks * heads) by segment; the pieces before each segment
    and in all, each lane counting a run of segments in 32 bits."""
    segs = len(work)
    run = -(-segs // 32)
    first, total = [0] * segs, 0
    for lane in range(32):
        mine = 0
        for s in range(min(segs, lane * run), min(segs, lane * run + run)):
            first[s] = total + mine
            mine = min(mine + work[s][0] * work[s][1], cap) if cap else mine + work[s][0] * work[s][1]
        total += mine
    wrap = lambda v: (v + (1 << 31)) % (1 << 32) - (1 << 31)  # noqa: E731
    return [wrap(v) for v in first] + [wrap(total)]


@pytest.mark.parametrize("segs", [1, 3, 32, 33, 1000, 4096])
def test_the_plan_ascends_whatever_the_lists_say(segs):
    """Also where every sequence claims all rows there can be (2^30 row-heads): a count that wrapped around
    would name pieces and rows before the workspace."""
    rnd = random.Random(segs)
    fair = [(rnd.randint(0, 9), rnd.randint(0, 40)) for _ in range(segs)]
    assert plan(fair) == plan(fair, cap=None) and plan(fair)[-1] == sum(a * b for a, b in fair)
    wild = [(rnd.choice((0, 1, 1 << 10, 1 << 24)), rnd.choice((0, 8, 1 << 20, 1 << 27))) for _ in range(segs)]
    for work in (wild, [(1 << 24, 1 << 27)] * segs, [(1, 1 << 27)] * segs):
        first = plan(work)
        assert all(0 <= a <= b for a, b in zip(first, first[1:]))
    assert segs < 32 or min(plan([(1, 1 << 27)] * segs, cap=None)) < 0


def marker(pieces, bars, seed, ring=2):
    """prefix_kernel's rows and the warp that marks NaN values behind them, over a ring of `ring` pieces and
    `bars` barriers: how far the rows get ahead, and whether a wait could see a phase past the one it is for."""
    rnd = random.Random(seed)
    given = taken = stored = marked = 0  # pieces: handed out, taken by the rows, stored, taken by the marker
    waiting, ahead, alias = None, 0, False
    done = [0] * bars  # completed phases
    while marked < pieces or waiting is not None:
        step = rnd.choice(("give", "take", "store", "mark", "wait"))
        if step == "give" and given < pieces and given < min(taken, marked) + ring:
            given += 1
        elif step == "take" and taken == stored and taken < given:
            taken += 1
        elif step == "store" and stored < taken:
            done[stored % bars] += 1
            stored += 1
        elif step == "mark" and waiting is None and marked < given:
            waiting, marked = marked, marked + 1
        elif step == "wait" and waiting is not None:
            phases = done[waiting % bars] - waiting // bars  # 1: complete; 2 would look like 0
            ahead, alias = max(ahead, stored - waiting), alias or phases > 1
            if phases >= 1:
                waiting = None
    return ahead, alias


@pytest.mark.parametrize("pieces", [1, 2, 3, 9, 30])
def test_the_marking_warp_never_mistakes_a_phase(pieces):
    runs = [marker(pieces, 4, seed) for seed in range(300)]
    assert max(a for a, _ in runs) <= 3 and not any(alias for _, alias in runs)
    assert pieces < 9 or any(alias for _, alias in (marker(pieces, 1, seed) for seed in range(300)))
