"""CPU model of the barrier protocol of the 4-bit prefill kernel (csrc/kv4_prefill.cu) under random schedules.

Roles are generators that yield (barrier, parity) to wait; barriers count arrivals like mbarriers, and a wait by
parity succeeds exactly when the current phase has the other parity (so one that is two phases late hangs, and one
whose phase before has not completed passes too early: both show).  MMAs complete at random times, S before an earlier P V as well.
Checked: no deadlock; every MMA reads the block it means; no buffer is overwritten before its reader is
done; O is rescaled only between P V of the blocks around it; the end reads O complete.  Three planted mistakes
are caught."""
import random

import pytest

NSTG, NKV = 4, 3


class Barrier:
    def __init__(self, count):
        self.count, self.pending, self.phase = count, count, 0

    def arrive(self):
        self.pending -= 1
        assert self.pending >= 0, "more arrivals than a phase has"
        if self.pending == 0:
            self.pending, self.phase = self.count, self.phase + 1

    def done(self, parity):
        return (self.phase & 1) != parity


class Mistake(AssertionError):
    pass


def check(ok, what):
    if not ok:
        raise Mistake(what)


def simulate(nblk, seed, plant=None, rescale=0.3):
    r = random.Random(seed)
    B = dict(e_full=[Barrier(1) for _ in range(NSTG)], e_empty=[Barrier(4) for _ in range(NSTG)],
             kv_full=[Barrier(4) for _ in range(NKV)], kv_empty=[Barrier(1) for _ in range(NKV)],
             s_full=[[Barrier(2), Barrier(2)] for _ in range(2)], p_full=[[Barrier(4), Barrier(4)] for _ in range(2)],
             o_done=[Barrier(1), Barrier(1)], o_last=[Barrier(1), Barrier(1)], q_ready=Barrier(8))
    stage, conv, slot = [None] * NSTG, [[None] * 4 for _ in range(NKV)], [None] * NKV
    sbuf = [[None, None], [None, None]]      # ("S" | "P", block), P a count of warps
    o_pv = [-1, -1]                          # last P V completed
    queue = []                               # MMAs and commits, in order

    def producer():
        for j in range(nblk):
            s = j % NSTG
            if j >= NSTG:
                yield B["e_empty"][s], ((j // NSTG) - 1) & 1
            stage[s] = j
            B["e_full"][s].arrive()

    def converter(w):
        for j in range(nblk):
            s, kb = j % NSTG, j % NKV
            yield B["e_full"][s], (j // NSTG) & 1
            if j >= NKV and plant != "kv_empty":
                yield B["kv_empty"][kb], ((j // NKV) - 1) & 1
            check(stage[s] == j, "staging overwritten")
            check(not any(kind in ("S", "PV") and k % NKV == kb and k != j for kind, _, k in queue if kind != "commit"),
                  "operands overwritten under an MMA")
            conv[kb][w] = j
            yield None
            B["kv_full"][kb].arrive()
            B["e_empty"][s].arrive()

    def issuer():
        def s_of(j):
            for t in range(2):
                queue.append(("S", t, j))
                queue.append(("commit", B["s_full"][t][j & 1], None))
                B["s_full"][t][j & 1].arrive()

        yield B["q_ready"], 0
        yield B["kv_full"][0], 0
        s_of(0)
        for j in range(nblk):
            if j + 1 < nblk:
                yield B["kv_full"][(j + 1) % NKV], ((j + 1) // NKV) & 1
                if j > 0 and plant != "issuer":
                    yield B["o_done"][0], (j - 1) & 1
                    yield B["o_done"][1], (j - 1) & 1
                s_of(j + 1)
            for t in range(2):
                yield B["p_full"][t][j & 1], (j >> 1) & 1
                queue.append(("PV", t, j))
                queue.append(("commit", B["o_done"][t], None))
                if j + 1 == nblk:
                    queue.append(("commit", B["o_last"][t], None))
            queue.append(("commit", B["kv_empty"][j % NKV], None))

    def softmax(t, w):
        B["q_ready"].arrive()
        for j in range(nblk):
            yield B["s_full"][t][j & 1], (j >> 1) & 1
            check(sbuf[t][j & 1] in (("S", j), ("P", j)), "scores of another block")
            check(conv[j % NKV] == [j] * 4, "flags of another block")
            yield None
            sbuf[t][j & 1] = ("P", j)
            if j > 0 and r.random() < rescale:
                yield B["o_done"][t], (j - 1) & 1
                check(o_pv[t] == j - 1, "O rescaled while P V runs")
            yield None
            B["p_full"][t][j & 1].arrive()
        if plant == "end":
            yield B["o_done"][t], (nblk - 1) & 1
        else:
            yield B["o_last"][t], 0
        check(o_pv[t] == nblk - 1, "O read before the last P V")

    def tensor():
        while True:
            if queue and r.random() < 0.7:
                # (the order of MMAs of different shapes is not promised: an S may pass P V before it)
                at = 0
                if r.random() < 0.3:
                    at = next((i for i, q in enumerate(queue) if q[0] == "S"), 0)
                kind, t, j = queue[at]
                if kind == "commit":
                    t.arrive()
                elif kind == "S":
                    check(conv[j % NKV] == [j] * 4, "S of another block's keys")
                    check(sbuf[t][j & 1] is None or sbuf[t][j & 1] == ("P", j - 2), "S over scores in use")
                    check(o_pv[t] >= j - 2, "S over probabilities that P V has yet to read")
                    sbuf[t][j & 1] = ("S", j)
                else:
                    check(conv[j % NKV] == [j] * 4, "P V of another block's values")
                    check(sbuf[t][j & 1] == ("P", j), "P V of another block's probabilities")
                    check(o_pv[t] == j - 1, "P V out of order")
                    o_pv[t] = j
                queue.pop(at)
            yield None

    roles = {"producer": producer(), "issuer": issuer()}
    roles |= {f"conv{w}": converter(w) for w in range(4)}
    roles |= {f"soft{t}{w}": softmax(t, w) for t in range(2) for w in range(4)}
    machine = tensor()
    waits, speed = dict.fromkeys(roles), {k: r.choice((1.0, 1.0, 0.2, 0.03)) for k in roles}
    idle = 0
    while roles:
        next(machine)
        moved = bool(queue)
        for k in r.sample(list(roles), len(roles)):
            w = waits[k]
            if w is not None and not w[0].done(w[1]):
                continue
            moved = True
            if r.random() > speed[k]:
                continue
            try:
                waits[k] = next(roles[k])
            except StopIteration:
                del roles[k]
        idle = 0 if moved else idle + 1
        check(idle < 3, f"deadlock: {sorted(roles)}")


@pytest.mark.parametrize("nblk", [1, 2, 3, 4, 5, 9, 24])
def test_random_schedules(nblk):
    for seed in range(40):
        simulate(nblk, 1000 * nblk + seed)
    for seed in range(12):
        simulate(nblk, seed, rescale=0.0)
        simulate(nblk, seed, rescale=1.0)


@pytest.mark.parametrize("plant,nblk", [("end", 2), ("issuer", 6), ("kv_empty", 9)])
def test_planted_mistakes_are_caught(plant, nblk):
    caught = 0
    for seed in range(200):
        try:
            simulate(nblk, seed, plant, rescale=0.0)
        except (Mistake, AssertionError):
            caught += 1
    assert caught > 0
