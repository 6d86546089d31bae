"""CPU model of the barrier protocol of the 4-bit prefill kernel (csrc/kv4_prefill.cu) under random schedules.

Roles are generators that yield (barrier, parity) to wait; barriers count arrivals like mbarriers, and a wait by
parity succeeds exactly when the current phase has the other parity (so one that is two phases late hangs, and one
whose phase before has not completed passes too early: both show).  MMAs complete at random times, those of the two issuers in any order.
Checked: no deadlock; every MMA reads the block it means; no buffer is overwritten before its reader is
done; O is rescaled only between P V of the blocks around it; the end reads O complete.  Three planted mistakes
are caught."""
import random

import pytest

NKV = 3


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
    B = dict(kv_empty=[Barrier(1) for _ in range(NKV)], s_go=[[Barrier(5) for _ in range(NKV)] for _ in range(2)],
             s_full=[[Barrier(2), Barrier(2)] for _ in range(2)], p_full=[[Barrier(4), Barrier(4)] for _ in range(2)],
             o_last=[Barrier(1), Barrier(1)], q_ready=Barrier(8))
    conv = [[None] * 4 for _ in range(NKV)]
    sbuf = [[None, None], [None, None]]      # block of a tile's scores
    pbuf = [[[None] * 4, [None] * 4] for _ in range(2)]  # block of a warp's probabilities (over the scores)
    o_pv = [-1, -1]                          # last P V completed
    queues = [], []                          # MMAs and commits of the two issuers, each in order

    def converter(w):
        for j in range(nblk):
            kb = j % NKV
            if j >= NKV and plant != "kv_empty":
                yield B["kv_empty"][kb], ((j // NKV) - 1) & 1
            check(not any(kind in ("S", "PV") and k % NKV == kb and k != j for kind, _, k in queues[0] + queues[1]
                      if kind != "commit"),
                  "operands overwritten under an MMA")
            conv[kb][w] = j
            yield None
            B["s_go"][0][kb].arrive()
            B["s_go"][1][kb].arrive()

    def issuer_s():
        yield B["q_ready"], 0
        for t in range(2):
            B["s_go"][t][0].arrive()
            B["s_go"][t][1].arrive()
        for j in range(nblk):
            for t in range(2):
                yield B["s_go"][t][j % NKV], (j // NKV) & 1
                queues[0].append(("S", t, j))
                queues[0].append(("commit", B["s_full"][t][j & 1], None))
                B["s_full"][t][j & 1].arrive()

    def issuer_pv():
        for j in range(nblk):
            for t in range(2):
                yield B["p_full"][t][j & 1], (j >> 1) & 1
                if plant == "p_read" and j + 1 < nblk:
                    B["s_go"][t][(j + 2) % NKV].arrive()
                queues[1].append(("PV", t, j))
                if j + 1 == nblk:
                    queues[1].append(("commit", B["o_last"][t], None))
                elif plant != "p_read":
                    queues[1].append(("commit", B["s_go"][t][(j + 2) % NKV], None))
            queues[1].append(("commit", B["kv_empty"][j % NKV], None))

    def softmax(t, w):
        B["q_ready"].arrive()
        for j in range(nblk):
            yield B["s_full"][t][j & 1], (j >> 1) & 1
            check(sbuf[t][j & 1] == j, "scores of another block")
            check(conv[j % NKV] == [j] * 4, "flags of another block")
            yield None
            check(sbuf[t][j & 1] == j and conv[j % NKV] == [j] * 4, "scores or flags of another block")
            pbuf[t][j & 1][w] = j
            if j > 0 and r.random() < rescale:
                yield B["kv_empty"][(j - 1) % NKV], ((j - 1) // NKV) & 1
                check(o_pv[t] == j - 1, "O rescaled while P V runs")
            yield None
            B["p_full"][t][j & 1].arrive()
        if plant == "end":
            yield B["kv_empty"][(nblk - 2) % NKV], (max(nblk - 2, 0) // NKV) & 1
        else:
            yield B["o_last"][t], 0
        check(o_pv[t] == nblk - 1, "O read before the last P V")

    def tensor():
        while True:
            # (the order of the two issuers' MMAs is not promised; a commit waits for its own issuer's)
            queue = r.choice(queues)
            if queue and r.random() < 0.7:
                kind, t, j = queue.pop(0)
                if kind == "commit":
                    t.arrive()
                elif kind == "S":
                    check(conv[j % NKV] == [j] * 4, "S of another block's keys")
                    check(pbuf[t][j & 1] == [j - 2 if j > 1 else None] * 4, "S over scores in use")
                    check(o_pv[t] >= j - 2, "S over probabilities that P V has yet to read")
                    sbuf[t][j & 1] = j
                else:
                    check(conv[j % NKV] == [j] * 4, "P V of another block's values")
                    check(pbuf[t][j & 1] == [j] * 4, "P V of another block's probabilities")
                    check(o_pv[t] == j - 1, "P V out of order")
                    o_pv[t] = j
            yield None

    roles = {"issuer_s": issuer_s(), "issuer_pv": issuer_pv()}
    roles |= {f"conv{w}": converter(w) for w in range(4)}
    roles |= {f"soft{t}{w}": softmax(t, w) for t in range(2) for w in range(4)}
    machine = tensor()
    waits, speed = dict.fromkeys(roles), {k: r.choice((1.0, 1.0, 0.2, 0.03)) for k in roles}
    idle = 0
    while roles:
        next(machine)
        moved = any(queues)
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


@pytest.mark.parametrize("plant,nblk", [("end", 3), ("kv_empty", 9), ("p_read", 9)])
def test_planted_mistakes_are_caught(plant, nblk):
    caught = 0
    for seed in range(200):
        try:
            simulate(nblk, seed, plant, rescale=0.0)
        except (Mistake, AssertionError):
            caught += 1
    assert caught > 0
