"""CPU model of a prefill warp whose bounded wait runs out (csrc/kv4_prefill.cu, csrc/prefill_attention.cu).

A wait ends lane by lane: one lane may see the phase complete where another sees the CTA's abort flag or its own
limit.  Lanes that leave the role's loop go to the CTA's last barrier and stay there, so a warp collective (shuffle,
ballot, __syncwarp, with all lanes in its mask) behind them is never complete: the kernel that meant to give up hangs.
The outcome must be agreed on first.  The events of a role's loop are read from the source in their order."""
import os
import random
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "adallm_b200", "csrc")
EVENT = re.compile(r"(?P<vote>__all_sync\(0xffffffffu, (?:ok && )?wait_b\(|\bwait_w\()|(?P<leave>!wait_b\()|"
                   r"(?P<warp>__shfl_sync|__ballot_sync|__all_sync|__any_sync|__syncwarp|\bfetch\(j)")


def loop_events(name, role):
    """Events of the first loop over blocks in the section that starts with the role's comment."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//(?! -{8}).*", "", f.read())
    section = text[text.index(f"// ---------------- {role}"):]
    section = section[section.index("for (int j = 0; j < nblk; ++j) {"):]
    depth, end = 0, 0
    for end, c in enumerate(section):
        depth += (c == "{") - (c == "}")
        if c == "}" and depth == 0:
            break
    return [m.lastgroup for m in EVENT.finditer(section[:end])]


class Hang(AssertionError):
    pass


def give_up(events, seed, blocks=6):
    """One warp through the loop; some wait runs out for some of its lanes."""
    r = random.Random(seed)
    here = set(range(32))  # the others are at the CTA's last barrier
    bad = r.randrange(blocks * sum(e in ("vote", "leave") for e in events))
    waits, lost = 0, False
    for _ in range(blocks):
        for e in events:
            if e == "leave" or e == "vote":
                if e == "vote" and len(here) < 32:
                    raise Hang("a vote of a part of a warp")
                lost = lost or waits == bad
                waits += 1
                out = {x for x in here if lost and r.random() < 0.5}
                if e == "vote":
                    here = set() if out else here
                else:
                    here -= out
            elif len(here) < 32:
                raise Hang("a collective of a part of a warp")
            if not here:
                return


ROLES = [("kv4_prefill.cu", "converters"), ("kv4_prefill.cu", "softmax"), ("prefill_attention.cu", "converters"),
         ("prefill_attention.cu", "softmax")]


@pytest.mark.parametrize("name,role", ROLES)
def test_lanes_give_up_together(name, role):
    events = loop_events(name, role)
    assert "warp" in events and ("vote" in events or "leave" in events)
    for seed in range(300):
        give_up(events, seed)


def test_a_lane_that_leaves_alone_is_caught():
    caught = 0
    for seed in range(100):
        try:
            give_up(["leave", "warp"], seed)
        except Hang:
            caught += 1
    assert caught > 0
