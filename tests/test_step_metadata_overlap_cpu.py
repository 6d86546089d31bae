"""Outputs of a step's metadata that lie in its inputs are refused, also by a part (CTAs read the one while another
writes the other).  Pointers are placeholders: the refusals come before any CUDA call, and what is not refused here
stops at the device query, where there is no GPU, or is not called."""
import pytest
import torch

from adallm_b200 import _native as N
from adallm_b200 import build as B

REQUESTS, TOKENS, FREE = 6, 10, 9
READ = dict(c=(1 << 12, 4 * REQUESTS), n=(2 << 12, 4 * REQUESTS), free=(3 << 12, 4 * FREE), start=(4 << 12, 4))
MADE = dict(pos=(5 << 12, 8 * TOKENS), slots=(6 << 12, 4 * TOKENS), cq=(7 << 12, 4 * (REQUESTS + 1)),
            ck=(8 << 12, 4 * (REQUESTS + 1)), ctx=(9 << 12, 4 * REQUESTS), nxt=(10 << 12, 4))


@pytest.fixture(scope="module")
def entry():
    B.build()
    return N.lib().ada_step_metadata


def call(entry, **change):
    p = {k: v[0] for k, v in {**READ, **MADE}.items()} | change
    return entry(p["c"], p["n"], REQUESTS, 11 << 12, 4, 4, p["free"], p.get("nf", FREE), p["start"], 16, TOKENS, p["pos"],
                 p["slots"], p["cq"], p["ck"], p["ctx"], p["nxt"], None, None)


@pytest.mark.parametrize("made", MADE)
@pytest.mark.parametrize("read", READ)
def test_overlaps_are_refused(entry, made, read):
    (at, n), (_, m) = READ[read], MADE[made]
    unit = 8 if made == "pos" else 4
    inside = {at, at + (n - 1) // unit * unit, at - m + unit}  # its start, its last word, all but the first word before it
    for p in sorted(inside):
        assert p < at + n and at < p + m
        assert call(entry, **{made: p}) == N.ADA_ERR_INVALID_ARG, p


@pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused would launch")
def test_neighbours_and_empty_lists_are_not(entry):
    assert call(entry) == N.ADA_ERR_CUDA
    for made, (_, m) in MADE.items():
        for at, n in READ.values():
            if made != "pos" or n % 8 == 0:
                assert call(entry, **{made: at + n}) == N.ADA_ERR_CUDA
            assert call(entry, **{made: at - m}) == N.ADA_ERR_CUDA
    assert call(entry, free=MADE["cq"][0] + 8, nf=0) == N.ADA_ERR_CUDA
