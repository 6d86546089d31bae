"""ada_call hands every word to the argument it is meant for: each entry is called both ways with one argument
changed, and the change alone decides the status.

Unchanged, a call passes every check and stops at its first CUDA call (there is no GPU; with one these calls would
launch, and the tests are skipped).  For each argument that a check depends on there is a change whose status is not
that of the unchanged call.  To show that the cases have the power to notice, words are swapped on purpose: any
two neighbours that do not share their checks must change some status."""
import math

import pytest
import torch

from adallm_b200 import _native as N
from adallm_b200 import build as B

BAD, UNSUP, ALIGN, WS = N.ADA_ERR_INVALID_ARG, N.ADA_ERR_UNSUPPORTED, N.ADA_ERR_ALIGNMENT, N.ADA_ERR_WORKSPACE
pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="calls that pass every check would launch")

# name: (unchanged value, changed value or None for no check, status of the change)
META = dict(c=(1 << 12, 0, BAD), n=(2 << 12, 18, ALIGN), b=(2, -1, BAD), bt=(3 << 12, 6, ALIGN), bts=(4, 3, BAD),
            mp=(4, 5, BAD), free=(4 << 12, 0, BAD), nf=(9, -1, BAD), start=(5 << 12, 0, BAD), page=(16, 0, BAD),
            t=(8, 1 << 31, UNSUP), pos=(6 << 12, 4 + (6 << 12), ALIGN),
            # outputs that reach into c by their last word: each is longer than its neighbour
            slots=(7 << 12, (1 << 12) - 28, BAD), cq=(8 << 12, (1 << 12) - 8, BAD), ck=(9 << 12, (1 << 12) - 8, BAD),
            ctx=(10 << 12, (1 << 12) - 4, BAD), nxt=(11 << 12, 5 << 12, BAD),
            err=(12 << 12, 1, ALIGN), stream=(0, None, 0))
ROTARY = dict(pos=(16, 12, ALIGN), q=(32, 40, ALIGN), qst=(4096, 4, ALIGN), qsh=(128, 4, ALIGN), k=(48, 0, BAD),
              kst=(1024, 12, ALIGN), ksh=(128, 12, ALIGN), qo=(64, 32, BAD), ko=(80, 48, BAD), t=(3, 0, 0),
              hq=(32, -1, BAD), hkv=(8, -1, BAD), d=(128, 2048, UNSUP), table=(16, 18, ALIGN), maxp=(10, 0, BAD),
              rot=(64, 24, UNSUP), inter=(1, None, 0), dt=(1, 2, BAD), stream=(0, None, 0))
STORE = dict(pos=(16, 12, ALIGN), q=(32, 40, ALIGN), qst=(4096, 4, ALIGN), qsh=(128, 4, ALIGN), k=(48, 0, BAD),
             kst=(1024, 12, ALIGN), ksh=(128, 12, ALIGN), v=(64, 72, ALIGN), vst=(1024, 20, ALIGN), vsh=(128, 20, ALIGN),
             qo=(80, 32, BAD), t=(3, 0, 0), hq=(32, -1, BAD), hkv=(8, 0, BAD), d=(128, 64, UNSUP),
             table=(16, 18, ALIGN), maxp=(10, 0, BAD), rot=(128, 24, UNSUP), inter=(0, None, 0), slots=(16, 0, BAD),
             kc=(16, 24, ALIGN), vc=(32, 0, BAD), sp=(8 * 1152, 8 * 1152 + 8, ALIGN), sh=(1152, 1136, BAD), pages=(4, 0, BAD),
             page=(16, 8, UNSUP), ks=(1.0, -1.0, BAD), vs=(1.0, math.inf, BAD), dt=(0, 2, BAD), stream=(0, None, 0))
READ = dict(kc=(16, 24, ALIGN), vc=(32, 0, BAD), sp=(8 * 1152, 8 * 1152 + 8, ALIGN), sh=(1152, 1136, BAD), pages=(4, 0, BAD),
            page=(16, 8, UNSUP), hkv=(8, 0, BAD), d=(128, 64, UNSUP), slots=(16, 18, ALIGN), t=(3, -1, BAD),
            ks=(1.0, -1.0, BAD), vs=(1.0, math.inf, BAD), k=(48, 0, BAD), v=(64, 72, ALIGN), dt=(0, 2, BAD), stream=(0, None, 0))
ATTEND = dict(k=(16, 24, ALIGN), v=(32, 0, BAD), sp=(8 * 1152, 8 * 1152 + 8, ALIGN), sh=(1152, 1136, BAD), pages=(4, 0, BAD),
              bt=(16, 18, ALIGN), bts=(200, 199, BAD), mp=(200, 1 << 27, BAD))
HEADS = dict(hq=(32, 31, BAD), hkv=(8, 0, BAD), d=(128, 64, UNSUP), page=(16, 8, UNSUP), scale=(0.1, 0.0, BAD),
             ks=(1.0, -1.0, BAD), vs=(1.0, math.inf, BAD), window=(0, -1, BAD))
DECODE = dict(q=(32, 40, ALIGN), qd=(0, 2, BAD), qsb=(4096, 4, ALIGN), qsh=(128, 4, ALIGN), **ATTEND, ctx=(64, 0, BAD),
              batch=(1, 8193, UNSUP), **HEADS, out=(64, 72, ALIGN), od=(1, 3, BAD), osb=(4096, 12, ALIGN), osh=(128, 12, ALIGN),
              ws=(16, 24, ALIGN), wsb=(1 << 30, 1, WS), stream=(0, None, 0))
PREFILL = dict(q=(32, 40, ALIGN), qd=(0, 2, BAD), qst=(4096, 4, ALIGN), qsh=(128, 4, ALIGN), **ATTEND, cq=(64, 0, BAD),
               ck=(80, 82, ALIGN), batch=(1, 70000, UNSUP), total=(50, -1, BAD), most=(50, (1 << 30) + 1, UNSUP), **HEADS,
               out=(64, 72, ALIGN), od=(1, 3, BAD), ost=(4096, 12, ALIGN), osh=(128, 12, ALIGN), ws=(16, 24, ALIGN),
               wsb=(1 << 30, 1, WS), err=(16, 2, ALIGN), stream=(0, None, 0))
ENTRIES = {"step_metadata": ("ada_step_metadata", META), "rotary": ("ada_rotary", ROTARY), "kv4_store": ("ada_kv4_store", STORE),
           "kv4_read": ("ada_kv4_read", READ), "kv4_paged_decode": ("ada_kv4_paged_decode", DECODE),
           "kv4_paged_prefill": ("ada_kv4_paged_prefill", PREFILL)}


@pytest.fixture(scope="module")
def lib():
    B.build()
    return N.lib()


def cases(table):
    """The unchanged call, then each argument changed: (name, values, status or None)."""
    good = {k: v[0] for k, v in table.items()}
    return [(None, good, None)] + [(k, {**good, k: v[1]}, v[2]) for k, v in table.items() if v[1] is not None]


def packed(lib, name, values, swap=None):
    p = getattr(N, name)
    words = list(values)
    if swap is not None:
        words[swap], words[swap + 1] = words[swap + 1], words[swap]
    return lib.ada_call(p.entry, p.pack(*words))


@pytest.mark.parametrize("name", ENTRIES)
def test_every_argument_decides_alike(lib, name):
    entry, table = ENTRIES[name]
    fn = getattr(lib, entry)
    assert len(table) == len(fn.argtypes)
    unchanged = None
    for changed, values, status in cases(table):
        # (a 32-bit argument past its range is refused by ada_call alone)
        direct = fn(*values.values())
        if changed is None:
            unchanged = direct
            assert direct in (N.ADA_ERR_CUDA, N.ADA_ERR_LAUNCH)
        else:
            assert direct == status != unchanged, changed
        assert packed(lib, name, values.values()) == direct, changed


# Neighbours with the same checks: the numerical GPU tests tell them apart (the public calls go through ada_call).
ALIKE = [("qst", "qsh"), ("qsb", "qsh"), ("kst", "ksh"), ("vst", "vsh"), ("sp", "sh"), ("ost", "osh"), ("osb", "osh"), ("k", "v"),
         ("kc", "vc"), ("cq", "ck"), ("c", "n"), ("ks", "vs"), ("scale", "ks"), ("hq", "hkv"), ("free", "nf")]


@pytest.mark.parametrize("name", ENTRIES)
def test_swapped_words_are_noticed(lib, name):
    entry, table = ENTRIES[name]
    fn = getattr(lib, entry)
    names = list(table)
    for i in range(len(names) - 1):
        a, b = table[names[i]], table[names[i + 1]]
        if isinstance(a[0], float) != isinstance(b[0], float) or (names[i], names[i + 1]) in ALIKE:
            continue  # (the binding packs no float where an integer goes)
        assert any(packed(lib, name, v.values(), swap=i) != fn(*v.values()) for _, v, _ in cases(table)), names[i:i + 2]
