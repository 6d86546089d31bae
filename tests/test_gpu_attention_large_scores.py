"""Two keys whose scores lie 16 (log2) apart near 2^27, where fp32 counts in sixteens.

A running reference that moves when a score passes it by more than 8 must not round that sum up to the next score: the
weight would be 2^16, which fp16 does not have.  q . k is exact here (multiples of 16 below 2^28) and the scale is the
fp32 ln 2, which makes the factor of log2 exactly 1, so the weights are 1 : 2^16 and all other keys have none.

Tolerance: the weights' fp16 rounding, exp2 and fp32 sums (2^-11 + 2^-20) and the output's half step."""
import math

import pytest
import torch

from adallm_b200 import kvcache_fp4 as kv
from adallm_b200.attention import paged_prefill
from adallm_b200.shared_prefix import shared_prefix_decode
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16
LN2 = float(torch.tensor(math.log(2.0)))
WANT = (1.0 + 2.0 * 2.0 ** 16) / (1.0 + 2.0 ** 16)  # value 1 at the first key, 2 at the second


def near(out):
    half = torch.finfo(out.dtype).eps / 2
    assert out.isfinite().all()
    assert ((out.double() - WANT).abs() <= (2.0 ** -11 + 2.0 ** -20 + half) * WANT).all(), (float(out.min()), float(out.max()))


def caches4(sequences, keys, page, at):
    """4-bit caches of one head: key rows of 0, but 1024 in element 0 and 1 or 2 in element 16 of the keys at `at`."""
    pages = -(-keys // page)
    kc, vc = kv.empty_kvcache_fp4(sequences * pages, 1, page, dev())
    one, big = (int(torch.tensor(x).to(torch.float8_e4m3fn).view(torch.uint8)) for x in (1.0, 256.0))
    for key, code in zip(at, (2, 4)):  # e2m1 codes of 1 and 2
        p, r = torch.arange(sequences, device=dev()) * pages + key // page, key % page
        kc[p, 0, r * 64] = 6           # 4.0, element 0
        kc[p, 0, r * 64 + 8] = code    # element 16
        kc[p, 0, page * 64 + r * 8] = big
        kc[p, 0, page * 64 + r * 8 + 1] = one
        vc[p, 0, r * 64:r * 64 + 64] = code * 17
        vc[p, 0, page * 64 + r * 8:page * 64 + r * 8 + 8] = one
    return kc, vc, torch.arange(sequences * pages, dtype=torch.int32, device=dev()).view(sequences, pages)


def queries4(rows, heads):
    q = torch.zeros((rows, heads, 128), dtype=BF16, device=dev())
    q[..., 0], q[..., 16] = 2.0 ** 17, 16.0
    return q


@pytest.mark.parametrize("sequences,keys,wide", [(1, 600, 0), (300, 2000, 0), (700, 600, 200)])
def test_4_bit_decode(sequences, keys, wide):
    """Both keys in one warp's range: one launch, and the steps of many sequences shared out."""
    kc, vc, tables = caches4(sequences, keys, 16, (0, 40))
    tables = torch.nn.functional.pad(tables, (0, wide), value=-1)
    out = kv.paged_decode_fp4(queries4(sequences, 4), kc, vc, tables,
                              torch.full((sequences,), keys, dtype=torch.int32, device=dev()), LN2, out=torch.empty(
                                  (sequences, 4, 128), dtype=F16, device=dev()))
    near(out)


@pytest.mark.parametrize("sequences,keys,new", [(400, 1500, 2), (1, 600, 300), (1, 4000, 40)])
def test_4_bit_prefill(sequences, keys, new):
    """A few rows a sequence, a prompt, keys shared by CTAs."""
    kc, vc, tables = caches4(sequences, keys, 16, (0, 70 if new > 2 else 40))
    cu = torch.arange(sequences + 1, dtype=torch.int32, device=dev())
    out = kv.paged_prefill_fp4(queries4(sequences * new, 4), kc, vc, tables, cu * new, cu * keys, new, LN2,
                               out=torch.empty((sequences * new, 4, 128), dtype=F16, device=dev()))
    near(out)


def caches8(keys, page, at):
    """e4m3 caches of one head: key rows of 0, but 256 in elements 0 to 15 and 1 or 2 in element 16 of the keys at `at`."""
    pages = -(-keys // page)
    k, v = (torch.zeros((pages * page, 1, 128), device=dev()) for _ in range(2))
    for key, value in zip(at, (1.0, 2.0)):
        k[key, :, :16], k[key, :, 16], v[key] = 256.0, value, value
    return *(x.to(torch.float8_e4m3fn).view(pages, page, 1, 128) for x in (k, v)), torch.arange(
        pages, dtype=torch.int32, device=dev())[None]


def queries8(rows, heads):
    q = torch.zeros((rows, heads, 128), dtype=BF16, device=dev())
    q[..., :16], q[..., 16] = 2.0 ** 15, 16.0
    return q


@pytest.mark.parametrize("keys,new", [(600, 300), (3000, 64)])
def test_e4m3_prefill(keys, new):
    kc, vc, tables = caches8(keys, 16, (3, 100))
    cu = torch.arange(2, dtype=torch.int32, device=dev())
    out = paged_prefill(queries8(new, 4), kc, vc, tables, cu * new, cu * keys, new, LN2,
                        out=torch.empty((new, 4, 128), dtype=F16, device=dev()))
    near(out)


@pytest.mark.parametrize("sequences,prefix", [(4, 700), (64, 8192), (200, 20000)])
def test_shared_prefix(sequences, prefix):
    """Both keys in the prefix; the sequences' own keys are the row of zeros behind it."""
    kc, vc, tables = caches8(prefix + 16, 16, (3, 140))
    own = torch.full((sequences, 1), prefix // 16, dtype=torch.int32, device=dev())
    out = shared_prefix_decode(queries8(sequences, 4), kc, vc, tables[:, :prefix // 16],
                               torch.tensor([prefix // 16 * 16], dtype=torch.int32, device=dev()), None, own,
                               torch.ones(sequences, dtype=torch.int32, device=dev()), LN2,
                               out=torch.empty((sequences, 4, 128), dtype=F16, device=dev()))
    near(out)
