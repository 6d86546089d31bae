"""One key that takes most of the weight and has no value, thousands behind it that take 2^-22 to 2^-30 of it each: what
comes out is theirs.  4-bit decode and prefill against 64 bits, within oracle/kv4.py's bound and the output's half
step (the scores are exact: one product each)."""
import pytest
import torch

from adallm_b200 import kvcache_fp4 as kv
from oracle import kv4
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu
BF16 = torch.bfloat16


def setting(sequences, keys, new, heads, page=16):
    """Keys 0 but for the first, whose element 0 is 6; values 1 but for the first, which is 0; queries 16 in element 0."""
    pages = -(-keys // page)
    kc, vc = kv.empty_kvcache_fp4(sequences * pages, 2, page, dev())
    one = int(torch.tensor(1.0).to(torch.float8_e4m3fn).view(torch.uint8))
    first = torch.arange(sequences, device=dev()) * pages
    kc[first, :, 0], kc[first, :, page * 64] = 7, one
    vc[:, :, :page * 64], vc[:, :, page * 64:] = 0x22, one
    vc[first, :, :64] = 0
    q = torch.zeros((sequences * new, heads, 128), dtype=BF16, device=dev())
    q[..., 0] = 16.0
    return q, kc, vc, torch.arange(sequences * pages, dtype=torch.int32, device=dev()).view(sequences, pages)


def check(out, q, kc, vc, tables, sequences, keys, new, scale, decode):
    want, err = kv4.attention(q[:new], kc, vc, tables[:1], [new], [keys], scale, decode=decode)  # (all sequences are alike)
    tol = err + torch.finfo(out.dtype).eps / 2 * (want.abs() + err)
    assert (want > tol).all()  # zeros would be noticed
    off = (out.view(sequences, *want.shape).double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("gap", [15.5, 17.6, 20.0])
@pytest.mark.parametrize("sequences,keys,wide", [(1, 1200, 0), (148, 1200, 0), (300, 3000, 0), (2000, 700, 100)])
def test_decode(sequences, keys, wide, gap):
    q, kc, vc, tables = setting(sequences, keys, 1, 4)
    wider = torch.nn.functional.pad(tables, (0, wide), value=-1)
    out = kv.paged_decode_fp4(q, kc, vc, wider, torch.full((sequences,), keys, dtype=torch.int32, device=dev()), gap / 96)
    check(out, q, kc, vc, tables, sequences, keys, 1, gap / 96, True)


@pytest.mark.parametrize("gap", [15.5, 17.6, 20.0])
@pytest.mark.parametrize("sequences,keys,new", [(300, 1200, 2), (1, 3000, 300), (1, 8000, 40), (3, 600, 600)])
def test_prefill(sequences, keys, new, gap):
    """A few rows a sequence, a chunk of a prompt, keys shared by CTAs, whole prompts."""
    q, kc, vc, tables = setting(sequences, keys, new, 4)
    cu = torch.arange(sequences + 1, dtype=torch.int32, device=dev())
    out = kv.paged_prefill_fp4(q, kc, vc, tables, cu * new, cu * keys, new, gap / 96)
    if new == keys:  # (the first rows see too few of the small ones to tell)
        first, rest = out.view(sequences, new, 4, 128)[:, :200], out.view(sequences, new, 4, 128)[:, 200:]
        assert (first >= 0).all() and (first <= 200 * 2.0 ** -21).all()
        q, out, new = q[200:], rest, new - 200
    check(out, q, kc, vc, tables, sequences, keys, new, gap / 96, False)
