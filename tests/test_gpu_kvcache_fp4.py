"""The 4-bit KV cache: store and read-back (equal to the definition bit by bit), decode and prefill attention
(against 64 bits, within oracle/kv4.py's bound), and a serving step of all of them together."""
import math

import pytest
import torch

from adallm_b200 import kvcache_fp4 as kv
from adallm_b200.rotary_embedding import apply_rotary
from adallm_b200.step_metadata import step_metadata
from oracle import kv4
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu
BF16, F16 = torch.bfloat16, torch.float16


def gen(seed):
    return torch.Generator(device=dev()).manual_seed(seed)


def randn(shape, g, spread=1.0, dtype=BF16):
    return (spread * torch.randn(shape, generator=g, device=dev())).to(dtype)


# ---- store and read ----
@pytest.mark.parametrize("t,hkv,page,dtype,ks,vs,spread", [
    (1, 1, 16, BF16, 1.0, 1.0, 1.0), (7, 8, 16, F16, 1.0, 1.0, 0.02), (300, 8, 64, BF16, 0.37, 0.05, 1.0),
    (1000, 3, 48, F16, 2.0, 0.5, 30.0), (129, 16, 256, BF16, 1.0, 3.0, 1000.0), (65, 2, 32, BF16, 1.0, 1.0, 1e-3)])
def test_store_and_read(t, hkv, page, dtype, ks, vs, spread):
    g = gen(t)
    k, v = randn((t, hkv, 128), g, spread, dtype), randn((t, hkv, 128), g, spread / 3, dtype)
    pages = -(-t // page) + 2
    kc, vc = kv.empty_kvcache_fp4(pages, hkv, page, dev())
    kc.fill_(0xA5)
    vc.fill_(0xA5)
    slots = torch.randperm(pages * page, generator=g, device=dev())[:t].to(torch.int32)
    if t > 5:
        slots[2] = -1
        slots[5] = pages * page  # behind the cache
    kv.store_kvcache_fp4(k, v, kc, vc, slots, ks, vs)
    ko, vo = kv.read_kvcache_fp4(kc, vc, slots, dtype, ks, vs)
    there = ((slots >= 0) & (slots < pages * page))[:, None, None]
    for x, o, s, cache in ((k, ko, ks, kc), (v, vo, vs, vc)):
        want = torch.where(there, kv4.stored(x, s), torch.zeros((), dtype=torch.float64, device=dev()))
        assert torch.equal(o, want.float().to(dtype))
        # the bytes themselves, and everything else as it was
        data, scale = kv4.pack(x.float() / torch.tensor(s, device=dev()))
        full = torch.full_like(cache, 0xA5)
        dv, sv = full[:, :, :page * 64].unflatten(2, (page, 64)), full[:, :, page * 64:].unflatten(2, (page, 8))
        ok = there.flatten()
        at = slots[ok].long()
        dv.transpose(1, 2)[at // page, at % page] = data[ok]
        sv.transpose(1, 2)[at // page, at % page] = scale[ok]
        # (a zero that was negative keeps its sign bit in the cache)
        same = cache == full
        nib = cache[:, :, :page * 64][~same[:, :, :page * 64]] ^ full[:, :, :page * 64][~same[:, :, :page * 64]]
        assert same[:, :, page * 64:].all() and ((nib & 0x77) == 0).all()


def test_ties_and_borders_go_to_the_even_code():
    """Rows of exact midpoints, of their neighbours in bf16, and of every magnitude, under many scales."""
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    rows = []
    for e in range(-6, 7):
        for s in (1.0, 1.125, 1.25, 1.375, 1.5, 1.625, 1.75, 1.875):
            x = torch.cat((mids, mids * (1 + 2.0 ** -7), -mids * (1 - 2.0 ** -7), -mids, torch.tensor(kv4.MAG)[1:]))
            x = torch.nn.functional.pad(x, (0, 45 - x.numel())).view(3, 15)
            rows.append(torch.cat((torch.full((3, 1), 6.0), x), 1).flatten() * s * 2.0 ** e)
    x = torch.stack(rows).to(dev())
    x = torch.nn.functional.pad(x, (0, 80)).view(-1, 1, 128)
    for dtype in (BF16, F16):
        y = x.to(dtype)
        kc, vc = kv.empty_kvcache_fp4(-(-x.shape[0] // 16), 1, 16, dev())
        slots = torch.arange(x.shape[0], dtype=torch.int32, device=dev())
        kv.store_kvcache_fp4(y, -y, kc, vc, slots)
        a, b = kv.read_kvcache_fp4(kc, vc, slots, dtype)
        want = kv4.stored(y).to(dtype)
        assert torch.equal(a, want) and torch.equal(b, -want)


def test_zeros_infinities_nan_and_extremes():
    x = torch.zeros((6, 1, 128), dtype=BF16, device=dev())
    x[1, 0, 5] = math.inf
    x[1, 0, 6] = -math.inf
    x[1, 0, 7] = 3.0
    x[2, 0, 20] = math.nan
    x[2, 0, 21] = 2.0
    x[3] = 3e38
    x[4, 0, :16] = 1e-4      # below the smallest scale: zeros
    x[5, 0, 0] = 2688.0
    x[5, 0, 1] = -3000.0
    kc, vc = kv.empty_kvcache_fp4(1, 1, 16, dev())
    slots = torch.arange(6, dtype=torch.int32, device=dev())
    kv.store_kvcache_fp4(x, x, kc, vc, slots)
    for o in kv.read_kvcache_fp4(kc, vc, slots, BF16):
        assert (o[0] == 0).all()
        assert o[1, 0, 5] == 2688 and o[1, 0, 6] == -2688 and (o[1, 0, 16:] == 0).all() and o[1, 0, 7] == 0
        assert o[2, 0, 16:32].isnan().all() and o[2].isnan().sum() == 16
        assert (o[3] == 2688).all()
        assert (o[4] == 0).all()
        assert o[5, 0, 0] == 2688 and o[5, 0, 1] == -2688


@pytest.mark.parametrize("t,hq,hkv,r,inter,dtype", [(1, 32, 8, 128, False, BF16), (19, 16, 2, 64, True, F16),
                                                    (700, 12, 4, 32, False, BF16), (3, 8, 8, 128, True, BF16)])
def test_rotary_store_is_rotary_then_store(t, hq, hkv, r, inter, dtype):
    g = gen(t + hq)
    qkv = randn((t, hq + 2 * hkv, 128), g, 1.0, dtype)
    q, k, v = qkv.split((hq, hkv, hkv), 1)
    pos = torch.randint(0, 4000, (t,), generator=g, device=dev())
    a = torch.randn((4000, r), generator=g, device=dev()).clamp(-1, 1)
    page = 32
    pages = t // page + 1
    slots = torch.randperm(pages * page, generator=g, device=dev())[:t].to(torch.int32)
    if t > 2:
        slots[1] = -1
    one, two = kv.empty_kvcache_fp4(pages, hkv, page, dev()), kv.empty_kvcache_fp4(pages, hkv, page, dev())
    qo = kv.rotary_store_kvcache_fp4(pos, q, k, v, a, *one, slots, inter, 0.5, 0.7)
    want_q, want_k = apply_rotary(pos, q, k, a, inter)
    kv.store_kvcache_fp4(want_k, v, *two, slots, 0.5, 0.7)
    assert torch.equal(qo, want_q) and all(torch.equal(x, y) for x, y in zip(one, two))


def test_strided_caches():
    """Pages of several layers in one pool, heads of two caches side by side."""
    g = gen(5)
    t, hkv, page, pages = 40, 4, 16, 5
    pool = torch.zeros((pages, 3, 2 * hkv, page * 72), dtype=torch.uint8, device=dev())
    kc, vc = pool[:, 1, :hkv], pool[:, 1, hkv:]
    k, v = randn((t, hkv, 128), g), randn((t, hkv, 128), g)
    slots = torch.randperm(pages * page, generator=g, device=dev())[:t].to(torch.int32)
    kv.store_kvcache_fp4(k, v, kc, vc, slots)
    assert (pool[:, 0] == 0).all() and (pool[:, 2] == 0).all()
    a, b = kv.read_kvcache_fp4(kc, vc, slots, F16)
    assert torch.equal(a, kv4.stored(k).half()) and torch.equal(b, kv4.stored(v).half())


def test_caches_past_32_bits():
    """Pages and heads further apart than 32 bits count, and a page of more rows than 16 bits count."""
    g = gen(9)
    hkv, page, lens = 2, 16, [40, 17]
    far = torch.empty(11 << 30, dtype=torch.uint8, device=dev())
    t, slots = 57, torch.tensor([*range(40), *range(64, 81)], dtype=torch.int32, device=dev())
    k, v, q = randn((t, hkv, 128), g), randn((t, hkv, 128), g), randn((2, 8, 128), g)
    tables = torch.tensor([[0, 1, 2], [4, 5, -1]], dtype=torch.int32, device=dev())
    ctx, i32 = torch.tensor(lens, dtype=torch.int32, device=dev()), dict(dtype=torch.int32, device=dev())
    kc, vc = (far[o:].as_strided((6, hkv, page * 72), ((1 << 30) + 32, (5 << 30) + (1 << 21), 1)) for o in (0, 1 << 20))
    near = [torch.zeros((6, hkv, page * 72), dtype=torch.uint8, device=dev()) for _ in range(2)]
    outs = []
    for c in ((kc, vc), near):
        kv.store_kvcache_fp4(k, v, *c, slots)
        outs.append((*kv.read_kvcache_fp4(*c, slots), kv.paged_decode_fp4(q, *c, tables, ctx, 0.1),
                     kv.paged_prefill_fp4(q, *c, tables, torch.tensor([0, 1, 2], **i32), torch.tensor([0, 40, 57], **i32), 1, 0.1)))
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    rows = 80000  # one page
    kc, vc = (far[o:o + rows * 72].view(1, 1, rows * 72) for o in (0, rows * 72))
    slots = torch.arange(rows - t, rows, **i32)
    kv.store_kvcache_fp4(k[:, :1], v[:, :1], kc, vc, slots)
    assert torch.equal(kv.read_kvcache_fp4(kc, vc, slots, F16)[0], kv4.stored(k[:, :1]).half())


# ---- attention ----
def make(seed, lens, new, hq, hkv, page, dtype=BF16, q_spread=1.5, k_spread=1.0, extra=3):
    """Caches whose rows behind a sequence's end are NaN, scattered pages, -1 behind them."""
    g = gen(seed)
    pages = [-(-n // page) for n in lens]
    pool = sum(pages) + extra
    kc = kv4.make_cache(pool, hkv, page, g, dev(), k_spread)
    vc = kv4.make_cache(pool, hkv, page, g, dev())
    ids = torch.randperm(pool, generator=g, device=dev()).tolist()
    tables = torch.full((len(lens), max(pages + [1]) + 1), -1, dtype=torch.int32, device=dev())
    at = 0
    for b, n in enumerate(lens):
        tables[b, :pages[b]] = torch.tensor(ids[at:at + pages[b]], dtype=torch.int32)
        at += pages[b]
        if n % page:
            for c in (kc, vc):
                blk = c[int(tables[b, n // page])]
                blk[:, (n % page) * 64:page * 64] = 0xFF
                blk[:, page * 64 + (n % page) * 8:] = 0x7F
    spare = torch.tensor(ids[at:], device=dev())
    kc[spare], vc[spare] = 0x7F, 0x7F  # pages of nobody
    q = randn((sum(new), hq, 128), g, q_spread, dtype)
    i32 = dict(dtype=torch.int32, device=dev())
    cu = lambda x: torch.tensor([0] + torch.tensor(x).cumsum(0).tolist(), **i32)  # noqa: E731
    return dict(q=q, k=kc, v=vc, tables=tables, lens=lens, new=new, ctx=torch.tensor(lens, **i32), cu_q=cu(new),
                cu_k=cu(lens))


def behind_long_tables(c, pages=64):
    """The same sequences with wider tables: what selects the forms that share keys out."""
    return dict(c, tables=torch.nn.functional.pad(c["tables"], (0, pages), value=-1))


def assert_near(out, want, err, dtype=None):
    half = torch.finfo(dtype or out.dtype).eps / 2
    tol = err + half * (want.abs() + err) + torch.finfo(dtype or out.dtype).smallest_normal
    off = (out.double() - want).abs()
    assert out.isfinite().all()
    assert (off <= tol).all(), f"worst {float((off / tol).max())} of the bound"


def run_decode(c, window=0, ks=1.0, vs=1.0, scale=128 ** -0.5, **kw):
    out = kv.paged_decode_fp4(c["q"], c["k"], c["v"], c["tables"], c["ctx"], scale, window, ks, vs, **kw)
    torch.cuda.synchronize()
    return out


def want_of(c, window=0, ks=1.0, vs=1.0, scale=128 ** -0.5, decode=True):
    return kv4.attention(c["q"], c["k"], c["v"], c["tables"], c["new"], c["lens"], scale, window, decode, ks, vs)


DECODE = [  # lens, hq, hkv, page, window, dtype
    ([1], 8, 8, 16, 0, BF16), ([0, 1, 0], 32, 8, 16, 0, BF16), ([15, 16, 17, 31, 33], 32, 8, 16, 0, F16),
    ([700], 32, 8, 16, 0, BF16), ([5, 1000, 64, 0, 129], 32, 4, 32, 0, BF16), ([3000, 100], 16, 2, 64, 100, BF16),
    ([1, 40, 41, 300], 12, 4, 48, 17, F16), ([2048] * 3, 32, 16, 256, 1024, F16), ([777, 1], 6, 2, 16, 1, BF16),
    ([257, 513], 32, 2, 16, 0, BF16), ([400, 90], 24, 2, 16, 30, F16), ([20000, 3, 8191], 32, 8, 16, 0, BF16),
    ([100] * 70, 4, 1, 16, 0, BF16), ([33, 500], 33, 1, 16, 0, BF16), ([9000], 40, 1, 16, 5000, F16)]


@pytest.mark.parametrize("lens,hq,hkv,page,window,dtype", DECODE)
def test_decode_matches_64_bits(lens, hq, hkv, page, window, dtype):
    c = make(len(lens) + lens[-1] + hq, lens, [1] * len(lens), hq, hkv, page, dtype)
    assert_near(run_decode(c, window), *want_of(c, window))


def test_decode_scales_output_type_strides_and_workspace():
    c = make(3, [100, 600], [1, 1], 16, 4, 16)
    wide = torch.full((2, 20, 144), 7.0, dtype=F16, device=dev())
    ws = torch.full((max(16, kv.paged_decode_fp4_workspace_bytes(2, 16, 4, c["tables"].shape[1], 16)),), 0xFF, dtype=torch.uint8, device=dev())
    q = c["q"]
    c["q"] = torch.nn.functional.pad(q, (0, 8, 1, 1))[:, 1:17, :128]
    out = run_decode(c, 0, 0.37, 0.05, 0.2, out=wide[:, 2:18, 8:136], workspace=ws)
    assert_near(out, *want_of(c, 0, 0.37, 0.05, 0.2))
    assert (wide[:, :2] == 7).all() and (wide[:, 18:] == 7).all() and (wide[..., :8] == 7).all()


def test_decode_forms_agree():
    """The same sequences behind tables that select one launch and two (lengths 0, 1, whole steps, ragged)."""
    for lens, window in (([1280, 0, 1, 31, 32, 33, 64, 777], 0), ([5000, 1279, 40, 0], 1200)):
        c = make(41, lens, [1] * len(lens), 16, 4, 16)
        if window == 0:
            c["tables"] = c["tables"][:, :80].contiguous()
        assert kv.paged_decode_fp4_workspace_bytes(len(lens), 16, 4, c["tables"].shape[1], 16, window) == 0
        want, err = want_of(c, window)
        assert_near(run_decode(c, window), want, err)
        wide = dict(c, tables=torch.nn.functional.pad(c["tables"], (0, 200), value=-1))
        if window == 0:
            assert kv.paged_decode_fp4_workspace_bytes(len(lens), 16, 4, wide["tables"].shape[1], 16) > 0
            assert_near(run_decode(wide), want, err)


def test_decode_batch_of_thousands():
    lens = [(i * 37) % 70 for i in range(3000)]
    c = make(6, lens, [1] * 3000, 4, 2, 16)
    assert_near(run_decode(c), *want_of(c))


@pytest.mark.parametrize("decode", [True, False])
def test_holes_and_bad_page_ids_are_masked(decode):
    c = make(7, [200, 64, 33], [1, 1, 1], 8, 2, 16)
    c["tables"][0, 3] = -1
    c["tables"][0, 5] = c["k"].shape[0]
    c["tables"][0, 7] = 2 ** 31 - 1
    c["tables"][1, :] = -1  # nothing there: zeros
    want, err = want_of(c, decode=decode)
    for d in (c, behind_long_tables(c, 100)):
        out = run_decode(d) if decode else run_prefill(d)
        assert_near(out, want, err)
        assert (out[1] == 0).all()


def test_lengths_beyond_the_table():
    c = make(8, [64, 64], [1, 1], 8, 2, 16)
    c["tables"] = c["tables"][:, :3].contiguous()
    c["ctx"] += 1000
    c["cu_k"][1] += 1000
    c["cu_k"][2] += 2000
    want = dict(c, lens=[48, 48])
    assert_near(run_decode(c), *want_of(want))
    assert_near(run_prefill(c), *want_of(want, decode=False))


def test_large_and_extreme_queries():
    """bf16 queries far beyond fp16, rows of tiny ones: the scores decide as in 64 bits."""
    for dtype, big in ((BF16, 1e37), (F16, 60000.0)):
        c = make(9, [300, 50], [1, 1], 16, 4, 16, dtype)
        for factor in (big, 1e-3 if dtype is F16 else 1e-30):
            d = dict(c, q=(c["q"].float().clamp(-1, 1) * factor).to(dtype))
            scale = 1.0 if factor > 1 else 128 ** -0.5
            want, err = want_of(d, 0, scale=scale)
            for out in (run_decode(d, scale=scale), run_prefill(d, scale=scale)):
                if factor > 1:  # one key takes all; the bound's score term says nothing here
                    half = torch.finfo(dtype).eps / 2
                    assert ((out.double() - want).abs() <= (2.0 ** -10 + half) * want.abs() + 1e-30).all()
                else:
                    assert_near(out, want, err)


def test_a_nan_reaches_the_rows_that_see_it():
    """NaN in a key: every element of its rows; in a value: the 16 elements of its block."""
    c = make(10, [100, 100, 40], [1, 1, 1], 16, 4, 16)
    page_of = lambda b, t: int(c["tables"][b, t // 16])  # noqa: E731
    c["k"][page_of(0, 20), 1, 16 * 64 + (20 % 16) * 8 + 3] = 0x7F
    c["v"][page_of(1, 99), 2, 16 * 64 + (99 % 16) * 8 + 5] = 0x7F
    out = run_decode(c)
    bad = out.isnan()
    assert bad[0, 4:8].all() and bad[0].sum() == 4 * 128
    assert bad[1, 8:12, 80:96].all() and bad[1].sum() == 4 * 16
    assert not bad[2].any()
    out = run_decode(c, 50)  # the window leaves the key out, the value in
    assert not out[0].isnan().any() and out[1].isnan().sum() == 64


def run_prefill(c, window=0, ks=1.0, vs=1.0, scale=128 ** -0.5, most=None, **kw):
    err = torch.zeros(1, dtype=torch.int32, device=dev())
    out = kv.paged_prefill_fp4(c["q"], c["k"], c["v"], c["tables"], c["cu_q"], c["cu_k"],
                               max(c["new"]) if most is None else most, scale, window, ks, vs, err=err, **kw)
    torch.cuda.synchronize()
    assert int(err) == 0
    return out


PREFILL = [  # cached, new, hq, hkv, page, window, dtype
    ([0], [1], 8, 8, 16, 0, BF16), ([0, 37, 300, 5], [50, 1, 129, 0], 32, 8, 16, 0, BF16),
    ([0, 37, 300, 5], [50, 1, 129, 0], 32, 8, 16, 40, F16), ([100, 0], [77, 200], 32, 4, 64, 0, BF16),
    ([15], [70], 12, 4, 32, 0, F16), ([3], [130], 4, 4, 16, 17, BF16), ([1024], [512], 32, 8, 16, 0, BF16),
    ([0], [700], 16, 1, 16, 0, BF16), ([500, 0, 63], [65, 64, 1], 32, 16, 256, 128, F16), ([7], [300], 33, 1, 48, 0, BF16),
    ([2000], [3], 32, 8, 16, 0, F16), ([0, 0, 0], [16, 17, 15], 32, 2, 16, 1, BF16),
    # few rows a KV head: the keys shared out as for decode
    ([700, 0, 33], [8, 5, 1], 16, 4, 16, 0, BF16), ([9000, 3], [4, 2], 32, 4, 64, 0, F16),
    ([300, 20, 0], [7, 3, 1], 12, 4, 48, 13, F16), ([1, 30, 31, 32] * 12, [1, 2, 3, 4] * 12, 8, 8, 16, 0, BF16),
    ([64, 500], [0, 2], 32, 2, 32, 1, BF16), ([100], [32], 2, 2, 16, 40, BF16)]


@pytest.mark.parametrize("cached,new,hq,hkv,page,window,dtype", PREFILL)
def test_prefill_matches_64_bits(cached, new, hq, hkv, page, window, dtype):
    lens = [a + b for a, b in zip(cached, new)]
    c = make(sum(lens) + hq, lens, new, hq, hkv, page, dtype)
    want, err = want_of(c, window, decode=False)
    assert_near(run_prefill(c, window), want, err)
    assert_near(run_prefill(behind_long_tables(c), window), want, err)


def test_prefill_scales_output_type_strides_and_rows_left_alone():
    c = make(21, [90, 40], [50, 30], 16, 4, 16)
    n = 80
    wide = torch.full((n + 6, 20, 144), 7.0, dtype=F16, device=dev())
    q = torch.nn.functional.pad(c["q"], (0, 8, 1, 1, 0, 6))[:, 1:17, :128]
    d = dict(c, q=q)
    out = run_prefill(d, 20, 0.37, 0.05, 0.2, out=wide[:, 2:18, 8:136], most=64)
    assert_near(out[:n], *want_of(c, 20, 0.37, 0.05, 0.2, decode=False))
    assert (wide[n:] == 7).all() and (wide[:, :2] == 7).all() and (wide[..., :8] == 7).all()


def test_prefill_rows_without_keys_are_zeros():
    """More new tokens than keys: the rows before the first key."""
    c = make(22, [20, 64], [30, 64], 8, 2, 16)
    out = run_prefill(c)
    assert (out[:10] == 0).all()
    want, err = kv4.attention(torch.cat((c["q"][10:30], c["q"][30:])), c["k"], c["v"], c["tables"], [20, 64], [20, 64],
                              128 ** -0.5)
    assert_near(out[10:], want, err)


def test_prefill_lists_that_do_not_ascend_stay_inside():
    c = make(23, [64, 64], [40, 40], 8, 2, 16)
    out = torch.full_like(c["q"], 7.0)
    c["cu_q"] = torch.tensor([60, 20, 2 ** 30], dtype=torch.int32, device=dev())
    run_prefill(c, out=out, most=100)
    c["cu_q"] = torch.tensor([-50, 30, 90], dtype=torch.int32, device=dev())
    run_prefill(c, out=out, most=100)
    c = behind_long_tables(c)
    for cu in ([60, 20, 2 ** 30], [-50, 30, 90], [2 ** 31 - 1, -2 ** 31, 7]):  # and with few rows
        c["cu_q"] = torch.tensor(cu, dtype=torch.int32, device=dev())
        run_prefill(c, out=out, most=8)
    c["cu_q"] = torch.tensor([0, 4, 8], dtype=torch.int32, device=dev())
    c["cu_k"] = torch.tensor([0, 2 ** 31 - 1, -5], dtype=torch.int32, device=dev())
    run_prefill(c, out=out, most=4)


@pytest.mark.parametrize("where", ["k", "v"])
def test_few_rows_nan_reaches_the_rows_that_see_it(where):
    """NaN at key 97 of 100 with 6 new (94..99), and in the middle: elements as the formula has them."""
    for key, window in ((97, 0), (97, 2), (50, 0), (93, 5)):
        c = behind_long_tables(make(26, [100, 90], [6, 2], 16, 4, 16))
        cache = c[where]
        cache[int(c["tables"][0, key // 16]), 1, 16 * 64 + (key % 16) * 8 + 3] = 0x7F
        out = run_prefill(c, window)
        rows = torch.arange(6, device=dev()) + 94
        sees = (rows >= key) & ((rows <= key + window) if window else True)
        bad = out.isnan()
        want = torch.zeros_like(bad)
        want[:6, 4:8, (48 if where == "v" else 0):(64 if where == "v" else 128)] = sees[:, None, None]
        assert torch.equal(bad, want)


def test_few_rows_without_keys_scales_and_workspace():
    c = behind_long_tables(make(27, [3, 64, 0], [8, 2, 3], 8, 2, 16))
    size = kv.paged_prefill_fp4_workspace_bytes(3, 13, 8, 8, 2, c["tables"].shape[1], 16)
    assert size > 0 and kv.paged_prefill_fp4_workspace_bytes(3, 13, 9, 8, 2, 16, 16) == 0
    out = torch.full((15, 8, 128), 7.0, dtype=F16, device=dev())
    q = torch.nn.functional.pad(c["q"], (0, 0, 0, 0, 0, 2))
    run_prefill(dict(c, q=q), 0, 0.5, 0.3, 0.2, out=out, workspace=torch.full((size,), 0xFF, dtype=torch.uint8, device=dev()))
    assert (out[:5] == 0).all() and (out[10:13] == 0).all() and (out[13:] == 7).all()
    want, err = kv4.attention(c["q"][5:10], c["k"], c["v"], c["tables"], [3, 2], [3, 64], 0.2, k_scale=0.5, v_scale=0.3)
    assert_near(out[5:10], want, err)
    short = torch.empty(size - 1, dtype=torch.uint8, device=dev())
    with pytest.raises(ValueError):
        run_prefill(c, workspace=short)


SHARED = [  # cached, new, hq, hkv, page, window, dtype: few query blocks whose keys several CTAs share
    ([3000], [40], 32, 8, 16, 0, BF16), ([2000, 0, 700], [64, 9, 100], 12, 4, 48, 0, F16), ([1030], [70], 64, 1, 64, 0, BF16),
    ([5000], [33], 16, 16, 16, 900, F16), ([0, 2500], [300, 40], 8, 8, 16, 0, BF16), ([600], [33], 6, 6, 256, 0, F16)]


@pytest.mark.parametrize("cached,new,hq,hkv,page,window,dtype", SHARED)
def test_prefill_with_shared_keys(cached, new, hq, hkv, page, window, dtype):
    lens = [a + b for a, b in zip(cached, new)]
    c = make(sum(lens) + hq, lens, new, hq, hkv, page, dtype)
    size = kv.paged_prefill_fp4_workspace_bytes(len(new), sum(new), max(new), hq, hkv, c["tables"].shape[1], page)
    assert size > 0
    want, err = want_of(c, window, decode=False)
    out = torch.full((sum(new) + 3, hq, 128), 7.0, dtype=dtype, device=dev())
    q = torch.nn.functional.pad(c["q"], (0, 0, 0, 0, 0, 3))
    ws = torch.full((size,), 0xFF, dtype=torch.uint8, device=dev())
    run_prefill(dict(c, q=q), window, out=out, workspace=ws)
    assert_near(out[:-3], want, err)
    assert (out[-3:] == 7).all() and torch.equal(run_prefill(c, window), out[:-3])
    with pytest.raises(ValueError):
        kv.paged_prefill_fp4(c["q"], c["k"], c["v"], c["tables"], c["cu_q"], c["cu_k"], max(new), 0.1,
                             workspace=ws[:size // 2 // 16 * 16])


def test_shared_keys_with_holes_nan_and_rows_without_keys():
    c = make(50, [3000, 1500, 20], [60, 40, 50], 16, 4, 16)  # (the last sequence's first 30 rows see no key)
    c["tables"][0, 10:100] = -1
    c["tables"][1, :] = -1
    want, err = want_of(c, decode=False)
    out = run_prefill(c)
    assert_near(out, want, err)
    assert (out[60:130] == 0).all()
    key, block = 2980, 5  # a value that the last 20 rows see
    page = c["v"][int(c["tables"][0, key // 16])]
    page[:, 16 * 64 + (key % 16) * 8 + block] = 0x7F
    got = run_prefill(c)
    nan = got.isnan()
    assert nan[40:60, :, 80:96].all() and int(nan.sum()) == 20 * 16 * 16
    assert_near(torch.where(nan, want.to(got.dtype), got), want, err)


@pytest.mark.parametrize("where", ["k", "v"])
def test_prefill_nan_reaches_the_rows_that_see_it(where):
    """NaN in row 70 of 100 keys with 50 new: rows 20.. of the new see it; with a window the last do not."""
    c = make(24, [100, 90], [50, 20], 16, 4, 16)
    cache = c[where]
    cache[int(c["tables"][0, 70 // 16]), 1, 16 * 64 + (70 % 16) * 8 + 3] = 0x7F
    for window in (0, 13):
        out = run_prefill(c, window)
        bad = out.isnan().any(-1)
        rows = torch.arange(50, device=dev()) + 50
        sees = (rows >= 70) & ((rows <= 70 + 13) if window else True)
        assert torch.equal(bad[:50, 4:8], sees[:, None].expand(50, 4))
        assert not bad[:50, :4].any() and not bad[:50, 8:].any() and not bad[50:].any()


def test_split_prefill_and_decode_agree_with_one_prefill():
    """A prompt in one chunk, in two, and its last token by decode."""
    c = make(25, [333], [333], 32, 8, 16)
    want, err = want_of(c, decode=False)
    one = run_prefill(c)
    assert_near(one, want, err)
    tail = dict(c, q=c["q"][200:], new=[133], cu_q=torch.tensor([0, 133], dtype=torch.int32, device=dev()))
    assert_near(run_prefill(tail), want[200:], err[200:])
    last = dict(c, q=c["q"][332:], new=[1])
    assert_near(run_decode(last), want[332:], err[332:])


def test_attention_directly_behind_the_metadata_that_extends_its_tables():
    """No launch in between: the tables' new entries are seen, next to old ones that the first launch reads."""
    g = gen(40)
    d, i32, page, hq, hkv = dev(), dict(dtype=torch.int32, device=dev()), 16, 16, 4
    cached, new = [16 * (i % 5) for i in range(12)], [1 + 40 * (i % 3) for i in range(12)]
    lens = [a + b for a, b in zip(cached, new)]
    kc, vc = kv4.make_cache(200, hkv, page, g, d), kv4.make_cache(200, hkv, page, g, d)
    old = torch.full((12, 12), -1, **i32)
    for b, n in enumerate(cached):
        old[b, :n // page] = torch.arange(10 * b, 10 * b + n // page)
    free, start = torch.arange(150, 200, **i32), torch.zeros(1, **i32)
    q = randn((sum(new), hq, 128), g)
    one, wide = randn((12, hq, 128), g), torch.full((12, 12 + 128), -1, **i32)
    a, b = torch.tensor(cached, **i32), torch.tensor(new, **i32)
    for tables in (wide[:, :12], wide):
        for _ in range(5):
            wide.fill_(-1)
            wide[:, :12] = old
            torch.cuda.synchronize()
            m = step_metadata(a, b, tables, free, start, page, sum(new))
            pre = kv.paged_prefill_fp4(q, kc, vc, tables, m.cu_seqlens_q, m.cu_seqlens_k, max(new), 0.1)
            wide.fill_(-1)
            wide[:, :12] = old
            torch.cuda.synchronize()
            m = step_metadata(a, b, tables, free, start, page, sum(new))
            dec = kv.paged_decode_fp4(one, kc, vc, tables, m.context_lens, 0.1)
            assert (tables >= 0).sum().item() == sum(-(-n // page) for n in lens)
            assert_near(pre, *kv4.attention(q, kc, vc, tables, new, lens, 0.1))
            assert_near(dec, *kv4.attention(one, kc, vc, tables, [1] * 12, lens, 0.1, decode=True))


def test_output_over_the_queries():
    c = make(42, [900, 33, 0, 500], [3, 1, 0, 2], 16, 4, 16)
    for d in (c, behind_long_tables(c)):
        want = run_prefill(d)
        q = d["q"].clone()
        out = run_prefill(dict(d, q=q), out=q)
        assert out is q and torch.equal(q, want)
    c = make(43, [900, 33, 0, 500], [1] * 4, 16, 4, 16)
    want = run_decode(c)
    q = c["q"].clone()
    assert torch.equal(run_decode(dict(c, q=q), out=q), want)


def test_streams_graphs_and_two_calls_at_once():
    a, b = (make(s, [2900, 3, 250], [1, 1, 1], 32, 8, 16) for s in (31, 32))
    wa, wb = run_decode(a), run_decode(b)
    pa = run_prefill(a)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    call = lambda c, **kw: kv.paged_decode_fp4(c["q"], c["k"], c["v"], c["tables"], c["ctx"], 128 ** -0.5, **kw)  # noqa: E731
    for _ in range(20):
        with torch.cuda.stream(s1):
            x = call(a)
        with torch.cuda.stream(s2):
            y = call(b)
        torch.cuda.synchronize()
        assert torch.equal(x, wa) and torch.equal(y, wb)
    # two graphs with one workspace, replayed in turn
    size = kv.paged_decode_fp4_workspace_bytes(3, 32, 8, a["tables"].shape[1], 16)
    assert size > 0 and size == kv.paged_decode_fp4_workspace_bytes(3, 32, 8, b["tables"].shape[1], 16)
    ws = torch.empty(size, dtype=torch.uint8, device=dev())
    outs, graphs = [], []
    for c in (a, b):
        o = torch.zeros_like(c["q"])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call(c, out=o, workspace=ws)
        outs.append(o)
        graphs.append(g)
    for _ in range(5):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    assert torch.equal(outs[0], wa) and torch.equal(outs[1], wb)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        o = kv.paged_prefill_fp4(a["q"], a["k"], a["v"], a["tables"], a["cu_q"], a["cu_k"], 1, 128 ** -0.5)
    o.zero_()
    g.replay()
    torch.cuda.synchronize()
    assert torch.equal(o, pa)


def test_results_do_not_change_between_runs():
    c = make(33, [5000, 70, 2222, 1], [1] * 4, 32, 8, 16)
    first = run_decode(c)
    assert all(torch.equal(first, run_decode(c)) for _ in range(5))
    for lens, new in (([85], [70]), ([64, 128, 192, 300], [33, 128, 20, 250]), ([2000], [3])):  # one, two, more key blocks
        c = make(36, lens, new, 12, 4, 32)
        first = run_prefill(c)
        assert_near(first, *want_of(c, decode=False))
        assert all(torch.equal(first, run_prefill(c)) for _ in range(25))


def test_refusals():
    c = make(34, [40, 40], [1, 1], 8, 2, 16)
    q, k, v, t, ctx = c["q"], c["k"], c["v"], c["tables"], c["ctx"]
    i32 = torch.int32

    def bad(fn, *args, error=ValueError, **kw):
        with pytest.raises(error):
            fn(*args, **kw)

    dec, pre = kv.paged_decode_fp4, kv.paged_prefill_fp4
    for args in ((q.float(), k, v, t, ctx), (q[..., :64], k, v, t, ctx), (q, k[..., :-8], v[..., :-8], t, ctx),
                 (q, k, v[1:], t, ctx), (q, k.view(torch.int8), v, t, ctx), (q, k, v, t.long(), ctx),
                 (q, k, v, t, ctx.long()), (q, k, v, t, ctx[:1]), (q, k, v, t[:1], ctx), (q[:, :7], k, v, t, ctx),
                 (q, k[:, :, :72 * 8].contiguous(), v[:, :, :72 * 8].contiguous(), t, ctx)):
        bad(dec, *args, 0.1)
    bad(dec, q, k, v, t, ctx, 0.1, window=-1)
    bad(dec, q, k, v, t, ctx, 0.0)
    bad(dec, q, k, v, t, ctx, 0.1, k_scale=-1.0)
    bad(dec, q, k, v, t, ctx, 0.1, v_scale=0.0)
    bad(dec, q, k, v, t, ctx, 0.1, out=torch.empty((2, 8, 64), dtype=BF16, device=dev()))
    wide = torch.nn.functional.pad(t, (0, 200), value=-1)
    bad(dec, q, k, v, wide, ctx, 0.1, workspace=torch.empty(8, dtype=torch.uint8, device=dev()))
    bad(dec, q, k, v, t.cpu(), ctx, 0.1, error=RuntimeError)
    cu = torch.tensor([0, 1, 2], dtype=i32, device=dev())
    bad(pre, q, k, v, t, cu.long(), cu, 1, 0.1)
    bad(pre, q, k, v, t, cu, cu[:2], 1, 0.1)
    bad(pre, q, k, v, t[:1], cu, cu, 1, 0.1)
    bad(pre, q, k, v, t, cu, cu, -1, 0.1)
    bad(pre, q, k, v, t, cu, cu, 1, 0.1, window=-2)
    rows = randn((3, 2, 128), gen(1))
    slots = torch.zeros(3, dtype=i32, device=dev())
    st = kv.store_kvcache_fp4
    bad(st, rows, rows[:2], k, v, slots)
    bad(st, rows, rows.half(), k, v, slots)
    bad(st, rows.float(), rows.float(), k, v, slots)
    bad(st, rows[:, :1], rows[:, :1], k, v, slots)
    bad(st, rows, rows, k, v, slots[:2])
    bad(st, rows, rows, k, v, slots.long())
    bad(st, rows, rows, k, v, slots, 0.0)
    bad(st, rows, rows, k, v, slots, 1e-39)
    pos, table = torch.zeros(3, dtype=torch.int64, device=dev()), torch.zeros(64, device=dev())
    bad(kv.rotary_store_kvcache_fp4, pos, rows, rows, rows, table, k, v, slots)
    bad(kv.read_kvcache_fp4, k, v, slots, torch.float32)
    bad(kv.empty_kvcache_fp4, 1, 1, 8)


def test_empty_calls():
    c = make(35, [40], [1], 8, 2, 16)
    z = c["q"][:0]
    zero = torch.zeros(0, dtype=torch.int32, device=dev())
    assert kv.paged_decode_fp4(z, c["k"], c["v"], c["tables"][:0], zero, 0.1).shape == (0, 8, 128)
    one = torch.zeros(1, dtype=torch.int32, device=dev())
    assert kv.paged_prefill_fp4(z, c["k"], c["v"], c["tables"][:0], one, one, 0, 0.1).shape == (0, 8, 128)
    kv.store_kvcache_fp4(z[:, :2], z[:, :2], c["k"], c["v"], zero)
    assert kv.read_kvcache_fp4(c["k"], c["v"], zero)[0].shape == (0, 2, 128)
