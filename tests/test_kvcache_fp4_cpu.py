"""The 4-bit cache's, rotary and metadata entries without a GPU: every refusal comes before any CUDA call
(pointers are placeholders, never dereferenced), the binding refuses CPU tensors, and the oracle's pieces agree with
independent forms."""
import math

import pytest
import torch

from adallm_b200 import _native as N
from adallm_b200 import build as B
from adallm_b200 import kvcache_fp4 as kv
from adallm_b200.rotary_embedding import apply_rotary, build_cos_sin_cache
from adallm_b200.step_metadata import step_metadata
from oracle import kv4

BAD, UNSUP, ALIGN, WS = N.ADA_ERR_INVALID_ARG, N.ADA_ERR_UNSUPPORTED, N.ADA_ERR_ALIGNMENT, N.ADA_ERR_WORKSPACE


@pytest.fixture(scope="module")
def lib():
    B.build()
    return N.lib()


def refuse(fn, good, cases):
    """good: the arguments of an accepted call by name (in order); cases: ({name: value}, status)."""
    for change, want in cases:
        assert set(change) <= set(good)
        assert fn(*{**good, **change}.values()) == want, change


DECODE = dict(q=16, qd=0, qsb=1024, qsh=128, k=16, v=16, sp=8 * 1152, sh=1152, pages=4, bt=16, bts=4, mp=4, ctx=16,
              batch=1, hq=32, hkv=8, d=128, page=16, scale=0.1, ks=1.0, vs=1.0, window=0, out=32, od=0, osb=4096, osh=128,
              ws=16, wsb=1 << 30, stream=None)


def test_decode_refusals(lib):
    assert lib.ada_kv4_paged_decode(*{**DECODE, "batch": 0}.values()) == 0
    refuse(lib.ada_kv4_paged_decode, DECODE, [
        (dict(batch=-1), BAD), (dict(q=None), BAD), (dict(k=None), BAD), (dict(v=None), BAD), (dict(bt=None), BAD),
        (dict(ctx=None), BAD), (dict(out=None), BAD), (dict(qd=2), BAD), (dict(od=-1), BAD), (dict(d=64), UNSUP),
        (dict(page=24), UNSUP), (dict(page=0), BAD), (dict(hq=31), BAD), (dict(hkv=0), BAD), (dict(hq=0), BAD),
        (dict(window=-1), BAD), (dict(bts=3), BAD), (dict(mp=0), BAD), (dict(pages=0), BAD), (dict(scale=0.0), BAD),
        (dict(scale=math.nan), BAD), (dict(scale=math.inf), BAD), (dict(ks=-1.0), BAD), (dict(vs=0.0), BAD),
        (dict(ks=math.inf), BAD), (dict(ks=1e-39), BAD), (dict(vs=math.inf), BAD),
        (dict(page=1 << 25, sp=1 << 36, sh=1 << 32), UNSUP), (dict(hq=1 << 30, hkv=1 << 30, mp=1 << 26, bts=1 << 26), UNSUP), (dict(q=8), ALIGN), (dict(k=8), ALIGN),
        (dict(out=24), ALIGN), (dict(qsh=132), ALIGN), (dict(osb=4100), ALIGN), (dict(sh=1160, sp=9999), ALIGN),
        (dict(sp=8 * 1152 + 8), ALIGN), (dict(sh=1136), BAD), (dict(bt=18), ALIGN), (dict(ctx=17), ALIGN),
        (dict(mp=1 << 27, bts=1 << 27), UNSUP), (dict(mp=200, bts=200, ws=None), WS),
        (dict(mp=200, bts=200, wsb=1), WS), (dict(mp=200, bts=200, ws=24), ALIGN), (dict(batch=8193), UNSUP)])
    size = lib.ada_kv4_paged_decode_workspace_size
    assert size(0, 32, 8, 100, 16, 0) == 0 and size(16, 32, 8, 100, 16, 0) > 0
    assert size(1, 32, 8, 80, 16, 0) == 0 and size(1, 32, 8, 81, 16, 0) > 0 and size(37, 32, 8, 81, 16, 1000) == 0


PREFILL = dict(q=16, qd=0, qst=1024, qsh=128, k=16, v=16, sp=8 * 1152, sh=1152, pages=4, bt=16, bts=4, mp=4, cq=16, ck=16,
               batch=1, total=50, most=50, hq=32, hkv=8, d=128, page=16, scale=0.1, ks=1.0, vs=1.0, window=0, out=32, od=0,
               ost=4096, osh=128, ws=None, wsb=0, err=None, stream=None)


def test_prefill_refusals(lib):
    for k in ("batch", "total", "most"):
        assert lib.ada_kv4_paged_prefill(*{**PREFILL, k: 0}.values()) == 0
        assert lib.ada_kv4_paged_prefill(*{**PREFILL, k: -1}.values()) == BAD
    refuse(lib.ada_kv4_paged_prefill, PREFILL, [
        (dict(q=None), BAD), (dict(k=None), BAD), (dict(bt=None), BAD), (dict(cq=None), BAD), (dict(ck=None), BAD),
        (dict(out=None), BAD), (dict(qd=2), BAD), (dict(d=256), UNSUP), (dict(page=8), UNSUP), (dict(hq=33), BAD),
        (dict(window=-1), BAD), (dict(scale=-0.1), BAD), (dict(vs=math.nan), BAD), (dict(q=8), ALIGN), (dict(v=4), ALIGN),
        (dict(ost=4), ALIGN), (dict(cq=18), ALIGN), (dict(err=2), ALIGN), (dict(batch=70000), UNSUP),
        (dict(most=8, mp=40, bts=40), WS), (dict(most=8, mp=40, bts=40, ws=16, wsb=100), WS),
        (dict(most=8, mp=40, bts=40, ws=8, wsb=1 << 30), ALIGN), (dict(total=3, mp=40, bts=40), WS), (dict(mp=40, bts=40), WS),
        (dict(mp=40, bts=40, ws=16, wsb=1 << 20), WS), (dict(mp=40, bts=40, ws=8, wsb=1 << 30), ALIGN)])
    size = lib.ada_kv4_paged_prefill_workspace_size
    assert size(1, 50, 50, 32, 8, 20, 16) == 0 and size(1, 50, 50, 32, 8, 40, 16) > 0 and size(1, 50, 8, 32, 8, 40, 16) > 0
    assert size(1, 50, 8, 32, 8, 16, 16) == 0 and size(1, 0, 8, 32, 8, 40, 16) == 0
    assert size(8000, 8000, 1, 1 << 30, 1 << 30, 1 << 26, 16) == 0 and size(1, 1, 1, 8, 8, 1 << 30, 1 << 30) == 0


STORE = dict(pos=16, q=32, qst=4096, qsh=128, k=48, kst=1024, ksh=128, v=64, vst=1024, vsh=128, qo=80, t=3, hq=32, hkv=8,
             d=128, table=16, maxp=10, rot=128, inter=0, slots=16, kc=16, vc=16, sp=8 * 1152, sh=1152, pages=4, page=16,
             ks=1.0, vs=1.0, dt=0, stream=None)


def test_store_refusals(lib):
    assert lib.ada_kv4_store(*{**STORE, "t": 0}.values()) == 0
    refuse(lib.ada_kv4_store, STORE, [
        (dict(t=-1), BAD), (dict(q=None), BAD), (dict(qo=None), BAD), (dict(qo=32), BAD), (dict(k=None), BAD),
        (dict(v=None), BAD), (dict(slots=None), BAD), (dict(kc=None), BAD), (dict(table=None), BAD), (dict(maxp=0), BAD),
        (dict(rot=0), BAD), (dict(rot=144), BAD), (dict(rot=40), UNSUP), (dict(d=64), UNSUP), (dict(page=20), UNSUP),
        (dict(ks=0.0), BAD), (dict(vs=math.nan), BAD), (dict(ks=math.inf), BAD), (dict(vs=1e-39), BAD),
        (dict(page=1 << 25, sp=1 << 36, sh=1 << 32), UNSUP), (dict(dt=2), BAD), (dict(q=8), ALIGN), (dict(kst=1020), ALIGN),
        (dict(vsh=4), ALIGN), (dict(kc=8), ALIGN), (dict(table=18), ALIGN), (dict(pos=12), ALIGN)])


def test_rotary_and_read_refusals(lib):
    good = dict(pos=16, q=32, qst=4096, qsh=128, k=48, kst=1024, ksh=128, qo=64, ko=80, t=3, hq=32, hkv=8, d=128, table=16,
                maxp=10, rot=64, inter=1, dt=1, stream=None)
    assert lib.ada_rotary(*{**good, "t": 0}.values()) == 0
    refuse(lib.ada_rotary, good, [
        (dict(pos=None), BAD), (dict(q=None), BAD), (dict(k=None), BAD), (dict(qo=None), BAD), (dict(ko=None), BAD),
        (dict(qo=32), BAD), (dict(ko=48), BAD), (dict(d=120), UNSUP), (dict(d=2048), UNSUP), (dict(rot=8), UNSUP),
        (dict(rot=256), BAD), (dict(dt=2), BAD), (dict(t=-2), BAD), (dict(hq=-1), BAD), (dict(qsh=4), ALIGN),
        (dict(ko=88), ALIGN)])
    good = dict(kc=16, vc=16, sp=8 * 1152, sh=1152, pages=4, page=16, hkv=8, d=128, slots=16, t=3, ks=1.0, vs=1.0, k=16,
                v=32, dt=0, stream=None)
    assert lib.ada_kv4_read(*{**good, "t": 0}.values()) == 0
    refuse(lib.ada_kv4_read, good, [
        (dict(kc=None), BAD), (dict(slots=None), BAD), (dict(k=None), BAD), (dict(v=40), ALIGN), (dict(dt=2), BAD),
        (dict(d=96), UNSUP), (dict(page=15), UNSUP), (dict(ks=0.0), BAD), (dict(vs=math.inf), BAD), (dict(t=-1), BAD)])


def test_metadata_refusals(lib):
    good = dict(c=16, n=20, b=2, bt=16, bts=4, mp=4, free=16, nf=9, start=24, page=16, t=8, pos=16, slots=16, cq=16, ck=16,
                ctx=32, nxt=28, err=None, stream=None)
    refuse(lib.ada_step_metadata, good, [
        (dict(b=-1), BAD), (dict(b=8193), UNSUP), (dict(page=0), BAD), (dict(t=-1), BAD), (dict(c=None), BAD),
        (dict(bt=None), BAD), (dict(bts=3), BAD), (dict(free=None), BAD), (dict(start=None), BAD), (dict(pos=None), BAD),
        (dict(slots=None), BAD), (dict(cq=None), BAD), (dict(ck=None), BAD), (dict(ctx=None), BAD), (dict(nxt=None), BAD),
        (dict(nxt=24), BAD), (dict(ctx=16), BAD), (dict(ctx=20), BAD), (dict(pos=12), ALIGN), (dict(slots=18), ALIGN),
        (dict(t=1 << 31), UNSUP)])


def test_packed_calls_are_the_entries_themselves(lib):
    """Every entry's refusals come back the same through ada_call, argument by argument."""
    store = dict(STORE)
    cases = [(N.kv4_paged_decode, lib.ada_kv4_paged_decode, DECODE), (N.kv4_paged_prefill, lib.ada_kv4_paged_prefill, PREFILL),
             (N.kv4_store, lib.ada_kv4_store, store)]
    for packed, entry, good in cases:
        assert len(good) == len(entry.argtypes)
        for name in good:
            for value in (-1, 0, 3, 7.5 if isinstance(good[name], float) else 1 << 40):
                change = {**good, name: value}
                if value == 1 << 40 and entry.argtypes[list(good).index(name)] in (N.I32, N.INT):
                    assert lib.ada_call(packed.entry, packed.pack(*(v or 0 for v in change.values()))) == UNSUP
                    continue
                if isinstance(good[name], float):
                    value = change[name] = float(value)
                change["page"] = 20  # (no call is good, but for those that have nothing to do)
                want = entry(*change.values())
                assert lib.ada_call(packed.entry, packed.pack(*(v or 0 for v in change.values()))) == want, (name, value)
    assert lib.ada_call(0, b"\0" * 300) == BAD and lib.ada_call(7, b"\0" * 300) == BAD
    assert lib.ada_call(1, None) == BAD


def test_cpu_tensors_are_refused():
    k, v = kv.empty_kvcache_fp4(2, 2, 16)
    q = torch.zeros((1, 4, 128), dtype=torch.bfloat16)
    one = torch.ones(1, dtype=torch.int32)
    with pytest.raises(RuntimeError):
        kv.paged_decode_fp4(q, k, v, one[:, None], one, 0.1)
    with pytest.raises(RuntimeError):
        kv.store_kvcache_fp4(q[:, :2], q[:, :2], k, v, one)
    with pytest.raises(RuntimeError):
        apply_rotary(one.long(), q, q, torch.zeros((4, 64)))
    with pytest.raises(RuntimeError):
        step_metadata(one, one, one[:, None], one, one, 16, 4)
    with pytest.raises(ValueError):
        kv.empty_kvcache_fp4(2, 2, 24)


def test_error_words_name_their_bits():
    assert N.describe_error_word(0x100).startswith("the free list")
    assert N.describe_error_word(0x600).count(";") == 1
    assert "prefill" in N.describe_error_word(0x70)


def test_quantiser_against_every_neighbour():
    """No other code is nearer, and a tie has the even code."""
    g = torch.Generator().manual_seed(0)
    x = torch.cat((torch.randn((200, 16), generator=g), torch.randn((200, 16), generator=g).to(torch.bfloat16).float(),
                   torch.randint(-24, 25, (200, 16), generator=g) / 4.0))
    code, scale = kv4.quantise(x)
    s = scale.view(torch.float8_e4m3fn).double()
    lut = torch.tensor(kv4.MAG + tuple(-m for m in kv4.MAG), dtype=torch.float64)
    off = (x.double()[..., None] / s[..., None] - lut).abs()
    best = off.amin(-1)
    mine = off.gather(-1, code.long()[..., None])[..., 0]
    assert (mine <= best).all()
    tie = (off == best[..., None])[..., :8].sum(-1) > 1
    assert tie.any() and (code[tie] % 2 == 0).all()
    assert torch.equal(s[:, 0], (x.abs().amax(-1) / 6).to(torch.float8_e4m3fn).double())


def test_yarn_table():
    """Pairs of many turns keep their angles, pairs of less than one are slowed, both times the amplitude."""
    yarn = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 1024}
    t = build_cos_sin_cache(128, 4096, 1e6, yarn)
    assert t.shape == (4096, 1, 128) and t.dtype == torch.float32
    amp = 0.1 * math.log(4.0) + 1
    pos = torch.arange(4096, dtype=torch.float64)
    for pair, slow in ((0, 1.0), (5, 1.0), (40, 4.0), (63, 4.0)):
        a = pos * 1e6 ** (-pair / 64) / slow
        assert torch.allclose(t[:, 0, pair].double(), a.cos() * amp, atol=1e-7 * amp, rtol=0)
        assert torch.allclose(t[:, 0, 64 + pair].double(), a.sin() * amp, atol=1e-7 * amp, rtol=0)
    with pytest.raises(ValueError):
        build_cos_sin_cache(128, 16, 1e6, {"rope_type": "other", "factor": 2.0})


def test_attention_oracle_against_a_direct_sum():
    g = torch.Generator().manual_seed(1)
    k, v = kv4.make_cache(3, 1, 16, g), kv4.make_cache(3, 1, 16, g)
    q = torch.randn((2, 2, 128), generator=g)
    table = torch.tensor([[2, 0, -1]])
    out, err = kv4.attention(q, k, v, table, [2], [20], 0.1, window=3)
    kk, there = kv4.rows_of(k, table[0], 20)
    vv, _ = kv4.rows_of(v, table[0], 20)
    assert there.all() and (err > 0).all()
    for i, seen in ((0, range(15, 19)), (1, range(16, 20))):
        for h in range(2):
            w = torch.tensor([float(q[i, h].double() @ kk[t, 0]) * 0.1 for t in seen], dtype=torch.float64).exp()
            want = sum(w[j] * vv[t, 0] for j, t in enumerate(seen)) / w.sum()
            assert torch.allclose(out[i, h], want, atol=1e-12)
    dec, _ = kv4.attention(q[1:], k, v, table, [1], [20], 0.1, window=4, decode=True)
    assert torch.allclose(dec[0], out[1])
