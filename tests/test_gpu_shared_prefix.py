"""Shared-prefix decode attention (through the C ABI) vs its definition in 64 bits.

Tolerances.  Inputs are exact on both sides (bf16/fp16 queries, e4m3 cache); what is left is the
fp32 score (relative 2^-20 or so), probabilities held in no fewer than 11 bits for P.V (at most
2^-11 of each weight) and the output's own rounding (at most 2^-8 relative for bf16, 2^-11 fp16).
Element-wise: 2^-8 (2^-11) of the element plus 2^-10 of the largest |v| of the case (weights sum to
one, so their rounding moves an element by at most 2^-11 max|v|; doubled for the row sum and the
scores).  Over all elements: roundings are spread evenly below their bounds, so the relative
2-norm is below 2^-8.5 (bf16) and 2^-10 (fp16)."""
import pytest
import torch

from adallm_b200.shared_prefix import shared_prefix_decode, shared_prefix_workspace_bytes
from oracle import speculative as osp
from tests.gpu_util import dev, rel_l2

pytestmark = pytest.mark.gpu

REL = {torch.bfloat16: 2 ** -8.5, torch.float16: 2 ** -10}
ULP = {torch.bfloat16: 2 ** -8, torch.float16: 2 ** -11}


REACH = 0


@pytest.fixture(params=[0, 1 << 18], ids=["", "wide"], autouse=True)
def reach(request):
    """Every test also with prefix tables padded to a long reach: from 33 rows a prefix on, the
    library then takes the tensor-core kernel for the prefixes whatever their lengths."""
    global REACH
    REACH = request.param
    yield
    REACH = 0


def _to_gpu(case):
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in case.items()}
    pad = REACH // c["k_cache"].shape[1] - c["prefix_tables"].shape[1]
    if pad > 0:
        c["prefix_tables"] = torch.nn.functional.pad(c["prefix_tables"], (0, pad), value=-1)
    return c


def _args(c, **kw):
    a = dict(cu_seqlens_q=c["cu_seqlens_q"])
    a.update(kw)
    return (c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"], c["cu_groups"],
            c["block_tables"], c["context_lens"], c["scale"]), a


def _check(out, ref, case, v_scale=1.0):
    out = out.cpu()
    assert bool(torch.isfinite(out.float()).all())
    dt = out.dtype
    bits = case["v_cache"].view(torch.uint8)
    vmax = float(torch.where((bits & 0x7F) == 0x7F, torch.zeros_like(bits), bits).view(torch.float8_e4m3fn)
                 .float().abs().max()) * abs(v_scale)
    off = (out.double() - ref).abs() - ULP[dt] * ref.abs() - 2 ** -10 * vmax
    assert float(off.max()) <= 0, float(off.max())
    if float(ref.norm()) > 0:
        assert rel_l2(out, ref) < REL[dt]
    dead = ref.abs().amax(dim=(1, 2)) == 0
    assert not bool(out[dead].any())


def _run(case, **kw):
    a, k = _args(_to_gpu(case), **kw)
    out = shared_prefix_decode(*a, **k)
    torch.cuda.synchronize()
    ref_a, ref_k = _args(case, **kw)
    _check(out, osp.shared_prefix_decode(*ref_a, **ref_k), case, kw.get("v_scale", 1.0))
    return out


@pytest.mark.parametrize("hq,hkv,page", [(32, 8, 16), (32, 16, 32), (8, 8, 256), (32, 2, 16), (16, 2, 48)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_heads_and_pages(hq, hkv, page, dtype):
    _run(osp.make_shared_prefix_case(1, [333], [5], [1, 16, 17, 100, 250], [1] * 5, hq, hkv, page, dtype))


@pytest.mark.parametrize("prefix", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 255, 257, 1000])
@pytest.mark.parametrize("rows", [[1, 1, 1], [9, 3, 1], [30, 35, 2]])
def test_prefix_lengths(prefix, rows):
    _run(osp.make_shared_prefix_case(2, [prefix], [3], [9, 2, 40], rows, 32, 8, 16))


@pytest.mark.parametrize("own", [0, 1, 15, 16, 17, 63, 64, 65, 127, 128, 129, 400])
def test_own_lengths(own):
    """Own keys from none (the query then stands on the prefix's last key) to several tiles."""
    _run(osp.make_shared_prefix_case(3, [70], [2], [own, 33], [1, 1], 32, 8, 16))


@pytest.mark.parametrize("rows", [[1, 2, 3, 5], [9, 1, 0, 4], [40, 33, 1, 7], [0, 0, 1, 0]])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_rows_of_drafts(rows, dtype):
    """Several rows a sequence (and none), causal among the newest tokens."""
    _run(osp.make_shared_prefix_case(4, [190], [4], [50, 64, 3, 90], rows, 32, 8, 16, dtype))


def test_more_rows_than_own_keys():
    """Rows older than the own keys stand inside the prefix; before position 0 they see nothing."""
    _run(osp.make_shared_prefix_case(5, [3, 40], [1, 1], [2, 1], [8, 5], 32, 8, 16))


@pytest.mark.parametrize("sizes,prefixes", [([3, 4, 1], [100, 7, 300]), ([0, 8, 0], [50, 60, 70]),
                                            ([2, 2, 2], [0, 513, 0])])
def test_groups(sizes, prefixes):
    n = 8
    for rows in ([1, 2, 1, 1, 3, 1, 1, 2], [17, 20, 40, 1, 9, 30, 3, 16]):
        _run(osp.make_shared_prefix_case(6, prefixes, sizes, [5, 30, 64, 1, 129, 17, 70, 16], rows, 32, 8, 16)
             | {"n": n})


def test_many_groups_and_sequences():
    g = torch.Generator().manual_seed(0)
    sizes = torch.randint(0, 6, (40,), generator=g).tolist()
    n = sum(sizes) + 3
    prefixes = torch.randint(0, 150, (40,), generator=g).tolist()
    own = torch.randint(0, 60, (n,), generator=g).tolist()
    rows = torch.randint(0, 4, (n,), generator=g).tolist()
    _run(osp.make_shared_prefix_case(7, prefixes, sizes, own, rows, 16, 4, 16))


def test_wide_batches_fill_several_row_blocks():
    n = 70
    _run(osp.make_shared_prefix_case(8, [300], [n], [1 + (7 * i) % 50 for i in range(n)], [1 + i % 3 for i in range(n)],
                                     32, 8, 16))


@pytest.mark.parametrize("window", [1, 2, 17, 64, 130, 1024])
@pytest.mark.parametrize("rows", [[1, 1, 1], [4, 2, 5], [30, 9, 40]])
def test_window(window, rows):
    """Windows inside the own keys, across the prefix's end and over everything."""
    _run(osp.make_shared_prefix_case(9, [200], [3], [5, 60, 150], rows, 32, 16, 16), window=window)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_holes_in_the_tables(dtype):
    for seed, rows in enumerate(([1, 2, 1, 3], [20, 2, 1, 3], [12, 30, 9, 30])):
        _run(osp.make_shared_prefix_case(10 + seed, [430, 340], [2, 2], [20, 70, 0, 33], rows, 32, 8, 16, dtype,
                                         holes=12))
    # every page a hole: nothing to see, zeros
    case = osp.make_shared_prefix_case(14, [40], [2], [20, 30], [1, 2], 32, 8, 16)
    case["prefix_tables"].fill_(-1)
    case["block_tables"].fill_(1 << 30)
    assert not bool(_run(case).any())


def test_lengths_past_the_tables_are_cut_off():
    case = osp.make_shared_prefix_case(15, [64], [2], [32, 32], [1, 1], 32, 8, 16)
    case["prefix_tables"] = case["prefix_tables"][:, :4].contiguous()
    case["block_tables"] = case["block_tables"][:, :2].contiguous()
    full = _run(case)
    if not REACH:
        case["prefix_lens"] += 1000
    case["context_lens"] += 5000
    assert torch.equal(_to_gpu_run(case), full)
    case["prefix_lens"].fill_(-5)
    case["context_lens"].fill_(-5)
    assert not bool(_to_gpu_run(case).any())


def _to_gpu_run(case, **kw):
    a, k = _args(_to_gpu(case), **kw)
    out = shared_prefix_decode(*a, **k)
    torch.cuda.synchronize()
    return out


@pytest.mark.parametrize("rows", [[2, 1, 1], [20, 11, 3]])
def test_peaked_and_flat_scores(rows):
    """Large scores (one key takes all the weight; rising maxima along the keys) and none (q = 0)."""
    case = osp.make_shared_prefix_case(16, [500], [3], [40, 80, 3], rows, 32, 8, 16, q_gain=12.0)
    _run(case)
    case["q"].zero_()
    _run(case)
    rising = osp.make_shared_prefix_case(17, [512], [2], [64, 10], [30, 9] if rows[0] > 2 else [1, 1], 8, 8, 16)
    order = rising["prefix_tables"][0]
    k = rising["k_cache"].float()
    for j in range(512):  # scores grow steadily: the running maximum moves in every tile
        k[order[j // 16], j % 16] = rising["q"][0].float() * (0.02 * j - 4.0) / 8.0
    rising["q"][1:] = rising["q"][:1] * torch.linspace(0.5, 1.0, len(rising["q"]) - 1)[:, None, None]
    rising["k_cache"] = k.to(torch.float8_e4m3fn)
    _run(rising)


def test_scales_and_output_type():
    case = osp.make_shared_prefix_case(18, [100], [2], [20, 30], [1, 2], 32, 8, 16, torch.float16)
    _run(case, k_scale=0.25, v_scale=3.0)
    c = _to_gpu(case)
    a, k = _args(c)
    out = torch.empty(c["q"].shape, dtype=torch.bfloat16, device=dev())
    shared_prefix_decode(*a, **k, out=out)
    ref_a, ref_k = _args(case)
    _check(out, osp.shared_prefix_decode(*ref_a, **ref_k), case)


def test_strides():
    """q and out inside wider rows, heads apart; caches inside a [2, layers, ...] buffer."""
    case = osp.make_shared_prefix_case(19, [90], [3], [20, 30, 5], [2, 1, 1], 32, 8, 16)
    c = _to_gpu(case)
    wide = torch.zeros((4, 40, 144), dtype=torch.bfloat16, device=dev())
    wide[:, 3:35, :128] = c["q"]
    kv = torch.full((2, 3) + tuple(c["k_cache"].shape), osp.NAN_BYTE, dtype=torch.uint8, device=dev())
    kv[0, 1] = c["k_cache"].view(torch.uint8)
    kv[1, 1] = c["v_cache"].view(torch.uint8)
    kv = kv.view(torch.float8_e4m3fn)
    out = torch.full((4, 33, 136), 7.0, dtype=torch.bfloat16, device=dev())
    c2 = dict(c, q=wide[:, 3:35, :128], k_cache=kv[0, 1], v_cache=kv[1, 1])
    a, k = _args(c2)
    shared_prefix_decode(*a, **k, out=out[:, :32, :128])
    ref_a, ref_k = _args(case)
    _check(out[:, :32, :128], osp.shared_prefix_decode(*ref_a, **ref_k), case)
    assert bool((out[:, 32:] == 7).all()) and bool((out[:, :, 128:] == 7).all())


def test_cache_offsets_past_32_bits():
    """Pages 500 MB apart: the last one starts past 2^32 bytes."""
    case = osp.make_shared_prefix_case(20, [100], [2], [30, 20], [1, 2], 32, 8, 16)
    pages = case["k_cache"].shape[0]
    step = 5 * 10 ** 8 // 16 * 16
    buf = torch.empty(step * pages + (1 << 20), dtype=torch.uint8, device=dev())
    size = (pages, 16, 8, 128)
    k = torch.as_strided(buf, size, (step, 1024, 128, 1), 0)
    v = torch.as_strided(buf, size, (step, 1024, 128, 1), 65536)
    k.copy_(case["k_cache"].view(torch.uint8))
    v.copy_(case["v_cache"].view(torch.uint8))
    assert step * (pages - 1) > 1 << 32
    c = dict(_to_gpu(case), k_cache=k.view(torch.float8_e4m3fn), v_cache=v.view(torch.float8_e4m3fn))
    a, kw = _args(c)
    out = shared_prefix_decode(*a, **kw)
    ref_a, ref_k = _args(case)
    _check(out, osp.shared_prefix_decode(*ref_a, **ref_k), case)


def test_defaults_and_rows_of_no_sequence():
    """One group without cu_groups, one row each without cu_seqlens_q, no prefix, padding rows."""
    case = osp.make_shared_prefix_case(21, [50], [4], [20, 30, 1, 9], [1] * 4, 32, 8, 16)
    full = _to_gpu_run(case)
    c = _to_gpu(case)
    a, _ = _args(c)
    assert torch.equal(shared_prefix_decode(*a[:5], None, *a[6:]), full)
    none = torch.empty(0, dtype=torch.int32, device=dev())
    alone = shared_prefix_decode(*a[:3], c["prefix_tables"][:0], none, None, *a[6:])
    zero = dict(case, prefix_lens=torch.zeros(1, dtype=torch.int32))
    ref_a, ref_k = _args(zero)
    _check(alone, osp.shared_prefix_decode(*ref_a, **ref_k), case)
    padded = dict(c, q=torch.cat((c["q"], c["q"][:2])))
    a, k = _args(padded)
    out = shared_prefix_decode(*a, **k)
    assert torch.equal(out[:4], full) and not bool(out[4:].any())


def test_same_result_twice_on_another_stream_and_in_a_graph():
    case = osp.make_shared_prefix_case(22, [700, 90], [6, 2], [5, 100, 64, 1, 30, 70, 20, 33], [1, 3, 1, 2, 1, 1, 4, 1],
                                       32, 8, 16)
    c = _to_gpu(case)
    a, k = _args(c)
    first = shared_prefix_decode(*a, **k)
    assert torch.equal(shared_prefix_decode(*a, **k), first)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = shared_prefix_decode(*a, **k)
    side.synchronize()
    assert torch.equal(other, first)
    need = shared_prefix_workspace_bytes(first.shape[0], 2, 8, 32, 8, 128)
    ws = torch.empty(need, dtype=torch.uint8, device=dev())
    out = torch.zeros_like(first)
    with torch.cuda.stream(side):
        shared_prefix_decode(*a, **k, out=out, workspace=ws)
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            shared_prefix_decode(*a, **k, out=out, workspace=ws)
    ws.fill_(0xFF)  # whatever an earlier use left behind
    out.zero_()
    for _ in range(3):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, first)
    # lengths are read on the device: the graph follows them
    c["context_lens"].sub_(1)
    c["prefix_lens"].sub_(3)
    graph.replay()
    torch.cuda.synchronize()
    moved = dict(case, context_lens=case["context_lens"] - 1, prefix_lens=case["prefix_lens"] - 3)
    ref_a, ref_k = _args(moved)
    _check(out, osp.shared_prefix_decode(*ref_a, **ref_k), case)


def test_agrees_with_the_decode_and_prefill_entries():
    """With the prefix's pages in front of the own table, the single-sequence entries see the same keys."""
    from adallm_b200.attention import paged_decode, paged_prefill
    case = _to_gpu(osp.make_shared_prefix_case(23, [96], [3], [20, 64, 7], [1, 1, 1], 32, 8, 16))
    a, k = _args(case)
    out = shared_prefix_decode(*a, **k)
    joined = torch.cat((case["prefix_tables"][:, :6].expand(3, -1), case["block_tables"]), 1).contiguous()
    one = paged_decode(case["q"], case["k_cache"], case["v_cache"], joined, case["context_lens"] + 96, case["scale"])
    assert rel_l2(out, one) < 2 * REL[torch.bfloat16]
    case = _to_gpu(osp.make_shared_prefix_case(24, [96], [3], [20, 64, 7], [3, 1, 5], 32, 8, 16))
    a, k = _args(case)
    out = shared_prefix_decode(*a, **k)
    joined = torch.cat((case["prefix_tables"][:, :6].expand(3, -1), case["block_tables"]), 1).contiguous()
    cu_k = torch.tensor([0, 116, 276, 379], dtype=torch.int32, device=dev())
    many = paged_prefill(case["q"], case["k_cache"], case["v_cache"], joined, case["cu_seqlens_q"], cu_k, 5,
                         case["scale"])
    assert rel_l2(out, many) < 2 * REL[torch.bfloat16]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_queries_of_any_size(dtype):
    """Rows scaled from the smallest normal numbers to the largest, and rows with one large element."""
    case = osp.make_shared_prefix_case(26, [200], [3], [20, 33, 40], [20, 16, 9], 32, 8, 16, dtype)
    top = 1e30 if dtype == torch.bfloat16 else 6e4
    gain = torch.logspace(-4.0, 0.0, 45)
    case["q"] = (case["q"].float() * gain[:, None, None]).to(dtype)
    case["q"][3, :, 5] = 30.0
    case["q"][7, :, 77] = -200.0
    _run(case)
    case["q"][0] = top / 8 * torch.sign(case["q"][0].float() + 1e-9).to(dtype)  # one key takes it all
    a, k = _args(_to_gpu(case))
    out = shared_prefix_decode(*a, **k)
    assert bool(torch.isfinite(out[0].float()).all())
    case["q"][1, 2, 3] = float("inf")
    case["q"][2, 4, 100] = float("nan")
    a, k = _args(_to_gpu(case))
    out = shared_prefix_decode(*a, **k).float().cpu()
    assert bool(torch.isnan(out[1, 2]).all()) and bool(torch.isnan(out[2, 4]).all())
    assert int(torch.isnan(out).any(-1).sum()) == 2  # and no other row


def test_empty_calls():
    case = _to_gpu(osp.make_shared_prefix_case(25, [20], [2], [5, 6], [1, 1], 32, 8, 16))
    a, k = _args(case)
    k = {"cu_seqlens_q": torch.zeros(3, dtype=torch.int32, device=dev())}
    assert shared_prefix_decode(case["q"][:0], *a[1:], **k).shape == (0, 32, 128)
    assert not bool(shared_prefix_decode(*a, **k).any())  # rows, but none of them owned


def test_as_many_sequences_as_there_may_be():
    """4,095 sequences behind one prefix; one more is refused."""
    n = 4095
    case = osp.make_shared_prefix_case(26, [20], [n], [1 + i % 3 for i in range(n)], [1] * n, 2, 2, 16)
    out = _run(case)
    c = _to_gpu(case)
    with pytest.raises(ValueError):
        shared_prefix_decode(out[:1].expand(n + 1, -1, -1), c["k_cache"], c["v_cache"], c["prefix_tables"],
                             c["prefix_lens"], None, c["block_tables"][:1].expand(n + 1, -1),
                             c["context_lens"][:1].repeat(n + 1), 1.0)


def test_refusals():
    case = _to_gpu(osp.make_shared_prefix_case(27, [20], [2], [5, 6], [1, 1], 32, 8, 16))
    good = dict(zip(("q", "k_cache", "v_cache", "prefix_tables", "prefix_lens", "cu_groups", "block_tables",
                     "context_lens", "scale"), _args(case)[0]))
    need = shared_prefix_workspace_bytes(2, 1, 2, 32, 8, 128)
    q, k, v = good["q"], good["k_cache"], good["v_cache"]
    wrong = [dict(q=q.float()), dict(q=q[..., :64]), dict(q=q[:1]), dict(q=q[:, :30]), dict(k_cache=k.view(torch.uint8)),
             dict(v_cache=v[:, :, :4]), dict(prefix_tables=good["prefix_tables"].long()),
             dict(prefix_lens=good["prefix_lens"].long()), dict(prefix_lens=good["prefix_lens"].repeat(2)),
             dict(cu_groups=good["cu_groups"][:1]), dict(block_tables=good["block_tables"][:1]),
             dict(context_lens=good["context_lens"].float()), dict(scale=0.0), dict(scale=float("nan")),
             dict(scale=-1.0), dict(window=-1), dict(cu_seqlens_q=torch.zeros(2, dtype=torch.int32, device=dev())),
             dict(out=q.float()), dict(out=q[:1]), dict(workspace=torch.empty(need - 256, dtype=torch.uint8, device=dev()))]
    for kw in wrong:
        with pytest.raises(ValueError):
            shared_prefix_decode(**{**good, **kw})
    for name in ("q", "k_cache", "v_cache", "prefix_tables", "prefix_lens", "block_tables", "context_lens", "cu_groups"):
        with pytest.raises(RuntimeError, match="CUDA"):
            shared_prefix_decode(**{**good, name: good[name].cpu()})
    with pytest.raises(RuntimeError, match="CUDA"):
        shared_prefix_decode(**good, workspace=torch.empty(need, dtype=torch.uint8))
    assert bool(torch.isfinite(shared_prefix_decode(**good).float()).all())


def test_many_segments_give_the_same_every_time():
    """More segments than the split length is searched over: all warps still agree on one."""
    n = 320
    case = osp.make_shared_prefix_case(28, [900, 1200, 40, 300, 1], [64] * 5, [1 + (37 * i) % 700 for i in range(n)],
                                       [1] * n, 8, 8, 16)
    out = _run(case)
    a, k = _args(_to_gpu(case))
    for _ in range(200):
        assert torch.equal(shared_prefix_decode(*a, **k), out)


@pytest.mark.parametrize("prefixes,sizes", [([3000], [4]), ([6000], [4]), ([700, 2500], [3, 1])])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_long_prefixes(prefixes, sizes, dtype):
    """Blocks of keys for half of the SMs (several each) and for all of them, ranges that cross units."""
    _run(osp.make_shared_prefix_case(29, prefixes, sizes, [5, 64, 3, 90], [12, 3, 1, 9], 32, 8, 16, dtype))
