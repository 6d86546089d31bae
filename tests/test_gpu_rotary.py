"""Rotary positions in both layouts against 64 bits.

Tolerance: the table holds cos and sin in fp32 (error e <= 2^-24 A, A the amplitude, given the exact angle), two
products and a sum in fp32 (2^-24 each of |x1 cos| + |x2 sin|), one rounding to the type:
|error| <= half * |y| + 4 * 2^-24 * A * (|x1| + |x2|); the half step counts also for the value it rounds."""
import math

import pytest
import torch

from adallm_b200.rotary_embedding import RotaryEmbedding, apply_rope, apply_rotary, build_cos_sin_cache
from oracle import kv4
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu
BASE = 1e6


def inv_freq(r):
    return BASE ** (-torch.arange(r // 2, dtype=torch.float64) / (r // 2))


def table_of(inv, reach, amplitude=1.0):
    a = torch.arange(reach, dtype=torch.float64)[:, None] * inv
    return (torch.cat((a.cos(), a.sin()), -1) * amplitude).float().to(dev())


def check(x, y, positions, inv, interleaved, amplitude=1.0):
    want = kv4.rotate(x, positions, inv.to(x.device), interleaved, amplitude)
    half = torch.finfo(x.dtype).eps / 2
    r = 2 * inv.shape[0]
    part = x[..., :r].double().abs()
    both = part[..., 0::2] + part[..., 1::2] if interleaved else sum(part.chunk(2, -1))
    both = both.repeat_interleave(2, -1) if interleaved else torch.cat((both, both), -1)
    tol = half * (1 + half) * want.abs()
    tol[..., :r] += 4 * 2.0 ** -24 * amplitude * both
    tol[..., r:] = 0
    tiny = torch.finfo(x.dtype).smallest_normal * torch.finfo(x.dtype).eps  # half a step of a subnormal, doubled
    assert ((y.double() - want).abs() <= tol + tiny).all()


CASES = [  # tokens, q heads, kv heads, head size, rotary, interleaved, reach, dtype
    (1, 32, 8, 128, 128, False, 131072, torch.bfloat16), (1, 1, 1, 16, 16, True, 10, torch.float16),
    (5, 8, 8, 128, 64, True, 4096, torch.bfloat16), (16, 32, 4, 128, 32, False, 262144, torch.float16),
    (700, 3, 1, 80, 48, False, 1024, torch.bfloat16), (33, 7, 5, 96, 96, True, 5000, torch.float16),
    (1100, 32, 8, 128, 128, False, 8192, torch.bfloat16), (9, 16, 2, 256, 128, True, 300, torch.bfloat16),
    (3, 5, 0, 1024, 1024, False, 64, torch.float16), (130, 64, 8, 64, 16, False, 2048, torch.bfloat16)]


@pytest.mark.parametrize("t,hq,hk,d,r,inter,reach,dtype", CASES)
def test_matches_the_formula(t, hq, hk, d, r, inter, reach, dtype):
    g = torch.Generator().manual_seed(t + d + r)
    pos = torch.randint(0, reach, (t,), generator=g)
    pos[-1] = reach - 1
    q = (torch.randn((t, hq, d), generator=g) * 3).to(dtype).to(dev())
    k = torch.randn((t, hk, d), generator=g).to(dtype).to(dev())
    inv = inv_freq(r)
    qo, ko = apply_rotary(pos.to(dev()), q, k, table_of(inv, reach), inter)
    assert qo.shape == q.shape and ko.shape == k.shape and qo.dtype == dtype
    check(q, qo, pos.to(dev()), inv, inter)
    if hk:
        check(k, ko, pos.to(dev()), inv, inter)


@pytest.mark.parametrize("inter", [False, True])
def test_fused_rows_strides_and_given_outputs(inter):
    """q and k as slices of one projection, heads apart, int32 positions, outputs given."""
    g = torch.Generator().manual_seed(3)
    t, hq, hk, d = 21, 6, 2, 128
    qkv = torch.randn((t, hq + 2 * hk, d + 8), generator=g).to(torch.bfloat16).to(dev())
    q, k = qkv[:, :hq, :d], qkv[:, hq:hq + hk, :d]
    pos = torch.randint(0, 500, (t,), generator=g, dtype=torch.int32).to(dev())
    inv = inv_freq(64)
    qo, ko = torch.empty((t, hq, d), dtype=q.dtype, device=dev()), torch.empty((t, hk, d), dtype=q.dtype, device=dev())
    a, b = apply_rotary(pos, q, k, table_of(inv, 500), inter, q_out=qo, k_out=ko)
    assert a is qo and b is ko
    check(q, qo, pos, inv, inter)
    check(k, ko, pos, inv, inter)


def test_half_layout_equals_the_drop_in_kernel_and_positions_are_clamped():
    g = torch.Generator().manual_seed(4)
    q = torch.randn((37, 32, 128), generator=g).to(torch.bfloat16).to(dev())
    k = torch.randn((37, 8, 128), generator=g).to(torch.bfloat16).to(dev())
    pos = torch.randint(0, 1000, (37,), generator=g).to(dev())
    pos[0], pos[1] = -5, 10 ** 12
    table = build_cos_sin_cache(128, 1000, BASE).to(dev())
    for a, b in zip(apply_rope(pos, q, k, table), apply_rotary(pos, q, k, table)):
        assert torch.equal(a, b)


def test_infinities_and_nan_stay_in_their_pair():
    q = torch.ones((1, 2, 128), dtype=torch.bfloat16, device=dev())
    q[0, 0, 3], q[0, 1, 100] = math.inf, math.nan
    k = torch.ones((1, 1, 128), dtype=torch.bfloat16, device=dev())
    pos = torch.tensor([7], device=dev())
    qo, ko = apply_rotary(pos, q, k, table_of(inv_freq(64), 16), True)
    bad = ~qo.isfinite()
    assert bad[0, 0].nonzero().flatten().tolist() == [2, 3] and bad[0, 1].nonzero().flatten().tolist() == [100]
    assert ko.isfinite().all()


@pytest.mark.parametrize("scaling", [None, {"rope_type": "linear", "factor": 8.0},
                                     {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048}])
@pytest.mark.parametrize("r,inter", [(128, False), (64, True)])
def test_module_with_scaled_tables(scaling, r, inter):
    g = torch.Generator().manual_seed(5)
    reach = 8192
    m = RotaryEmbedding(128, r, reach, BASE, scaling, interleaved=inter).to(dev())
    pos = torch.randint(0, reach, (19,), generator=g).to(dev())
    q = torch.randn((19, 4 * 128), generator=g).to(torch.float16).to(dev())
    k = torch.randn((19, 128), generator=g).to(torch.float16).to(dev())
    qo, ko = m(pos, q, k)
    assert qo.shape == q.shape and ko.shape == k.shape
    inv, amp = inv_freq(r), 1.0
    if scaling and scaling["rope_type"] == "linear":
        inv = inv / 8
    elif scaling:
        amp = 0.1 * math.log(4.0) + 1
        turns = 2048 * inv_freq(r) / (2 * math.pi)
        edge = [r / 2 * math.log(2048 / (n * 2 * math.pi)) / math.log(BASE) for n in (32.0, 1.0)]
        low, high = math.floor(edge[0]), math.ceil(edge[1])
        keep = 1 - ((torch.arange(r // 2, dtype=torch.float64) - low) / (high - low)).clamp(0, 1)
        assert (keep[turns > 33] > 0.9).all() and (keep[turns < 0.9] < 0.1).all()
        inv = inv * keep + inv / 4 * (1 - keep)
    if scaling and scaling["rope_type"] == "yarn":
        check(q.view(19, 4, 128), qo.view(19, 4, 128), pos, inv, inter, amp)
        check(k.view(19, 1, 128), ko.view(19, 1, 128), pos, inv, inter, amp)
    else:
        # these tables keep the reference's 32-bit angles: position * frequency is off by 2^-22 of itself at most
        want = kv4.rotate(q.view(19, 4, 128), pos, inv.to(dev()), inter)
        assert ((qo.view(19, 4, 128).double() - want).abs() <= 8 * (reach * 2.0 ** -22) + 2.0 ** -11 * want.abs()).all()


def test_graph_and_streams():
    g = torch.Generator().manual_seed(6)
    q = torch.randn((64, 32, 128), generator=g).to(torch.bfloat16).to(dev())
    k = torch.randn((64, 8, 128), generator=g).to(torch.bfloat16).to(dev())
    pos = torch.randint(0, 1000, (64,), generator=g).to(dev())
    table = table_of(inv_freq(128), 1000)
    want = apply_rotary(pos, q, k, table)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = apply_rotary(pos, q, k, table)
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = apply_rotary(pos, q, k, table)
    for o in out:
        o.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_empty_and_refusals():
    d = dev()
    q = torch.zeros((4, 2, 128), dtype=torch.bfloat16, device=d)
    k, pos, table = q[:, :1], torch.zeros(4, dtype=torch.int64, device=d), table_of(inv_freq(64), 8)
    assert apply_rotary(pos[:0], q[:0], k[:0], table)[0].shape == (0, 2, 128)
    for args in ((pos, q, k.half(), table), (pos, q.float(), k.float(), table), (pos[:3], q, k, table),
                 (pos, q, k, table.double()), (pos, q, k, table[:, ::2]), (pos, q, k[:3], table),
                 (pos, q[..., :64], k, table), (pos, q.flatten(1), k.flatten(1), table),
                 (pos, q, k, table[:, :40].contiguous()), (pos, q[..., :16].contiguous(), k[..., :16].contiguous(), table),
                 (pos, q[..., :72].contiguous(), k[..., :72].contiguous(), table)):
        with pytest.raises(ValueError):
            apply_rotary(*args)
    for bad in (table[0], table[:, None].expand(8, 2, 64).contiguous()):  # [width], [positions, 2, width]
        with pytest.raises(ValueError):
            apply_rotary(pos, q, k, bad)
    with pytest.raises(ValueError):  # in place: a pair's halves belong to two threads
        apply_rotary(pos, q, k, table, q_out=q)
    with pytest.raises(ValueError):
        apply_rotary(pos, q, k, table, q_out=torch.empty((4, 2, 64), dtype=q.dtype, device=d))
    with pytest.raises(RuntimeError):
        apply_rotary(pos, q.cpu(), k, table)
