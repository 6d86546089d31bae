"""Shared-prefix decode, sampling and verification where calls meet: several threads on one stream,
calls of different size in turn, and inputs at the ends of their ranges.

Tolerances are those of the operators' own tests (tests/test_gpu_shared_prefix.py,
tests/test_gpu_sampling.py); where two runs of one call are compared they have to be equal."""
import functools
import math
import threading

import numpy as np
import pytest
import torch

from adallm_b200.attention import paged_decode, paged_prefill
from adallm_b200.sampler import sample, verify_drafts
from adallm_b200.shared_prefix import shared_prefix_decode
from oracle import speculative as osp
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _in_threads(*functions):
    """Runs each in a thread of its own, all at once; the first failure is raised."""
    failed = []

    def run(f):
        try:
            f()
        except BaseException as e:  # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=run, args=(f,)) for f in functions]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if failed:
        raise failed[0]


@pytest.mark.parametrize("entry", ["shared", "decode", "prefill"])
def test_a_threads_first_cuda_call(entry):
    """Everything is allocated, so that the library's own calls are the first that need a context."""
    c = osp.make_shared_prefix_case(1, [96], [3], [20, 64, 7], [1, 1, 1], 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    room = torch.empty(1 << 26, dtype=torch.uint8, device=dev())
    out = torch.empty_like(c["q"])
    cu_q = torch.arange(4, dtype=torch.int32, device=dev())
    cu_k = torch.tensor([0, 20, 84, 91], dtype=torch.int32, device=dev())
    call = {"shared": lambda: shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"],
                                                   c["prefix_lens"], c["cu_groups"], c["block_tables"],
                                                   c["context_lens"], c["scale"], out=out, workspace=room),
            "decode": lambda: paged_decode(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], c["context_lens"],
                                           c["scale"], out=out, workspace=room),
            "prefill": lambda: paged_prefill(c["q"], c["k_cache"], c["v_cache"], c["block_tables"], cu_q, cu_k, 1,
                                             c["scale"], out=out)}[entry]
    call()
    want = out.clone()
    out.zero_()
    torch.cuda.synchronize()
    _in_threads(call)
    torch.cuda.synchronize()
    assert torch.equal(out, want)


def _attention(seed, prefix, n, rows, reach=0):
    c = osp.make_shared_prefix_case(seed, [prefix], [n], [3 + (7 * i) % 90 for i in range(n)], [rows] * n, 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    if reach:  # a table of this many pages: enough rows then go to the tensor-core kernel
        c["prefix_tables"] = torch.nn.functional.pad(c["prefix_tables"], (0, reach), value=-1)
    return lambda: (shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"],
                                         c["cu_groups"], c["block_tables"], c["context_lens"], c["scale"],
                                         cu_seqlens_q=c["cu_seqlens_q"]),)


def _verification(seed, batch, drafts, vocab):
    g = torch.Generator().manual_seed(seed)
    n = batch * (drafts + 1)
    target = 3 * torch.randn((n, vocab), generator=g)
    ids = target.roll(1, 0).argmax(-1)  # likely tokens: some are accepted
    a = [t.to(dev()) for t in (target, ids, torch.arange(0, n + 1, drafts + 1, dtype=torch.int32), torch.full((batch,), 0.3),
                               torch.rand((batch, drafts), generator=g),
                               torch.empty((batch, vocab)).exponential_(1.0, generator=g))]
    return lambda: verify_drafts(*a)


def _calls():
    return [_attention(1, 300, 5, 1), _verification(2, 3, 4, 5003), _attention(3, 900, 24, 3, reach=1 << 14),
            _verification(4, 40, 2, 1009), _attention(5, 64, 60, 2), _verification(6, 1, 1, 90001)]


def test_threads_on_one_stream_get_their_own_results():
    calls = _calls()
    alone = [tuple(t.clone() for t in f()) for f in calls]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(calls)), []

    def caller(i):
        start.wait(timeout=60)
        for _ in range(150):
            got = calls[i]()
            if not all(torch.equal(a, b) for a, b in zip(got, alone[i])):
                wrong.append(i)

    _in_threads(*(functools.partial(caller, i) for i in range(len(calls))))
    torch.cuda.synchronize()
    assert not wrong, wrong


def test_calls_of_different_sizes_in_turn():
    """No host wait between them: each one's launches follow the one's before on the stream."""
    calls = _calls()
    alone = [tuple(t.clone() for t in f()) for f in calls]
    torch.cuda.synchronize()
    order = np.random.default_rng(0).integers(0, len(calls), 400).tolist()
    got = [(i, calls[i]()) for i in order]
    torch.cuda.synchronize()
    for i, out in got:
        assert all(torch.equal(a, b) for a, b in zip(out, alone[i])), i


@pytest.mark.parametrize("reach", [0, 1 << 14])
@pytest.mark.parametrize("rows", [[1, 2], [40, 33], [3, 0]])
def test_windows_wider_than_all_positions(rows, reach):
    """Prefixes and contexts with fewer keys than rows; from the reach of the tables on a window cuts nothing."""
    c = osp.make_shared_prefix_case(7, [20], [2], [2, 30], rows, 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    c["prefix_tables"] = torch.nn.functional.pad(c["prefix_tables"], (0, reach), value=-1)

    def run(window):
        return shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"],
                                    c["cu_groups"], c["block_tables"], c["context_lens"], c["scale"],
                                    cu_seqlens_q=c["cu_seqlens_q"], window=window)

    want = run(0)
    reached = (c["prefix_tables"].shape[1] + c["block_tables"].shape[1]) * 16
    for window in (50, reached - 1, reached, 1 << 30, 2 ** 31 - 40, 2 ** 31 - 1, 2 ** 31, 2 ** 32 + 3, 1 << 62):
        got = run(window)
        assert float((got - want).float().abs().max()) <= 2 ** -8 * float(want.float().abs().max()), window
        if window >= reached:
            assert torch.equal(got, want), window


@pytest.mark.parametrize("cu", [[0, 5, 3, 8], [-3, 4, 6, 8], [0, 2 ** 31 - 1, -2 ** 31, 8], [8, 6, 2, 0], [5, 5, 9, 12]])
@pytest.mark.parametrize("temperature", [0.0, 0.7])
def test_verify_lists_that_do_not_ascend(cu, temperature):
    """Such a list has no meaning, but the call stays inside its tensors: tokens of the vocabulary or -1,
    whatever the workspace held before."""
    g = torch.Generator().manual_seed(3)
    v = 1003
    a = [t.to(dev()) for t in (torch.randn((8, v), generator=g), torch.randint(0, v, (8,), generator=g),
                               torch.tensor(cu, dtype=torch.int32), torch.full((3,), temperature),
                               torch.rand((3, 2), generator=g), torch.empty((3, v)).exponential_(1.0, generator=g))]
    for fill in (0x00, 0x7F, 0xFF):
        room = torch.full((1 << 16,), fill, dtype=torch.uint8, device=dev())
        tokens, accepted, _ = verify_drafts(*a, workspace=room)
        assert bool(((tokens >= -1) & (tokens < v)).all())
        assert bool(((accepted >= 0) & (accepted <= 2)).all())


@pytest.mark.parametrize("reach", [0, 1 << 14])
def test_attention_lists_that_do_not_ascend(reach):
    """Rows and sequences claimed several times over, or before and past all there are: the call stays inside
    its tensors, and lists in order give what they gave."""
    n = 12
    c = osp.make_shared_prefix_case(9, [100, 60], [7, 5], [5 + i for i in range(n)], [4] * n, 32, 8, 16)
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    c["prefix_tables"] = torch.nn.functional.pad(c["prefix_tables"], (0, reach), value=-1)

    def run(**kw):
        a = {**c, **kw}
        return shared_prefix_decode(a["q"], a["k_cache"], a["v_cache"], a["prefix_tables"], a["prefix_lens"],
                                    a["cu_groups"], a["block_tables"], a["context_lens"], a["scale"],
                                    cu_seqlens_q=a["cu_seqlens_q"])

    want = run()
    i32 = dict(dtype=torch.int32, device=dev())
    low, high = -2 ** 31, 2 ** 31 - 1
    for cu_q in ([0, 48] * 6 + [0], [48] * 6 + [0] * 7, [low, high] * 6 + [low], list(range(24, -2, -2))):
        assert run(cu_seqlens_q=torch.tensor(cu_q, **i32)).shape == want.shape
    for cu_g in ([0, 12, 0], [12, 0, 12], [low, high, low], [5, 5, 3]):
        assert run(cu_groups=torch.tensor(cu_g, **i32)).shape == want.shape
    torch.cuda.synchronize()
    assert torch.equal(run(), want)


def _matches(out, ref, vmax):
    """NaN where the definition is NaN, and elsewhere the tolerance of tests/test_gpu_shared_prefix.py."""
    out = out.cpu()
    assert torch.equal(out.isnan(), ref.isnan())
    ulp = 2 ** -8 if out.dtype == torch.bfloat16 else 2 ** -11
    off = ((out.double() - ref).abs() - ulp * ref.abs() - 2 ** -10 * vmax).nan_to_num(nan=-1.0)
    assert float(off.max()) <= 0, float(off.max())


@pytest.mark.parametrize("reach", [0, 1 << 14])
@pytest.mark.parametrize("rows", [[1, 1, 1], [4, 3, 1], [40, 30, 9]])
@pytest.mark.parametrize("window", [0, 64])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_nan_keys_and_values_reach_the_rows_that_see_them_alone(rows, window, reach, dtype):
    """Single elements and whole keys: before the windows, at their edges, among the newest tokens, in pages
    that end inside a tile."""
    c = osp.make_shared_prefix_case(11, [301], [3], [50, 90, 33], rows, 32, 8, 16, dtype)
    vmax = float(c["v_cache"].float().nan_to_num(0.0).abs().max())
    d = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    d["prefix_tables"] = torch.nn.functional.pad(d["prefix_tables"], (0, reach), value=-1)

    def place(table, key):
        return int(table[key // 16]), key % 16

    spots = [("v_cache", place(c["prefix_tables"][0], k), h, at) for k, h, at in
             ((5, slice(None), slice(None)), (230, 2, 17), (250, 0, 127), (290, 7, 64), (300, 3, 5))]
    spots += [("v_cache", place(c["block_tables"][0], k), h, at) for k, h, at in
              ((49, 1, 0), (48, slice(None), slice(None)), (46, 5, 33), (20, 6, 100))]
    spots += [("v_cache", place(c["block_tables"][2], 32), 4, 77), ("k_cache", place(c["block_tables"][1], 89), 2, 9),
              ("k_cache", place(c["prefix_tables"][0], 7), slice(None), slice(None))]
    if window == 0:  # without a window the rows see all of the prefix: leave it some finite output
        spots = [s for s in spots if s[2] != slice(None)]
    for some in (spots[:1], spots[4:7], spots):
        for cache in ("k_cache", "v_cache"):
            d[cache].copy_(c[cache].to(dev()))
        host = {n: c[n].clone() for n in ("k_cache", "v_cache")}
        for name, (block, row), head, at in some:
            host[name].view(torch.uint8)[block, row, head, at] = osp.NAN_BYTE
        for cache in host:
            d[cache].copy_(host[cache].to(dev()))
        out = shared_prefix_decode(d["q"], d["k_cache"], d["v_cache"], d["prefix_tables"], d["prefix_lens"],
                                   d["cu_groups"], d["block_tables"], d["context_lens"], d["scale"],
                                   cu_seqlens_q=d["cu_seqlens_q"], window=window)
        ref = osp.shared_prefix_decode(c["q"], host["k_cache"], host["v_cache"], c["prefix_tables"], c["prefix_lens"],
                                       c["cu_groups"], c["block_tables"], c["context_lens"], c["scale"],
                                       cu_seqlens_q=c["cu_seqlens_q"], window=window)
        assert not bool(ref.isnan().all())
        _matches(out, ref, vmax)


@pytest.mark.parametrize("reach", [0, 1 << 14])
def test_nan_values_in_many_short_prefixes(reach):
    """Several pieces a CTA and a warp, of which some hold NaN values behind the windows of some rows."""
    groups, rng = 40, np.random.default_rng(5)
    prefixes = rng.integers(1, 260, groups).tolist()
    own = rng.integers(9, 60, groups).tolist()
    c = osp.make_shared_prefix_case(12, prefixes, [1] * groups, own, rng.integers(20, 50, groups).tolist(), 8, 4, 16)
    vmax = float(c["v_cache"].float().nan_to_num(0.0).abs().max())
    for g in range(0, groups, 3):
        key = int(rng.integers(0, prefixes[g]))
        c["v_cache"].view(torch.uint8)[int(c["prefix_tables"][g, key // 16]), key % 16, g % 4, rng.integers(0, 128, 5)] = 0xFF
    for g in range(1, groups, 4):
        key = int(rng.integers(0, own[g]))
        c["v_cache"].view(torch.uint8)[int(c["block_tables"][g, key // 16]), key % 16, g % 4, 64:] = 0x7F
    d = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    d["prefix_tables"] = torch.nn.functional.pad(d["prefix_tables"], (0, reach), value=-1)
    for window in (0, 30, 100):
        def run(a):
            f = shared_prefix_decode if a is d else osp.shared_prefix_decode
            return f(a["q"], a["k_cache"], a["v_cache"], a["prefix_tables"], a["prefix_lens"], a["cu_groups"],
                     a["block_tables"], a["context_lens"], a["scale"], cu_seqlens_q=a["cu_seqlens_q"], window=window)

        out, ref = run(d), run(c)
        assert bool(ref.isnan().any())
        _matches(out, ref, vmax)
        assert torch.equal(torch.nan_to_num(run(d), 7.0), torch.nan_to_num(out, 7.0))


@pytest.mark.parametrize("rows", [1, 3, 700])
def test_greedy_takes_the_largest_float_before_a_later_infinity(rows):
    """+inf is read as the largest float, so the two tie: in packets of one lane, of one warp and apart."""
    v, top = 70001, torch.finfo(torch.float32).max
    logits = torch.randn((rows, v), generator=torch.Generator().manual_seed(1)).to(dev())
    first = (torch.arange(rows, device=dev()) * 7 + 5) % 1000
    r = torch.arange(rows, device=dev())
    zero, noise = torch.zeros(rows, device=dev()), torch.ones((rows, v), device=dev())
    one = torch.arange(rows + 1, dtype=torch.int32, device=dev())
    for step in (1, 4, 128, 1024, 4096, 8192, 16384, 65536):
        x = logits.clone()
        x[r, first] = top
        x[r, first + step] = torch.inf
        assert torch.equal(sample(x, zero, noise)[0], first), step
        ids = torch.zeros(rows, dtype=torch.int64, device=dev())
        tokens, _, _ = verify_drafts(x, ids, one, zero, zero[:, None][:, :0], noise)
        assert torch.equal(tokens[:, 0], first), step


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("t", [0.25, 0.9, 1.0, 2.0])
def test_drafts_that_infinities_make_certain(dtype, t):
    """A drafter that forces a token by +inf: its normaliser stays finite at every temperature, the draft's
    probability is 1, and it is accepted as often as the target would draw it."""
    g = torch.Generator().manual_seed(2)
    n, v, at = 64, 1003, 7
    target = torch.randn((2 * n, v), generator=g).to(dtype)
    target[::2, at] = torch.linspace(-3, 9, n).to(dtype)  # from hardly ever to nearly always
    draft = torch.randn((n, v), generator=g).to(dtype)
    draft[:, at] = torch.inf
    temps, u = torch.full((n,), t), torch.rand((n, 1), generator=g)
    noise = torch.empty((n, v)).exponential_(1.0, generator=g)
    drawn, logprobs, lse = sample(draft.to(dev()), temps.to(dev()), noise.to(dev()))
    assert drawn.tolist() == [at] * n and not bool(logprobs.any()) and bool(torch.isfinite(lse).all())
    ids = torch.zeros(2 * n, dtype=torch.int64)
    ids[1::2] = at
    sure = 0
    for given in (lse, torch.full_like(lse, torch.inf) if t < 1 else lse):  # as a plain logsumexp has it
        tokens, accepted, lp = verify_drafts(target.to(dev()), ids.to(dev()),
                                             torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=dev()),
                                             temps.to(dev()), u.to(dev()), noise.to(dev()),
                                             draft_logits=draft[:, None].to(dev()), draft_lse=given[:, None])
        for i in range(n):
            want, count, want_lp, margin = osp.verify(target[2 * i:2 * i + 2].double().numpy(), [0, at], t, u[i].tolist(),
                                                      noise[i].numpy(), draft[i:i + 1].double().numpy(), [float(lse[i])], 1)
            if margin < 2 ** -17:
                continue
            sure += 1
            assert tokens[i].tolist() == want + [-1] * (2 - len(want)) and int(accepted[i]) == count, i
            assert all(abs(a - b) <= 2 ** -20 * 60 + 2 ** -19 for a, b in zip(lp[i].tolist(), want_lp))
        assert int(accepted.sum()) < n and (t > 1 or int(accepted.sum()) > 0)  # (at 2 no target is above 1 in 10)
    assert sure > n


@pytest.mark.parametrize("reach", [0, 1 << 18])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_huge_queries_take_the_key_with_the_largest_score(dtype, reach):
    """Queries near the top of their type: the scores of a head are so far apart that its output is the value of
    its best key.  A score is a sum of 128 products in 32 bits, off by 2^-20 of the sum of their sizes at most;
    heads whose best two scores are closer than twice that and 64 powers of two are left out."""
    c = osp.make_shared_prefix_case(26, [200], [3], [20, 33, 40], [20, 16, 9], 32, 8, 16, dtype)
    top = 1e30 if dtype == torch.bfloat16 else 6e4
    g = torch.Generator().manual_seed(4)
    size = 2.0 ** -torch.randint(0, 4, c["q"].shape, generator=g).float()
    c["q"] = (top * size * torch.sign(c["q"].float() + 1e-9)).to(dtype)
    c["scale"] = 128 ** -0.5 * (1.0 if dtype == torch.bfloat16 else 64.0)
    d = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    pad = reach // 16 - d["prefix_tables"].shape[1]
    d["prefix_tables"] = torch.nn.functional.pad(d["prefix_tables"], (0, max(pad, 0)), value=-1)
    out = shared_prefix_decode(d["q"], d["k_cache"], d["v_cache"], d["prefix_tables"], d["prefix_lens"], d["cu_groups"],
                               d["block_tables"], d["context_lens"], d["scale"], cu_seqlens_q=d["cu_seqlens_q"]).cpu()
    ulp = 2 ** -8 if dtype == torch.bfloat16 else 2 ** -11
    sure = 0
    for b in range(3):
        begin, end, own = int(c["cu_seqlens_q"][b]), int(c["cu_seqlens_q"][b + 1]), int(c["context_lens"][b])
        keys = [(c["prefix_tables"][0, j // 16], j % 16) for j in range(200)]
        keys += [(c["block_tables"][b, j // 16], j % 16) for j in range(own)]
        k, v = (torch.stack([c[n][int(p), r].double() for p, r in keys]) for n in ("k_cache", "v_cache"))
        for n in range(begin, end):
            see = 200 + own - (end - begin) + (n - begin) + 1
            q = c["q"][n].double().view(8, 4, 128)
            s = torch.einsum("hgd,lhd->hgl", q, k[:see]) * c["scale"] / np.log(2)
            err = 2.0 ** -20 * torch.einsum("hgd,lhd->hgl", q.abs(), k[:see].abs()).amax(-1) * c["scale"] / np.log(2)
            best = s.topk(2, dim=-1)
            clear = best.values[..., 0] - best.values[..., 1] > 2 * err + 64
            want = v[best.indices[..., 0], torch.arange(8)[:, None]]
            got = out[n].double().view(8, 4, 128)
            assert bool(((got - want).abs() <= ulp * want.abs())[clear].all()), n
            sure += int(clear.sum())
    assert sure > 32 * 45 // 2


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("t", [1e-4, 0.3, 1.0, 3.0])
def test_rows_masked_by_the_lowest_value_alone(dtype, t):
    """Every logit the type's lowest: all tokens alike, so the noise decides, log-probability -ln n; the
    normaliser is not the -inf of a row without a possible token, and a draft drawn from such a row never makes
    the verified tokens anything but the target's (here certain ones)."""
    n, v = 5, 300
    g = torch.Generator().manual_seed(6)
    low = torch.full((n, v), torch.finfo(dtype).min, dtype=dtype)
    low[3, 10:] = -torch.inf
    low[4] = -torch.inf
    temps, noise = torch.full((n,), t, device=dev()), torch.empty((n, v)).exponential_(1.0, generator=g)
    tokens, logprobs, lse = (x.cpu() for x in sample(low.to(dev()), temps, noise.to(dev())))
    want = [int(noise[r].argmin()) for r in range(3)] + [int(noise[3, :10].argmin()), -1]
    assert tokens.tolist() == want
    off = logprobs - torch.tensor([-math.log(v)] * 3 + [-math.log(10), 0.0])
    assert float(off.abs().max()) <= 2 ** -20 * math.log(v) + 2 ** -19
    assert bool(torch.isfinite(lse[:4]).all()) and float(lse[4]) == -math.inf
    target = torch.zeros((2 * n, v), dtype=dtype)
    target[torch.arange(2 * n), torch.arange(2 * n)] = 20000.0
    ids = torch.stack((torch.zeros(n, dtype=torch.long), tokens), 1).reshape(-1)
    got, accepted, _ = verify_drafts(target.to(dev()), ids.to(dev()),
                                     torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=dev()), temps,
                                     torch.rand((n, 1), generator=g).to(dev()), noise.to(dev()),
                                     draft_logits=low[:, None].to(dev()), draft_lse=lse[:, None].to(dev()))
    for r in range(n):
        assert got[r].tolist() == ([2 * r, 2 * r + 1] if int(accepted[r]) else [2 * r, -1])
