"""Sampling and draft verification (through the C ABI) vs their definitions in 64 bits.

Tolerances.  z = x / T is rounded to 24 bits, and exp(z - max) with |z - max| up to about 32 where
it matters carries a relative error of at most 2^-19 or so; scores that decide a draw, and the two
sides of an acceptance, can therefore differ by 2^-17 relative before the choice itself may differ:
a row whose margin in 64 bits is below 2^-17 may go either way, every other one has to agree.
lse and logprobs: a few roundings of values up to |lse| + |z|, so 2^-20 of that sum, plus the sum's
own error 2^-19."""
import math

import numpy as np
import pytest
import torch

from adallm_b200.sampler import Sampler, sample, verify_drafts
from oracle import speculative as osp
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu
MARGIN = 2 ** -17


def _tol(lse, z):
    return 2 ** -20 * (abs(lse) + abs(z)) + 2 ** -19


def _exp(shape, g):
    return torch.empty(shape).exponential_(1.0, generator=g)


def _check_sample(logits, temps, noise, got):
    tokens, logprobs, lse = (t.cpu() for t in got)
    for r in range(logits.shape[0]):
        k, lp, l, margin = osp.sample(logits[r].double().numpy(), float(temps[r]), noise[r].numpy())
        if l == -math.inf:
            assert int(tokens[r]) == -1 and float(lse[r]) == -math.inf and float(logprobs[r]) == 0.0
            continue
        assert abs(float(lse[r]) - l) <= _tol(l, 0)
        if margin < MARGIN:
            continue
        assert int(tokens[r]) == k, (r, int(tokens[r]), k, margin)
        assert abs(float(logprobs[r]) - lp) <= _tol(l, lp + l)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 2), (5, 7), (2, 31), (4, 255), (1, 1000), (3, 4099), (7, 32003),
                                        (2, 151936), (200, 513), (1, 70001)])
def test_sample(rows, vocab, dtype):
    g = torch.Generator().manual_seed(rows * 7 + vocab)
    logits = (3 * torch.randn((rows, vocab), generator=g)).to(dtype)
    temps = 0.3 + torch.rand(rows, generator=g)
    temps[rows // 2:][::3] = 0.0
    noise = _exp((rows, vocab), g)
    got = sample(logits.to(dev()), temps.to(dev()), noise.to(dev()))
    _check_sample(logits, temps, noise, got)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample_masks_infinities_and_nan(dtype):
    g = torch.Generator().manual_seed(5)
    v = 5003
    logits = (3 * torch.randn((12, v), generator=g)).to(dtype)
    low = torch.finfo(dtype).min
    logits[0] = -math.inf                      # nothing possible
    logits[1] = -math.inf
    logits[1, 4711] = -3.0                     # one token possible
    logits[2] = low                            # masked by the lowest value, all alike
    logits[3, 1:] = low
    logits[4, 100] = math.inf                  # one certain
    logits[5, 17:40] = math.inf                # several share it
    logits[6, ::2] = math.nan                  # NaN in masked places
    logits[7] = math.nan
    logits[8] = 0.0                            # flat
    logits[9, 5:] = -math.inf
    logits[10, 2500:] = math.nan
    temps = torch.ones(12)
    temps[8] = 1e-10
    temps[10] = 0.0
    temps[11] = 1e-4                           # z in the ten thousands
    noise = _exp((12, v), g)
    noise[1, 4711] = 1e5
    noise[3, 7] = 0.0                          # read as 1e-10
    got = sample(logits.to(dev()), temps.to(dev()), noise.to(dev()))
    _check_sample(logits, temps, noise, got)
    assert int(got[0][8]) == 0 and int(got[0][4]) == 100


def test_sample_greedy_takes_the_first_maximum():
    g = torch.Generator().manual_seed(6)
    logits = torch.randint(-3, 4, (33, 20011), generator=g).to(torch.bfloat16)
    zero = torch.zeros(33, device=dev())
    tokens, _, _ = sample(logits.to(dev()), zero, _exp((33, 20011), g).to(dev()))
    assert torch.equal(tokens.cpu(), logits.float().argmax(-1))


def test_sample_equal_scores_take_the_lowest_index():
    logits = torch.zeros((4, 3001), dtype=torch.float32)
    noise = torch.full((4, 3001), 2.0)
    noise[1, 1500:] = 1.0
    noise[2, 3000] = 1.0
    noise[3, [7, 2999]] = 0.5
    tokens, _, _ = sample(logits.to(dev()), torch.ones(4, device=dev()), noise.to(dev()))
    assert tokens.tolist() == [0, 1500, 3000, 7]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_sample_strided_rows_and_odd_starts(dtype):
    g = torch.Generator().manual_seed(8)
    for pad, shift in ((1, 1), (3, 2), (8, 5), (0, 0)):
        base = torch.randn((9, 4001 + pad + shift), generator=g).to(dtype).to(dev())
        noise = _exp((9, 4001 + 5), g).to(dev())
        x, e = base[:, shift:shift + 4001], noise[:, 3:4004]
        temps = torch.full((9,), 0.8, device=dev())
        _check_sample(x.cpu(), temps.cpu(), e.cpu(), sample(x, temps, e))
    wide = torch.randn((50, 6), generator=g).to(dtype).to(dev())
    _check_sample(wide.t().cpu(), torch.ones(6), noise[:6, :50].cpu(),
                  sample(wide.t(), torch.ones(6, device=dev()), noise[:6, :50]))


def test_sample_draws_from_the_distribution():
    """20,000 draws of one row of 12 tokens: counts within 5 standard deviations."""
    g = torch.Generator().manual_seed(9)
    n = 20000
    row = torch.randn(12, generator=g)
    tokens, _, _ = sample(row.expand(n, -1).contiguous().to(dev()), torch.full((n,), 0.7, device=dev()),
                          _exp((n, 12), g).to(dev()))
    p = torch.softmax(row.double() / 0.7, 0)
    count = torch.bincount(tokens.cpu(), minlength=12).double()
    assert bool(((count - n * p).abs() < 5 * (n * p * (1 - p)).sqrt()).all())


def test_sampler_module():
    torch.manual_seed(0)
    logits = torch.full((64, 1000), -20.0, device=dev(), dtype=torch.bfloat16)
    logits[torch.arange(64), torch.arange(64) * 7] = 20.0
    assert torch.equal(Sampler()(logits, torch.full((64,), 0.6, device=dev())).cpu(), torch.arange(64) * 7)


# ---- verification ----------------------------------------------------------------------------
def _make(seed, counts, vocab, dtype, drafter=True, greedy=(), keep=1.0, near=0.5, most=None):
    g = torch.Generator().manual_seed(seed)
    b, most = len(counts), max(counts + [0]) if most is None else most
    rows = [c + 1 if c >= 0 else 0 for c in counts]  # -1: an empty sequence
    cu = [0] + np.cumsum(rows).tolist()
    target = 3 * torch.randn((cu[-1], vocab), generator=g)
    if keep < 1:
        target = torch.where(torch.rand(target.shape, generator=g) < keep, target, torch.tensor(-math.inf))
        target[:, 0] = 1.0
    temps = 0.4 + torch.rand(b, generator=g)
    temps[list(greedy)] = 0.0
    draft = torch.zeros((b, most, vocab))
    lse = torch.zeros((b, most))
    ids = torch.randint(0, vocab, (cu[-1],), generator=g)
    for i, c in enumerate(counts):
        for j in range(min(c, most)):
            x = (target[cu[i] + j] + near * torch.randn(vocab, generator=g)).to(dtype)
            draft[i, j] = x.float()
            z = x.double() / (temps[i].double() if temps[i] > 0 else 1.0)
            lse[i, j] = torch.logsumexp(z, 0).float()
            score = (z - z.max()).exp() / (_exp((vocab,), g).double() if temps[i] > 0 else 1.0)
            ids[cu[i] + j + 1] = int(score.argmax())
    return dict(target=target.to(dtype), ids=ids, cu=torch.tensor(cu, dtype=torch.int32), temps=temps,
                u=torch.rand((b, most), generator=g), noise=_exp((b, vocab), g),
                draft=draft.to(dtype) if drafter else None, lse=lse if drafter else None)


def _verify(c):
    c = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    return verify_drafts(c["target"], c["ids"], c["cu"], c["temps"], c["u"], c["noise"], draft_logits=c["draft"],
                         draft_lse=c["lse"])


def _check_verify(c, got):
    tokens, accepted, logprobs = (t.cpu() for t in got)
    b, most = c["u"].shape
    sure = 0
    for i in range(b):
        lo, hi = int(c["cu"][i]), int(c["cu"][i + 1])
        if hi <= lo:
            assert int(accepted[i]) == 0 and bool((tokens[i] == -1).all()) and not bool(logprobs[i].any())
            continue
        want, count, lp, margin = osp.verify(
            c["target"][lo:hi].double().numpy(), c["ids"][lo:hi].tolist(), float(c["temps"][i]), c["u"][i].tolist(),
            c["noise"][i].numpy(), None if c["draft"] is None else c["draft"][i].double().numpy(),
            None if c["lse"] is None else c["lse"][i].tolist(), most)
        if margin < MARGIN:
            continue
        sure += 1
        pad = most + 1 - len(want)
        assert tokens[i].tolist() == want + [-1] * pad, (i, margin)
        assert int(accepted[i]) == count
        for a, e in zip(logprobs[i].tolist(), lp + [0.0] * pad):
            assert abs(a - e) <= _tol(30, 30)
    return sure


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("drafter", [True, False])
@pytest.mark.parametrize("counts,vocab", [([4], 4099), ([0, 1, 2, 3, 8, -1, 5], 1000), ([1], 2), ([3, 3], 1),
                                          ([2] * 40, 777), ([4, 2], 151936), ([0], 33)])
def test_verify(counts, vocab, drafter, dtype):
    c = _make(sum(counts) + vocab, counts, vocab, dtype, drafter, greedy=(len(counts) - 1,) if len(counts) > 2 else ())
    sure = _check_verify(c, _verify(c))
    assert sure >= len(counts) // 2


@pytest.mark.parametrize("drafter", [True, False])
def test_verify_masked(drafter):
    c = _make(3, [3, 4, 0, 2, 5], 3001, torch.float32, drafter, greedy=(1,), keep=0.05)
    assert _check_verify(c, _verify(c)) >= 3


def test_verify_empty_and_odd_rows():
    """A target row without a possible token, NaN and infinities in masked places, a draft outside
    the vocabulary, equal distributions (nothing is left to draw from after a refusal)."""
    c = _make(4, [2, 2, 2, 2, 1, 1], 700, torch.float32, True, near=0.0)
    cu = c["cu"].tolist()
    c["target"][cu[0]] = -math.inf                 # refused at once, no token
    c["target"][cu[1] + 1, ::2] = math.nan
    c["draft"][1, 1, 1::2] = math.nan
    c["ids"][cu[2] + 1] = 700                      # outside: refused
    c["ids"][cu[3] + 2] = -1
    c["target"][cu[4], 5] = math.inf
    c["u"][5, 0] = 2.0                             # refused although p = q: drawn from p
    c["draft"][5, 0] = c["target"][cu[5]]
    c["lse"][5, 0] = torch.logsumexp(c["target"][cu[5]].double() / c["temps"][5].double(), 0).float() - 1e-3
    got = _verify(c)
    _check_verify(c, got)
    assert got[0][0].tolist() == [-1, -1, -1]


def test_verify_accepts_all_with_the_same_distribution():
    c = _make(5, [6] * 8, 2000, torch.bfloat16, True, near=0.0)
    _, accepted, _ = _verify(c)
    assert accepted.tolist() == [6] * 8


def test_verify_greedy_ties_take_the_first_maximum():
    c = _make(6, [3] * 4, 900, torch.bfloat16, True, greedy=(0, 1, 2, 3))
    c["target"] = torch.randint(-2, 3, c["target"].shape).to(torch.bfloat16)
    first = c["target"].float().argmax(-1)
    c["ids"][1:4] = first[0:3]                     # all right
    c["ids"][5:8] = first[4:7]
    c["ids"][6] = int((c["target"][5].float() == 2).nonzero()[1])  # an equal maximum, but not the first
    assert _check_verify(c, _verify(c)) == 4


def test_verify_more_drafts_than_asked_for():
    """Rows past max_drafts drafts are not looked at."""
    c = _make(7, [5, 2], 500, torch.bfloat16, True, near=0.0, most=3)
    _check_verify(c, _verify(c))
    c = _make(8, [2, 0], 500, torch.bfloat16, False, most=0)
    c["u"] = torch.zeros((2, 0))
    _check_verify(c, _verify(c))


def test_verify_strided_inputs():
    """Step-major draft logits (as a drafting loop stacks them), padded rows, odd starts."""
    c = _make(9, [3, 1, 2, 0], 1003, torch.bfloat16)
    want = _verify(c)
    g = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}
    steps = torch.empty((3, 4, 1009), dtype=torch.bfloat16, device=dev())
    steps[:, :, 3:1006] = g["draft"].transpose(0, 1)
    lse = g["lse"].t().contiguous().t()
    target = torch.zeros((g["target"].shape[0], 1010), dtype=torch.bfloat16, device=dev())
    target[:, 1:1004] = g["target"]
    noise = torch.zeros((4, 1007), device=dev())
    noise[:, 2:1005] = g["noise"]
    got = verify_drafts(target[:, 1:1004], g["ids"], g["cu"], g["temps"], g["u"], noise[:, 2:1005],
                        draft_logits=steps[:, :, 3:1006].transpose(0, 1), draft_lse=lse)
    assert all(torch.equal(x, y) for x, y in zip(got[:2], want[:2]))
    assert torch.allclose(got[2], want[2], rtol=0, atol=_tol(30, 30))


def test_verify_keeps_the_target_distribution():
    """First tokens of 40,000 sequences with one draft: distributed as the target, whatever the draft."""
    g = torch.Generator().manual_seed(10)
    n, v = 40000, 8
    target, draft = torch.randn((2, v), generator=g), torch.randn(v, generator=g)
    q = torch.softmax(draft, 0)
    x = torch.multinomial(q, n, replacement=True, generator=g)
    ids = torch.stack((torch.zeros(n, dtype=torch.long), x), 1).reshape(-1)
    tokens, _, _ = verify_drafts(
        target.repeat(n, 1).to(dev()), ids.to(dev()), torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device=dev()),
        torch.ones(n, device=dev()), torch.rand((n, 1), generator=g).to(dev()), _exp((n, v), g).to(dev()),
        draft_logits=draft.repeat(n, 1, 1).view(n, 1, v).to(dev()),
        draft_lse=torch.logsumexp(draft, 0).repeat(n, 1).to(dev()))
    p = torch.softmax(target[0].double(), 0)
    count = torch.bincount(tokens[:, 0].cpu(), minlength=v).double()
    assert bool(((count - n * p).abs() < 5 * (n * p * (1 - p)).sqrt()).all())


def test_same_result_twice_on_another_stream_and_in_a_graph():
    c = _make(11, [4, 0, 2, 3], 40009, torch.bfloat16, greedy=(3,))
    g = {k: v.to(dev()) if isinstance(v, torch.Tensor) else v for k, v in c.items()}

    def both():
        return sample(g["target"], g["target"].new_full((g["target"].shape[0],), 0.7, dtype=torch.float32),
                      noise) + _verify(g)

    noise = _exp(tuple(c["target"].shape), torch.Generator().manual_seed(1)).to(dev())
    first = both()
    assert all(torch.equal(a, b) for a, b in zip(both(), first))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = both()
        side.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            held = both()
    assert all(torch.equal(a, b) for a, b in zip(other, first))
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(held, first))


def test_refusals():
    x = torch.zeros((3, 50), device=dev())
    t, e = torch.ones(3, device=dev()), torch.ones((3, 50), device=dev())
    for a in ((x.double(), t, e), (x, t, e.half()), (x, t, e[:, :49]), (x, t[:2], e), (x, t.double(), e)):
        with pytest.raises(ValueError):
            sample(*a)
    with pytest.raises(RuntimeError, match="CUDA"):
        sample(x, t.cpu(), e)
    good = dict(target_logits=x, input_ids=torch.zeros(3, dtype=torch.int64, device=dev()),
                cu_seqlens_q=torch.tensor([0, 3], dtype=torch.int32, device=dev()), temperatures=t[:1],
                uniforms=torch.zeros((1, 2), device=dev()), noise=e[:1], draft_logits=x[None, :2],
                draft_lse=torch.zeros((1, 2), device=dev()))
    wrong = [dict(target_logits=x.double()), dict(input_ids=good["input_ids"].int()), dict(input_ids=good["input_ids"][:2]),
             dict(cu_seqlens_q=good["cu_seqlens_q"][:1]), dict(cu_seqlens_q=good["cu_seqlens_q"].long()),
             dict(temperatures=t), dict(uniforms=good["uniforms"].half()), dict(noise=e), dict(draft_lse=None),
             dict(draft_logits=None), dict(draft_logits=x[None]), dict(draft_logits=x[None, :2].half()),
             dict(draft_lse=torch.zeros((1, 3), device=dev())),
             dict(workspace=torch.empty(16, dtype=torch.uint8, device=dev()))]
    for kw in wrong:
        with pytest.raises(ValueError):
            verify_drafts(**{**good, **kw})
    for name in good:
        with pytest.raises(RuntimeError, match="CUDA"):
            verify_drafts(**{**good, name: good[name].cpu()})
    verify_drafts(**good)
