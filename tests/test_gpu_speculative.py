"""The speculative sampling example end to end: shared-prefix decode, sampling and verification
together, against a plain 32-bit forward over the same e4m3 keys and values.

Tolerance: the example's logits are bf16 products of bf16 activations, attention outputs rounded to
bf16 (2^-8 relative) and a bf16 sum: roundings of up to 2^-8 of the largest logit at three places.
A token counts as the maximum when its 32-bit logit is within 3 * 2^-8 of the largest size of it."""
import importlib.util
import os

import pytest
import torch

from tests.conftest import ROOT
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("speculative_sampling",
                                                  os.path.join(ROOT, "examples", "speculative_sampling.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain_logits(target, ids):
    """Logits of every position of one token list: full causal attention in fp32, e4m3 keys and values."""
    x, q, k, v = target.qkv(ids)
    k, v = (t.to(torch.float8_e4m3fn).float().repeat_interleave(4, 1) for t in (k, v))
    s = torch.einsum("qhd,khd->hqk", q.float(), k) * 128 ** -0.5
    s = s.masked_fill(torch.ones(len(ids), len(ids), device=ids.device).triu(1).bool(), float("-inf"))
    out = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)
    return (x.float() + out.reshape(len(ids), -1) @ target.wo.float().t()) @ target.head.float().t()


def test_greedy_speculation_gives_the_targets_own_tokens():
    m = _example()
    steps, drafts = 6, 3
    session, prompt = m.make(sequences=3, drafts=drafts, steps=steps, temperature=0.0, device=dev())
    session.bigram[::4] = session.bigram[::4].roll(1, 1)  # a quarter of the drafts are wrong
    results = [session.step() for _ in range(steps)]
    counts = torch.stack([n for _, n, _ in results])
    assert 0 < int(counts.sum()) < 3 * drafts * steps  # some drafts accepted, some replaced
    for b in range(3):
        last = prompt[-1]
        for t, n, _ in results:
            match = 0  # the drafts are the bigram's own greedy chain; its agreement with the tokens is the count
            while match < drafts and int(session.bigram[last].argmax()) == int(t[b, match]):
                last, match = t[b, match], match + 1
            assert int(n[b]) == match
            last = t[b, match]
        new = torch.cat([t[b, :int(n[b]) + 1] for t, n, _ in results])
        assert int(session.stored[b]) == len(new) and bool((new >= 0).all())
        ids = torch.cat((prompt, new))
        z = _plain_logits(session.target, ids)[len(prompt) - 1:-1]
        assert float((z.max(-1).values - z.gather(1, new[:, None])[:, 0]).max()) <= 3 * 2 ** -8 * float(z.abs().max())


def test_sampled_speculation_scores_its_tokens():
    """Log-probabilities of the emitted tokens agree with the plain forward's at the same temperature."""
    m = _example()
    session, prompt = m.make(sequences=4, drafts=4, steps=5, temperature=0.7, device=dev())
    results = [session.step() for _ in range(5)]
    off, size = [], 0.0
    assert 0 < int(sum(n.sum() for _, n, _ in results)) < 4 * 4 * 5  # some drafts accepted, some replaced
    for b in range(4):
        new = torch.cat([t[b, :int(n[b]) + 1] for t, n, _ in results])
        lp = torch.cat([p[b, :int(n[b]) + 1] for _, n, p in results])
        ids = torch.cat((prompt, new))
        z = _plain_logits(session.target, ids)[len(prompt) - 1:-1] / 0.7
        size = max(size, float(z.abs().max()))
        z = torch.log_softmax(z, -1)
        off.append((lp - z.gather(1, new[:, None])[:, 0]).abs().max())
    assert float(torch.stack(off).max()) <= 2 * 3 * 2 ** -8 * size  # the token's logit and the normaliser


def test_a_step_runs_from_a_cuda_graph():
    m = _example()
    session, _ = m.make(sequences=4, drafts=2, steps=40, device=dev())
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            session.step()
        side.synchronize()
        last = session.last.clone()
        graph = torch.cuda.CUDAGraph()
        graph.register_generator_state(session.generator)
        with torch.cuda.graph(graph, stream=side):
            session.last = last
            tokens, accepted, _ = session.step()
            last.copy_(session.last)
    seen, stored = [], session.stored.clone()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        seen.append(tokens.clone())
        stored += accepted + 1
    assert torch.equal(session.stored, stored)
    assert not all(torch.equal(seen[0], s) for s in seen[1:])
    assert all(bool((t[:, 0] >= 0).all()) for t in seen)
