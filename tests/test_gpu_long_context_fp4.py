"""Step metadata, rotation, the 4-bit cache's store and its prefill and decode attention together: the example, and
the Attention module over a 4-bit cache, against a plain forward over the same packed keys and values.

Tolerance of the example: its logits are bf16 products of bf16 activations, attention outputs rounded to bf16
(2^-8 relative) and a bf16 sum: roundings of up to 2^-8 of the largest logit at three places.  A token counts
as the maximum when its 32-bit logit is within 3 * 2^-8 of the largest size of it."""
import importlib.util
import os

import pytest
import torch

from adallm_b200 import kvcache_fp4 as kv
from adallm_b200.attention import Attention
from adallm_b200.context import reset_context, set_context
from adallm_b200.rotary_embedding import apply_rotary
from adallm_b200.step_metadata import step_metadata
from oracle import kv4
from tests.conftest import ROOT
from tests.gpu_util import dev

pytestmark = pytest.mark.gpu


def _example():
    spec = importlib.util.spec_from_file_location("long_context_fp4",
                                                  os.path.join(ROOT, "examples", "long_context_fp4.py"))
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def _plain_logits(m, server, ids):
    x, q, k, v = server.layer.qkv(ids)
    pos = torch.arange(len(ids), device=ids.device)
    q, k = apply_rotary(pos, q.contiguous(), k.contiguous(), server.table, True)
    k, v = (kv4.stored(t).float().repeat_interleave(m.HEADS // m.KV_HEADS, 1) for t in (k, v))
    s = torch.einsum("qhd,khd->hqk", q.float(), k) * m.HEAD_DIM ** -0.5
    s = s.masked_fill(torch.ones(len(ids), len(ids), device=ids.device).triu(1).bool(), float("-inf"))
    out = torch.einsum("hqk,khd->qhd", torch.softmax(s, -1), v)
    layer = server.layer
    return (x.float() + out.reshape(len(ids), -1) @ layer.wo.float().t()) @ layer.head.float().t()


@pytest.mark.parametrize("chunk", [7, 64, 500])
def test_example_gives_the_layers_own_tokens(chunk):
    m = _example()
    lens, steps = [150, 1, 64, 33], 20
    server, prompts = m.make(lens, max(lens) + steps, dev(), seed=chunk)
    tokens = server.decode(server.prompt(prompts, chunk), steps)
    torch.cuda.synchronize()
    assert int(server.err) == 0 and server.cached.tolist() == [n + steps - 1 for n in lens]
    used = server.tables[server.tables >= 0].tolist()
    assert len(set(used)) == len(used) == sum(-(-(n + steps - 1) // m.PAGE) for n in lens)
    for b, p in enumerate(prompts):
        every = torch.cat((p, tokens[b]))
        logits = _plain_logits(m, server, every[:-1])[len(p) - 1:]
        mine = logits.gather(1, tokens[b][:, None])[:, 0]
        assert (mine >= logits.amax(-1) - 3 * 2.0 ** -8 * logits.abs().amax(-1)).all()


def test_example_runs_from_the_command_line(capsys, monkeypatch):
    m = _example()
    monkeypatch.setattr("sys.argv", ["x", "--requests", "3", "--prompt", "90", "--chunk", "40", "--steps", "5"])
    m.main()
    assert "error word 0" in capsys.readouterr().out


def test_attention_module_over_a_4_bit_cache():
    """Prefill of ragged requests behind cached prefixes, then decode, through Attention.forward."""
    d, page, hq, hkv, scale = dev(), 32, 16, 4, 0.1
    g = torch.Generator(device=d).manual_seed(1)
    i32 = dict(dtype=torch.int32, device=d)
    attn = Attention(hq, 128, scale, hkv, sliding_window=50)
    attn.k_cache, attn.v_cache = kv.empty_kvcache_fp4(40, hkv, page, d)
    attn.k_scale, attn.v_scale = 0.5, 0.25
    tables = torch.full((3, 8), -1, **i32)
    cached, start, free = torch.zeros(3, **i32), torch.zeros(1, **i32), torch.randperm(40, device=d).to(torch.int32)
    keys = [torch.zeros((0, hkv, 128), device=d, dtype=torch.bfloat16) for _ in range(3)]
    values = [k.clone() for k in keys]
    try:
        for new in ([40, 3, 0], [20, 70, 5], [1, 1, 1], [1, 1, 1], [2, 0, 90], [1, 1, 1]):
            n = sum(new)
            q, k, v = (torch.randn((n, h, 128), generator=g, device=d).to(torch.bfloat16) for h in (hq, hkv, hkv))
            m = step_metadata(cached, torch.tensor(new, **i32), tables, free, start, page, n)
            prefill = max(new) > 1
            set_context(prefill, m.cu_seqlens_q, m.cu_seqlens_k, max(new), 0, m.slot_mapping, m.context_lens, tables)
            out = attn(q, k, v)
            cached.copy_(m.context_lens)
            start.copy_(m.free_next)
            at = 0
            for b, t in enumerate(new):
                keys[b] = torch.cat((keys[b], k[at:at + t]))
                values[b] = torch.cat((values[b], v[at:at + t]))
                at += t
            lens = [len(x) for x in keys]
            want, err = kv4.attention(q, attn.k_cache, attn.v_cache, tables, new, lens, scale, 50, not prefill, 0.5, 0.25)
            half = torch.finfo(torch.bfloat16).eps / 2
            assert ((out.double() - want).abs() <= err + half * (want.abs() + err) + 1e-30).all()
        for b in range(3):  # the cache holds what was given
            got, there = kv4.rows_of(attn.k_cache, tables[b], len(keys[b]))
            assert there.all() and torch.equal(got * 0.5, kv4.stored(keys[b], 0.5))
            got, _ = kv4.rows_of(attn.v_cache, tables[b], len(values[b]))
            assert torch.equal(got * 0.25, kv4.stored(values[b], 0.25))
    finally:
        reset_context()
