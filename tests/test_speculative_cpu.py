"""Shared-prefix decode, sampling and verification without a GPU: what the C ABI and the Python
layer refuse (before any CUDA call; pointers are placeholders), and the 64-bit oracles."""
import math

import numpy as np
import pytest
import torch

from adallm_b200 import _native as N
from adallm_b200 import build as B
from oracle import attention as oa
from oracle import speculative as osp

P = 1 << 20


@pytest.fixture(scope="module")
def lib():
    B.build()
    return N.lib()


def test_shared_prefix_argument_errors(lib):
    need = lib.ada_fp8_shared_prefix_decode_workspace_size(6, 1, 4, 32, 8, 128)
    assert need > 0 and lib.ada_fp8_shared_prefix_decode_workspace_size(0, 1, 4, 32, 8, 128) == 0

    def call(**kw):
        a = dict(q=P, q_dtype=0, q_st=4096, q_sh=128, k=P, v=P, s_page=16384, s_tok=1024, s_head=128, num_pages=64,
                 pt=P, pt_stride=9, max_pp=8, plens=P, cu_g=P, groups=1, bt=P, bt_stride=8, max_pages=8, ctx=P, cu_q=P,
                 batch=4, total_q=6, hq=32, hkv=8, d=128, page=16, scale=0.088, ks=1.0, vs=1.0, window=0, out=P,
                 out_dtype=0, o_st=4096, o_sh=128, ws=P, ws_bytes=need, err=None, stream=None)
        a.update(kw)
        return lib.ada_fp8_shared_prefix_decode(*a.values())

    assert call(total_q=0) == 0 and call(batch=0) == 0                 # nothing to do
    for name in ("q", "k", "v", "plens", "pt", "bt", "ctx", "out", "ws"):
        assert call(**{name: None}) == N.ADA_ERR_INVALID_ARG, name
    assert call(cu_g=None, groups=2) == N.ADA_ERR_INVALID_ARG          # several groups need their bounds
    assert call(cu_q=None) == N.ADA_ERR_INVALID_ARG                    # six rows of four sequences
    assert call(hq=30) == N.ADA_ERR_INVALID_ARG
    assert call(q_dtype=2) == N.ADA_ERR_INVALID_ARG and call(out_dtype=5) == N.ADA_ERR_INVALID_ARG
    assert call(scale=0.0) == N.ADA_ERR_INVALID_ARG and call(scale=math.nan) == N.ADA_ERR_INVALID_ARG
    assert call(window=-1) == N.ADA_ERR_INVALID_ARG
    assert call(bt_stride=7) == N.ADA_ERR_INVALID_ARG and call(pt_stride=7) == N.ADA_ERR_INVALID_ARG
    assert call(total_q=-1) == N.ADA_ERR_INVALID_ARG and call(num_pages=0) == N.ADA_ERR_INVALID_ARG
    assert call(d=64) == N.ADA_ERR_UNSUPPORTED and call(page=24) == N.ADA_ERR_UNSUPPORTED
    assert call(hq=256, hkv=1) == N.ADA_ERR_UNSUPPORTED
    assert call(batch=4096, total_q=4096) == N.ADA_ERR_UNSUPPORTED     # 4,097 prefixes and sequences
    assert call(max_pp=1 << 27, pt_stride=1 << 27) == N.ADA_ERR_UNSUPPORTED
    assert call(q=P + 8) == N.ADA_ERR_ALIGNMENT and call(k=P + 8) == N.ADA_ERR_ALIGNMENT
    assert call(s_tok=1032) == N.ADA_ERR_ALIGNMENT and call(q_sh=100) == N.ADA_ERR_ALIGNMENT
    assert call(o_st=4092) == N.ADA_ERR_ALIGNMENT and call(out=P + 2) == N.ADA_ERR_ALIGNMENT
    assert call(ws=P + 16) == N.ADA_ERR_ALIGNMENT and call(err=P + 1) == N.ADA_ERR_ALIGNMENT
    assert call(ws_bytes=need - 1) == N.ADA_ERR_WORKSPACE


def test_sample_argument_errors(lib):
    def call(**kw):
        a = dict(x=P, dtype=0, ld=1000, rows=4, vocab=1000, temps=P, noise=P, ld_noise=1000, tokens=P, lp=P, lse=P,
                 stream=None)
        a.update(kw)
        return lib.ada_sample(*a.values())

    assert call(rows=0) == 0
    for name in ("x", "temps", "noise", "tokens"):
        assert call(**{name: None}) == N.ADA_ERR_INVALID_ARG, name
    assert call(vocab=0) == N.ADA_ERR_INVALID_ARG and call(rows=-1) == N.ADA_ERR_INVALID_ARG
    assert call(ld=999) == N.ADA_ERR_INVALID_ARG and call(ld_noise=999) == N.ADA_ERR_INVALID_ARG
    assert call(dtype=3) == N.ADA_ERR_INVALID_ARG
    assert call(rows=(1 << 20) + 1) == N.ADA_ERR_UNSUPPORTED
    assert call(x=P + 1) == N.ADA_ERR_ALIGNMENT and call(x=P + 2, dtype=2) == N.ADA_ERR_ALIGNMENT
    assert call(noise=P + 2) == N.ADA_ERR_ALIGNMENT and call(tokens=P + 4) == N.ADA_ERR_ALIGNMENT


def test_verify_argument_errors(lib):
    need = lib.ada_verify_drafts_workspace_size(10, 4, 1000, 0)
    assert need > 0 and lib.ada_verify_drafts_workspace_size(10, 0, 1000, 0) == 0

    def call(**kw):
        a = dict(x=P, dtype=0, ld=1000, total=10, vocab=1000, ids=P, cu=P, batch=4, most=3, temps=P, u=P, ld_u=3,
                 noise=P, ld_noise=1000, draft=P, d_sb=3000, d_sd=1000, lse=P, l_sb=3, l_sd=1, tokens=P, acc=P, lp=P,
                 ws=P, ws_bytes=need, stream=None)
        a.update(kw)
        return lib.ada_verify_drafts(*a.values())

    assert call(batch=0) == 0
    for name in ("x", "ids", "cu", "temps", "u", "noise", "tokens", "acc", "lp", "ws"):
        assert call(**{name: None}) == N.ADA_ERR_INVALID_ARG, name
    assert call(draft=None) == N.ADA_ERR_INVALID_ARG and call(lse=None) == N.ADA_ERR_INVALID_ARG
    assert call(d_sd=-1) == N.ADA_ERR_INVALID_ARG
    assert call(ld_u=2) == N.ADA_ERR_INVALID_ARG and call(dtype=4) == N.ADA_ERR_INVALID_ARG
    assert call(most=1025, ld_u=1025) == N.ADA_ERR_UNSUPPORTED
    assert call(ws_bytes=need - 1) == N.ADA_ERR_WORKSPACE and call(ws=P + 8) == N.ADA_ERR_ALIGNMENT
    assert call(draft=P + 1) == N.ADA_ERR_ALIGNMENT and call(ids=P + 4) == N.ADA_ERR_ALIGNMENT


def test_python_layer_needs_cuda_tensors():
    from adallm_b200.sampler import sample, verify_drafts
    from adallm_b200.shared_prefix import shared_prefix_decode
    x, t = torch.zeros((2, 5)), torch.ones(2)
    with pytest.raises(RuntimeError, match="CUDA"):
        sample(x, t, x)
    with pytest.raises(RuntimeError, match="CUDA"):
        verify_drafts(x, torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32), t, x[:, :1], x)
    c = osp.make_shared_prefix_case(0, [4], [1], [3], [1], 8, 8, 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"], None,
                             c["block_tables"], c["context_lens"], 1.0)


@pytest.mark.parametrize("window", [0, 40])
def test_oracle_is_the_decode_oracle_over_joined_pages(window):
    """With the prefix filling whole pages, the joined page lists give oracle.attention's decode."""
    c = osp.make_shared_prefix_case(1, [64], [3], [5, 16, 33], [1, 1, 1], 8, 2, 16)
    got = osp.shared_prefix_decode(c["q"], c["k_cache"], c["v_cache"], c["prefix_tables"], c["prefix_lens"], None,
                                   c["block_tables"], c["context_lens"], c["scale"], window=window)
    joined = torch.cat((c["prefix_tables"][:, :4].expand(3, -1), c["block_tables"]), 1).numpy()
    want = oa.paged_decode(c["q"].float().numpy(), c["k_cache"].view(torch.uint8).numpy(),
                           c["v_cache"].view(torch.uint8).numpy(), joined, c["context_lens"].numpy() + 64, c["scale"],
                           window)
    assert float(np.abs(got.numpy() - want).max()) < 1e-5


def test_oracle_verification_keeps_the_target_distribution():
    """Exact over all outcomes of one draft: sum_x q(x) accept(x) and the drawn rest give p."""
    rng = np.random.default_rng(0)
    target, draft = rng.standard_normal((2, 6)), rng.standard_normal(6)
    p = np.exp(target[0]) / np.exp(target[0]).sum()
    q = np.exp(draft) / np.exp(draft).sum()
    lse = float(np.log(np.exp(draft).sum()))
    n, count = 4000, np.zeros(6)
    for _ in range(n):
        x = rng.choice(6, p=q)
        tokens, accepted, _, _ = osp.verify(target, [0, x], 1.0, [rng.random()], rng.exponential(size=6), [draft], [lse])
        assert accepted in (0, 1) and len(tokens) == accepted + 1
        count[tokens[0]] += 1
    assert (np.abs(count - n * p) < 5 * np.sqrt(n * p * (1 - p))).all()
