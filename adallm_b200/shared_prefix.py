"""Decode attention for batches that share prompt prefixes, on the FP8 paged cache.

``shared_prefix_decode`` reads the keys and values of a prefix once for all the sequences behind
it (parallel samples of a prompt, a common system prompt), joins them with each sequence's own
pages, and takes one or several query rows a sequence (the rows of drafted tokens).  The
reference has no such form: its decode reads a cached prefix once per sequence
(adallm/ops/attention.py:359-414)."""
from __future__ import annotations

import functools

import torch

from . import _native as N


@functools.lru_cache(maxsize=512)
def shared_prefix_workspace_bytes(total_q: int, num_groups: int, batch: int, num_heads: int, num_kv_heads: int,
                                  head_dim: int) -> int:
    return int(N.lib().ada_fp8_shared_prefix_decode_workspace_size(total_q, num_groups, batch, num_heads,
                                                                   num_kv_heads, head_dim))


I32 = torch.int32


def _lengths(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dtype is not I32 or not t.is_contiguous():
        raise ValueError(f"{name} must be int32 with unit stride")
    return t


def shared_prefix_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, prefix_tables: torch.Tensor,
                         prefix_lens: torch.Tensor, cu_groups: torch.Tensor | None, block_tables: torch.Tensor,
                         context_lens: torch.Tensor, scale: float, cu_seqlens_q: torch.Tensor | None = None,
                         window: int = 0, k_scale: float = 1.0, v_scale: float = 1.0,
                         out: torch.Tensor | None = None, workspace: torch.Tensor | None = None,
                         err: torch.Tensor | None = None) -> torch.Tensor:
    """Attention of each sequence's newest tokens over its group's prefix and its own keys.

    q [N, Hq, 128] bf16/fp16; k_cache/v_cache [num_pages, page, Hkv, 128] e4m3;
    prefix_tables int32 [G, pages], prefix_lens int32 [G]: the prefix pages of each group;
    cu_groups int32 [G + 1]: group g is sequences cu_groups[g]..cu_groups[g+1] (None: one group
    of all); block_tables int32 [B, pages], context_lens int32 [B]: each sequence's own keys
    behind the prefix, its new tokens included (store_kvcache runs first);
    cu_seqlens_q int32 [B + 1]: sequence b's rows of q are its newest tokens (None: one each).
    Row i of t attends to positions <= prefix + context - t + i, with window W > 0 to the last W
    of them.  Rows that see no key are zeros.
    Returns [N, Hq, 128] in q.dtype.  workspace: at least shared_prefix_workspace_bytes(...) bytes
    (default: allocated for the call).  At most 4096 prefixes and sequences together.  err: optional
    int32 [1] device word; 0x90 is OR-ed in if a tile wait ran out."""
    if not (q.is_cuda and k_cache.is_cuda and v_cache.is_cuda and prefix_tables.is_cuda and prefix_lens.is_cuda
            and block_tables.is_cuda and context_lens.is_cuda):
        raise RuntimeError("shared_prefix_decode requires CUDA tensors")
    total_q, hq, d = q.shape
    pages, page, hkv, dk = shape = k_cache.shape
    if q.stride(-1) != 1:
        q = q.contiguous()
    qs, ks, pts, bts = q.stride(), k_cache.stride(), prefix_tables.stride(), block_tables.stride()
    code = N.DT.get(q.dtype)
    if code is None or (out is not None and out.dtype not in N.DT):
        raise ValueError("q and out must be bf16 or fp16")
    if dk != d or shape != v_cache.shape or ks != v_cache.stride() or ks[3] != 1:
        raise ValueError("k_cache and v_cache must share a [pages, page, Hkv, D] layout with q's head size")
    if k_cache.dtype is not torch.float8_e4m3fn or v_cache.dtype is not torch.float8_e4m3fn:
        raise ValueError("the shared-prefix decode reads a float8_e4m3fn cache")
    if prefix_tables.dtype is not I32 or block_tables.dtype is not I32 or pts[1] != 1 or bts[1] != 1:
        raise ValueError("prefix_tables and block_tables must be int32 with unit stride")
    _lengths(prefix_lens, "prefix_lens")
    _lengths(context_lens, "context_lens")
    cu_g = cu_q = None
    if cu_groups is not None:
        N.require_cuda(cu_groups, what="shared_prefix_decode")
        cu_g = _lengths(cu_groups, "cu_groups").data_ptr()
    if cu_seqlens_q is not None:
        N.require_cuda(cu_seqlens_q, what="shared_prefix_decode")
        cu_q = _lengths(cu_seqlens_q, "cu_seqlens_q").data_ptr()
    groups, batch = prefix_lens.numel(), context_lens.numel()
    (pt_rows, pt_pages), (bt_rows, bt_pages) = prefix_tables.shape, block_tables.shape
    if pt_rows != groups or bt_rows != batch:
        raise ValueError("page tables must have one row per prefix and per sequence")
    if groups > 1 if cu_groups is None else cu_groups.numel() != groups + 1:
        raise ValueError("cu_groups must hold the first sequence of each group and the end (None for one group)")
    if total_q != batch if cu_seqlens_q is None else cu_seqlens_q.numel() != batch + 1:
        raise ValueError("cu_seqlens_q must have batch + 1 entries (None for one row per sequence)")
    window = min(int(window), 0x7FFFFFFF)  # (past any position; the foreign call would take the low 32 bits)
    device = q.device
    if out is None:
        out = q.new_empty((total_q, hq, d))
        os, out_code = (hq * d, d), code
    else:
        N.require_cuda(out, what="shared_prefix_decode")
        os, out_code = out.stride(), N.DT[out.dtype]
        if out.shape != q.shape or os[2] != 1:
            raise ValueError("out must have q's shape and unit stride in the head dimension")
    if total_q == 0:
        return out
    if batch == 0:
        return out.zero_()
    stream = N.stream_ptr(device)
    need = shared_prefix_workspace_bytes(total_q, groups, batch, hq, hkv, d)
    if workspace is None:
        # one of its own: the launches of another thread's call on this stream may fall between this call's
        workspace = torch.empty(need, dtype=torch.uint8, device=device)
    else:
        N.require_cuda(workspace, what="shared_prefix_decode")
    if err is not None:
        N.require_cuda(err, what="shared_prefix_decode")
    st = N.lib().ada_fp8_shared_prefix_decode(
        q.data_ptr(), code, qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), ks[0], ks[1], ks[2], pages,
        prefix_tables.data_ptr(), pts[0], pt_pages, prefix_lens.data_ptr(), cu_g, groups,
        block_tables.data_ptr(), bts[0], bt_pages, context_lens.data_ptr(), cu_q, batch,
        total_q, hq, hkv, d, page, float(scale), float(k_scale), float(v_scale), window, out.data_ptr(), out_code,
        os[0], os[1], workspace.data_ptr(), workspace.nbytes, N.ptr(err), stream)
    if st:
        N.check(st, "shared-prefix decode attention")
    return out
