"""The paged KV cache in 4 bits: store, read-back, decode and prefill attention.

Beside the e4m3 cache of ``attention.py`` (128 bytes a row and head) this one holds a row in 72:
e2m1 codes with an e4m3 scale for every 16 elements, the format of the NVFP4 weights.  The reference
has no such cache (its decode reads e4m3, adallm/ops/attention.py:359-414).

A cache is uint8 [num_pages, Hkv, page * 72] (any strides over pages and heads that are multiples of
16): a block of one page and head holds its rows' codes, 64 bytes a row with the even element in the low
nibble, then the rows' 8 scales.  Page tables, slots and masks are those of ``attention.py``."""
from __future__ import annotations

import functools

import torch

from . import _native as N

I32 = torch.int32
HEAD_DIM = 128
ROW_BYTES = 72


def empty_kvcache_fp4(num_pages: int, num_kv_heads: int, page_size: int, device=None) -> tuple:
    """(k_cache, v_cache) of num_pages pages, zeros."""
    if page_size <= 0 or page_size % 16:
        raise ValueError("page_size must be a multiple of 16")
    shape = (2, num_pages, num_kv_heads, page_size * ROW_BYTES)
    return tuple(torch.zeros(shape, dtype=torch.uint8, device=device).unbind(0))


def _cache(k_cache: torch.Tensor, v_cache: torch.Tensor):
    """(num_pages, KV heads, page size, page stride, head stride) of a cache."""
    shape, strides = k_cache.shape, k_cache.stride()
    if k_cache.dtype is not torch.uint8 or v_cache.dtype is not torch.uint8:
        raise ValueError("the 4-bit KV cache is held as uint8")
    if len(shape) != 3 or shape != v_cache.shape or strides != v_cache.stride() or strides[2] != 1:
        raise ValueError("k_cache and v_cache must share a [pages, Hkv, page * 72] layout")
    page, rest = divmod(shape[2], ROW_BYTES)
    if rest:
        raise ValueError("a block of the 4-bit KV cache has 72 bytes a row")
    return shape[0], shape[1], page, strides[0], strides[1]


def _rows(t: torch.Tensor, name: str) -> torch.Tensor:
    if t.dim() != 3 or t.shape[2] != HEAD_DIM:
        raise ValueError(f"{name} must be [tokens, heads, 128]")
    return t if t.stride(2) == 1 else t.contiguous()


def _slots(slot_mapping: torch.Tensor, tokens: int) -> torch.Tensor:
    if slot_mapping.numel() != tokens:
        raise ValueError("slot_mapping must have one entry per token")
    if slot_mapping.dtype is not I32:
        raise ValueError("slot_mapping must be int32")
    return slot_mapping if slot_mapping.is_contiguous() else slot_mapping.contiguous()


def _store(positions, query, key, value, cos_sin, k_cache, v_cache, slot_mapping, interleaved, k_scale, v_scale, q_out,
           device):
    pages, hkv, page, s_page, s_head = _cache(k_cache, v_cache)
    key, value = _rows(key, "key"), _rows(value, "value")
    tokens = key.shape[0]
    code = N.DT.get(key.dtype)
    if code is None or value.dtype is not key.dtype:
        raise ValueError("key/value must be bf16 or fp16")
    if key.shape != value.shape or key.shape[1] != hkv:
        raise ValueError("key and value must be [tokens, Hkv, 128] with the cache's heads")
    slots = _slots(slot_mapping, tokens)
    ks, vs = key.stride(), value.stride()
    if query is None:
        q_args = (None, None, 0, 0)
        hq, table_args = 0, (None, 0, 0, 0)
    else:
        qs = query.stride()
        q_args = (positions.data_ptr(), query.data_ptr(), qs[0], qs[1])
        hq = query.shape[1]
        table_args = (cos_sin.data_ptr(), cos_sin.shape[0], cos_sin.shape[-1], interleaved)
    st = N.call(N.lib().ada_kv4_store, device, *q_args, key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1],
                N.ptr(q_out), tokens, hq, hkv, HEAD_DIM, *table_args, slots.data_ptr(), k_cache.data_ptr(),
                v_cache.data_ptr(), s_page, s_head, pages, page, k_scale, v_scale, code, N.stream_ptr(device))
    if st:
        N.check(st, "store_kvcache_fp4")


def store_kvcache_fp4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, k_scale: float = 1.0, v_scale: float = 1.0) -> None:
    """Pack key / k_scale and value / v_scale [T, Hkv, 128] (bf16/fp16) at every slot of the cache.

    slot = page * page_size + row; slots outside the cache (-1 among them) are skipped, and a slot
    given twice holds a mix of both rows.  Of each 16 elements: scale = e4m3(max |x| / 6), codes = the nearest e2m1
    to x / scale; infinities saturate, a NaN makes its 16 elements read as NaN."""
    device = N.one_device("store_kvcache_fp4", key, value, k_cache, v_cache, slot_mapping)
    _store(None, None, key, value, None, k_cache, v_cache, slot_mapping, False, k_scale, v_scale, None, device)


def rotary_store_kvcache_fp4(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                             cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                             slot_mapping: torch.Tensor, interleaved: bool = False, k_scale: float = 1.0,
                             v_scale: float = 1.0, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """apply_rotary on query and key, and store_kvcache_fp4 of the rotated key and the value, in one launch.

    query [T, Hq, 128], key/value [T, Hkv, 128]; the rest as in rotary_embedding.apply_rotary and
    store_kvcache_fp4.  Returns the rotated query (q_out, contiguous, if given)."""
    device = N.one_device("rotary_store_kvcache_fp4", key, query, value, positions, cos_sin_cache, k_cache, v_cache,
                          slot_mapping, q_out)
    query = _rows(query, "query")
    shape = query.shape
    if shape[0] != key.shape[0] or positions.numel() != shape[0] or query.dtype is not key.dtype:
        raise ValueError("positions, query and key must describe the same tokens in one type")
    if cos_sin_cache.dtype is not torch.float32 or not cos_sin_cache.is_contiguous():
        raise ValueError("cos_sin_cache must be contiguous fp32")
    if positions.dtype is not torch.int64 or not positions.is_contiguous():
        positions = positions.to(torch.int64).contiguous()
    if q_out is None:
        q_out = query.new_empty(shape)
    elif q_out.shape != shape or q_out.dtype is not query.dtype or not q_out.is_contiguous():
        raise ValueError("q_out must be contiguous with query's shape and type")
    _store(positions, query, key, value, cos_sin_cache, k_cache, v_cache, slot_mapping, interleaved, k_scale, v_scale,
           q_out, device)
    return q_out


def read_kvcache_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                     dtype: torch.dtype = torch.bfloat16, k_scale: float = 1.0, v_scale: float = 1.0,
                     out: tuple | None = None) -> tuple:
    """The keys and values at the slots, [T, Hkv, 128] each in bf16/fp16; zeros for slots outside the cache."""
    k_out, v_out = out if out is not None else (None, None)
    device = N.one_device("read_kvcache_fp4", k_cache, v_cache, slot_mapping, k_out, v_out)
    pages, hkv, page, s_page, s_head = _cache(k_cache, v_cache)
    code = N.DT.get(dtype)
    if code is None:
        raise ValueError("the cache is read as bf16 or fp16")
    tokens = slot_mapping.numel()
    slots = _slots(slot_mapping, tokens)
    shape = (tokens, hkv, HEAD_DIM)
    if out is None:
        k_out, v_out = torch.empty((2,) + shape, dtype=dtype, device=device).unbind(0)
    else:
        for t in out:
            if t.shape != shape or t.dtype is not dtype or not t.is_contiguous():
                raise ValueError("out must be two contiguous [tokens, Hkv, 128] tensors of dtype")
    st = N.call(N.lib().ada_kv4_read, device, k_cache.data_ptr(), v_cache.data_ptr(), s_page, s_head, pages, page, hkv,
                HEAD_DIM, slots.data_ptr(), tokens, k_scale, v_scale, k_out.data_ptr(), v_out.data_ptr(), code,
                N.stream_ptr(device))
    if st:
        N.check(st, "read_kvcache_fp4")
    return k_out, v_out


@functools.lru_cache(maxsize=512)
def paged_decode_fp4_workspace_bytes(batch: int, num_heads: int, num_kv_heads: int) -> int:
    return int(N.lib().ada_kv4_paged_decode_workspace_size(batch, num_heads, num_kv_heads))


def _attention(q, k_cache, v_cache, block_tables, out, *lists):
    """Checks that decode and prefill share."""
    layout = _cache(k_cache, v_cache)
    q = _rows(q, "q")
    code = N.DT.get(q.dtype)
    if code is None or (out is not None and out.dtype not in N.DT):
        raise ValueError("q and out must be bf16 or fp16")
    if block_tables.dtype is not I32 or block_tables.dim() != 2 or block_tables.stride(1) != 1:
        raise ValueError("block_tables must be int32 [sequences, pages] with unit stride")
    for t, name in lists:
        if t.dtype is not I32 or not t.is_contiguous():
            raise ValueError(f"{name} must be int32 with unit stride")
    if out is None:
        out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.stride(2) != 1:
        raise ValueError("out must have q's shape and unit stride in the head dimension")
    return layout, q, code, out


def paged_decode_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, scale: float, window: int = 0, k_scale: float = 1.0,
                     v_scale: float = 1.0, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of one query token per sequence against the 4-bit paged cache.

    q [B, Hq, 128] bf16/fp16; k_cache/v_cache uint8 [pages, Hkv, page * 72]; block_tables int32 [B, max_pages]
    (ids outside the cache are masked); context_lens int32 [B], the new token included.  window W > 0: the last
    W tokens.  Returns [B, Hq, 128] in q.dtype; a sequence without keys gives zeros.  workspace: at
    least paged_decode_fp4_workspace_bytes(B, Hq, Hkv) bytes (default: allocated for the call)."""
    device = N.one_device("paged_decode_fp4", q, k_cache, v_cache, block_tables, context_lens, out, workspace)
    (pages, hkv, page, s_page, s_head), q, code, out = _attention(q, k_cache, v_cache, block_tables, out,
                                                                  (context_lens, "context_lens"))
    batch, hq, d = q.shape
    if context_lens.numel() != batch or block_tables.shape[0] != batch:
        raise ValueError("block_tables and context_lens must have one entry per sequence")
    if batch == 0:
        return out
    if workspace is None:
        # one of its own: the launches of another thread's call on this stream may fall between this call's
        workspace = torch.empty(paged_decode_fp4_workspace_bytes(batch, hq, hkv), dtype=torch.uint8, device=device)
    qs, os = q.stride(), out.stride()
    st = N.call(N.lib().ada_kv4_paged_decode, device, q.data_ptr(), code, qs[0], qs[1], k_cache.data_ptr(),
                v_cache.data_ptr(), s_page, s_head, pages, block_tables.data_ptr(), block_tables.stride(0),
                block_tables.shape[1], context_lens.data_ptr(), batch, hq, hkv, d, page, scale, k_scale, v_scale,
                min(int(window), 0x7FFFFFFF), out.data_ptr(), N.DT[out.dtype], os[0], os[1], workspace.data_ptr(),
                workspace.nbytes, N.stream_ptr(device))
    if st:
        N.check(st, "4-bit KV decode kernel")
    return out


def paged_prefill_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                      cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, max_seqlen_q: int, scale: float,
                      window: int = 0, k_scale: float = 1.0, v_scale: float = 1.0, out: torch.Tensor | None = None,
                      err: torch.Tensor | None = None) -> torch.Tensor:
    """Causal prefill attention of the new tokens against the 4-bit paged cache.

    The arguments of attention.paged_prefill with a 4-bit cache: q [total_q, Hq, 128]; the cache holds every
    sequence's cached prefix and new tokens; max_seqlen_q must be at least every sequence's new tokens.
    window W > 0: a row sees its own position and the W before it.  Rows behind the last sequence are left as
    they are in ``out`` (unset without it)."""
    device = N.one_device("paged_prefill_fp4", q, k_cache, v_cache, block_tables, cu_seqlens_q, cu_seqlens_k, out, err)
    (pages, hkv, page, s_page, s_head), q, code, out = _attention(q, k_cache, v_cache, block_tables, out,
                                                                  (cu_seqlens_q, "cu_seqlens_q"),
                                                                  (cu_seqlens_k, "cu_seqlens_k"))
    total_q, hq, d = q.shape
    batch = cu_seqlens_q.numel() - 1
    if cu_seqlens_k.numel() != batch + 1 or block_tables.shape[0] < batch:
        raise ValueError("cu_seqlens_q, cu_seqlens_k and block_tables must describe the same sequences")
    if err is not None and (err.dtype is not I32 or err.numel() != 1):
        raise ValueError("err must be one int32")
    if total_q == 0 or batch <= 0:
        return out
    qs, os = q.stride(), out.stride()
    st = N.call(N.lib().ada_kv4_paged_prefill, device, q.data_ptr(), code, qs[0], qs[1], k_cache.data_ptr(),
                v_cache.data_ptr(), s_page, s_head, pages, block_tables.data_ptr(), block_tables.stride(0),
                block_tables.shape[1], cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), batch, total_q,
                int(max_seqlen_q), hq, hkv, d, page, scale, k_scale, v_scale, min(int(window), 0x7FFFFFFF),
                out.data_ptr(), N.DT[out.dtype], os[0], os[1], N.ptr(err), N.stream_ptr(device))
    if st:
        N.check(st, "4-bit KV prefill kernel")
    return out
