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
from .rotary_embedding import check_table

I32, U8 = torch.int32, torch.uint8
LARGEST = 0x7FFFFFFF  # windows past any position
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
    if k_cache.dtype is not U8 or v_cache.dtype is not U8:
        raise ValueError("the 4-bit KV cache is held as uint8")
    if len(shape) != 3 or shape != v_cache.shape or strides != v_cache.stride() or strides[2] != 1:
        raise ValueError("k_cache and v_cache must share a [pages, Hkv, page * 72] layout")
    pages, hkv, block = shape
    page = block // ROW_BYTES
    if page * ROW_BYTES != block:
        raise ValueError("a block of the 4-bit KV cache has 72 bytes a row")
    return pages, hkv, page, strides[0], strides[1]


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


def _store(device, rotation, key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale):
    """rotation: None, or (positions, query, cos_sin, interleaved, q_out)."""
    pages, hkv, page, s_page, s_head = _cache(k_cache, v_cache)
    key, value = _rows(key, "key"), _rows(value, "value")
    shape, ks, vs, dtype = key.shape, key.stride(), value.stride(), key.dtype
    tokens = shape[0]
    code = N.DT.get(dtype)
    if code is None or value.dtype is not dtype:
        raise ValueError("key/value must be bf16 or fp16")
    if shape != value.shape or shape[1] != hkv:
        raise ValueError("key and value must be [tokens, Hkv, 128] with the cache's heads")
    slots = _slots(slot_mapping, tokens)
    pos = q = qs0 = qs1 = out = hq = table = reach = width = turn = 0
    if rotation is not None:
        positions, query, cos_sin, turn, q_out = rotation
        pos, q, out, table = positions.data_ptr(), query.data_ptr(), q_out.data_ptr(), cos_sin.data_ptr()
        qs0, qs1, _ = query.stride()
        hq = query.shape[1]
        size = cos_sin.shape
        reach, width = size[0], size[-1]  # [positions, (1,) width]
    st = N.kv4_store(device, pos, q, qs0, qs1, key.data_ptr(), ks[0], ks[1], value.data_ptr(), vs[0], vs[1], out, tokens,
                     hq, hkv, HEAD_DIM, table, reach, width, turn, slots.data_ptr(), k_cache.data_ptr(),
                     v_cache.data_ptr(), s_page, s_head, pages, page, k_scale, v_scale, code, N.raw_stream(device))
    if st:
        N.check(st, "store_kvcache_fp4")


def store_kvcache_fp4(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                      slot_mapping: torch.Tensor, k_scale: float = 1.0, v_scale: float = 1.0) -> None:
    """Pack key / k_scale and value / v_scale [T, Hkv, 128] (bf16/fp16) at every slot of the cache.

    slot = page * page_size + row; slots outside the cache (-1 among them) are skipped, and a slot
    given twice holds a mix of both rows.  Of each 16 elements: scale = e4m3(max |x| / 6), codes = the nearest e2m1
    to x / scale; infinities saturate, a NaN makes its 16 elements read as NaN.  k_scale and v_scale: 1e-30 to 1e30."""
    device = N.one_device("store_kvcache_fp4", key, value, k_cache, v_cache, slot_mapping)
    _store(device, None, key, value, k_cache, v_cache, slot_mapping, k_scale, v_scale)


def rotary_store_kvcache_fp4(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, value: torch.Tensor,
                             cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                             slot_mapping: torch.Tensor, interleaved: bool = False, k_scale: float = 1.0,
                             v_scale: float = 1.0, q_out: torch.Tensor | None = None) -> torch.Tensor:
    """apply_rotary on query and key, and store_kvcache_fp4 of the rotated key and the value, in one launch.

    query [T, Hq, 128], key/value [T, Hkv, 128]; the rest as in rotary_embedding.apply_rotary and
    store_kvcache_fp4.  Returns the rotated query (q_out, contiguous, if given; no input may lie in it)."""
    device = N.one_device("rotary_store_kvcache_fp4", key, query, value, positions, cos_sin_cache, k_cache, v_cache,
                          slot_mapping)
    query = _rows(query, "query")
    shape, dtype = query.shape, query.dtype
    if shape[0] != key.shape[0] or positions.numel() != shape[0] or dtype is not key.dtype:
        raise ValueError("positions, query and key must describe the same tokens in one type")
    check_table(cos_sin_cache)
    if positions.dtype is not torch.int64 or not positions.is_contiguous():
        positions = positions.to(torch.int64).contiguous()
    if q_out is None:
        q_out = query.new_empty(shape)
    elif q_out.shape != shape or q_out.dtype is not dtype or not q_out.is_contiguous() or q_out.get_device() != device:
        raise ValueError("q_out must be contiguous with query's shape, type and device")
    _store(device, (positions, query, cos_sin_cache, interleaved, q_out), key, value, k_cache, v_cache, slot_mapping,
           k_scale, v_scale)
    return q_out


def read_kvcache_fp4(k_cache: torch.Tensor, v_cache: torch.Tensor, slot_mapping: torch.Tensor,
                     dtype: torch.dtype = torch.bfloat16, k_scale: float = 1.0, v_scale: float = 1.0,
                     out: tuple | None = None) -> tuple:
    """The keys and values at the slots, [T, Hkv, 128] each in bf16/fp16; zeros for slots outside the cache."""
    device = N.one_device("read_kvcache_fp4", k_cache, v_cache, slot_mapping)
    pages, hkv, page, s_page, s_head = _cache(k_cache, v_cache)
    code = N.DT.get(dtype)
    if code is None:
        raise ValueError("the cache is read as bf16 or fp16")
    tokens = slot_mapping.numel()
    slots = _slots(slot_mapping, tokens)
    shape = (tokens, hkv, HEAD_DIM)
    if out is None:
        k_out, v_out = torch.empty((2, tokens, hkv, HEAD_DIM), dtype=dtype, device=k_cache.device).unbind(0)
    else:
        k_out, v_out = out
        for t in out:
            if t.shape != shape or t.dtype is not dtype or not t.is_contiguous() or t.get_device() != device:
                raise ValueError("out must be two contiguous [tokens, Hkv, 128] tensors of dtype on the cache's device")
    st = N.kv4_read(device, k_cache.data_ptr(), v_cache.data_ptr(), s_page, s_head, pages, page, hkv, HEAD_DIM,
                    slots.data_ptr(), tokens, k_scale, v_scale, k_out.data_ptr(), v_out.data_ptr(), code,
                    N.raw_stream(device))
    if st:
        N.check(st, "read_kvcache_fp4")
    return k_out, v_out


@functools.lru_cache(maxsize=512)
def paged_decode_fp4_workspace_bytes(batch: int, num_heads: int, num_kv_heads: int, max_pages: int, page_size: int,
                                     window: int = 0) -> int:
    """0 where one launch does it (short tables and windows)."""
    return int(N.lib().ada_kv4_paged_decode_workspace_size(batch, num_heads, num_kv_heads, max_pages, page_size,
                                                           min(window, LARGEST)))


def _attention(device, q, block_tables, out, *lists):
    """Checks that decode and prefill share: (q, its type's code, out, out's code)."""
    q = _rows(q, "q")
    code = N.DT.get(q.dtype)
    if code is None:
        raise ValueError("q must be bf16 or fp16")
    if block_tables.dtype is not I32 or block_tables.dim() != 2 or block_tables.stride(1) != 1:
        raise ValueError("block_tables must be int32 [sequences, pages] with unit stride")
    for t in lists:
        if t.dtype is not I32 or not t.is_contiguous():
            raise ValueError("context_lens, cu_seqlens_q and cu_seqlens_k must be int32 with unit stride")
    if out is None:
        return q, code, q.new_empty(q.shape), code
    out_code = N.DT.get(out.dtype)
    if out_code is None or out.shape != q.shape or out.stride(2) != 1 or out.get_device() != device:
        raise ValueError("out must be bf16 or fp16 with q's shape and device and unit stride in the head dimension")
    return q, code, out, out_code


def paged_decode_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                     context_lens: torch.Tensor, scale: float, window: int = 0, k_scale: float = 1.0,
                     v_scale: float = 1.0, out: torch.Tensor | None = None,
                     workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Decode attention of one query token per sequence against the 4-bit paged cache.

    q [B, Hq, 128] bf16/fp16; k_cache/v_cache uint8 [pages, Hkv, page * 72]; block_tables int32 [B, max_pages]
    (ids outside the cache are masked); context_lens int32 [B], the new token included.  window W > 0: the last
    W tokens.  Returns [B, Hq, 128] in q.dtype; a sequence without keys gives zeros.  workspace: at
    least paged_decode_fp4_workspace_bytes(...) bytes (default: allocated for the call)."""
    device = N.one_device("paged_decode_fp4", q, k_cache, v_cache, block_tables, context_lens)
    pages, hkv, page, s_page, s_head = _cache(k_cache, v_cache)
    q, code, out, out_code = _attention(device, q, block_tables, out, context_lens)
    batch, hq, d = q.shape
    rows, max_pages = block_tables.shape
    if context_lens.numel() != batch or rows != batch:
        raise ValueError("block_tables and context_lens must have one entry per sequence")
    if batch == 0:
        return out
    at = 0
    if workspace is None:
        size = paged_decode_fp4_workspace_bytes(batch, hq, hkv, max_pages, page, window)
        if size:
            # one of its own: the launches of another thread's call on this stream may fall between this call's
            workspace = k_cache.new_empty(size)
            at = workspace.data_ptr()
    else:
        size, at = workspace.nbytes, workspace.data_ptr()
        if workspace.get_device() != device or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous on q's device")
    qs, os = q.stride(), out.stride()
    st = N.kv4_paged_decode(device, q.data_ptr(), code, qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), s_page,
                            s_head, pages, block_tables.data_ptr(), block_tables.stride(0), max_pages,
                            context_lens.data_ptr(), batch, hq, hkv, d, page, scale, k_scale, v_scale,
                            window if window < LARGEST else LARGEST, out.data_ptr(), out_code, os[0], os[1],
                            at, size, N.raw_stream(device))
    if st:
        N.check(st, "4-bit KV decode kernel")
    return out


@functools.lru_cache(maxsize=512)
def paged_prefill_fp4_workspace_bytes(batch: int, total_q: int, max_seqlen_q: int, num_heads: int, num_kv_heads: int,
                                      max_pages: int, page_size: int) -> int:
    """0 where one launch does it: full grids, short tables."""
    return int(N.lib().ada_kv4_paged_prefill_workspace_size(batch, total_q, max_seqlen_q, num_heads, num_kv_heads,
                                                            max_pages, page_size))


def paged_prefill_fp4(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, block_tables: torch.Tensor,
                      cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor, max_seqlen_q: int, scale: float,
                      window: int = 0, k_scale: float = 1.0, v_scale: float = 1.0, out: torch.Tensor | None = None,
                      err: torch.Tensor | None = None, workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Causal prefill attention of the new tokens against the 4-bit paged cache.

    The arguments of attention.paged_prefill with a 4-bit cache: q [total_q, Hq, 128]; the cache holds every
    sequence's cached prefix and new tokens; max_seqlen_q must be at least every sequence's new tokens.
    window W > 0: a row sees its own position and the W before it.  Rows behind the last sequence are left as
    they are in ``out`` (unset without it).  workspace: at least paged_prefill_fp4_workspace_bytes(...) bytes, which few
    rows behind long tables need (default: allocated for the call)."""
    device = N.one_device("paged_prefill_fp4", q, k_cache, v_cache, block_tables, cu_seqlens_q, cu_seqlens_k)
    pages, hkv, page, s_page, s_head = _cache(k_cache, v_cache)
    q, code, out, out_code = _attention(device, q, block_tables, out, cu_seqlens_q, cu_seqlens_k)
    total_q, hq, d = q.shape
    rows, max_pages = block_tables.shape
    batch = cu_seqlens_q.numel() - 1
    if cu_seqlens_k.numel() != batch + 1 or rows < batch:
        raise ValueError("cu_seqlens_q, cu_seqlens_k and block_tables must describe the same sequences")
    word = 0
    if err is not None:
        if err.dtype is not I32 or err.numel() != 1 or err.get_device() != device:
            raise ValueError("err must be one int32 on q's device")
        word = err.data_ptr()
    if total_q == 0 or batch <= 0:
        return out
    at = 0
    if workspace is None:
        size = paged_prefill_fp4_workspace_bytes(batch, total_q, max_seqlen_q, hq, hkv, max_pages, page)
        if size:
            workspace = k_cache.new_empty(size)
            at = workspace.data_ptr()
    else:
        size, at = workspace.nbytes, workspace.data_ptr()
        if workspace.get_device() != device or not workspace.is_contiguous():
            raise ValueError("workspace must be contiguous on q's device")
    qs, os = q.stride(), out.stride()
    st = N.kv4_paged_prefill(device, q.data_ptr(), code, qs[0], qs[1], k_cache.data_ptr(), v_cache.data_ptr(), s_page,
                             s_head, pages, block_tables.data_ptr(), block_tables.stride(0), max_pages,
                             cu_seqlens_q.data_ptr(), cu_seqlens_k.data_ptr(), batch, total_q, max_seqlen_q, hq, hkv, d,
                             page, scale, k_scale, v_scale, window if window < LARGEST else LARGEST, out.data_ptr(),
                             out_code, os[0], os[1], at, size, word, N.raw_stream(device))
    if st:
        N.check(st, "4-bit KV prefill kernel")
    return out
