"""A serving step's metadata (positions, slots, prefix sums, block tables) built on the GPU.

The reference builds it with host loops and copies it over every step
(adallm/runtime/model_runner.py:234-300), and its block manager hands out pages on the host.  Here a
step's lengths stay on the device: one launch extends the block tables from a free list and writes
what RoPE, the KV store and the attention of the step read, so a captured decode step needs no host
work between its replays."""
from __future__ import annotations

from typing import NamedTuple

import torch

from . import _native as N

I32 = torch.int32


class StepMetadata(NamedTuple):
    positions: torch.Tensor     # int64 [num_tokens]
    slot_mapping: torch.Tensor  # int32 [num_tokens], -1: not stored
    cu_seqlens_q: torch.Tensor  # int32 [B + 1]
    cu_seqlens_k: torch.Tensor  # int32 [B + 1]
    context_lens: torch.Tensor  # int32 [B]
    free_next: torch.Tensor     # int32 [1]


def empty_step_metadata(requests: int, num_tokens: int, device) -> StepMetadata:
    """Buffers for step_metadata's ``out`` (a captured step keeps one)."""
    return StepMetadata(torch.empty(num_tokens, dtype=torch.int64, device=device),
                        *(torch.empty(n, dtype=I32, device=device)
                          for n in (num_tokens, requests + 1, requests + 1, requests, 1)))


def step_metadata(cached_lens: torch.Tensor, new_lens: torch.Tensor, block_tables: torch.Tensor,
                  free_pages: torch.Tensor, free_start: torch.Tensor, page_size: int, num_tokens: int,
                  out: StepMetadata | tuple | None = None, err: torch.Tensor | None = None) -> StepMetadata:
    """Metadata of one step: requests with ``cached_lens`` stored and ``new_lens`` new tokens.

    cached_lens, new_lens int32 [B]; block_tables int32 [B, max_pages]: the pages of the cached tokens;
    the pages the new tokens need are written behind them, taken off free_pages int32 [F] from
    free_start int32 [1] on in request order, and ``free_next`` says where the next step starts.
    num_tokens: what the outputs are laid out for, at least the sum of new_lens; further tokens are
    padding with position 0 and slot -1.  A token without a page (free list at its end, table too narrow)
    gets slot -1, and its table entry is -1 (so it stays without one in the steps behind).  err: optional int32 [1] device word; 0x100 (free list), 0x200 (table) and 0x400 (more
    tokens than num_tokens) are OR-ed in.  The inputs, block_tables apart, are left as they are: for the
    next step copy free_next to free_start and context_lens to cached_lens.  At most 8192 requests."""
    tensors = (cached_lens, new_lens, free_pages, free_start)
    device = N.one_device("step_metadata", *tensors, block_tables)
    for t in tensors:
        if t.dtype is not I32 or not t.is_contiguous():
            raise ValueError("cached_lens, new_lens, free_pages and free_start must be int32 with unit stride")
    requests = cached_lens.numel()
    if new_lens.numel() != requests or free_start.numel() != 1:
        raise ValueError("cached_lens and new_lens must have one entry per request, free_start one")
    if block_tables.dtype is not I32 or block_tables.dim() != 2:
        raise ValueError("block_tables must be int32 [requests, pages]")
    (rows, max_pages), (row_stride, unit) = block_tables.shape, block_tables.stride()
    if rows != requests or (unit != 1 and max_pages > 1):
        raise ValueError("block_tables must have one row of unit stride per request")
    if num_tokens < 0:
        raise ValueError("num_tokens must not be negative")
    word = 0
    if err is not None:
        N.one_device("step_metadata", err, cached_lens)
        if err.dtype is not I32 or err.numel() != 1:
            raise ValueError("err must be one int32")
        word = err.data_ptr()
    if out is None:
        out = empty_step_metadata(requests, num_tokens, cached_lens.device)
    else:
        if type(out) is not StepMetadata:
            out = StepMetadata(*out)
        for t, n in zip(out, (num_tokens, num_tokens, requests + 1, requests + 1, requests, 1)):
            if t.numel() != n or t.dtype is not (I32 if t is not out[0] else torch.int64) or not t.is_contiguous() \
                    or t.get_device() != device:
                raise ValueError("out must hold contiguous tensors as empty_step_metadata makes them")
    positions, slots, cu_q, cu_k, context, free_next = out
    st = N.step_metadata(device, cached_lens.data_ptr(), new_lens.data_ptr(), requests, block_tables.data_ptr(),
                         max_pages if requests == 1 else row_stride, max_pages, free_pages.data_ptr(),
                         free_pages.numel(), free_start.data_ptr(), page_size, num_tokens, positions.data_ptr(),
                         slots.data_ptr(), cu_q.data_ptr(), cu_k.data_ptr(), context.data_ptr(), free_next.data_ptr(),
                         word, N.raw_stream(device))
    if st:
        N.check(st, "step_metadata")
    return out
