"""Sampling at a temperature and verification of drafted tokens (B200 kernels).

  * sample: the reference's Sampler.forward (adallm/ops/sampler.py:10-15: softmax(logits / T)
    divided by Exp(1) noise, argmax) with the noise given, and the log-normaliser of every row
  * verify_drafts: acceptance of drafted tokens against the target's probabilities, given the
    draft's logits and their log-normalisers (what ``sample`` returned when it drew them)
  * Sampler: the reference's module on these kernels
"""
from __future__ import annotations

import functools

import torch
from torch import nn

from . import _native as N


F32 = torch.float32


def _unit(t: torch.Tensor) -> torch.Tensor:
    """t with unit stride in its last dimension."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _dense(t: torch.Tensor, name: str, dtype: torch.dtype, n: int) -> torch.Tensor:
    if t.dtype is not dtype or t.numel() != n:
        raise ValueError(f"{name} must be {dtype} with {n} entries")
    return t if t.is_contiguous() else t.contiguous()


def sample(logits: torch.Tensor, temperatures: torch.Tensor,
           noise: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """One token per row of logits [R, V] (bf16/fp16/fp32; rows may be strided).

    temperatures fp32 [R] (<= 1e-10: greedy); noise fp32 [R, V]: Exp(1) draws.
    Returns (tokens int64 [R], logprobs fp32 [R], lse fp32 [R]): the draw, its log-probability
    and the row's log-normaliser, both at the row's temperature (1 where greedy).  A row whose
    logits are all -inf gives -1, 0 and -inf."""
    if not (logits.is_cuda and temperatures.is_cuda and noise.is_cuda):
        raise RuntimeError("sample requires CUDA tensors")
    r, v = logits.shape
    code = N.DT_LOGITS.get(logits.dtype)
    if code is None or noise.dtype is not F32 or noise.shape != logits.shape:
        raise ValueError("logits must be bf16, fp16 or fp32, and noise fp32 with one entry per logit")
    logits, noise = _unit(logits), _unit(noise)
    temperatures = _dense(temperatures, "temperatures", F32, r)
    tokens = temperatures.new_empty(r, dtype=torch.int64)
    logprobs, lse = temperatures.new_empty(r), temperatures.new_empty(r)
    if r == 0:
        return tokens, logprobs, lse
    # (a single row may have any stride)
    ld, ld_noise = (logits.stride(0), noise.stride(0)) if r > 1 else (v, v)
    st = N.lib().ada_sample(logits.data_ptr(), code, ld, r, v, temperatures.data_ptr(), noise.data_ptr(), ld_noise,
                            tokens.data_ptr(), logprobs.data_ptr(), lse.data_ptr(), N.stream_ptr(logits.device))
    if st:
        N.check(st, "sampling kernel")
    return tokens, logprobs, lse


@functools.lru_cache(maxsize=512)
def verify_workspace_bytes(total_q: int, batch: int, vocab: int, dtype: torch.dtype) -> int:
    return int(N.lib().ada_verify_drafts_workspace_size(total_q, batch, vocab, N.DT_LOGITS[dtype]))


def verify_drafts(target_logits: torch.Tensor, input_ids: torch.Tensor, cu_seqlens_q: torch.Tensor,
                  temperatures: torch.Tensor, uniforms: torch.Tensor, noise: torch.Tensor,
                  draft_logits: torch.Tensor | None = None, draft_lse: torch.Tensor | None = None,
                  workspace: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Accepts each sequence's drafted tokens up to the first refusal and draws the token after them.

    target_logits [N, V] (bf16/fp16/fp32): the target's logits of the rows input_ids int64 [N];
    cu_seqlens_q int32 [B + 1]: sequence b's rows are its last known token and then its drafts;
    temperatures fp32 [B] (<= 1e-10: greedy); uniforms fp32 [B, D] in [0, 1); noise fp32 [B, V]
    Exp(1); draft_logits [B, D, V] (target's dtype, any strides with unit stride in V) and
    draft_lse fp32 [B, D]: the logits each draft was drawn from and their log-normaliser at the
    sequence's temperature (``sample`` returns it); both None for drafts without a distribution.
    workspace: at least verify_workspace_bytes(...) bytes (default: allocated for the call).
    Returns (tokens int64 [B, D + 1], accepted int32 [B], logprobs fp32 [B, D + 1]): the accepted
    drafts and the drawn token with their log-probabilities under the target, then -1 and 0."""
    drafter = draft_logits is not None
    if not (target_logits.is_cuda and input_ids.is_cuda and cu_seqlens_q.is_cuda and temperatures.is_cuda
            and uniforms.is_cuda and noise.is_cuda):
        raise RuntimeError("verify_drafts requires CUDA tensors")
    (n, v), (b, most) = target_logits.shape, uniforms.shape
    dtype = target_logits.dtype
    code = N.DT_LOGITS.get(dtype)
    if code is None or noise.dtype is not F32 or uniforms.dtype is not F32 or noise.shape != (b, v):
        raise ValueError("target_logits must be bf16, fp16 or fp32, uniforms and noise [batch, vocab] fp32")
    target_logits, noise, uniforms = _unit(target_logits), _unit(noise), _unit(uniforms)
    temperatures = _dense(temperatures, "temperatures", F32, b)
    input_ids = _dense(input_ids, "input_ids", torch.int64, n)
    cu_seqlens_q = _dense(cu_seqlens_q, "cu_seqlens_q", torch.int32, b + 1)
    if drafter != (draft_lse is not None):
        raise ValueError("draft_logits and draft_lse come together")
    if drafter:
        if not (draft_logits.is_cuda and draft_lse.is_cuda):
            raise RuntimeError("verify_drafts requires CUDA tensors")
        if (draft_logits.dtype is not dtype or draft_logits.shape != (b, most, v) or draft_lse.shape != (b, most)
                or draft_lse.dtype is not F32):
            raise ValueError("draft_logits must be [batch, drafts, vocab] like the target's, draft_lse fp32 "
                             "[batch, drafts]")
        draft_logits = _unit(draft_logits)
        (db, dd, _), (lb, ld) = draft_logits.stride(), draft_lse.stride()
        draft, lse = draft_logits.data_ptr(), draft_lse.data_ptr()
    else:
        db = dd = lb = ld = 0
        draft = lse = None
    tokens = temperatures.new_empty((b, most + 1), dtype=torch.int64)
    logprobs = temperatures.new_empty((b, most + 1))
    accepted = cu_seqlens_q.new_empty(b)
    if b == 0:
        return tokens, accepted, logprobs
    device = target_logits.device
    stream = N.stream_ptr(device)
    if workspace is None:
        # one of its own: the launches of another thread's call on this stream may fall between this call's
        workspace = torch.empty(verify_workspace_bytes(n, b, v, dtype), dtype=torch.uint8, device=device)
    else:
        N.require_cuda(workspace, what="verify_drafts")
    # (a single row may have any stride)
    ld_u, ld_noise = (uniforms.stride(0), noise.stride(0)) if b > 1 else (most, v)
    st = N.lib().ada_verify_drafts(
        target_logits.data_ptr(), code, target_logits.stride(0) if n > 1 else v, n, v, input_ids.data_ptr(),
        cu_seqlens_q.data_ptr(), b, most, temperatures.data_ptr(), uniforms.data_ptr(), ld_u, noise.data_ptr(),
        ld_noise, draft, db, dd, lse, lb, ld, tokens.data_ptr(), accepted.data_ptr(), logprobs.data_ptr(),
        workspace.data_ptr(), workspace.nbytes, stream)
    if st:
        N.check(st, "draft verification kernel")
    return tokens, accepted, logprobs


class Sampler(nn.Module):
    """Drop-in for adallm.ops.sampler.Sampler: one token per row at its temperature (the reference
    refuses greedy rows; here a temperature of 0 takes the first maximum)."""

    def forward(self, logits: torch.Tensor, temperatures: torch.Tensor) -> torch.Tensor:
        noise = torch.empty(logits.shape, dtype=torch.float32, device=logits.device).exponential_(1.0)
        return sample(logits, temperatures.float(), noise)[0]
