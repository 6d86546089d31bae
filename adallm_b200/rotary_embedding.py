"""Rotary embedding on the B200 kernel (adallm_b200 C ABI ``ada_rope``).

Same constructor, cache and forward contract as the reference
(adallm/ops/rotary_embedding.py:17-90): an fp32 cos/sin cache
[max_position, 1, head_size] = [cos | sin] with optional linear scaling,
NeoX rotate-half applied in fp32 and cast back, new q / k returned.

``apply_rotary`` (``ada_rotary``) takes what the reference does not: interleaved pairs, a rotated part
of the head narrower than the head, strided heads.  ``build_cos_sin_cache`` also makes YaRN's table.
"""
from __future__ import annotations

import math
from functools import lru_cache

import torch
from torch import nn

from . import _native as N


_YARN_KEYS = {"rope_type", "type", "rope_theta", "factor", "original_max_position_embeddings", "beta_fast", "beta_slow",
              "attention_factor", "mscale", "mscale_all_dim", "truncate",
              "partial_rotary_factor"}  # (the table's width is an argument)


def _yarn_cos_sin_cache(rotary_dim: int, max_position: int, base: float, rope_scaling: dict, device=None):
    """YaRN (Peng et al. 2023): pairs that turn more than beta_fast times over the trained length keep their
    frequency, those below beta_slow turns are slowed by `factor`, a linear ramp lies between (its ends on whole
    pairs unless `truncate` is false); cos and sin are multiplied by the attention factor: 0.1 ln(factor) + 1, or with
    mscale m and mscale_all_dim n (0.1 m ln(factor) + 1) / (0.1 n ln(factor) + 1).  Angles in 64 bits, the table in
    fp32.  The table has factor x original_max_position_embeddings rows at least (where that is not given it is
    max_position / factor), as positions behind its last row are clamped to it.  Keys that would change the table in
    a way not known here are refused."""
    given = {k: v for k, v in rope_scaling.items() if v is not None}
    unknown = sorted(set(given) - _YARN_KEYS)
    if unknown:
        raise ValueError(f"yarn rope_scaling: unknown {', '.join(unknown)}")
    if float(given.get("rope_theta", base)) != float(base):
        raise ValueError("yarn rope_scaling: rope_theta is not the table's base")
    if "factor" not in given:
        raise ValueError("yarn rope_scaling needs its factor")
    factor = float(given["factor"])
    if not 0.0 < factor < math.inf:
        raise ValueError("yarn rope_scaling: factor must be positive")
    trained = float(given.get("original_max_position_embeddings", max_position / factor))
    fast, slow = float(given.get("beta_fast", 32.0)), float(given.get("beta_slow", 1.0))
    if not (0.0 < trained < math.inf and 0.0 < slow <= fast < math.inf):
        raise ValueError("yarn rope_scaling: original_max_position_embeddings must be positive, 0 < beta_slow <= beta_fast")
    scales = [k for k in ("attention_factor", "mscale", "mscale_all_dim") if k in given]
    if not all(0.0 < float(given[k]) < math.inf for k in scales):
        raise ValueError("yarn rope_scaling: attention_factor, mscale and mscale_all_dim must be positive")
    if ("mscale" in given) != ("mscale_all_dim" in given):
        raise ValueError("yarn rope_scaling: mscale and mscale_all_dim go together")  # (one alone is read in two ways)
    stretch = 0.1 * math.log(max(factor, 1.0))
    m, n = (stretch * float(given.get(k, d)) + 1.0 for k, d in (("mscale", 1.0), ("mscale_all_dim", 0.0)))
    amplitude = float(given.get("attention_factor", m / n))
    half = rotary_dim // 2

    def pair(turns):
        return half * math.log(trained / (turns * 2 * math.pi)) / math.log(base)

    low, high = pair(fast), pair(slow)
    if given.get("truncate", True):
        low, high = math.floor(low), math.ceil(high)
    low, high = max(low, 0), min(high, rotary_dim - 1)
    i = torch.arange(half, dtype=torch.float64, device=device)
    keep = 1.0 - ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    inv_freq = base ** (-i / half)
    inv_freq = inv_freq * keep + inv_freq / factor * (1.0 - keep)
    rows = max(max_position, math.ceil(factor * trained)) if "original_max_position_embeddings" in given else max_position
    angle = torch.arange(rows, dtype=torch.float64, device=device)[:, None] * inv_freq
    return (torch.cat((angle.cos(), angle.sin()), -1) * amplitude).float().unsqueeze_(1)


def build_cos_sin_cache(head_size: int, max_position: int, base: float, rope_scaling: dict | None = None,
                        device=None) -> torch.Tensor:
    """fp32 [max_position, 1, head_size]; same arithmetic as rotary_embedding.py:26-43.  A yarn table has
    factor x original_max_position_embeddings rows where that is more."""
    if rope_scaling is not None and rope_scaling.get("rope_type", rope_scaling.get("type")) == "yarn":
        return _yarn_cos_sin_cache(head_size, max_position, base, rope_scaling, device)
    inv_freq = 1.0 / (base ** (torch.arange(0, head_size, 2, dtype=torch.float) / head_size))
    t = torch.arange(max_position, dtype=torch.float)
    if rope_scaling is not None:
        rope_type = rope_scaling.get("rope_type", rope_scaling.get("type", "linear"))
        if rope_type != "linear":
            raise ValueError(f"Unsupported rope_scaling type: {rope_type}")
        t = t / float(rope_scaling.get("factor", 1.0))
    freqs = torch.einsum("i,j -> ij", t, inv_freq)
    cache = torch.cat((freqs.cos(), freqs.sin()), dim=-1).unsqueeze_(1)
    return cache if device is None else cache.to(device)


def _heads(x: torch.Tensor, positions: torch.Tensor, d: int) -> torch.Tensor:
    """x as [tokens, heads, d], the heads counted: without tokens there is nothing to infer them from."""
    t = positions.numel()
    if x.numel():
        return x.reshape(t, -1, d)
    return x.reshape(t, 0 if t else math.prod(x.shape[positions.dim():]) // d, d)


def apply_rope(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, cos_sin_cache: torch.Tensor,
               q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    N.require_cuda(positions, query, key, cos_sin_cache, what="rotary_embedding")
    if query.dtype not in N.DT or key.dtype != query.dtype:
        raise ValueError("rotary embedding expects bf16/fp16 q and k")
    d = cos_sin_cache.shape[-1]
    t = positions.numel()
    q3, k3 = _heads(query, positions, d), _heads(key, positions, d)
    if q3.stride(1) != d or k3.stride(1) != d or q3.stride(2) != 1 or k3.stride(2) != 1:
        q3, k3 = q3.contiguous(), k3.contiguous()
    if cos_sin_cache.dtype != torch.float32 or not cos_sin_cache.is_contiguous():
        raise ValueError("cos_sin_cache must be contiguous fp32")
    pos = positions if positions.dtype == torch.int64 else positions.to(torch.int64)
    qo = q_out if q_out is not None else torch.empty(q3.shape, dtype=query.dtype, device=query.device)
    ko = k_out if k_out is not None else torch.empty(k3.shape, dtype=key.dtype, device=key.device)
    st = N.lib().ada_rope(pos.data_ptr(), q3.data_ptr(), q3.stride(0), k3.data_ptr(), k3.stride(0), qo.data_ptr(),
                          ko.data_ptr(), t, q3.shape[1], k3.shape[1], d, cos_sin_cache.data_ptr(),
                          cos_sin_cache.shape[0], N.DT[query.dtype], N.stream_ptr(query.device))
    N.check(st, "rotary_embedding")
    return qo.view(query.shape), ko.view(key.shape)


def check_table(cos_sin_cache: torch.Tensor) -> None:
    shape = cos_sin_cache.shape
    if cos_sin_cache.dtype is not torch.float32 or not cos_sin_cache.is_contiguous():
        raise ValueError("cos_sin_cache must be contiguous fp32")
    if len(shape) < 2 or shape[0] * shape[-1] != cos_sin_cache.numel():
        raise ValueError("cos_sin_cache must be [max_position, (1,) rotated width]")


def apply_rotary(positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor, cos_sin_cache: torch.Tensor,
                 interleaved: bool = False, q_out: torch.Tensor | None = None, k_out: torch.Tensor | None = None):
    """Rotate the first r = cos_sin_cache.shape[-1] elements of each head; the others are copied.

    positions [T] (clamped to the table); query [T, Hq, D], key [T, Hkv, D] bf16/fp16, any strides over tokens and
    heads that are multiples of 8; cos_sin_cache fp32 [max_position, (1,) r] = [cos | sin] of r / 2 pairs.  Pairs are
    (i, i + r / 2), or (2i, 2i + 1) with interleaved.  Returns new contiguous tensors (q_out, k_out if given; no input may
    lie in them)."""
    device = N.one_device("rotary_embedding", query, positions, key, cos_sin_cache)
    dtype = query.dtype
    code = N.DT.get(dtype)
    if code is None or key.dtype is not dtype:
        raise ValueError("rotary embedding expects bf16/fp16 q and k")
    if query.dim() != 3 or key.dim() != 3:
        raise ValueError("query and key must be [tokens, heads, head size]")
    qs, ks = query.stride(), key.stride()
    if qs[2] != 1:
        query = query.contiguous()
        qs = query.stride()
    if ks[2] != 1:
        key = key.contiguous()
        ks = key.stride()
    t, hq, d = q_shape = query.shape
    tk, hk, dk = k_shape = key.shape
    if tk != t or positions.numel() != t or dk != d:
        raise ValueError("positions, query and key must describe the same tokens")
    check_table(cos_sin_cache)
    if positions.dtype is not torch.int64 or not positions.is_contiguous():
        positions = positions.to(torch.int64).contiguous()
    if q_out is None:
        q_out = query.new_empty(q_shape)
    elif q_out.shape != q_shape or q_out.dtype is not dtype or not q_out.is_contiguous() \
            or q_out.get_device() != device:
        raise ValueError("q_out must be contiguous with query's shape, type and device")
    if k_out is None:
        k_out = key.new_empty(k_shape)
    elif k_out.shape != k_shape or k_out.dtype is not dtype or not k_out.is_contiguous() \
            or k_out.get_device() != device:
        raise ValueError("k_out must be contiguous with key's shape, type and device")
    table = cos_sin_cache.shape
    st = N.rotary(device, positions.data_ptr(), query.data_ptr(), qs[0], qs[1], key.data_ptr(), ks[0], ks[1],
                  q_out.data_ptr(), k_out.data_ptr(), t, hq, hk, d, cos_sin_cache.data_ptr(), table[0], table[-1],
                  interleaved, code, N.raw_stream(device))
    if st:
        N.check(st, "rotary_embedding")
    return q_out, k_out


class RotaryEmbedding(nn.Module):
    """Drop-in for adallm.ops.rotary_embedding.RotaryEmbedding; rotary_dim below head_size rotates a part of the
    head, interleaved pairs neighbours."""

    def __init__(self, head_size: int, rotary_dim: int, max_position_embeddings: int, base: float,
                 rope_scaling: dict | None = None, interleaved: bool = False) -> None:
        super().__init__()
        self.head_size = head_size
        self.rotary_dim = rotary_dim
        self.interleaved = interleaved
        assert rotary_dim <= head_size
        self.register_buffer("cos_sin_cache", build_cos_sin_cache(rotary_dim, max_position_embeddings, base,
                                                                  rope_scaling), persistent=False)

    def forward(self, positions: torch.Tensor, query: torch.Tensor, key: torch.Tensor):
        if self.rotary_dim == self.head_size and not self.interleaved:
            return apply_rope(positions, query, key, self.cos_sin_cache)
        d = self.head_size
        q, k = apply_rotary(positions, _heads(query, positions, d), _heads(key, positions, d), self.cos_sin_cache,
                            self.interleaved)
        return q.view(query.shape), k.view(key.shape)


@lru_cache(1)
def _get_rope_cached(head_size, rotary_dim, max_position, base, rope_scaling_key, interleaved):
    rope_scaling = dict(rope_scaling_key) if rope_scaling_key is not None else None
    return RotaryEmbedding(head_size, rotary_dim, max_position, base, rope_scaling=rope_scaling, interleaved=interleaved)


def get_rope(head_size: int, rotary_dim: int, max_position: int, base: float, rope_scaling: dict | None = None,
             interleaved: bool = False):
    key = None if rope_scaling is None else tuple(sorted(rope_scaling.items()))
    return _get_rope_cached(head_size, rotary_dim, max_position, base, key, bool(interleaved))
