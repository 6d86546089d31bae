"""Shared-prefix decode attention, sampling and draft verification from their definitions, in
64 bits on the CPU (no counterpart in the reference beyond adallm/ops/sampler.py:10-15)."""
from __future__ import annotations

import math

import numpy as np
import torch

NAN_BYTE = 0x7F  # e4m3 NaN: what rows past the last token of a page may hold


def _keys(cache: torch.Tensor, table, length: int):
    """Rows 0..length-1 of a page list as float64 [length, Hkv, D], and which of them exist."""
    page = cache.shape[1]
    out = torch.zeros((length,) + tuple(cache.shape[2:]), dtype=torch.float64)
    there = torch.zeros(length, dtype=torch.bool)
    for j in range(0, length, page):
        blk = int(table[j // page])
        if 0 <= blk < cache.shape[0]:
            n = min(page, length - j)
            out[j:j + n] = cache[blk, :n].double()
            there[j:j + n] = True
    return out, there


def shared_prefix_decode(q, k_cache, v_cache, prefix_tables, prefix_lens, cu_groups, block_tables, context_lens,
                         scale, cu_seqlens_q=None, window=0, k_scale=1.0, v_scale=1.0) -> torch.Tensor:
    """float64 [N, Hq, D]; CPU tensors (caches float8_e4m3fn), tables and lengths as the kernel takes them."""
    n, hq, d = q.shape
    hkv, page = k_cache.shape[2], k_cache.shape[1]
    groups, batch = len(prefix_lens), len(context_lens)
    cu_g = [0, batch] if cu_groups is None else [int(x) for x in cu_groups]
    cu_q = list(range(batch + 1)) if cu_seqlens_q is None else [int(x) for x in cu_seqlens_q]
    out = torch.zeros((n, hq, d), dtype=torch.float64)
    cached = {}
    for b in range(batch):
        g = next((i for i in range(groups) if cu_g[i] <= b < cu_g[i + 1]), None)
        if g not in cached:
            length = 0 if g is None else min(int(prefix_lens[g]), prefix_tables.shape[1] * page)
            table = [] if g is None else prefix_tables[g]
            cached[g] = _keys(k_cache, table, length) + _keys(v_cache, table, length)[:1]
        pk, pthere, pv = cached[g]
        own = min(int(context_lens[b]), block_tables.shape[1] * page)
        ok, othere = _keys(k_cache, block_tables[b], own)
        ov, _ = _keys(v_cache, block_tables[b], own)
        k, v, there = torch.cat((pk, ok)) * k_scale, torch.cat((pv, ov)) * v_scale, torch.cat((pthere, othere))
        t = cu_q[b + 1] - cu_q[b]
        for i in range(t):
            pos = len(k) - t + i
            j = torch.arange(len(k))
            see = there & (j <= pos)
            if window > 0:
                see &= j > pos - window
            if not bool(see.any()):
                continue
            qi = q[cu_q[b] + i].double().view(hkv, hq // hkv, d)
            s = torch.einsum("hgd,lhd->hgl", qi, k[see]) * scale
            out[cu_q[b] + i] = torch.einsum("hgl,lhd->hgd", torch.softmax(s, -1), v[see]).reshape(hq, d)
    return out


def make_shared_prefix_case(seed: int, prefix_lens, group_sizes, context_lens, rows, hq: int, hkv: int, page: int,
                            dtype=torch.bfloat16, d: int = 128, q_gain: float = 1.0, holes: int = 0) -> dict:
    """Random paged caches (unused rows hold NaN), shuffled pages, -1 padded tables."""
    g = torch.Generator().manual_seed(seed)
    lens = list(prefix_lens) + list(context_lens)
    pages = [-(-n // page) for n in lens]
    width = max(max(pages), 1) + 1
    pool = sum(pages) + 2
    order = torch.randperm(pool, generator=g).tolist()
    caches = [torch.full((pool, page, hkv, d), NAN_BYTE, dtype=torch.uint8) for _ in range(2)]
    tables = torch.full((len(lens), width), -1, dtype=torch.int32)
    at = 0
    for i, n in enumerate(lens):
        for j in range(pages[i]):
            blk = order[at]
            at += 1
            tables[i, j] = blk
            rows_here = min(page, n - j * page)
            for c in caches:
                c[blk, :rows_here] = torch.randn((rows_here, hkv, d), generator=g).to(
                    torch.float8_e4m3fn).view(torch.uint8)
    for _ in range(holes):  # block ids that name no page
        i = int(torch.randint(len(lens), (1,), generator=g))
        if pages[i]:
            tables[i, int(torch.randint(pages[i], (1,), generator=g))] = pool + 7
    q = (q_gain * torch.randn((sum(rows), hq, d), generator=g)).to(dtype)
    i32 = torch.int32
    ng = len(prefix_lens)
    return dict(q=q, k_cache=caches[0].view(torch.float8_e4m3fn), v_cache=caches[1].view(torch.float8_e4m3fn),
                prefix_tables=tables[:ng].contiguous(), prefix_lens=torch.tensor(list(prefix_lens), dtype=i32),
                cu_groups=torch.tensor([0] + np.cumsum(list(group_sizes)).tolist(), dtype=i32),
                block_tables=tables[ng:].contiguous(), context_lens=torch.tensor(list(context_lens), dtype=i32),
                cu_seqlens_q=torch.tensor([0] + np.cumsum(list(rows)).tolist(), dtype=i32), scale=d ** -0.5)


# ---- sampling -------------------------------------------------------------------------------
GREEDY = float(np.float32(1e-10))  # temperatures are fp32
FLOAT_MAX = float(np.finfo(np.float32).max)


def _z(logits, t: float) -> np.ndarray:
    x = np.asarray(logits, np.float64)
    x = np.where(np.isnan(x), -np.inf, np.minimum(x, FLOAT_MAX))
    with np.errstate(over="ignore"):
        return np.minimum(x / (t if t > GREEDY else 1.0), FLOAT_MAX)


def _lse(z: np.ndarray) -> float:
    top = z.max()
    return -math.inf if top == -math.inf else float(top + np.log(np.exp(z - top).sum()))


def _probs(z: np.ndarray) -> np.ndarray:
    top = z.max()
    if top == -math.inf:
        return np.zeros_like(z)
    e = np.exp(z - top)
    return e / e.sum()


def _race(w: np.ndarray, e) -> tuple[int, float]:
    """(winner or -1, how far the second best score is behind, relative)."""
    s = w / np.maximum(np.asarray(e, np.float64), np.float64(np.float32(1e-10)))
    k = int(s.argmax())
    if not s[k] > 0:
        return -1, 1.0
    rest = np.delete(s, k)
    return k, 1.0 - float(rest.max()) / float(s[k]) if rest.size else 1.0


def sample(logits, temperature: float, noise):
    """(token, logprob, lse, margin) of one row."""
    z = _z(logits, temperature)
    lse = _lse(z)
    if lse == -math.inf:
        return -1, 0.0, lse, 1.0
    k, margin = _race(_probs(z), noise) if temperature > GREEDY else (int(z.argmax()), 1.0)
    return k, float(z[k] - lse), lse, margin


def verify(target, ids, temperature: float, uniforms, noise, draft=None, draft_lse=None, max_drafts=None):
    """(tokens, accepted, logprobs, margin) of one sequence: target [rows, V], ids [rows]."""
    drafts = min(len(ids) - 1, len(uniforms) if max_drafts is None else max_drafts)
    greedy = not temperature > GREEDY
    tokens, logprobs, margin = [], [], 1.0
    for i in range(drafts + 1):
        z = _z(target[i], temperature)
        p, lse = _probs(z), _lse(z)
        q = np.zeros_like(p)
        if i < drafts:
            x = int(ids[i + 1])
            inside = 0 <= x < len(p)
            if draft is not None:
                q = np.exp(_z(draft[i], temperature) - float(draft_lse[i]))
            elif inside:
                q[x] = 1.0
            if greedy:
                ok = lse > -math.inf and x == int(z.argmax())
            else:
                ok = inside and float(uniforms[i]) * q[x] < p[x]
                if inside and p[x] > 0:
                    margin = min(margin, abs(float(uniforms[i]) * q[x] / p[x] - 1.0))
            if ok:
                tokens.append(x)
                logprobs.append(float(z[x] - lse))
                continue
        if greedy:
            k = int(z.argmax()) if lse > -math.inf else -1
        else:
            left = np.maximum(p - q, 0.0)
            if i < drafts and (p > 0).any():
                # p - q cancels where they are alike: whether anything is left at all
                margin = min(margin, float((np.abs(p - q)[p > 0] / p[p > 0]).max()))
            if not (left > 0).any():
                left = p
            k, far = _race(left, noise)
            # and the weight's error is relative to p
            margin = min(margin, far * (left[k] / p[k] if k >= 0 else 1.0))
        return tokens + [k], i, logprobs + [float(z[k] - lse) if k >= 0 else 0.0], margin
    raise AssertionError
