"""The 4-bit paged KV cache, rotary layouts and step metadata in 64 bits (torch, any device).
Test infrastructure only.

Definitions of this package (the reference holds its cache in e4m3, adallm/ops/attention.py:11-31,
rotates whole heads in halves, adallm/ops/rotary_embedding.py:6-56, and builds a step's metadata with
host loops, adallm/runtime/model_runner.py:234-300):
  * a block of the cache: page rows of 64 bytes (e2m1, even element in the low nibble), then page rows
    of 8 e4m3 scales; value = code * scale * tensor scale
  * decode sees keys [max(ctx - W, 0), ctx); row i of t new tokens of a prefill sees keys
    [max(n - t + i - W, 0), n - t + i] of n; a row without keys gives zeros."""
from __future__ import annotations

import math

import torch

MAG = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def quantise(x: torch.Tensor):
    """codes uint8 [..., D] and e4m3 scales [..., D / 16] of fp32 values (already over the tensor's scale)."""
    b = x.float().double().unflatten(-1, (-1, 16))
    nan = b.isnan().any(-1)
    top = b.abs().amax(-1)
    scale = (top / 6).clamp(max=448.0).float().to(torch.float8_e4m3fn)
    s = scale.double()[..., None]
    mag = torch.tensor(MAG, dtype=torch.float64, device=x.device)
    y = torch.where(s > 0, (b.abs() / s).nan_to_num(0.0, posinf=1e9), torch.zeros_like(b)).contiguous()
    hi = torch.searchsorted(mag, y).clamp(1, 7)
    low, high = y - mag[hi - 1], mag[hi] - y
    code = torch.where((high < low) | ((high == low) & (hi % 2 == 0)), hi, hi - 1).to(torch.uint8)
    code = code | ((b < 0) & (code > 0)).to(torch.uint8) << 3
    bits = scale.view(torch.uint8)
    return code.flatten(-2), torch.where(nan, torch.full_like(bits, 0x7F), bits)


def pack(x: torch.Tensor):
    """Packed rows uint8 [..., 64] and scale bytes [..., 8] of [..., 128]."""
    code, scale = quantise(x)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def values(data: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp64 [..., 128] of packed rows and scale bytes."""
    lut = torch.tensor(MAG + tuple(-m for m in MAG), dtype=torch.float64, device=data.device)
    x = torch.stack((lut[(data & 15).long()], lut[(data >> 4).long()]), -1).flatten(-2)
    return x * scale.contiguous().view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)


def stored(x: torch.Tensor, scale: float = 1.0) -> torch.Tensor:
    """What the cache holds of rows x [..., 128] under a tensor scale, as fp64 values."""
    t = torch.tensor(scale, dtype=torch.float32, device=x.device)
    return values(*pack(x.float() / t)) * t.double()


def make_cache(pages: int, hkv: int, page: int, gen: torch.Generator, device="cpu", spread: float = 1.0):
    """A cache of quantised Gaussian rows."""
    data, scale = pack(spread * torch.randn((pages, hkv, page, 128), generator=gen, device=device))
    return torch.cat((data.flatten(2), scale.flatten(2)), 2)


def rows_of(cache: torch.Tensor, table: torch.Tensor, n: int):
    """fp64 [n, Hkv, 128] of one sequence, and whether each row is there (its page is in the cache)."""
    page = cache.shape[2] // 72
    pos = torch.arange(n, device=cache.device)
    col = pos // page
    there = col < table.shape[0]
    block = table[col.clamp(max=max(table.shape[0] - 1, 0))].long()
    there = there & (block >= 0) & (block < cache.shape[0])
    block = torch.where(there, block, torch.zeros_like(block))
    r = pos % page
    data = cache[:, :, :page * 64].unflatten(2, (page, 64)).transpose(1, 2)[block, r]
    scale = cache[:, :, page * 64:].unflatten(2, (page, 8)).transpose(1, 2)[block, r]
    return values(data, scale), there


def attention(q, k_cache, v_cache, block_tables, new, lens, scale, window=0, decode=False, k_scale=1.0, v_scale=1.0):
    """fp64 [sum(new), Hq, 128] and the elementwise error bound of the kernels (see ``bound``) without the output's
    own rounding; new / lens: new tokens and all keys of each sequence (host lists)."""
    outs, bounds, at = [], [], 0
    hkv = k_cache.shape[1]
    for b, (m, n) in enumerate(zip(new, lens)):
        if m == 0:
            continue
        qi = q[at:at + m].double()
        at += m
        hq, d = qi.shape[1], qi.shape[2]
        if n == 0:
            outs.append(torch.zeros_like(qi))
            bounds.append(torch.zeros_like(qi))
            continue
        k, there = rows_of(k_cache, block_tables[b], n)
        v, _ = rows_of(v_cache, block_tables[b], n)
        qi = qi.view(m, hkv, hq // hkv, d).permute(1, 2, 0, 3)
        kt = (k * k_scale).transpose(0, 1)[:, None].transpose(-1, -2)
        vt = (v * v_scale).transpose(0, 1)[:, None]
        x = torch.matmul(qi, kt) * scale
        last = n - m + torch.arange(m, device=q.device)[:, None]
        key = torch.arange(n, device=q.device)
        see = there & (key <= last)
        if window > 0:
            see = see & (key >= last - window + (1 if decode else 0))
        vis = torch.where(see.any(0)[:, None], vt, torch.zeros_like(vt))  # rows that nothing sees may hold NaN
        x = torch.where(see, x, torch.full_like(x, -math.inf))
        top = x.amax(-1, keepdim=True)
        e = torch.where(see, (x - torch.where(top > -math.inf, top, torch.zeros_like(top))).exp(), torch.zeros_like(x))
        total = e.sum(-1, keepdim=True)
        p = e / torch.where(total > 0, total, torch.ones_like(total))
        o = torch.matmul(p, vis)
        spread = torch.matmul(p, vis.abs())
        size = torch.where(see, torch.matmul(qi.abs(), kt.abs()) * scale, torch.zeros_like(x)).amax(-1, keepdim=True)
        err = bound(spread, size, n, vis.abs().amax(-2, keepdim=True))
        outs.append(o.permute(2, 0, 1, 3).reshape(m, hq, d))
        bounds.append(err.permute(2, 0, 1, 3).reshape(m, hq, d))
    return torch.cat(outs), torch.cat(bounds)


def bound(spread, size, keys, largest):
    """How far an output element may be from the exact one before it is rounded to its type.

    spread = sum p |v|, size = the row's largest scale * sum |q k|, largest = max |v|.
      * probabilities enter P.V in fp16: half a step 2^-11 of each, so 2^-11 spread; they are held times
        2^6 against the reference, so below fp16's normal range half of 2^-30 each, 2^-31 keys largest
      * a score is 128 products in 8 fp32 accumulations of 16: each at most 2^-23 of the partial sum, twice
        (truncation), 2^-19 size together; it moves p and the normaliser, 2 * 2^-19 size spread
      * the exponent's argument and exp2 (2^-22 each), fp32 sums of p and of P.V over the keys (2^-23 a step, at
        most keys / 16 steps in a row): (2^-20 + keys * 2^-26) spread."""
    return ((2.0 ** -11 + 2.0 ** -18 * size + 2.0 ** -20 + keys * 2.0 ** -26) * spread
            + keys * 2.0 ** -31 * largest)


def rotate(x, positions, inv_freq, interleaved=False, amplitude=1.0):
    """fp64 rotation of the first 2 * len(inv_freq) elements of x [T, heads, D]."""
    r = 2 * inv_freq.shape[0]
    a = positions.double()[:, None, None] * inv_freq.double()
    cos, sin = a.cos() * amplitude, a.sin() * amplitude
    part = x[..., :r].double()
    x1, x2 = (part[..., 0::2], part[..., 1::2]) if interleaved else part.chunk(2, -1)
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    y = torch.stack((y1, y2), -1).flatten(-2) if interleaved else torch.cat((y1, y2), -1)
    return torch.cat((y, x[..., r:].double()), -1)


def step_metadata(cached, new, tables, free, start, page, tokens):
    """Host lists of what step_metadata writes: (positions, slots, cu_q, cu_k, context, next, tables, err)."""
    tables = [list(t) for t in tables]
    width = len(tables[0]) if tables else 0
    pos, slots, cu_q, cu_k, context, err, at = [], [], [0], [0], [], 0, start
    for b, (c, n) in enumerate(zip(cached, new)):
        c, n = max(c, 0), max(n, 0)
        ids = {}
        for col in range(-(-c // page), -(-(c + n) // page)):
            if not 0 <= at < len(free):
                err |= 0x100
                if col < width:
                    tables[b][col] = -1
            elif col >= width:
                err |= 0x200
                ids[col] = -1
            else:
                tables[b][col] = ids[col] = free[at]
            at += 1
        for p in range(c, c + n):
            col = p // page
            owned = col < -(-c // page)
            block = (tables[b][col] if owned else ids.get(col, -1)) if col < width else -1
            if col >= width and len(pos) < tokens:
                err |= 0x200
            pos.append(p)
            slots.append(block * page + p % page if block >= 0 else -1)
        cu_q.append(cu_q[-1] + n)
        cu_k.append(cu_k[-1] + c + n)
        context.append(c + n)
    if cu_q[-1] > tokens:
        err |= 0x400
    pad = tokens - len(pos)
    pos, slots = (pos + [0] * pad)[:tokens], (slots + [-1] * pad)[:tokens]
    return pos, slots, cu_q, cu_k, context, max(min(at, len(free)), min(start, len(free))), tables, err
