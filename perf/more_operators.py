"""Measured cases of a serving step over a KV cache held in 4 bits: the step's metadata built on
the GPU, rotary positions (half or interleaved pairs, a part of the head, scaled for long
contexts), the 4-bit store with the rotation in front of it, and decode and prefill attention.

``run`` computes each operator in plain torch in 32 bits, or (``own``) through
``adallm_b200.step_metadata``, ``adallm_b200.rotary_embedding`` and ``adallm_b200.kvcache_fp4``.

The cache: uint8 [pages, KV heads, page * 72]; a block holds the page's rows of one head as 64
bytes of e2m1 pairs (even element in the low nibble), then the rows' 8 e4m3 scales, one for 16
elements.  A value is code * scale * the tensor's scale."""
import math
import random

import torch

own = False

HEAD_DIM = 128
FLOATS = {"bf16": torch.bfloat16, "f16": torch.float16}
MAGNITUDES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def listed():
    return [
        # one decode step of 16 requests: the latency of a call
        dict(name="meta_step", op="meta", requests=16, decoding=1.0, chunk=1, cached_hi=8192, page=16, shape_seed=1),
        # a step of 600 requests, most decoding, the others with a chunk of their prompt
        dict(name="meta_mixed", op="meta", requests=600, decoding=0.9, chunk=2048, cached_hi=16384, page=16,
             shape_seed=2),
        # a decode step of 16 tokens with the dense engine's heads, far into a YaRN-scaled context
        dict(name="rope_step", op="rope", tokens=16, heads=32, kv_heads=8, rotary=128, interleaved=False,
             scaling="yarn", factor=4.0, reach=131072, dtype="bf16"),
        # a prompt of 16K tokens, interleaved pairs in half of each head
        dict(name="rope_prompt", op="rope", tokens=16381, heads=32, kv_heads=8, rotary=64, interleaved=True,
             scaling="none", factor=1.0, reach=32768, dtype="f16"),
        # the new rows of a decode batch written to the cache, three of them padding
        dict(name="append_step", op="append", tokens=16, padded=3, heads=32, kv_heads=8, rotary=128, interleaved=False,
             scaling="yarn", factor=4.0, reach=131072, page=16, k_scale=1.0, v_scale=1.0, dtype="bf16"),
        # a prompt written to the cache, sixteen KV heads, tensor scales
        dict(name="append_prompt", op="append", tokens=8195, padded=0, heads=32, kv_heads=16, rotary=128,
             interleaved=False, scaling="linear", factor=8.0, reach=131072, page=64, k_scale=0.37, v_scale=0.05,
             dtype="bf16"),
        # one user's next token
        dict(name="decode_one", op="decode", batch=1, ctx_lo=700, ctx_hi=700, heads=32, kv_heads=8, page=16, window=0,
             dtype="bf16", shape_seed=7),
        # a batch of 16 chats
        dict(name="decode_batch", op="decode", batch=16, ctx_lo=512, ctx_hi=8192, heads=32, kv_heads=8, page=16,
             window=0, dtype="bf16", shape_seed=8),
        # a sliding-window layer, two heads a KV head, contexts that end inside a page
        dict(name="decode_window", op="decode", batch=4, ctx_lo=4096, ctx_hi=16384, heads=32, kv_heads=16, page=256,
             window=1024, dtype="f16", shape_seed=9),
        # 32 long contexts
        dict(name="decode_long", op="decode", batch=32, ctx_lo=32767, ctx_hi=32767, heads=32, kv_heads=8, page=16,
             window=0, dtype="bf16", shape_seed=10),
        # chunks of 2,048 prompt tokens behind 2,048 cached ones
        dict(name="prefill_chunk", op="prefill", batch=4, cached_lo=2048, cached_hi=2048, new_lo=2048, new_hi=2048,
             heads=32, kv_heads=8, page=16, window=0, dtype="bf16", shape_seed=11),
        # ragged prompts and prefixes, a window
        dict(name="prefill_odd", op="prefill", batch=7, cached_lo=0, cached_hi=1500, new_lo=1, new_hi=700, heads=32,
             kv_heads=16, page=64, window=1024, dtype="f16", shape_seed=12),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    seed = rng.randrange(1 << 30)
    op = rng.choice(("meta", "rope", "append", "decode", "decode", "prefill", "prefill"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    if op == "meta":
        requests = _log_uniform(rng, 1, 2048)
        return dict(op=op, requests=requests, decoding=rng.choice((0.0, 0.5, 0.9, 1.0)),
                    chunk=_log_uniform(rng, 1, max(1, min(4096, 65536 // requests))),
                    cached_hi=_log_uniform(rng, 1, 16384), page=rng.choice((16, 32, 64, 256)), shape_seed=seed)
    if op in ("rope", "append"):
        scaling = rng.choice(("none", "linear", "yarn"))
        heads, kv_heads = rng.choice(((32, 8), (32, 16), (32, 4), (8, 8), (16, 2)))
        c = dict(op=op, tokens=_log_uniform(rng, 1, 8195), heads=heads, kv_heads=kv_heads,
                 rotary=rng.choice((128, 128, 64, 32)), interleaved=rng.random() < 0.5, scaling=scaling,
                 factor=1.0 if scaling == "none" else rng.choice((2.0, 4.0, 8.0)), reach=rng.choice((16384, 131072)),
                 dtype=dtype, shape_seed=seed)
        if op == "append":
            c.update(padded=rng.choice((0, 0, 1)) * rng.randint(0, c["tokens"] // 2), page=rng.choice((16, 32, 64, 256)),
                     k_scale=rng.choice((1.0, 0.37, 2.0)), v_scale=rng.choice((1.0, 0.05)))
        return c
    heads, kv_heads = rng.choice(((32, 8), (32, 8), (32, 16), (32, 4), (8, 8), (16, 2)))
    c = dict(op=op, heads=heads, kv_heads=kv_heads, page=rng.choice((16, 32, 64, 256)),
             window=rng.choice((0, 0, 0, 100, 1024)), dtype=dtype, shape_seed=seed)
    if op == "decode":
        batch = _log_uniform(rng, 1, 64)
        hi = _log_uniform(rng, 1, 32768 if batch <= 16 else 32768 * 16 // batch)
        c.update(batch=batch, ctx_lo=max(1, int(hi * rng.uniform(0.1, 1.0))), ctx_hi=hi)
        return c
    batch = _log_uniform(rng, 1, 16)
    new_hi = _log_uniform(rng, 1, 4096 // batch)
    cached_hi = _log_uniform(rng, 1, 8192 // batch)
    c.update(batch=batch, cached_lo=int(cached_hi * rng.uniform(0.0, 1.0)), cached_hi=cached_hi,
             new_lo=max(1, int(new_hi * rng.uniform(0.1, 1.0))), new_hi=new_hi)
    return c


# ---- lengths of a case, on the host ----
def _requests(c):
    """(cached, new) lengths of a step's requests: decoding ones have one new token."""
    r = random.Random(c["shape_seed"])
    cached, new = [], []
    for _ in range(c["requests"]):
        decoding = r.random() < c["decoding"]
        new.append(1 if decoding else _log_uniform(r, 1, c["chunk"]))
        cached.append(r.randint(1 if decoding else 0, c["cached_hi"]))
    return cached, new


def _lens(c):
    r = random.Random(c["shape_seed"])
    if c["op"] == "decode":
        return [r.randint(c["ctx_lo"], c["ctx_hi"]) - 1 for _ in range(c["batch"])], [1] * c["batch"]
    cached = [r.randint(c["cached_lo"], c["cached_hi"]) for _ in range(c["batch"])]
    return cached, [r.randint(c["new_lo"], c["new_hi"]) for _ in range(c["batch"])]


def _sum(lens):
    total = [0]
    for n in lens:
        total.append(total[-1] + n)
    return total


def _capacity(new):
    """Tokens a step is laid out for: the next multiple of 64."""
    return max(64, -(-sum(new) // 64) * 64)


# ---- inputs ----
def _page_tables(pages, width, gen):
    """Pages of each sequence, scattered over a pool; -1 behind them.  Also the pages left over."""
    need = sum(pages)
    ids = torch.randperm(need + 5, generator=gen, device="cuda").to(torch.int32)
    tables = torch.full((len(pages), width), -1, dtype=torch.int32, device="cuda")
    first = torch.tensor(_sum(pages)[:-1], device="cuda")
    col = torch.arange(width, device="cuda")
    used = col < torch.tensor(pages, device="cuda")[:, None]
    tables[used] = ids[(first[:, None] + col)[used]]
    return tables, ids[need:], need + 5


def _quantise(x):
    """e2m1 codes (as bytes of two) and e4m3 scales of blocks of 16; fp32 quotients, ties to even."""
    b = x.float().unflatten(-1, (-1, 16))
    top = b.abs().amax(-1)
    scale = (top / torch.full_like(top, 6.0)).clamp(max=448.0).to(torch.float8_e4m3fn)
    s = scale.float()[..., None]
    y = torch.where(s > 0, b.abs() / s, torch.zeros_like(b))
    code = torch.zeros_like(y, dtype=torch.uint8)
    for limit, up in ((0.25, False), (0.75, True), (1.25, False), (1.75, True), (2.5, False), (3.5, True),
                      (5.0, False)):
        code += (y >= limit) if up else (y > limit)
    code |= (torch.signbit(b) & (s > 0)).to(torch.uint8) << 3
    code = code.flatten(-2)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale.view(torch.uint8)


def _random_cache(pool, c, gen):
    """A pool of quantised Gaussian rows."""
    page, hkv = c["page"], c["kv_heads"]
    cache = torch.empty((pool, hkv, page * 72), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (hkv * page * HEAD_DIM))
    for at in range(0, pool, step):
        n = min(step, pool - at)
        data, scale = _quantise(torch.randn((n, hkv, page, HEAD_DIM), generator=gen, device="cuda"))
        cache[at:at + n, :, :page * 64] = data.flatten(2)
        cache[at:at + n, :, page * 64:] = scale.flatten(2)
    return cache


def _spoil_tails(cache, tables, lens, page):
    """Rows behind a sequence's last one hold whatever was there before: here NaN."""
    for b, n in enumerate(lens):
        if n % page:
            block = cache[tables[b, n // page].long()]
            block[:, (n % page) * 64:page * 64] = 0xFF
            block[:, page * 64 + (n % page) * 8:] = 0x7F


def _prepare_meta(c, gen):
    cached, new = _requests(c)
    page = c["page"]
    before = [-(-n // page) for n in cached]
    after = [-(-(n + m) // page) for n, m in zip(cached, new)]
    tables, _, pool = _page_tables(before, max(after) + 3, gen)
    take = sum(after) - sum(before)
    free = pool + torch.randperm(take + 9, generator=gen, device="cuda").to(torch.int32)
    i32 = dict(dtype=torch.int32, device="cuda")
    n, tokens = len(cached), _capacity(new)
    out = (torch.empty(tokens, dtype=torch.int64, device="cuda"), torch.empty(tokens, **i32),
           torch.empty(n + 1, **i32), torch.empty(n + 1, **i32), torch.empty(n, **i32), torch.empty(1, **i32))
    return dict(op="meta", cached=torch.tensor(cached, **i32), new=torch.tensor(new, **i32), tables=tables, free=free,
                start=torch.full((1,), 4, **i32), page=page, tokens=tokens, out=out)


def _angles(c, dtype=torch.float64):
    """Angle of each pair of the rotated part per position step, and the table's amplitude."""
    half = c["rotary"] // 2
    i = torch.arange(half, dtype=dtype, device="cuda")
    base, factor = 1e6, c["factor"]
    inv = base ** (-i / half)
    if c["scaling"] == "linear":
        return inv / factor, 1.0
    if c["scaling"] == "none":
        return inv, 1.0
    trained = c["reach"] / factor

    def pair(turns):  # the pair that makes so many turns over the trained length
        return half * math.log(trained / (turns * 2 * math.pi)) / math.log(base)

    low, high = max(math.floor(pair(32.0)), 0), min(math.ceil(pair(1.0)), 2 * half - 1)
    ramp = ((i - low) / max(high - low, 0.001)).clamp(0, 1)
    return inv / factor * ramp + inv * (1 - ramp), 0.1 * math.log(factor) + 1.0


def _prepare_rope(c, gen):
    n, d = c["tokens"], "cuda"
    inv, amplitude = _angles(c)
    a = torch.arange(c["reach"], dtype=torch.float64, device=d)[:, None] * inv
    table = torch.cat((a.cos() * amplitude, a.sin() * amplitude), -1).float()
    dtype = FLOATS[c["dtype"]]
    first = torch.randint(0, c["reach"] - n + 1, (1,), generator=gen, device=d)
    if n <= 64:  # the newest tokens of as many sequences
        positions = torch.randint(0, c["reach"], (n,), generator=gen, device=d)
    else:
        positions = first + torch.arange(n, device=d)

    def rows(heads, spread):
        return (spread * torch.randn((n, heads, HEAD_DIM), generator=gen, device=d)).to(dtype)

    s = dict(op=c["op"], positions=positions, q=rows(c["heads"], 1.5), k=rows(c["kv_heads"], 1.2), table=table,
             interleaved=c["interleaved"])
    s["q_out"] = torch.empty_like(s["q"])
    if c["op"] == "rope":
        s["k_out"] = torch.empty_like(s["k"])
        return s
    page = c["page"]
    s["v"] = rows(c["kv_heads"], 0.3)
    stored = n - c["padded"]
    pool = -(-stored // page) + 4
    pages = torch.randperm(pool, generator=gen, device=d)
    at = 5 + torch.arange(n, device=d)
    slots = (pages[(at // page).clamp(max=pool - 1)] * page + at % page).to(torch.int32)
    slots[stored:] = -1
    for name in ("k_cache", "v_cache"):
        s[name] = torch.zeros((pool, c["kv_heads"], page * 72), dtype=torch.uint8, device=d)
    s.update(slots=slots, k_scale=c["k_scale"], v_scale=c["v_scale"],
             k_div=torch.tensor(c["k_scale"], device=d), v_div=torch.tensor(c["v_scale"], device=d))
    return s


def _prepare_attn(c, gen):
    cached, new = _lens(c)
    lens = [a + b for a, b in zip(cached, new)]
    page = c["page"]
    pages = [-(-n // page) for n in lens]
    tables, _, pool = _page_tables(pages, max(pages) + 1, gen)
    k, v = _random_cache(pool, c, gen), _random_cache(pool, c, gen)
    for cache in (k, v):
        _spoil_tails(cache, tables, lens, page)
    n = sum(new)
    q = (1.5 * torch.randn((n, c["heads"], HEAD_DIM), generator=gen, device="cuda")).to(FLOATS[c["dtype"]])
    i32 = dict(dtype=torch.int32, device="cuda")
    return dict(op=c["op"], q=q, k=k, v=v, tables=tables, lens=torch.tensor(lens, **i32), page=page,
                cu_q=torch.tensor(_sum(new), **i32), cu_k=torch.tensor(_sum(lens), **i32), window=c["window"],
                scale=HEAD_DIM ** -0.5, most_new=max(new), most=max(lens), out=torch.empty_like(q))


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    if case["op"] == "meta":
        return _prepare_meta(case, gen)
    return (_prepare_rope if case["op"] in ("rope", "append") else _prepare_attn)(case, gen)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end ----
def _plain_meta(s):
    cached, new = s["cached"].long().clamp(min=0), s["new"].long().clamp(min=0)
    page, tables = s["page"], s["tables"]
    i32 = torch.int32
    zero = torch.zeros(1, dtype=torch.int64, device=new.device)
    cu_q = torch.cat((zero, new.cumsum(0)))
    context = cached + new
    before, after = (cached + page - 1) // page, (context + page - 1) // page
    taken = (after - before).cumsum(0)
    first = s["start"].long() + taken - (after - before)
    col = torch.arange(tables.shape[1], device=new.device)
    fresh = (col >= before[:, None]) & (col < after[:, None])
    at = (first[:, None] + col - before[:, None]).clamp(0, s["free"].shape[0] - 1)
    tables = torch.where(fresh, s["free"][at], tables)
    t = torch.arange(s["tokens"], device=new.device)
    b = torch.searchsorted(cu_q[1:], t, right=True).clamp(max=new.shape[0] - 1)
    there = t < cu_q[-1]
    pos = torch.where(there, cached[b] + t - cu_q[b], torch.zeros_like(t))
    block = tables[b, (pos // page).clamp(max=tables.shape[1] - 1)].long()
    slot = torch.where(there & (block >= 0), block * page + pos % page, torch.full_like(t, -1))
    return {"positions": pos, "slots": slot.to(i32), "cu_q": cu_q.to(i32),
            "cu_k": torch.cat((zero, context.cumsum(0))).to(i32), "context": context.to(i32),
            "next": (s["start"] + taken[-1:]).to(i32), "tables": tables}


def _rotated(x, s):
    """x [n, heads, 128] in fp32 with the first part of each head rotated."""
    table = s["table"][s["positions"]]
    half = table.shape[-1] // 2
    cos, sin = table[:, None, :half], table[:, None, half:]
    x = x.float()
    part = x[..., :2 * half]
    x1, x2 = (part[..., 0::2], part[..., 1::2]) if s["interleaved"] else (part[..., :half], part[..., half:])
    y1, y2 = x1 * cos - x2 * sin, x2 * cos + x1 * sin
    turned = torch.stack((y1, y2), -1).flatten(-2) if s["interleaved"] else torch.cat((y1, y2), -1)
    return torch.cat((turned, x[..., 2 * half:]), -1)


def _plain_rope(s):
    return {"q": _rotated(s["q"], s).to(s["q"].dtype), "k": _rotated(s["k"], s).to(s["k"].dtype)}


def _pairs(device):
    """The two values of each byte."""
    lut = torch.tensor(MAGNITUDES + tuple(-m for m in MAGNITUDES), device=device)
    byte = torch.arange(256, device=device)
    return torch.stack((lut[byte & 15], lut[byte >> 4]), -1)


def _values(data, scale):
    """fp32 [..., 128] of packed rows [..., 64] and their scales [..., 8]."""
    x = _pairs(data.device).index_select(0, data.reshape(-1).int()).view(data.shape[:-1] + (8, 16))
    return (x * scale.contiguous().view(torch.float8_e4m3fn).float()[..., None]).flatten(-2)


def _as_stored(x, div, slots):
    data, scale = _quantise(x.float() / div)
    y = _values(data, scale) * div
    return torch.where((slots >= 0)[:, None, None], y, torch.zeros_like(y)).to(x.dtype)


def _plain_append(s):
    q, k = _plain_rope(s).values()
    return {"q": q, "k": _as_stored(k, s["k_div"], s["slots"]), "v": _as_stored(s["v"], s["v_div"], s["slots"])}


def _rows(cache, s):
    """fp32 keys or values of every sequence, [B, most, KV heads, 128], zeros where there is none."""
    page = s["page"]
    pos = torch.arange(s["most"], device=cache.device)
    block = s["tables"][:, (pos // page).clamp(max=s["tables"].shape[1] - 1)].long()
    there = (pos < s["lens"][:, None]) & (block >= 0)
    block, row = block.clamp(min=0), pos % page
    data = cache[:, :, :page * 64].unflatten(2, (page, 64)).transpose(1, 2)[block, row]
    scale = cache[:, :, page * 64:].unflatten(2, (page, 8)).transpose(1, 2)[block, row]
    scale = torch.where(there[..., None, None], scale, torch.zeros_like(scale))
    return _values(data, scale), there


def _plain_attn(s):
    q, (n, hq, dim), hkv = s["q"], s["q"].shape, s["k"].shape[1]
    dev = q.device
    k, there = _rows(s["k"], s)
    v, _ = _rows(s["v"], s)
    cu = s["cu_q"].long()
    r = torch.arange(n, device=dev)
    seq = torch.searchsorted(cu, r, right=True) - 1
    place = r - cu[seq]
    batch, rows = k.shape[0], s["most_new"]
    wide = torch.zeros((batch, rows, hkv, hq // hkv, dim), device=dev)
    wide[seq, place] = q.float().view(n, hkv, hq // hkv, dim) * s["scale"]
    score = torch.matmul(wide.permute(0, 2, 3, 1, 4).reshape(batch, hkv, -1, dim), k.permute(0, 2, 3, 1))
    score = score.view(batch, hkv, hq // hkv, rows, -1)
    new = cu[1:] - cu[:-1]
    last = (s["lens"].long() - new)[:, None] + torch.arange(rows, device=dev)  # the newest key that a row sees
    key = torch.arange(s["most"], device=dev)
    see = there[:, None] & (key <= last[..., None])
    if s["window"] > 0:  # a decode step sees W keys, a prefill row W keys and its own
        see &= key > last[..., None] - s["window"] - int(s["op"] == "prefill")
    score.masked_fill_(~see[:, None, None], -math.inf)
    top = score.amax(-1, keepdim=True)
    score -= torch.where(top > -math.inf, top, torch.zeros_like(top))
    score.exp_()
    total = score.sum(-1, keepdim=True)
    score /= torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(score.view(batch, hkv, -1, s["most"]), v.transpose(1, 2))
    out = out.view(batch, hkv, hq // hkv, rows, dim).permute(0, 3, 1, 2, 4)[seq, place]
    return {"out": out.reshape(n, hq, dim).to(q.dtype)}


def run(state):
    s = state
    if not own:
        if s["op"] in ("decode", "prefill"):
            return _plain_attn(s)
        return {"meta": _plain_meta, "rope": _plain_rope, "append": _plain_append}[s["op"]](s)
    if s["op"] == "meta":
        from adallm_b200.step_metadata import step_metadata
        m = step_metadata(s["cached"], s["new"], s["tables"], s["free"], s["start"], s["page"], s["tokens"],
                          out=s["out"])
        return {"positions": m.positions, "slots": m.slot_mapping, "cu_q": m.cu_seqlens_q, "cu_k": m.cu_seqlens_k,
                "context": m.context_lens, "next": m.free_next, "tables": s["tables"]}
    if s["op"] == "rope":
        from adallm_b200.rotary_embedding import apply_rotary
        q, k = apply_rotary(s["positions"], s["q"], s["k"], s["table"], s["interleaved"], q_out=s["q_out"],
                            k_out=s["k_out"])
        return {"q": q, "k": k}
    from adallm_b200 import kvcache_fp4 as kv
    if s["op"] == "append":
        q = kv.rotary_store_kvcache_fp4(s["positions"], s["q"], s["k"], s["v"], s["table"], s["k_cache"], s["v_cache"],
                                        s["slots"], s["interleaved"], s["k_scale"], s["v_scale"], q_out=s["q_out"])
        k, v = kv.read_kvcache_fp4(s["k_cache"], s["v_cache"], s["slots"], s["q"].dtype, s["k_scale"], s["v_scale"])
        return {"q": q, "k": k, "v": v}
    if s["op"] == "decode":
        return {"out": kv.paged_decode_fp4(s["q"], s["k"], s["v"], s["tables"], s["lens"], s["scale"], s["window"],
                                           out=s["out"])}
    return {"out": kv.paged_prefill_fp4(s["q"], s["k"], s["v"], s["tables"], s["cu_q"], s["cu_k"], s["most_new"],
                                        s["scale"], s["window"], out=s["out"])}


def work(case):
    c = case
    if c["op"] == "meta":
        cached, new = _requests(c)
        page = c["page"]
        taken = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(cached, new))
        return {"bytes": 8 * len(new) + 12 * _capacity(new) + 12 * (len(new) + 1) + 8 * taken,
                "flops": 4 * _capacity(new)}
    if c["op"] in ("rope", "append"):
        n, d, hq, hkv = c["tokens"], HEAD_DIM, c["heads"], c["kv_heads"]
        rope = {"bytes": n * (8 + 4 * c["rotary"] + 4 * d * (hq + hkv)), "flops": 3 * n * (hq + hkv) * c["rotary"]}
        if c["op"] == "rope":
            return rope
        # q through; k and v read, packed, and read back as values
        row = 2 * d + 72 + 72 + 2 * d
        return {"bytes": n * (16 + 4 * c["rotary"] + 4 * d * hq + 2 * hkv * row),
                "flops": rope["flops"] + 8 * n * 2 * hkv * d}
    cached, new = _lens(c)
    keys = pairs = 0
    for a, m in zip(cached, new):
        w = c["window"] + (c["op"] == "prefill") if c["window"] else 1 << 40
        keys += a + m - max(0, a + 1 - w)
        pairs += sum(min(a + i + 1, w) for i in range(m))
    n = sum(new)
    return {"bytes": keys * c["kv_heads"] * 144 + 4 * n * c["heads"] * HEAD_DIM,
            "flops": 4 * HEAD_DIM * c["heads"] * pairs}


# ---- the definitions in 64 bits ----
def _exact_rotate(x, c, positions):
    inv, amplitude = _angles(c)
    a = positions.double()[:, None, None] * inv
    z = torch.polar(torch.full_like(a, amplitude), a)
    part = x[..., :c["rotary"]].double()
    if c["interleaved"]:
        y = torch.view_as_real(torch.view_as_complex(part.unflatten(-1, (-1, 2)).contiguous()) * z).flatten(-2)
    else:
        y = torch.complex(*part.contiguous().chunk(2, -1)) * z
        y = torch.cat((y.real, y.imag), -1)
    return torch.cat((y, x[..., c["rotary"]:].double()), -1)


def _exact_stored(x, scale, slots):
    mag = torch.tensor(MAGNITUDES, dtype=torch.float64, device="cuda")
    scale = torch.tensor(scale, device="cuda")
    b = (x.float() / scale).double().unflatten(-1, (-1, 16))  # what is packed is the 32-bit quotient
    s = (b.abs().amax(-1, keepdim=True) / 6).clamp(max=448).float().to(torch.float8_e4m3fn).double()
    y = (b.abs() / s).nan_to_num(0.0).contiguous()
    hi = torch.searchsorted(mag, y).clamp(1, 7)
    below, above = y - mag[hi - 1], mag[hi] - y
    code = torch.where((above < below) | ((above == below) & (hi % 2 == 0)), hi, hi - 1)
    out = (mag[code] * b.sign() * s).flatten(-2) * scale.double()
    return torch.where((slots >= 0)[:, None, None], out, torch.zeros_like(out))


def _exact_attn(c, s):
    page, hkv, out = c["page"], c["kv_heads"], []
    cu = s["cu_q"].tolist()
    for b, n in enumerate(s["lens"].tolist()):
        blocks = s["tables"][b, :-(-n // page)].long()
        wide = []
        for cache in (s["k"], s["v"]):
            part = cache[blocks]
            data = part[..., :page * 64].unflatten(-1, (page, 64)).transpose(1, 2).flatten(0, 1)[:n]
            scale = part[..., page * 64:].unflatten(-1, (page, 8)).transpose(1, 2).flatten(0, 1)[:n]
            code = torch.stack((data & 15, data >> 4), -1).flatten(-2)
            size, sign = (code & 7).double(), 1.0 - 2.0 * (code >> 3).double()
            size = torch.where(size < 2, size / 2, (1 + (code & 1).double() / 2) * 2.0 ** ((code & 7) // 2).double() / 2)
            scale = scale.contiguous().view(torch.float8_e4m3fn).double().repeat_interleave(16, -1)
            wide.append((sign * size * scale).transpose(0, 1))
        q = s["q"][cu[b]:cu[b + 1]].double()
        m = q.shape[0]
        q = q.view(m, hkv, -1, HEAD_DIM).permute(1, 2, 0, 3)
        x = torch.matmul(q, wide[0].transpose(1, 2)[:, None]) * s["scale"]
        last = n - m + torch.arange(m, device="cuda")[:, None]
        key = torch.arange(n, device="cuda")
        hide = key > last
        if c["window"]:
            hide |= key < last - c["window"] + int(c["op"] == "decode")
        x = torch.softmax(x.masked_fill_(hide, -math.inf), -1)
        out.append(torch.matmul(x, wide[1][:, None]).permute(2, 0, 1, 3).reshape(m, -1, HEAD_DIM))
    return {"out": torch.cat(out)}


def exact(case, seed):
    if case["op"] == "meta":
        return None
    s = prepare(case, seed)
    if case["op"] in ("decode", "prefill"):
        return _exact_attn(case, s)
    q, k = (_exact_rotate(s[x], case, s["positions"]) for x in ("q", "k"))
    if case["op"] == "rope":
        return {"q": q, "k": k}
    # the rows are rounded to the model's type before they are stored
    return {"q": q, "k": _exact_stored(k.to(s["k"].dtype), case["k_scale"], s["slots"]),
            "v": _exact_stored(s["v"], case["v_scale"], s["slots"])}
