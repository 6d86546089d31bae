"""Measured cases of one step of sampled, speculative decoding over shared prompts: attention
that reads a prefix shared by several sequences once (FP8 paged cache), sampling at a
temperature, and the verification of drafted tokens.

``run`` computes each operator in plain torch in 32 bits, or (``own``) through
``adallm_b200.shared_prefix`` and ``adallm_b200.sampler``.
"""
import math
import random

import torch

own = False

HEAD_DIM = 128
FLOATS = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
VOCAB = 151936  # the Qwen3 vocabulary of this repository's decode workloads


def listed():
    return [
        # two continuations of one short prompt: the latency of a call
        dict(name="attn_two_short", op="attn", groups=1, samples=2, prefix_lo=96, prefix_hi=96, own_lo=1, own_hi=40,
             rows_lo=1, rows_hi=1, heads=32, kv_heads=8, page=16, window=0, dtype="bf16", shape_seed=1),
        # a system prompt in front of a batch of 16 chats, pages of 256 as the runtime's default
        dict(name="attn_system_prompt", op="attn", groups=1, samples=16, prefix_lo=2048, prefix_hi=2048, own_lo=1,
             own_hi=512, rows_lo=1, rows_hi=1, heads=32, kv_heads=8, page=256, window=0, dtype="bf16", shape_seed=2),
        # the same batch verifying up to four drafted tokens a sequence, prompt ending inside a page
        dict(name="attn_drafts_odd", op="attn", groups=1, samples=16, prefix_lo=8191, prefix_hi=8191, own_lo=5,
             own_hi=700, rows_lo=1, rows_hi=5, heads=32, kv_heads=8, page=16, window=0, dtype="f16", shape_seed=3),
        # eight samples of each of eight prompts, sliding-window layer with two heads a KV head
        dict(name="attn_samples_window", op="attn", groups=8, samples=8, prefix_lo=500, prefix_hi=4000, own_lo=1,
             own_hi=600, rows_lo=1, rows_hi=1, heads=32, kv_heads=16, page=16, window=1024, dtype="bf16", shape_seed=4),
        # 64 sequences behind one long document, three drafted tokens each
        dict(name="attn_long_document", op="attn", groups=1, samples=64, prefix_lo=32768, prefix_hi=32768, own_lo=256,
             own_hi=1024, rows_lo=4, rows_hi=4, heads=32, kv_heads=8, page=16, window=0, dtype="bf16", shape_seed=5),
        # one user's next token
        dict(name="sample_one", op="sample", rows=1, vocab=VOCAB, dtype="bf16", keep=1.0, greedy=0.0, pad=0,
             shape_seed=6),
        # a decode batch of 64, some of them greedy
        dict(name="sample_batch", op="sample", rows=64, vocab=VOCAB, dtype="bf16", keep=1.0, greedy=0.2, pad=0,
             shape_seed=7),
        # fp32 logits after a top-k filter (all but 1% masked), an odd vocabulary in padded rows
        dict(name="sample_filtered", op="sample", rows=33, vocab=32003, dtype="f32", keep=0.01, greedy=0.0, pad=13,
             shape_seed=8),
        # one sequence, four drafted tokens
        dict(name="verify_one", op="verify", batch=1, drafts_lo=4, drafts_hi=4, vocab=VOCAB, dtype="bf16", drafter=True,
             keep=1.0, greedy=0.0, shape_seed=9),
        # a serving batch with one to four drafted tokens a sequence, some of them greedy
        dict(name="verify_batch", op="verify", batch=64, drafts_lo=1, drafts_hi=4, vocab=VOCAB, dtype="bf16",
             drafter=True, keep=1.0, greedy=0.2, shape_seed=10),
        # drafts looked up in the prompt (no draft distribution), up to eight a sequence, some with none
        dict(name="verify_lookup", op="verify", batch=24, drafts_lo=0, drafts_hi=8, vocab=VOCAB, dtype="f16",
             drafter=False, keep=1.0, greedy=0.0, shape_seed=11),
        # fp32 logits after a top-k filter on both sides, odd vocabulary
        dict(name="verify_filtered", op="verify", batch=7, drafts_lo=2, drafts_hi=5, vocab=32003, dtype="f32",
             drafter=True, keep=0.02, greedy=0.0, shape_seed=12),
    ]


def _log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    seed = rng.randrange(1 << 30)
    op = rng.choice(("attn", "attn", "sample", "verify"))
    if op == "attn":
        groups = _log_uniform(rng, 1, 8)
        samples = _log_uniform(rng, 1, max(1, 64 // groups))
        rows_hi = rng.choice((1, 1, 2, 4, 5))
        prefix_hi = _log_uniform(rng, 16, 32768 // groups)
        own_hi = _log_uniform(rng, rows_hi, 1024)
        heads, kv_heads = rng.choice(((32, 8), (32, 8), (32, 16), (32, 4), (8, 8), (16, 2)))
        return dict(op=op, groups=groups, samples=samples, prefix_lo=max(1, int(prefix_hi * rng.uniform(0.3, 1.0))),
                    prefix_hi=prefix_hi, own_lo=rows_hi, own_hi=own_hi, rows_lo=rng.choice((1, rows_hi)),
                    rows_hi=rows_hi, heads=heads, kv_heads=kv_heads, page=rng.choice((16, 32, 256)),
                    window=rng.choice((0, 0, 0, 100, 1024)), dtype=rng.choice(("bf16", "bf16", "f16")),
                    shape_seed=seed)
    vocab = _log_uniform(rng, 1000, VOCAB)
    dtype = rng.choice(("bf16", "bf16", "f16", "f32"))
    keep = rng.choice((1.0, 1.0, 0.3, 0.02))
    greedy = rng.choice((0.0, 0.0, 0.3))
    if op == "sample":
        return dict(op=op, rows=_log_uniform(rng, 1, 64), vocab=vocab, dtype=dtype, keep=keep, greedy=greedy,
                    pad=rng.choice((0, 0, 1, 8)), shape_seed=seed)
    hi = rng.choice((1, 2, 3, 4, 8))
    return dict(op=op, batch=_log_uniform(rng, 1, 64 if hi <= 4 else 24), drafts_lo=rng.choice((0, 1)), drafts_hi=hi,
                vocab=vocab, dtype=dtype, drafter=rng.random() < 0.7, keep=keep, greedy=greedy, shape_seed=seed)


def _attn_lens(c):
    """Prefix length of each group, own length and query rows of each sequence."""
    r = random.Random(c["shape_seed"])
    prefix = [r.randint(c["prefix_lo"], c["prefix_hi"]) for _ in range(c["groups"])]
    n = c["groups"] * c["samples"]
    own_len = [r.randint(c["own_lo"], c["own_hi"]) for _ in range(n)]
    rows = [min(o, r.randint(c["rows_lo"], c["rows_hi"])) for o in own_len]
    return prefix, own_len, rows


def _draft_counts(c):
    r = random.Random(c["shape_seed"])
    return [r.randint(c["drafts_lo"], c["drafts_hi"]) for _ in range(c["batch"])]


def _sum(lens):
    total = [0]
    for n in lens:
        total.append(total[-1] + n)
    return total


def _prepare_attn(c, gen):
    d = "cuda"
    prefix, own_len, rows = _attn_lens(c)
    page, hkv = c["page"], c["kv_heads"]
    lens = prefix + own_len
    pages = [-(-n // page) for n in lens]
    need = sum(pages)
    pool = need + 3
    ids = torch.randperm(pool, generator=gen, device=d)[:need].to(torch.int32)
    tables = torch.full((len(lens), max(pages) + 1), -1, dtype=torch.int32, device=d)
    first = torch.tensor(_sum(pages)[:-1], device=d)
    count = torch.tensor(pages, device=d)
    col = torch.arange(tables.shape[1], device=d)
    used = col < count[:, None]
    tables[used] = ids[(first[:, None] + col)[used]]
    caches = []
    for _ in range(2):
        cache = torch.randn((pool, page, hkv, HEAD_DIM), generator=gen, device=d).to(torch.float8_e4m3fn)
        bits = cache.view(torch.uint8)
        # rows past a sequence's last token hold whatever was there before: here e4m3 NaN
        length = torch.tensor(lens, device=d)
        last = tables[torch.arange(len(lens), device=d), count - 1].long()
        left = length - (count - 1) * page
        stale = torch.arange(page, device=d) >= left[:, None]
        keep = bits[last].clone()
        keep[stale] = 0x7F
        bits[last] = keep
        caches.append(cache)
    n = sum(rows)
    q = (1.5 * torch.randn((n, c["heads"], HEAD_DIM), generator=gen, device=d)).to(FLOATS[c["dtype"]])
    i32 = dict(dtype=torch.int32, device=d)
    g = c["groups"]
    return dict(op="attn", q=q, k=caches[0], v=caches[1], prefix_tables=tables[:g], block_tables=tables[g:],
                prefix_lens=torch.tensor(prefix, **i32), context_lens=torch.tensor(own_len, **i32),
                cu_groups=torch.arange(0, g * c["samples"] + 1, c["samples"], **i32),
                cu_q=torch.tensor(_sum(rows), **i32), window=c["window"], scale=HEAD_DIM ** -0.5,
                most_prefix=max(prefix), most_own=max(own_len), most_rows=max(rows),
                most_group_rows=max(sum(rows[i * c["samples"]:(i + 1) * c["samples"]]) for i in range(g)))


def _temperatures(c, n, gen):
    t = 0.5 + torch.rand(n, generator=gen, device="cuda")
    return torch.where(torch.rand(n, generator=gen, device="cuda") < c["greedy"], torch.zeros_like(t), t)


def _exponential(shape, gen):
    return torch.empty(shape, device="cuda").exponential_(1.0, generator=gen)


def _filter(x, keep):
    """-inf outside the largest `keep` share of each row (a top-k filter)."""
    if keep >= 1.0:
        return x
    k = max(1, int(keep * x.shape[-1]))
    least = x.topk(k, dim=-1).values[..., -1:]
    return torch.where(x >= least, x, torch.full_like(x, -math.inf))


def _prepare_sample(c, gen):
    n, v = c["rows"], c["vocab"]
    full = 3.0 * torch.randn((n, v + c["pad"]), generator=gen, device="cuda")
    full[:, :v] = _filter(full[:, :v], c["keep"])
    noise = _exponential((n, v), gen)
    return dict(op="sample", logits=full.to(FLOATS[c["dtype"]])[:, :v], noise=noise, t=_temperatures(c, n, gen))


def _prepare_verify(c, gen):
    d = "cuda"
    counts = _draft_counts(c)
    b, most, v = c["batch"], max(1, c["drafts_hi"]), c["vocab"]
    cu = _sum([k + 1 for k in counts])
    cu_q = torch.tensor(cu, dtype=torch.int32, device=d)
    dtype = FLOATS[c["dtype"]]
    target = 3.0 * torch.randn((cu[-1], v), generator=gen, device=d)
    t = _temperatures(c, b, gen)
    row = (cu_q[:-1, None] + torch.arange(most, device=d)).clamp(max=cu[-1] - 1).long()
    # the drafter's logits: the target's, off by some noise
    draft = target[row] + 0.7 * torch.randn((b, most, v), generator=gen, device=d)
    target = _filter(target, c["keep"]).to(dtype)
    draft = _filter(draft, c["keep"]).to(dtype)
    z = draft.float() / torch.where(t > 0, t, torch.ones_like(t))[:, None, None]
    lse = torch.logsumexp(z, -1)
    drawn = torch.where((t > 0)[:, None], ((z - lse[..., None]).exp() / _exponential((b, most, v), gen)).argmax(-1),
                        z.argmax(-1))
    ids = torch.randint(0, v, (cu[-1],), generator=gen, device=d)
    at = torch.arange(most, device=d) < torch.tensor(counts, device=d)[:, None]
    ids[(cu_q[:-1, None] + 1 + torch.arange(most, device=d))[at].long()] = drawn[at]
    drafter = c["drafter"]
    return dict(op="verify", target=target, ids=ids, cu_q=cu_q, t=t, u=torch.rand((b, most), generator=gen, device=d),
                noise=_exponential((b, v), gen), draft=draft if drafter else None, lse=lse if drafter else None)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    return {"attn": _prepare_attn, "sample": _prepare_sample, "verify": _prepare_verify}[case["op"]](case, gen)


# ---- plain forms: elementary operations in 32 bits, rounded once at the end ----
def _gather(cache, tables, lens, most):
    page = cache.shape[1]
    pos = torch.arange(most, device=cache.device)
    block = tables[:, (pos // page).clamp(max=tables.shape[1] - 1)].long()
    there = (pos < lens[:, None]) & (block >= 0)
    rows = cache[block.clamp(min=0), pos % page].float()
    return torch.where(there[..., None, None], rows, torch.zeros_like(rows)), there


def _plain_attn(s):
    q, (n, hq, dim), hkv = s["q"].float(), s["q"].shape, s["k"].shape[2]
    dev = q.device
    cu_q, cu_g = s["cu_q"].long(), s["cu_groups"].long()
    r = torch.arange(n, device=dev)
    seq = torch.searchsorted(cu_q, r, right=True) - 1
    group = torch.searchsorted(cu_g, seq, right=True) - 1
    qr = q.view(n, hkv, hq // hkv, dim) * s["scale"]

    def part(tables, lens, most, owner, place, places):
        # the rows of each owner of pages side by side, scored against its keys, and back in order
        k, there = _gather(s["k"], tables, lens, most)
        v, _ = _gather(s["v"], tables, lens, most)
        padded = qr.new_zeros((lens.shape[0], places) + qr.shape[1:])
        padded[owner, place] = qr
        score = torch.einsum("orhgd,olhd->orhgl", padded, k)[owner, place]
        return score, v, there[owner], padded

    p_len, own_len = s["prefix_lens"].long()[group], s["context_lens"].long()[seq]
    place_g, place_s = r - cu_q[cu_g[group]], r - cu_q[seq]
    sp, vp, there_p, buf_p = part(s["prefix_tables"], s["prefix_lens"], s["most_prefix"], group, place_g,
                                  s["most_group_rows"])
    so, vo, there_o, buf_o = part(s["block_tables"], s["context_lens"], s["most_own"], seq, place_s, s["most_rows"])
    pos = (p_len + own_len - (cu_q[seq + 1] - r))[:, None]
    at_p = torch.arange(s["most_prefix"], device=dev)[None, :]
    at_o = p_len[:, None] + torch.arange(s["most_own"], device=dev)
    w = s["window"] if s["window"] > 0 else 1 << 30
    see_p = there_p & (at_p <= pos) & (at_p > pos - w)
    see_o = there_o & (at_o <= pos) & (at_o > pos - w)
    score = torch.cat((sp, so), -1).masked_fill_(~torch.cat((see_p, see_o), -1)[:, None, None, :], -math.inf)
    top = score.amax(-1, keepdim=True)
    e = (score - torch.where(top > -math.inf, top, torch.zeros_like(top))).exp()
    total = e.sum(-1, keepdim=True)
    e = e / torch.where(total > 0, total, torch.ones_like(total))
    wide_p = e.new_zeros(buf_p.shape[:-1] + (s["most_prefix"],))
    wide_p[group, place_g] = e[..., :s["most_prefix"]]
    wide_o = e.new_zeros(buf_o.shape[:-1] + (s["most_own"],))
    wide_o[seq, place_s] = e[..., s["most_prefix"]:]
    out = (torch.einsum("orhgl,olhd->orhgd", wide_p, vp)[group, place_g]
           + torch.einsum("orhgl,olhd->orhgd", wide_o, vo)[seq, place_s])
    return {"out": out.reshape(n, hq, dim).to(s["q"].dtype)}


def _softmax_parts(logits, t):
    z = logits.float() / torch.where(t > 0, t, torch.ones_like(t))
    top = z.amax(-1, keepdim=True)
    e = (z - top).exp()
    return z, top, e, e.sum(-1, keepdim=True)


def _plain_sample(s):
    t = s["t"][:, None]
    z, top, e, total = _softmax_parts(s["logits"], t)
    score = torch.where(t > 0, e / total / s["noise"], e)
    token = score.argmax(-1)
    lse = (top + total.log())[:, 0]
    return {"tokens": token, "logprobs": z.gather(1, token[:, None])[:, 0] - lse, "lse": lse}


def _plain_verify(s):
    b, most = s["u"].shape
    dev = s["u"].device
    cu = s["cu_q"].long()
    drafts = cu[1:] - cu[:-1] - 1
    place = torch.arange(most + 1, device=dev)
    rows = (cu[:-1, None] + place).clamp(max=s["target"].shape[0] - 1)
    t = s["t"][:, None, None]
    z, top, e, total = _softmax_parts(s["target"][rows], t)
    p = e / total
    x = s["ids"][(rows + 1).clamp(max=s["ids"].shape[0] - 1)[:, :most]]
    px = p[:, :most].gather(2, x[..., None])[..., 0]
    if s["draft"] is None:
        q = torch.zeros_like(p[:, :most]).scatter_(2, x[..., None], 1.0)
    else:
        q = (s["draft"].float() / torch.where(t > 0, t, torch.ones_like(t)) - s["lse"][..., None]).exp()
    qx = q.gather(2, x[..., None])[..., 0]
    greedy = s["t"][:, None] <= 0
    good = torch.where(greedy, x == z[:, :most].argmax(-1), s["u"] * qx < px) & (place[:most] < drafts[:, None])
    count = good.long().cumprod(1).sum(1)
    one = torch.arange(b, device=dev)
    pj = p[one, count]
    qj = torch.where((count < drafts)[:, None], q[one, count.clamp(max=most - 1)], torch.zeros_like(pj))
    left = (pj - qj).clamp(min=0)
    left = torch.where((left > 0).any(-1, keepdim=True), left, pj)
    score = torch.where(greedy, pj, left / s["noise"])
    last = score.argmax(-1)
    token = torch.where(place < count[:, None], torch.cat((x, x[:, :1]), 1), last[:, None])
    logprob = z.gather(2, token[..., None])[..., 0] - (top + total.log())[..., 0]
    written = place <= count[:, None]
    return {"tokens": torch.where(written, token, torch.full_like(token, -1)),
            "accepted": count.to(torch.int32),
            "logprobs": torch.where(written, logprob, torch.zeros_like(logprob))}


def run(state):
    s = state
    if not own:
        return {"attn": _plain_attn, "sample": _plain_sample, "verify": _plain_verify}[s["op"]](s)
    if s["op"] == "attn":
        from adallm_b200.shared_prefix import shared_prefix_decode
        return {"out": shared_prefix_decode(s["q"], s["k"], s["v"], s["prefix_tables"], s["prefix_lens"],
                                            s["cu_groups"], s["block_tables"], s["context_lens"], s["scale"],
                                            cu_seqlens_q=s["cu_q"], window=s["window"])}
    from adallm_b200 import sampler
    if s["op"] == "sample":
        tokens, logprobs, lse = sampler.sample(s["logits"], s["t"], s["noise"])
        return {"tokens": tokens, "logprobs": logprobs, "lse": lse}
    tokens, accepted, logprobs = sampler.verify_drafts(s["target"], s["ids"], s["cu_q"], s["t"], s["u"], s["noise"],
                                                       draft_logits=s["draft"], draft_lse=s["lse"])
    return {"tokens": tokens, "accepted": accepted, "logprobs": logprobs}


def work(case):
    c = case
    if c["op"] == "attn":
        prefix, own_len, rows = _attn_lens(c)
        w = c["window"] or 1 << 30
        pairs = keys = 0
        for g, p in enumerate(prefix):
            least = p  # first prefix key that any row of the group sees
            for b in range(g * c["samples"], (g + 1) * c["samples"]):
                low = own_len[b]
                for i in range(rows[b]):
                    pos = p + own_len[b] - rows[b] + i
                    lo = max(0, pos - w + 1)
                    pairs += pos + 1 - lo
                    least = min(least, lo)
                    low = min(low, max(0, lo - p))
                keys += own_len[b] - low
            keys += p - least
        n = sum(rows)
        return {"bytes": keys * c["kv_heads"] * HEAD_DIM * 2 + 4 * n * c["heads"] * HEAD_DIM,
                "flops": 4 * HEAD_DIM * c["heads"] * pairs}
    size = 4 if c["dtype"] == "f32" else 2
    if c["op"] == "sample":
        return {"bytes": c["rows"] * c["vocab"] * (size + 4), "flops": 5 * c["rows"] * c["vocab"]}
    rows = sum(_draft_counts(c)) + c["batch"]
    per = 4 + (size if c["drafter"] else 0)  # the noise and the draft's logits of the row that is drawn from
    return {"bytes": c["vocab"] * (rows * size + c["batch"] * per), "flops": 5 * c["vocab"] * (rows + c["batch"])}


# ---- the definitions in 64 bits ----
def _exact_attn(c, s):
    dim, page, w = HEAD_DIM, c["page"], c["window"] or 1 << 30
    prefix, own_len, rows = _attn_lens(c)
    out, at = [], 0
    for b, (mine, n) in enumerate(zip(own_len, rows)):
        g = b // c["samples"]
        length = prefix[g] + mine
        slots = torch.cat([s["prefix_tables"][g].repeat_interleave(page) * page
                           + torch.arange(page, device="cuda").repeat(s["prefix_tables"].shape[1]),
                           s["block_tables"][b].repeat_interleave(page) * page
                           + torch.arange(page, device="cuda").repeat(s["block_tables"].shape[1])])
        width = s["prefix_tables"].shape[1] * page
        take = torch.cat([slots[:prefix[g]], slots[width:width + mine]])
        k = s["k"].reshape(-1, c["kv_heads"], dim).view(torch.uint8)[take].view(torch.float8_e4m3fn).double()
        v = s["v"].reshape(-1, c["kv_heads"], dim).view(torch.uint8)[take].view(torch.float8_e4m3fn).double()
        for i in range(n):
            pos = length - n + i
            lo = max(0, pos - w + 1)
            qi = s["q"][at].double().view(c["kv_heads"], -1, dim)
            x = torch.matmul(qi, k[lo:pos + 1].permute(1, 2, 0)) * dim ** -0.5
            out.append(torch.matmul(torch.softmax(x, -1), v[lo:pos + 1].transpose(0, 1)).reshape(-1, dim))
            at += 1
    return {"out": torch.stack(out)}


def _exact_sample(s):
    rows = []
    for x, t in zip(s["logits"].double(), s["t"].double()):
        z = x / t if t > 0 else x
        rows.append((z, torch.logsumexp(z, 0), t))
    tokens = [int((z - torch.log(e.double())).argmax() if t > 0 else z.argmax())
              for (z, _, t), e in zip(rows, s["noise"])]
    return {"tokens": None, "logprobs": torch.stack([z[k] - lse for (z, lse, _), k in zip(rows, tokens)]),
            "lse": torch.stack([lse for _, lse, _ in rows])}


def _exact_verify(c, s):
    most = s["u"].shape[1]
    logprobs = torch.zeros((c["batch"], most + 1), dtype=torch.float64, device="cuda")
    at = 0
    for b, drafts in enumerate(_draft_counts(c)):
        t = s["t"][b].double()
        z = s["target"][at:at + drafts + 1].double() / (t if t > 0 else 1.0)
        logp = z - torch.logsumexp(z, -1, keepdim=True)
        for i in range(drafts + 1):
            if i < drafts:
                x = int(s["ids"][at + 1 + i])
                if s["draft"] is not None and t > 0:
                    q = (s["draft"][b, i].double() / t - s["lse"][b, i].double()).exp()
                else:
                    q = torch.zeros(c["vocab"], dtype=torch.float64, device="cuda")
                    q[x] = 1.0
                ok = x == int(z[i].argmax()) if t <= 0 else bool(s["u"][b, i].double() * q[x] < logp[i, x].exp())
                if ok:
                    logprobs[b, i] = logp[i, x]
                    continue
                left = (logp[i].exp() - q).clamp(min=0)
                left = left if bool((left > 0).any()) else logp[i].exp()
            else:
                left = logp[i].exp()
            k = int(z[i].argmax() if t <= 0 else (left / s["noise"][b].double()).argmax())
            logprobs[b, i] = logp[i, k]
            break
        at += drafts + 1
    return {"tokens": None, "accepted": None, "logprobs": logprobs}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attn":
        return _exact_attn(case, s)
    return _exact_sample(s) if case["op"] == "sample" else _exact_verify(case, s)
