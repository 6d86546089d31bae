"""Sampled, speculative decoding of several continuations of one prompt, on random weights.

    python examples/speculative_sampling.py [--sequences 8] [--drafts 4] [--steps 16]

One prompt is stored once in shared pages; every sequence continues it in pages of its own.  A
step drafts tokens with a bigram model (``sampler.sample``, which also gives the log-normaliser of
each draft's logits), runs the target on the last known token and the drafts of every sequence at
once (``store_kvcache``, ``shared_prefix_decode``), and accepts or replaces them
(``sampler.verify_drafts``).  Lengths and tokens stay on the device; nothing waits for the host
inside a step."""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from adallm_b200.attention import store_kvcache  # noqa: E402
from adallm_b200.sampler import sample, verify_drafts  # noqa: E402
from adallm_b200.shared_prefix import shared_prefix_decode  # noqa: E402

HEADS, KV_HEADS, HEAD_DIM, PAGE = 32, 8, 128, 16


class Target:
    """One attention layer between an embedding and a vocabulary projection."""

    def __init__(self, vocab: int, hidden: int, generator: torch.Generator, device):
        def weight(*shape):
            w = torch.randn(shape, generator=generator) * shape[-1] ** -0.5
            return w.to(torch.bfloat16).to(device)

        self.embed = hidden ** 0.5 * weight(vocab, hidden)
        self.wq, self.wk = weight(HEADS * HEAD_DIM, hidden), weight(KV_HEADS * HEAD_DIM, hidden)
        self.wv, self.wo = weight(KV_HEADS * HEAD_DIM, hidden), 4 * weight(hidden, HEADS * HEAD_DIM)
        self.head = 3 * weight(vocab, hidden)

    def qkv(self, ids: torch.Tensor):
        x = self.embed[ids]
        n = ids.shape[0]
        return (x, (x @ self.wq.t()).view(n, HEADS, HEAD_DIM), (x @ self.wk.t()).view(n, KV_HEADS, HEAD_DIM),
                (x @ self.wv.t()).view(n, KV_HEADS, HEAD_DIM))

    def logits(self, x: torch.Tensor, attended: torch.Tensor) -> torch.Tensor:
        return (x + attended.view(x.shape[0], -1) @ self.wo.t()) @ self.head.t()


class Session:
    """The continuations of one prompt: caches, page tables and the tokens known so far."""

    def __init__(self, target: Target, bigram: torch.Tensor, prompt: torch.Tensor, sequences: int, drafts: int,
                 temperatures: torch.Tensor, room: int, generator: torch.Generator):
        self.target, self.bigram, self.drafts, self.t = target, bigram, drafts, temperatures
        self.generator = generator  # on the device
        device = prompt.device
        i32 = dict(dtype=torch.int32, device=device)
        shared, own = -(-len(prompt) // PAGE), -(-room // PAGE)
        shape = (shared + sequences * own, PAGE, KV_HEADS, HEAD_DIM)
        self.k_cache = torch.zeros(shape, device=device).to(torch.float8_e4m3fn)
        self.v_cache = torch.zeros_like(self.k_cache)
        self.prefix_tables = torch.arange(shared, **i32)[None]
        self.block_tables = shared + torch.arange(sequences * own, **i32).view(sequences, own)
        # the prompt's last token is every sequence's first input; what is before it is the prefix
        self.prefix_lens = torch.tensor([len(prompt) - 1], **i32)
        _, _, k, v = target.qkv(prompt[:-1])
        store_kvcache(k, v, self.k_cache, self.v_cache, torch.arange(len(prompt) - 1, **i32))
        self.stored = torch.zeros(sequences, **i32)            # own keys whose tokens are final
        self.last = prompt[-1].repeat(sequences)
        self.cu_q = torch.arange(0, sequences * (drafts + 1) + 1, drafts + 1, **i32)

    def _exponential(self, *shape):
        return torch.empty(shape, device=self.last.device).exponential_(1.0, generator=self.generator)

    def step(self):
        """(tokens [B, drafts + 1] padded with -1, accepted [B], logprobs [B, drafts + 1])."""
        b, d, vocab = self.last.shape[0], self.drafts, self.bigram.shape[0]
        ids = torch.empty((b, d + 1), dtype=torch.int64, device=self.last.device)
        ids[:, 0] = self.last
        draft_logits = torch.empty((d, b, vocab), dtype=torch.bfloat16, device=self.last.device)
        draft_lse = torch.empty((d, b), device=self.last.device)
        for i in range(d):
            draft_logits[i] = self.bigram[ids[:, i]]
            ids[:, i + 1], _, draft_lse[i] = sample(draft_logits[i], self.t, self._exponential(b, vocab))
        x, q, k, v = self.target.qkv(ids.view(-1))
        place = self.stored[:, None].long() + torch.arange(d + 1, device=ids.device)
        slots = self.block_tables.gather(1, place // PAGE) * PAGE + place % PAGE
        store_kvcache(k, v, self.k_cache, self.v_cache, slots.view(-1).to(torch.int32))
        out = shared_prefix_decode(q, self.k_cache, self.v_cache, self.prefix_tables, self.prefix_lens, None,
                                   self.block_tables, self.stored + d + 1, HEAD_DIM ** -0.5, cu_seqlens_q=self.cu_q)
        logits = self.target.logits(x, out)
        tokens, accepted, logprobs = verify_drafts(
            logits, ids.view(-1), self.cu_q, self.t, torch.rand((b, d), device=ids.device, generator=self.generator),
            self._exponential(b, vocab), draft_logits=draft_logits.transpose(0, 1), draft_lse=draft_lse.t())
        # the last known token and the accepted drafts are stored; the rest is overwritten by the next step
        self.stored += accepted + 1
        self.last = tokens.gather(1, accepted[:, None].long())[:, 0]
        return tokens, accepted, logprobs


def make(vocab=4096, hidden=256, prompt_len=600, sequences=8, drafts=4, steps=16, temperature=0.8, seed=0,
         device="cuda"):
    g = torch.Generator().manual_seed(seed)
    target = Target(vocab, hidden, g, device)
    # the drafter: the target's own next-token logits without attention
    bigram = (target.embed.float() @ target.head.float().t()).to(torch.bfloat16)
    prompt = torch.randint(0, vocab, (prompt_len,), generator=g).to(device)
    on_device = torch.Generator(device=device).manual_seed(seed)
    t = torch.full((sequences,), float(temperature), device=device)
    return Session(target, bigram, prompt, sequences, drafts, t, steps * (drafts + 1) + 1, on_device), prompt


def main():
    p = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    p.add_argument("--sequences", type=int, default=8)
    p.add_argument("--drafts", type=int, default=4)
    p.add_argument("--steps", type=int, default=16)
    p.add_argument("--temperature", type=float, default=0.8)
    a = p.parse_args()
    session, _ = make(sequences=a.sequences, drafts=a.drafts, steps=a.steps, temperature=a.temperature)
    results = [session.step() for _ in range(a.steps)]
    tokens = torch.cat([t for t, _, _ in results], 1).cpu()
    accepted = torch.stack([n for _, n, _ in results]).float().mean().item()
    for b in range(a.sequences):
        print(b, tokens[b][tokens[b] >= 0].tolist())
    print(f"{accepted:.2f} of {a.drafts} drafts accepted a step")


if __name__ == "__main__":
    main()
