"""Serving over a KV cache held in 4 bits, on random weights: prompts in chunks, then decode steps from a CUDA graph.

    python examples/long_context_fp4.py [--requests 8] [--prompt 3000] [--chunk 512] [--steps 32]

A step knows its requests' lengths on the device only: ``step_metadata`` extends the block tables from the free
list and gives positions and slots, ``rotary_store_kvcache_fp4`` rotates (a YaRN table, half of each head in
interleaved pairs) and packs the new rows, and ``paged_prefill_fp4`` or ``paged_decode_fp4`` attends.
The decode step is captured once and replayed: nothing in it waits for the host."""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from adallm_b200 import kvcache_fp4 as kv  # noqa: E402
from adallm_b200.rotary_embedding import build_cos_sin_cache  # noqa: E402
from adallm_b200.step_metadata import empty_step_metadata, step_metadata  # noqa: E402

HEADS, KV_HEADS, HEAD_DIM, PAGE, ROTARY = 32, 8, 128, 16, 64
YARN = {"rope_type": "yarn", "factor": 4.0, "original_max_position_embeddings": 2048}


class Layer:
    """One attention layer between an embedding and a vocabulary projection."""

    def __init__(self, vocab: int, hidden: int, generator: torch.Generator, device):
        def weight(*shape):
            w = torch.randn(shape, generator=generator) * shape[-1] ** -0.5
            return w.to(torch.bfloat16).to(device)

        self.embed = hidden ** 0.5 * weight(vocab, hidden)
        self.wqkv = weight((HEADS + 2 * KV_HEADS) * HEAD_DIM, hidden)
        self.wo, self.head = 4 * weight(hidden, HEADS * HEAD_DIM), 3 * weight(vocab, hidden)

    def qkv(self, ids: torch.Tensor):
        x = self.embed[ids]
        return x, *(x @ self.wqkv.t()).view(-1, HEADS + 2 * KV_HEADS, HEAD_DIM).split((HEADS, KV_HEADS, KV_HEADS), 1)

    def logits(self, x: torch.Tensor, attended: torch.Tensor) -> torch.Tensor:
        return (x + attended.reshape(x.shape[0], -1) @ self.wo.t()) @ self.head.t()


class Server:
    """A batch of requests: caches, page tables, the free list and the lengths, all on the device."""

    def __init__(self, layer: Layer, requests: int, room: int, device):
        self.layer, self.requests, self.device = layer, requests, device
        width = -(-room // PAGE)
        i32 = dict(dtype=torch.int32, device=device)
        self.k_cache, self.v_cache = kv.empty_kvcache_fp4(requests * width, KV_HEADS, PAGE, device)
        self.tables = torch.full((requests, width), -1, **i32)
        self.free = torch.randperm(requests * width, device=device).to(torch.int32)
        self.start, self.cached = torch.zeros(1, **i32), torch.zeros(requests, **i32)
        self.table = build_cos_sin_cache(ROTARY, width * PAGE, 1e6, YARN, device)
        self.err = torch.zeros(1, **i32)

    def step(self, ids: torch.Tensor, new_lens: torch.Tensor, most: int, out=None) -> torch.Tensor:
        """Logits of the step's rows, request after request; ``most``: new tokens of a request at most."""
        m = step_metadata(self.cached, new_lens, self.tables, self.free, self.start, PAGE, ids.shape[0], out=out,
                          err=self.err)
        x, q, k, v = self.layer.qkv(ids)
        q = kv.rotary_store_kvcache_fp4(m.positions, q, k, v, self.table, self.k_cache, self.v_cache, m.slot_mapping,
                                        interleaved=True)
        scale = HEAD_DIM ** -0.5
        if most == 1 and ids.shape[0] == self.requests:
            o = kv.paged_decode_fp4(q, self.k_cache, self.v_cache, self.tables, m.context_lens, scale)
        else:
            o = kv.paged_prefill_fp4(q, self.k_cache, self.v_cache, self.tables, m.cu_seqlens_q, m.cu_seqlens_k, most,
                                     scale, err=self.err)
        self.cached.copy_(m.context_lens)
        self.start.copy_(m.free_next)
        return self.layer.logits(x, o)

    def prompt(self, prompts: list, chunk: int) -> torch.Tensor:
        """Takes the prompts in, `chunk` tokens of each a step; the first tokens that follow."""
        first = torch.zeros(self.requests, dtype=torch.int64, device=self.device)
        for at in range(0, max(len(p) for p in prompts), chunk):
            parts = [p[at:at + chunk] for p in prompts]
            new = [len(p) for p in parts]
            lens = torch.tensor(new, dtype=torch.int32, device=self.device)
            logits = self.step(torch.cat(parts), lens, max(new))
            last = (lens.long().cumsum(0) - 1).clamp(min=0)
            first = torch.where(lens > 0, logits[last].argmax(-1), first)
        return first

    def decode(self, first: torch.Tensor, steps: int) -> torch.Tensor:
        """Greedy tokens [requests, steps] behind the prompts, the step replayed from a graph."""
        ids, ones = first.clone(), torch.ones_like(self.cached)
        out = empty_step_metadata(self.requests, self.requests, self.device)
        state = [t.clone() for t in (self.cached, self.start, self.tables)]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ids.copy_(self.step(ids, ones, 1, out).argmax(-1))
        for t, s in zip((self.cached, self.start, self.tables), state):
            t.copy_(s)
        tokens = [first]
        for _ in range(steps - 1):
            graph.replay()
            tokens.append(ids.clone())
        return torch.stack(tokens, 1)


def make(prompts: list, room: int, device, seed: int = 0, vocab: int = 2000, hidden: int = 512):
    generator = torch.Generator().manual_seed(seed)
    layer = Layer(vocab, hidden, generator, device)
    ids = [torch.randint(0, vocab, (n,), generator=generator).to(device) for n in prompts]
    return Server(layer, len(prompts), room, device), ids


def main() -> None:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("--requests", 8), ("--prompt", 3000), ("--chunk", 512), ("--steps", 32)):
        p.add_argument(name, type=int, default=value)
    a = p.parse_args()
    lens = [max(1, a.prompt - 37 * i) for i in range(a.requests)]
    server, prompts = make(lens, max(lens) + a.steps, torch.device("cuda"))
    tokens = server.decode(server.prompt(prompts, a.chunk), a.steps)
    torch.cuda.synchronize()
    cached = int(server.cached.sum())
    print(f"{a.requests} requests, {cached} cached rows in {cached * KV_HEADS * 144 / 1e6:.1f} MB "
          f"({cached * KV_HEADS * 512 / 1e6:.1f} MB in 16 bits), error word {int(server.err)}")
    print(tokens[:, :12].tolist())


if __name__ == "__main__":
    main()
