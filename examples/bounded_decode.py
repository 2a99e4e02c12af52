"""Decode with a bounded paged cache: a stack of attention layers with random weights reads a
prompt, keeps the entries that its last queries attend to, and generates tokens while every
layer's cache stays within its budget.

    python examples/bounded_decode.py [--batch 4] [--prompt 2000] [--tokens 128] [--budget 512]

Every layer has a pool of pages; the block table, the lengths and the positions are shared by
all of them. Once the prompt is evicted, the calls get the columns of the table that a bounded
sequence can use: their plans follow the table's width. A decode step (append, attention with its
weights, the projections) is one CUDA graph; an eviction, another, runs once per page of new
tokens. Prints the time per step beside that of the whole cache, and how far the two streams of
hidden states drift apart.
"""
from __future__ import annotations

import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

from pseudobrain_b200.paged_cache import (PagedCache, paged_append_, paged_attend, paged_evict_,  # noqa: E402
                                          paged_observe_)
from pseudobrain_b200.transplant import causal_attention  # noqa: E402


class Layer:
    """One attention layer: projections with random weights and a pool of pages."""

    def __init__(self, hidden: int, heads: int, kv: int, hd: int, pages: int, page: int, gen: torch.Generator):
        rnd = lambda *s: (torch.randn(*s, generator=gen, device="cuda") * s[0] ** -0.5).to(torch.bfloat16)  # noqa: E731
        self.heads, self.kv, self.hd = heads, kv, hd
        self.qkv, self.out = rnd(hidden, (heads + 2 * kv) * hd), rnd(heads * hd, hidden)
        self.cache = PagedCache.allocate(pages, kv, page, hd)

    def project(self, x: torch.Tensor):
        h = torch.nn.functional.rms_norm(x, (x.shape[-1],))
        return (h @ self.qkv).unflatten(-1, (self.heads + 2 * self.kv, self.hd)).split((self.heads, self.kv, self.kv), -2)

    def prompt(self, x: torch.Tensor, table, lengths, seen, observe: int) -> torch.Tensor:
        """x [B, T, hidden] into the cache; its last `observe` queries' weights into the mass."""
        b, t, _ = x.shape
        q, k, v = self.project(x)
        cu = torch.arange(0, b * t + 1, t, dtype=torch.int32, device=x.device)
        paged_append_(self.cache, k.flatten(0, 1), v.flatten(0, 1), table, lengths, seen, cu)
        if observe:
            paged_observe_(self.cache, q[:, -observe:], table, lengths + t)
        o = causal_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2)).transpose(1, 2)
        return x + o.reshape(b, t, -1) @ self.out

    def step(self, x: torch.Tensor, table, before, seen, after, weights: bool) -> torch.Tensor:
        """One token per sequence, x [B, hidden]."""
        q, k, v = self.project(x)
        paged_append_(self.cache, k, v, table, before, seen)
        o, _ = paged_attend(self.cache, q, table, after, accumulate=weights)
        return x + o.flatten(1) @ self.out


class Decoder:
    def __init__(self, a: argparse.Namespace, budget: int | None):
        gen = torch.Generator(device="cuda").manual_seed(a.seed)
        width = -(-(a.prompt + a.tokens) // a.page)
        self.a, self.budget = a, budget
        self.layers = [Layer(a.hidden, a.heads, a.kv, 128, a.batch * width, a.page, gen) for _ in range(a.layers)]
        self.table = torch.randperm(a.batch * width, generator=gen, device="cuda").to(torch.int32).view(a.batch, width)
        # from the prompt's eviction on: the budget and the tokens until the next eviction
        self.used = self.table if budget is None else self.table[:, : -(-(budget + a.page) // a.page)]
        self.lengths = torch.zeros(a.batch, dtype=torch.int32, device="cuda")
        self.after = torch.zeros_like(self.lengths)
        self.seen = torch.zeros_like(self.lengths)
        self.x = torch.randn(a.batch, a.prompt, a.hidden, generator=gen, device="cuda").to(torch.bfloat16)

    def read_prompt(self) -> torch.Tensor:
        x = self.x
        for layer in self.layers:
            x = layer.prompt(x, self.table, self.lengths, self.seen, self.a.observe if self.budget else 0)
        self.lengths += self.a.prompt
        self.seen += self.a.prompt
        if self.budget:
            self.evict(self.table)
        return x[:, -1].clone()

    def evict(self, table: torch.Tensor) -> None:
        for layer in self.layers:
            paged_evict_(layer.cache, table, self.lengths, self.seen, self.budget, self.a.recent, self.a.sinks)
        self.lengths.clamp_(max=self.budget)

    def step(self, x: torch.Tensor) -> None:
        y = x
        torch.add(self.lengths, 1, out=self.after)
        for layer in self.layers:
            y = layer.step(y, self.used, self.lengths, self.seen, self.after, self.budget is not None)
        x.copy_(y / y.float().square().mean(-1, keepdim=True).sqrt())
        self.lengths += 1
        self.seen += 1

    def generate(self) -> tuple[torch.Tensor, float, int]:
        """(last hidden states of every step, ms per step, entries at the end)."""
        x = self.read_prompt()
        side, states = torch.cuda.Stream(), []
        state = [x, self.lengths, self.seen, *(layer.cache.mass for layer in self.layers)]
        keep = [t.clone() for t in state]
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            self.step(x)  # warm-up before the capture; its token is written again by the first replay
            for t, k in zip(state, keep):
                t.copy_(k)
            step, evict = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
            with torch.cuda.graph(step, stream=side):
                self.step(x)
            if self.budget:
                with torch.cuda.graph(evict, stream=side):
                    self.evict(self.used)
            start, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            start.record()
            for i in range(self.a.tokens):
                step.replay()
                states.append(x.clone())
                if self.budget and i % self.a.page == self.a.page - 1:
                    evict.replay()
            end.record()
        torch.cuda.synchronize()
        return torch.stack(states), start.elapsed_time(end) / self.a.tokens, int(self.lengths.max())


def main(argv: list[str] | None = None) -> dict:
    p = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("batch", 4), ("prompt", 2000), ("tokens", 128), ("budget", 512), ("recent", 64), ("sinks", 4),
                        ("observe", 32), ("page", 16), ("layers", 4), ("hidden", 1024), ("heads", 16), ("kv", 4), ("seed", 0)):
        p.add_argument(f"--{name}", type=int, default=value)
    a = p.parse_args(argv)
    whole, whole_ms, n_whole = Decoder(a, None).generate()
    bound, bound_ms, n_bound = Decoder(a, a.budget).generate()
    drift = 1 - torch.nn.functional.cosine_similarity(whole.float(), bound.float(), -1).mean(-1)
    print(f"whole cache:   {whole_ms:.3f} ms a step, {n_whole} entries a head at the end")
    print(f"bounded cache: {bound_ms:.3f} ms a step, {n_bound} entries a head at the end")
    print(f"1 - cosine of the hidden states: first step {drift[0]:.2e}, last step {drift[-1]:.2e}")
    return {"whole_ms": whole_ms, "bounded_ms": bound_ms, "whole": n_whole, "bounded": n_bound, "drift": drift.tolist()}


if __name__ == "__main__":
    main()
