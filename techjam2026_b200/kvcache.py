"""The layer stack served over an 8-bit key/value cache.

`FusedTransformer` runs whole sequences; a caller that extends them recomputes
every earlier token. `CachedStack` keeps each layer's K and V in an 8-bit cache
(`ops.KV8Cache`) and runs only the new tokens: a prompt in chunks of any
length, then one token at a time, each sequence of the batch at its own length.
With a `budget` it records the attention weight every cached token receives
and, when a sequence outgrows the budget, cuts its heads to their most recent
and their heaviest tokens.

    model = CachedStack(stack, batch=8, max_tokens=2048)
    out = model(prompt, counts=lengths)      # [B, T, d], ragged prompts
    out = model(token)                       # [B, 1, d], one more token each

`python -m techjam2026_b200.kvcache --config c2` runs a prompt and single
tokens of a benchmark configuration and compares them with the whole-sequence
forward. Causal stacks with head_dim 16 to 128; fp32, as the stack. The
reference recomputes the sequence (kernelforge/optimized.py:397-458).
"""
from __future__ import annotations

import itertools
from typing import List, Optional, Sequence

import torch

from .model import LayerStack
from .ops import (KV8Cache, add_mask_layernorm, kv8_append, kv8_attention, kv8_evict, linear)
from .ops.kv8 import HEAD_DIMS


class PagePool:
    """Which pages of a pool are free, and the page table of a batch.

    The table lives on the device; this is its host side. Pages are handed out
    and taken back between kernels of one stream, which the device then sees in
    order."""

    def __init__(self, pages: int, batch: int, blocks: int, block: int, device):
        self.block = block
        self.free = list(range(pages - 1, -1, -1))
        self.rows: List[List[int]] = [[] for _ in range(batch)]
        self.table = torch.zeros((batch, blocks), dtype=torch.int32, device=device)

    def take(self, n: int) -> List[int]:
        if n > len(self.free):
            raise RuntimeError(f"PagePool: {n} pages wanted, {len(self.free)} free")
        return [self.free.pop() for _ in range(n)]

    def reserve(self, tokens: Sequence[int]) -> None:
        """Pages for sequences of these lengths: for all of them, or an error
        and nothing changed."""
        if max(tokens) > self.table.shape[1] * self.block:
            raise RuntimeError(f"PagePool: a sequence of {max(tokens)} tokens does not fit "
                               f"{self.table.shape[1]} pages of {self.block}")
        more = [max(0, -(-n // self.block) - len(row)) for row, n in zip(self.rows, tokens)]
        if any(more):
            pages = iter(self.take(sum(more)))
            for row, n in zip(self.rows, more):
                row.extend(itertools.islice(pages, n))
            self._upload()

    def replace(self, rows: List[List[int]], which: Optional[Sequence[int]] = None) -> None:
        """New pages for every sequence, or for those in `which`; the old ones
        are free."""
        for i, row in zip(range(len(self.rows)) if which is None else which, rows):
            self.free.extend(self.rows[i])
            self.rows[i] = row
        self._upload()

    def _upload(self) -> None:
        host = torch.zeros(self.table.shape, dtype=torch.int32)
        for i, row in enumerate(self.rows):
            host[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        self.table.copy_(host)


class CachedStack:
    """A causal `LayerStack` over 8-bit caches, for a fixed batch of sequences.

    max_tokens  longest sequence a cache row holds
    code        torch.int8 or torch.float8_e4m3fn
    block       tokens that share a scale (a page)
    budget      None, or the most tokens a sequence holds between calls. One
                that has outgrown it is cut to budget - slack tokens, of which
                `recent` (or all, if that is more) are the latest
    slack       how far below the budget a cut goes, so that a sequence that is
                generated token by token is cut once in so many tokens: default
                a page, at most a quarter of the budget. A cut rounds the kept
                tokens again under the scales of their new pages: over 256
                tokens past a budget of 256, K and V went from 0.8 to 1.1 %
                off what was appended (int8), from 2.6 to 3.1 % (e4m3)"""

    def __init__(self, model: LayerStack, batch: int, max_tokens: int,
                 code: torch.dtype = torch.int8, block: int = 64, budget: Optional[int] = None,
                 recent: int = 0, device="cuda", slack: Optional[int] = None):
        cfg = model.config
        if not cfg.causal:
            raise ValueError("CachedStack: only a causal stack can be extended token by token")
        if budget is not None and not (0 < budget <= max_tokens and 0 <= recent <= budget):
            raise ValueError("CachedStack: needs 0 <= recent <= budget <= max_tokens, budget > 0")
        if slack is not None and (budget is None or not 0 <= slack < budget):
            raise ValueError("CachedStack: needs a budget and 0 <= slack < budget")
        self.heads, self.head_dim = cfg.num_heads, cfg.d_model // cfg.num_heads
        self.budget = budget
        if budget is not None:
            self.keep = budget - (min(block, budget // 4) if slack is None else slack)
            self.recent = min(recent, self.keep)
        device = torch.device(device, torch.cuda.current_device()) \
            if torch.device(device).index is None else torch.device(device)
        blocks = -(-max_tokens // block)
        if budget is not None and self.keep >= blocks * block:
            raise ValueError("CachedStack: a budget that fills the rows needs a slack")
        # an eviction writes the kept tokens before the old pages are free
        spare = -(-self.keep // block) if budget is not None else 0
        pages = batch * (blocks + spare)
        self.pool = PagePool(pages, batch, blocks, block, device)
        self.held = [0] * batch
        self.lens = torch.zeros(batch, dtype=torch.int32, device=device)
        self.caches = [KV8Cache.empty(pages, self.heads, block, self.head_dim, self.pool.table,
                                      self.lens, code, weight=budget is not None)
                       for _ in range(cfg.num_layers)]

        def dev(*ts):
            return torch.cat([t.detach() for t in ts], 0).to(device, torch.float32).contiguous()

        self.layers = [dict(
            wqkv=dev(a.q_proj.weight, a.k_proj.weight, a.v_proj.weight),
            bqkv=dev(a.q_proj.bias, a.k_proj.bias, a.v_proj.bias),
            wo=dev(a.out_proj.weight), bo=dev(a.out_proj.bias),
            w1=dev(m.ffn_in.weight), b1=dev(m.ffn_in.bias),
            w2=dev(m.ffn_out.weight), b2=dev(m.ffn_out.bias),
            n1=(dev(m.norm1.weight), dev(m.norm1.bias), m.norm1.eps),
            n2=(dev(m.norm2.weight), dev(m.norm2.bias), m.norm2.eps))
            for m in model.layers for a in (m.attention,)]
        self.final = (dev(model.final_norm.weight), dev(model.final_norm.bias),
                      model.final_norm.eps)

    def __call__(self, x: torch.Tensor, counts: Optional[Sequence[int]] = None) -> torch.Tensor:
        """Outputs [B, T, d] of the next T tokens of every sequence. `counts`
        (host integers): how many of the T each sequence takes, default all;
        the outputs of the others are 0."""
        B, T, d = x.shape
        if B != len(self.held):
            raise ValueError(f"CachedStack: a batch of {len(self.held)}, got {B}")
        counts = [T] * B if counts is None else [int(n) for n in counts]
        if len(counts) != B or min(counts) < 0 or max(counts) > T:
            raise ValueError(f"CachedStack: counts must be {B} numbers from 0 to {T}")
        if T == 0:
            return x
        if self.budget is not None:
            # a full row makes room first, if that is enough for every sequence
            reach = self.pool.table.shape[1] * self.pool.block
            full = [i for i, n in enumerate(counts) if self.held[i] + n > reach]
            if all(min(self.held[i], self.keep) + counts[i] <= reach for i in full):
                self._evict(full)
        self.pool.reserve([a + n for a, n in zip(self.held, counts)])
        new = torch.tensor(counts, dtype=torch.int32, device=x.device)
        keep = None
        if min(counts) < T:
            keep = (torch.arange(T, device=x.device) < new[:, None]).reshape(-1)
        longest = -(-max(a + n for a, n in zip(self.held, counts)) // 256) * 256
        res, y = x.reshape(B * T, d), None
        for p, cache in zip(self.layers, self.caches):
            res, h = add_mask_layernorm(res, y, keep, *p["n1"])
            qkv = linear(h, p["wqkv"], p["bqkv"]).view(B, T, 3, self.heads, self.head_dim)
            q, k, v = qkv.permute(2, 0, 3, 1, 4)
            kv8_append(cache, k, v, counts=new)
            ctx = torch.empty((B, T, self.heads, self.head_dim), device=x.device)
            kv8_attention(q, cache, counts=new, track=self.budget is not None, max_len=longest,
                          out=ctx.permute(0, 2, 1, 3))
            y = linear(ctx.view(B * T, d), p["wo"], p["bo"])
            res, h = add_mask_layernorm(res, y, keep, *p["n2"])
            y = linear(linear(h, p["w1"], p["b1"], gelu=True), p["w2"], p["b2"])
        _, out = add_mask_layernorm(res, y, keep, *self.final, mask_out=True)
        self.lens += new
        self.held = [a + n for a, n in zip(self.held, counts)]
        if self.budget is not None:
            self._evict([i for i, n in enumerate(self.held) if n > self.budget])
        return out.view(B, T, d)

    def _evict(self, which: List[int]) -> None:
        """Cuts the sequences in `which`; the others stay where they are."""
        if not which:
            return
        n = -(-self.keep // self.pool.block)
        pages = self.pool.take(n * len(which))
        rows = [pages[i * n:(i + 1) * n] for i in range(len(which))]
        table = torch.tensor(rows, dtype=torch.int32, device=self.lens.device)
        at = torch.tensor(which, device=self.lens.device)
        old, lens = self.pool.table[at], self.lens[at]
        for cache in self.caches:
            _, new = kv8_evict(cache.with_table(old, lens), table, self.keep, self.recent)
        self.lens.index_copy_(0, at, new.lens)
        for i in which:
            self.held[i] = self.keep
        self.pool.replace(rows, which)


def main(argv: Optional[Sequence[str]] = None) -> None:
    import argparse

    from .configs import WORKLOADS, init_params_
    from .fused import FusedTransformer

    ap = argparse.ArgumentParser(description="prompt, then single tokens, over an 8-bit cache")
    ap.add_argument("--config", default="c2", choices=sorted(
        name for name, w in WORKLOADS.items()
        if w.cfg.causal and w.cfg.d_model // w.cfg.num_heads in HEAD_DIMS))
    ap.add_argument("--tokens", type=int, default=16, help="single tokens after the prompt")
    ap.add_argument("--code", default="int8", choices=("int8", "float8_e4m3fn"))
    a = ap.parse_args(argv)
    cfg = WORKLOADS[a.config].cfg
    if not 0 < a.tokens < cfg.seq_len:
        ap.error(f"--tokens must be from 1 to {cfg.seq_len - 1}")
    warm = min(2, a.tokens - 1)      # single tokens before the timed ones
    stack = init_params_(LayerStack(cfg), 0)
    x = torch.randn(cfg.batch_size, cfg.seq_len, cfg.d_model,
                    generator=torch.Generator().manual_seed(1)).cuda()
    whole = FusedTransformer(cfg)
    whole.load_state_dict(stack.state_dict(), strict=True)
    want = whole(x, None)
    model = CachedStack(stack, cfg.batch_size, cfg.seq_len, getattr(torch, a.code))
    n = cfg.seq_len - a.tokens
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    outs = [model(x[:, :n])]
    for i in range(n, cfg.seq_len):
        if i == n + warm:
            begin.record()
        outs.append(model(x[:, i:i + 1]))
    end.record()
    got = torch.cat(outs, 1)
    torch.cuda.synchronize()
    rel = float((got - want).norm() / want.norm())
    ms = begin.elapsed_time(end) / (a.tokens - warm)
    print(f"{a.config}: {n} prompt tokens and {a.tokens} single ones of {cfg.batch_size} sequences, "
          f"{a.code} cache: relative difference from the whole-sequence forward {rel:.2e}, "
          f"{ms:.3f} ms a token")


if __name__ == "__main__":
    main()
