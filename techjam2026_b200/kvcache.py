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

Several sequences may continue one prompt: `fork` lets them share the pages that
they have in common (which are then also read once for all of them), `free` and
`compact` give pages back. `beam_search` puts these together.

    out = model(prompt, rows=[0])            # the prompt once
    model.fork([0] * 8)                      # eight samples of it
    tokens, scores = beam_search(model, prompts, lengths, embed, head, beams=4, steps=32)

`python -m techjam2026_b200.kvcache --config c2` runs a prompt and single
tokens of a benchmark configuration and compares them with the whole-sequence
forward; with `--beams 4` it runs beam search instead. Causal stacks with head_dim 16 to 128; fp32, as the stack. The
reference recomputes the sequence (kernelforge/optimized.py:397-458).
"""
from __future__ import annotations

import itertools
from typing import List, Optional, Sequence, Tuple

import torch

from .model import LayerStack
from .ops import (KV8Cache, add_mask_layernorm, beam_select, kv8_append, kv8_attention,
                  kv8_attention_shared, kv8_copy, kv8_evict, linear)
from .ops.beam import MAX_TAKE
from .ops.kv8 import HEAD_DIMS


class PagePool:
    """Which pages of a pool are free, and the page table of a batch.

    The table lives on the device; this is its host side. Pages are handed out
    and taken back between kernels of one stream, which the device then sees in
    order. After a fork, a page may be several sequences' (`uses`); it is free
    once it is nobody's."""

    def __init__(self, pages: int, batch: int, blocks: int, block: int, device):
        self.block = block
        self.free = list(range(pages - 1, -1, -1))
        self.uses = [0] * pages
        self.groups: Optional[Tuple[torch.Tensor, torch.Tensor, List[int]]] = None
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
                new = list(itertools.islice(pages, n))
                row.extend(new)
                self._use(new)
            self._upload()

    def replace(self, rows: List[List[int]], which: Optional[Sequence[int]] = None) -> None:
        """New pages for every sequence, or for those in `which`; the old ones
        are free."""
        for i, row in zip(range(len(self.rows)) if which is None else which, rows):
            self._use(row)
            self._drop(self.rows[i])
            self.rows[i] = row
        self._upload()

    def fork(self, parents: Sequence[int], held: Sequence[int], whole: bool = False
             ) -> List[Tuple[int, int, int]]:
        """Row i becomes row parents[i], of held[parents[i]] tokens. Full pages are
        shared; a last page that is not full stays the first child's, and the
        others get copies (whole: copies of all pages). Returns those copies,
        (from, to, tokens), or raises and changes nothing."""
        keep = [-(-held[p] // self.block) for p in parents]
        full = [0 if whole else held[p] // self.block for p in parents]
        first = {p: i for i, p in reversed(list(enumerate(parents)))}
        stay = set()
        for i, p in enumerate(parents):
            stay.update(self.rows[p][:keep[i] if first[p] == i else full[i]])
        gone = {q for row in self.rows for q in row} - stay
        need = sum(k - f for i, (k, f) in enumerate(zip(keep, full)) if first[parents[i]] != i)
        if need > len(self.free) + len(gone):
            raise RuntimeError(f"PagePool: {need} pages wanted, {len(self.free) + len(gone)} free")
        rows, old = [], self.rows
        for i, p in enumerate(parents):
            rows.append(list(old[p][:keep[i] if first[p] == i else full[i]]))
            self._use(rows[i])
        for row in old:
            self._drop(row)
        copies = []
        for i, p in enumerate(parents):
            for j in range(len(rows[i]), keep[i]):
                page = self.take(1)[0]
                rows[i].append(page)
                self._use([page])
                copies.append((old[p][j], page, min(self.block, held[p] - j * self.block)))
        self.rows = rows
        self._upload()
        return copies

    def compact(self) -> List[Tuple[int, int]]:
        """Moves the pages in use to the lowest numbers; returns the moves."""
        used = sum(n > 0 for n in self.uses)
        high = [p for p in range(used, len(self.uses)) if self.uses[p]]
        low = [p for p in range(used) if not self.uses[p]]
        to = dict(zip(high, low))
        if to:
            self.rows = [[to.get(p, p) for p in row] for row in self.rows]
            for a, b in to.items():
                self.uses[a], self.uses[b] = 0, self.uses[a]
            self._upload()
        self.free = list(range(len(self.uses) - 1, used - 1, -1))
        return list(to.items())

    def _use(self, pages: Sequence[int]) -> None:
        for p in pages:
            self.uses[p] += 1

    def _drop(self, pages: Sequence[int]) -> None:
        for p in pages:
            self.uses[p] -= 1
            if not self.uses[p]:
                self.free.append(p)

    def _group(self) -> None:
        """Groups of consecutive sequences that begin with the same pages, and how
        many leading tokens (of whole pages) each group shares. A sequence that has
        little in common with its neighbours does not join them: what a group shares
        is what all of it does."""
        self.groups = None
        if max(self.uses, default=0) < 2:
            return
        starts, common, run = [], [], []
        for i in range(1, len(self.rows) + 1):
            both = self._common(i, run[-1] if run else 0) if i < len(self.rows) else 0
            if both:
                run.append(both)
                continue
            at = i - 1 - len(run)         # sequences that begin with one page: from here on
            for m, n in _cut(run):
                starts.append(at)
                common.append(n)
                at += m
            run = []
        starts.append(len(self.rows))
        shared = [n * self.block for n in common]
        of = [n for n, (a, z) in enumerate(zip(starts, starts[1:])) for _ in range(z - a)]
        if not any(shared):
            return
        dev = self.table.device
        self.groups = (torch.tensor(starts, dtype=torch.int32).to(dev),
                       torch.tensor(shared, dtype=torch.int32).to(dev), [shared[n] for n in of])

    def _common(self, i: int, guess: int) -> int:
        """Leading pages that sequences i - 1 and i have in common."""
        a, b = self.rows[i - 1], self.rows[i]
        lo, hi = 0, min(len(a), len(b))
        if guess < hi and a[guess] != b[guess]:
            hi = guess                    # (siblings have what the pair before them has)
        if a[:hi] == b[:hi]:
            return hi
        while hi - lo > 1:                # a[:lo] == b[:lo], a[:hi] != b[:hi]
            mid = (lo + hi) // 2
            if a[lo:mid] == b[lo:mid]:
                lo = mid
            else:
                hi = mid
        return lo

    def _upload(self) -> None:
        host = torch.zeros(self.table.shape, dtype=torch.int32)
        for i, row in enumerate(self.rows):
            host[i, :len(row)] = torch.tensor(row, dtype=torch.int32)
        self.table.copy_(host)
        self._group()


def _cut(both: List[int]) -> List[Tuple[int, int]]:
    """Groups (members, pages that all of them share) of consecutive sequences of
    which neighbours have these numbers of leading pages in common. Reading them by
    groups saves (members - 1) * pages reads. One group of all, or what a pass along
    them finds better: a sequence joins the group before it, begins one, or takes
    the sequence before it along into a new one, as saves most."""
    if not both:
        return [(1, 0)]
    groups = [(2, both[0])]
    for b in both[1:]:
        m, n = groups[-1]
        join = m * min(n, b) if m > 1 else b
        along = (m - 2) * n + b if m > 1 else 0
        if join >= max((m - 1) * n, along):
            groups[-1] = (m + 1, min(n, b) if m > 1 else b)
        elif along > (m - 1) * n:
            groups[-1:] = [(m - 1, n if m > 2 else 0), (2, b)]
        else:
            groups.append((1, 0))
    if sum((m - 1) * n for m, n in groups) > len(both) * min(both):
        return groups
    return [(len(both) + 1, min(both))]


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

    def __call__(self, x: torch.Tensor, counts: Optional[Sequence[int]] = None,
                 rows: Optional[Sequence[int]] = None) -> torch.Tensor:
        """Outputs [B, T, d] of the next T tokens of every sequence. `counts`
        (host integers): how many of the T each sequence takes, default all;
        the outputs of the others are 0. `rows`: only these sequences, x and
        counts are theirs (a prompt that others will share is run once)."""
        B, T, d = x.shape
        which = list(range(len(self.held))) if rows is None else [int(i) for i in rows]
        if len(set(which)) != len(which) or any(not 0 <= i < len(self.held) for i in which):
            raise ValueError(f"CachedStack: rows must be different numbers from 0 to "
                             f"{len(self.held) - 1}")
        if B != len(which):
            raise ValueError(f"CachedStack: a batch of {len(which)}, got {B}")
        counts = [T] * B if counts is None else [int(n) for n in counts]
        if len(counts) != B or min(counts, default=0) < 0 or max(counts, default=0) > T:
            raise ValueError(f"CachedStack: counts must be {B} numbers from 0 to {T}")
        if T == 0 or B == 0:
            return x
        want = list(self.held)
        for i, n in zip(which, counts):
            want[i] += n
        if self.budget is not None:
            # a full row makes room first, if that is enough for every sequence
            reach = self.pool.table.shape[1] * self.pool.block
            full = [i for i in which if want[i] > reach]
            if all(min(self.held[i], self.keep) + want[i] - self.held[i] <= reach for i in full):
                self._evict(full)
                for i in full:
                    want[i] = self.held[i] + counts[which.index(i)]
        self.pool.reserve(want)
        new = torch.tensor(counts, dtype=torch.int32, device=x.device)
        keep = None
        if min(counts) < T:
            keep = (torch.arange(T, device=x.device) < new[:, None]).reshape(-1)
        caches, at = self.caches, None
        if rows is not None:
            at = torch.tensor(which, device=self.lens.device)
            table, lens = self.pool.table[at], self.lens[at]
            caches = [c.with_table(table, lens) for c in caches]
        groups = self.pool.groups if rows is None else None
        longest = -(-max(want[i] for i in which) // 256) * 256
        if groups is not None:
            own = -(-max(n - m for n, m in zip(want, groups[2])) // 256) * 256
        res, y = x.reshape(B * T, d), None
        for p, cache in zip(self.layers, caches):
            res, h = add_mask_layernorm(res, y, keep, *p["n1"])
            qkv = linear(h, p["wqkv"], p["bqkv"]).view(B, T, 3, self.heads, self.head_dim)
            q, k, v = qkv.permute(2, 0, 3, 1, 4)
            kv8_append(cache, k, v, counts=new)
            ctx = torch.empty((B, T, self.heads, self.head_dim), device=x.device)
            if groups is not None:
                # (every sequence of a group holds all that it shares: only full pages are
                # common, so nothing is cut and `own` bounds the rest)
                kv8_attention_shared(q, cache, groups[0], groups[1], counts=new,
                                     max_shared=max(groups[2]), max_own=own,
                                     out=ctx.permute(0, 2, 1, 3))
            else:
                kv8_attention(q, cache, counts=new, track=self.budget is not None, max_len=longest,
                              out=ctx.permute(0, 2, 1, 3))
            y = linear(ctx.view(B * T, d), p["wo"], p["bo"])
            res, h = add_mask_layernorm(res, y, keep, *p["n2"])
            y = linear(linear(h, p["w1"], p["b1"], gelu=True), p["w2"], p["b2"])
        _, out = add_mask_layernorm(res, y, keep, *self.final, mask_out=True)
        if at is None:
            self.lens += new
        else:
            self.lens.index_add_(0, at, new)
        self.held = want
        if self.budget is not None:
            self._evict([i for i in which if self.held[i] > self.budget])
        return out.view(B, T, d)

    def fork(self, parents: Sequence[int]) -> None:
        """Sequence i goes on from where sequence parents[i] stands (all at once;
        a sequence that is nobody's parent ends). Full pages are shared, a last
        one that is not full is copied; with a budget all pages are copied, since
        the record of weights belongs to the pages."""
        parents = [int(p) for p in parents]
        if len(parents) != len(self.held) or any(not 0 <= p < len(self.held) for p in parents):
            raise ValueError(f"CachedStack: parents must be {len(self.held)} sequences")
        copies = self.pool.fork(parents, self.held, whole=self.budget is not None)
        at = torch.tensor(parents, device=self.lens.device)
        if copies:
            src, dst, tokens = torch.tensor(copies, dtype=torch.int32).T.contiguous().to(
                self.lens.device)
            kv8_copy(self.caches, src, dst, tokens=tokens)
        self.lens.copy_(self.lens[at])
        self.held = [self.held[p] for p in parents]

    def free(self, which: Sequence[int]) -> None:
        """Ends these sequences: they hold no token, and their pages are free if
        no other sequence has them."""
        which = [int(i) for i in which]
        if any(not 0 <= i < len(self.held) for i in which):
            raise ValueError(f"CachedStack: sequences are 0 to {len(self.held) - 1}")
        self.pool.replace([[] for _ in which], which)
        for i in which:
            self.held[i] = 0
        if which:
            self.lens[torch.tensor(which, device=self.lens.device)] = 0

    def compact(self) -> int:
        """Moves the pages in use to the front of the pools; how many they are."""
        moves = self.pool.compact()
        if moves:
            src, dst = torch.tensor(moves, dtype=torch.int32).T.contiguous().to(self.lens.device)
            kv8_copy(self.caches, src, dst)
        return len(self.pool.uses) - len(self.pool.free)

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


def beam_search(model: CachedStack, prompts: torch.Tensor, lengths: Sequence[int],
                embed: torch.Tensor, head: torch.Tensor, beams: int, steps: int,
                end: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """The `beams` best continuations of each prompt that beam search finds.

    model    a CachedStack of N * beams sequences that hold nothing, beams at most
             128, without a budget; prompt n has the sequences n * beams and following
    prompts  [N, T, d] float32 embeddings, prompt n of lengths[n] >= 1 tokens
    embed    [V, d] float32, the embedding of each token
    head     [V, d] float32, the output projection
    steps    tokens to generate, with the prompts at most what the model's sequences
             hold and one; a beam that takes the token `end` stays as it is

    Returns (tokens [N, beams, steps] int32, scores [N, beams] float32: the sums of
    the tokens' log probabilities), best first. A beam that ended is filled with
    `end`; one for which there was no candidate has the score -inf."""
    N = prompts.shape[0]
    if len(model.held) != N * beams or any(model.held) or model.budget is not None:
        raise ValueError(f"beam_search: needs an empty CachedStack of {N * beams} sequences "
                         "without a budget")
    if len(lengths) != N or steps < 1 or any(not 0 < n <= prompts.shape[1] for n in lengths):
        raise ValueError("beam_search: needs a length of at least 1 for each prompt, and steps")
    dev, V = prompts.device, head.shape[0]
    reach = model.pool.table.shape[1] * model.pool.block
    if not 0 < beams <= MAX_TAKE or max(lengths, default=0) + steps - 1 > reach \
            or not (end is None or 0 <= end < V):
        raise ValueError(f"beam_search: needs 1 to {MAX_TAKE} beams, prompts that leave room for "
                         f"{steps} steps within {reach} tokens, and an end below {V}")
    first = [n * beams for n in range(N)]
    out = model(prompts, counts=lengths, rows=first)
    last = out[torch.arange(N, device=dev), torch.tensor(lengths, device=dev) - 1]
    model.fork([n for n in first for _ in range(beams)])
    logits = linear(last, head).view(N, 1, V)
    score = torch.zeros(N, 1, device=dev)
    base = torch.tensor(first, device=dev)[:, None]
    tokens = torch.zeros(N * beams, 0, dtype=torch.int32, device=dev)
    ended = None
    for step in range(steps):
        score, beam, token = beam_select(logits, score, beams, ended=ended,
                                         pad=end if end is not None else 0)
        parent = (base + beam.clamp(min=0)).view(-1)
        token = token.clamp(min=0).view(-1)
        tokens = torch.cat([tokens[parent], token[:, None]], 1)
        if end is not None:
            ended = (token == end).view(N, beams)
        if step + 1 == steps:
            break
        if step:                 # (after the first step all beams continue the prompt)
            model.fork(parent.tolist())
        out = model(embed[token][:, None])
        logits = linear(out.view(N * beams, -1), head).view(N, beams, V)
    return tokens.view(N, beams, steps), score


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
    ap.add_argument("--beams", type=int, default=0,
                    help="beam search with this many beams instead, random weights and embeddings")
    ap.add_argument("--vocab", type=int, default=8192, help="vocabulary of the beam search")
    a = ap.parse_args(argv)
    cfg = WORKLOADS[a.config].cfg
    if not 0 < a.tokens < cfg.seq_len:
        ap.error(f"--tokens must be from 1 to {cfg.seq_len - 1}")
    if a.beams < 0 or a.beams > 128 or (a.beams and a.vocab < 4):
        ap.error("--beams must be from 1 to 128, --vocab at least 4")
    if a.beams:
        return _beam_example(cfg, a)
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


def _beam_example(cfg, a) -> None:
    from .configs import init_params_

    stack = init_params_(LayerStack(cfg), 0)
    g = torch.Generator().manual_seed(1)
    n = cfg.seq_len - a.tokens
    x = torch.randn(cfg.batch_size, n, cfg.d_model, generator=g).cuda()
    embed = torch.randn(a.vocab, cfg.d_model, generator=g).cuda()
    model = CachedStack(stack, cfg.batch_size * a.beams, cfg.seq_len, getattr(torch, a.code))
    begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
    begin.record()
    tokens, scores = beam_search(model, x, [n] * cfg.batch_size, embed, embed, a.beams, a.tokens)
    end.record()
    torch.cuda.synchronize()
    pages = model.compact()
    alone = sum(-(-held // model.pool.block) for held in model.held)
    print(f"{a.config}: {cfg.batch_size} prompts of {n} tokens, {a.beams} beams, {a.tokens} tokens of "
          f"{a.vocab}, {a.code} cache: best scores {scores[:, 0].min():.2f} to "
          f"{scores[:, 0].max():.2f}, {begin.elapsed_time(end):.1f} ms, {pages} pages "
          f"({alone} without sharing)")


if __name__ == "__main__":
    main()
