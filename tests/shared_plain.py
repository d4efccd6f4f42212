"""Caches whose groups share pages, and float64 attention over them with the
bounds that the operator's roundings give, for the tests."""
from __future__ import annotations

import math

import torch

from techjam2026_b200 import ops

EPS_Q = {torch.float32: 2.0 ** -21, torch.bfloat16: 2.0 ** -23, torch.float16: 2.0 ** -23}
# one plane of P for bf16 (half of fp16's eps), two for the others
EPS_P = {torch.float32: 2.0 ** -21, torch.bfloat16: 2.0 ** -11, torch.float16: 2.0 ** -21}
EPS_OUT = {torch.float32: 2.0 ** -23, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


def make_groups(sizes, shared, own, heads=2, dim=64, block=16, dtype=torch.int8, room=32, seed=0,
                rest=0):
    """Groups of sizes[n] sequences (the last `rest` sequences are in none) whose
    first shared[n] tokens are on common pages; sequence b holds own[b] tokens
    more. Pages scattered over the pool; every slot and scale that holds no token
    is junk, NaN among it. Returns (cache, starts, shared)."""
    g = torch.Generator().manual_seed(seed)
    N, B = len(sizes), sum(sizes) + rest
    assert len(own) == B and all(s % block == 0 for s in shared)
    front = [s // block for s in shared]
    back = -(-(max(own) + room) // block) + 1
    blocks = max(front + [0]) + back
    pages = sum(front) + B * back + 5
    order = torch.randperm(pages, generator=g).to(torch.int32).tolist()
    table = torch.full((B, blocks), order[-1], dtype=torch.int32)
    common, group = [], []
    for n in range(N):
        common.append([order.pop() for _ in range(front[n])])
        group += [n] * sizes[n]
    group += [None] * rest
    for b, n in enumerate(group):
        row = (common[n] if n is not None else []) + [order.pop() for _ in range(back)]
        table[b, :len(row)] = torch.tensor(row, dtype=torch.int32)
    lens = torch.zeros(B, dtype=torch.int32, device="cuda")
    cache = ops.KV8Cache.empty(pages, heads, block, dim, table.cuda(), lens, dtype)
    cache.k.view(torch.uint8).fill_(0xFF)
    cache.v.view(torch.uint8).fill_(0x7F)
    cache.scale.fill_(math.nan)

    def tokens(n):
        x = torch.randn(2, 1, heads, n, dim, generator=g)
        return x[0].cuda(), x[1].cuda()

    for b, n in enumerate(group):
        one = cache.with_table(cache.table[b:b + 1], lens[b:b + 1])
        if n is not None and shared[n]:
            if b == sum(sizes[:n]):
                ops.kv8_append(one, *tokens(shared[n]))
            lens[b] = shared[n]
        if own[b]:
            ops.kv8_append(one, *tokens(own[b]))
            lens[b] += own[b]
    starts = torch.tensor([sum(sizes[:n]) for n in range(N + 1)], dtype=torch.int32, device="cuda")
    return cache, starts, torch.tensor(shared, dtype=torch.int32, device="cuda")


def attention64(q, cache, counts, causal, scale):
    """out, its bound, lse and its bound, in float64 on the GPU. The bounds are
    those of tests/kv8_plain.py: q off by eps_q and D products summed in fp32
    put a score off by at most d; a weight is off by e^(2 d), P by eps_p, the sum
    of m products by m steps of fp32; the smallest weights are lost below 2^-30
    (one plane) or 2^-34 of the largest V."""
    B, Hq, T, D = q.shape
    H, P = cache.kv_heads, cache.block
    G = Hq // H
    eps_q, eps_p, eps_out = EPS_Q[q.dtype], EPS_P[q.dtype], EPS_OUT[q.dtype]
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device="cuda")
    tol = torch.zeros_like(out)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device="cuda")
    tol_lse = torch.zeros_like(lse)
    for b in range(B):
        have = int(cache.lens[b])
        n = T if counts is None else int(counts[b])
        end = have + n
        if n <= 0 or end == 0:
            continue
        page = cache.table[b, :-(-end // P)].long()

        def values(pool, which):
            x = pool.view(torch.uint8)[page].view(pool.dtype).float()
            x = x.double() * cache.scale[page][:, :, which].double()[:, :, None, None]
            return x.permute(1, 0, 2, 3).reshape(H, -1, D)[:, :end]

        k, v = values(cache.k, 0), values(cache.v, 1)
        x = q[b, :, :n].double().reshape(H, G * n, D)
        s = (x @ k.transpose(1, 2)).view(H, G, n, end) * scale
        size = (x.abs() @ k.abs().transpose(1, 2)).view(H, G, n, end) * scale
        if causal:
            late = torch.arange(end, device="cuda") > have + torch.arange(n, device="cuda")[:, None]
            s = s.masked_fill(late, -math.inf)
            size = size.masked_fill(late, 0.0)
        d = (eps_q + (D + 4) * 2.0 ** -23) * size.amax(-1) + 2.0 ** -21
        l = torch.logsumexp(s, -1)
        p = torch.softmax(s, -1).view(H, G * n, end)
        o = (p @ v).view(Hq, n, D)
        mass = (p @ v.abs()).view(Hq, n, D)
        top = v.abs().amax(1).repeat_interleave(G, 0)[:, None]                  # [Hq, 1, D]
        rel = (2 * d + eps_p + (end + 16) * 2.0 ** -23).view(Hq, n, 1)
        small = 2.0 ** -30 if eps_p > 2.0 ** -20 else end * 2.0 ** -34
        out[b, :, :n] = o
        tol[b, :, :n] = mass * rel + o.abs() * eps_out + top * small + 1e-30
        lse[b, :, :n] = l.view(Hq, n)
        tol_lse[b, :, :n] = d.view(Hq, n) + 2.0 ** -20 * (1 + l.abs().view(Hq, n))
    return out, tol, lse, tol_lse
