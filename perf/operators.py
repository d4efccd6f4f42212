"""The operators of the 8-bit key/value cache, as cases to be measured.

A layer's cache holds K and V of B sequences in pages of `block` tokens, as
int8 or e4m3 codes with one scale for each page and head. Three kinds of case:

  append  a chunk of K/V is quantised into the cache and the touched pages are
          read back as values (kv8_append, kv8_read);
  attend  the queries of the newest tokens read the cache (kv8_attention), with
          `track` adding each key's attention weight to the cache's record;
  evict   each head keeps its most recent and its heaviest tokens, requantised
          into new pages (kv8_evict), and the result is read back (kv8_read).

`run` computes them with elementary torch operations in 32 bits where `own` is
false, and calls techjam2026_b200.ops where it is true. `exact` restates them
in 64 bits.
"""
import math

import torch

own = False

QMAX = {"int8": 127.0, "fp8": 448.0}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}
TINY = 2.0 ** -126          # a scale below the smallest normal number stands for a block of zeros


def listed():
    base = {"kind": "attend", "batch": 1, "heads": 8, "kv_heads": 8, "head_dim": 64, "block": 64,
            "format": "int8", "dtype": "float32", "cached_min": 0, "cached_max": 0, "new": 1,
            "ragged": False, "causal": True, "track": False, "budget": 0, "recent": 0}

    def case(name, **kw):
        return {"name": name, **base, **kw}

    return [
        # one generated token of each of 8 sequences enters the cache (stack of 8 heads of 64)
        case("append one token", kind="append", batch=8, cached_min=256, cached_max=511),
        # ragged chunks of a heavily padded batch (64 sequences, 12 heads of 64), fp32 as the stack
        case("append ragged chunks", kind="append", batch=64, heads=12, kv_heads=12,
             cached_min=1, cached_max=1271, new=777, ragged=True),
        # long prompts of a grouped-head model enter an empty e4m3 cache
        case("append prompts", kind="append", batch=16, heads=32, kv_heads=8, head_dim=128,
             format="fp8", dtype="bfloat16", new=4096),
        # one token of two short sequences: nothing but latency
        case("token, short", batch=2, heads=4, kv_heads=4, head_dim=32, block=16, cached_min=32,
             cached_max=63),
        # one token of each of 64 sequences of length 1 to 2048, fp32, weights recorded for eviction
        case("token, ragged batch, weights", batch=64, heads=12, kv_heads=12, cached_min=0,
             cached_max=2047, track=True),
        # one token of a long sequence, fp16: few rows, a long axis
        case("token, one long sequence", heads=16, kv_heads=16, dtype="float16", cached_min=65000,
             cached_max=65535),
        # one token of a batch of long grouped-head sequences: the largest reads
        case("token, long grouped batch", batch=16, heads=32, kv_heads=8, head_dim=128,
             format="fp8", dtype="bfloat16", cached_min=16384, cached_max=32767),
        # a chunk of a prompt over what the cache already holds, bf16
        case("chunk over a long cache", batch=2, heads=16, kv_heads=16, dtype="bfloat16",
             cached_min=8192, cached_max=30000, new=1024),
        # whole prompts of a grouped-head model, bf16 over e4m3
        case("prompts", batch=4, heads=32, kv_heads=8, head_dim=128, block=128, format="fp8",
             dtype="bfloat16", new=2048),
        # ragged fp32 chunks whose weights are recorded
        case("chunks, fp32, weights", batch=3, heads=16, kv_heads=4, head_dim=128, block=32,
             cached_min=1500, cached_max=4000, new=700, ragged=True, track=True),
        # a short cache is halved
        case("evict, short", kind="evict", batch=4, cached_min=400, cached_max=600, budget=256,
             recent=64),
        # long grouped-head caches are cut to a budget
        case("evict, long", kind="evict", batch=16, heads=32, kv_heads=8, head_dim=128,
             format="fp8", dtype="bfloat16", cached_min=16384, cached_max=32768, budget=8192,
             recent=1024),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = [work(c) for c in listed()]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while True:
        kind = rng.choice(["append", "attend", "attend", "attend", "evict"])
        kv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        group = rng.choice([1, 1, 2, 4, 8])
        c = {"kind": kind, "batch": _log(rng, 1, 64), "heads": kv * group, "kv_heads": kv,
             "head_dim": rng.choice([32, 64, 64, 128]), "block": rng.choice([16, 32, 64, 128]),
             "format": rng.choice(["int8", "fp8"]),
             "dtype": rng.choice(["float32", "bfloat16", "float16"]), "cached_min": 0,
             "cached_max": _log(rng, 40, 65536), "new": 1, "ragged": rng.random() < 0.5,
             "causal": rng.random() < 0.8, "track": False, "budget": 0, "recent": 0}
        c["cached_min"] = int(c["cached_max"] * rng.choice([0.0, 0.5, 0.99]))
        if kind == "append":
            c["new"] = _log(rng, 1, 4096)
        elif kind == "attend":
            c["new"] = rng.choice([1, 1, _log(rng, 1, 2048)])
            c["track"] = rng.random() < 0.4
        else:
            c["budget"] = max(1, int(c["cached_max"] * rng.uniform(0.1, 0.9)))
            c["recent"] = int(c["budget"] * rng.uniform(0.0, 1.0))
            c["ragged"] = False
        c["ragged"] = c["ragged"] and c["new"] > 1
        w = work(c)
        pool = c["batch"] * (c["cached_max"] + c["new"]) * kv * c["head_dim"]
        scores = c["batch"] * c["heads"] * c["new"] * (c["cached_max"] + c["new"])
        if (w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and pool <= 6e8
                and (kind != "attend" or scores <= 1.1e9)):
            return c


def work(case):
    """Bytes and products of one pass at the expected lengths."""
    B, T, D, H, Hq = (case[k] for k in ("batch", "new", "head_dim", "kv_heads", "heads"))
    size = 4 if case["dtype"] == "float32" else 2
    cached = (case["cached_min"] + case["cached_max"]) / 2
    new = T / 2 if case["ragged"] else T
    if case["kind"] == "append":
        # read the chunk, write its codes, read the touched pages and write their values
        touched = new + (case["block"] / 2 if case["cached_max"] else 0)
        return {"bytes": 2.0 * B * H * D * (new * (size + 1) + touched * (1 + size)),
                "flops": 2.0 * B * H * D * new}
    if case["kind"] == "evict":
        kept = min(case["budget"], cached)
        # all weights once, the kept tokens' codes and weights moved, their values read back
        return {"bytes": B * H * (4.0 * cached + 8 * kept + 4 * kept + 2 * D * kept * (3 + size)),
                "flops": 4.0 * B * H * D * kept}
    keys = cached + new
    pairs = new * (cached + (new + 1) / 2 if case["causal"] else keys)
    return {"bytes": B * (2.0 * H * D * keys + 2 * Hq * T * D * size
                          + (8.0 * H * keys if case["track"] else 0)),
            "flops": B * Hq * pairs * D * (6.0 if case["track"] and T > 1 else 4.0)}


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dev = torch.device("cuda")
    B, T, D, H, Hq, P = (case[k] for k in ("batch", "new", "head_dim", "kv_heads", "heads", "block"))
    dtype = getattr(torch, case["dtype"])
    lens = torch.randint(case["cached_min"], case["cached_max"] + 1, (B,), generator=g, device=dev,
                         dtype=torch.int32)
    counts = torch.full((B,), T, dtype=torch.int32, device=dev)
    if case["ragged"]:
        counts = torch.randint(0, T + 1, (B,), generator=g, device=dev, dtype=torch.int32)
    held = case["cached_max"] + (T if case["kind"] != "evict" else 0)
    blocks = held // P + 2          # a chunk that starts inside a page reaches one more
    spare = -(-case["budget"] // P) if case["kind"] == "evict" else 0
    pages = B * (blocks + spare)
    order = torch.randperm(pages, generator=g, device=dev).to(torch.int32).view(B, blocks + spare)
    k_codes, v_codes, scale = _pools(case, pages, g)
    state = {"case": dict(case), "k": k_codes, "v": v_codes, "scale": scale, "lens": lens,
             "counts": counts, "table": order[:, :blocks].contiguous(), "weight": None}
    if case["kind"] == "evict" or case["track"]:
        # heavy-tailed sums of attention weights, many of the light ones equal
        w = torch.randn(pages, H, P, generator=g, device=dev)
        state["weight"] = torch.floor(torch.exp(2 * w) * 64) / 64
    if case["kind"] == "evict":
        state["table_out"] = order[:, blocks:].contiguous()
        return state
    # the heads of a fused projection [B, T, 3 * heads, D], seen as [B, heads, T, D]
    qkv = torch.randn(B, T, Hq + 2 * H, D, generator=g, device=dev)
    qkv[:, :, Hq:Hq + H] *= 1.5
    qkv = qkv.to(dtype)
    state["q"] = qkv[:, :, :Hq].permute(0, 2, 1, 3)
    state["k_new"] = qkv[:, :, Hq:Hq + H].permute(0, 2, 1, 3)
    state["v_new"] = qkv[:, :, Hq + H:].permute(0, 2, 1, 3)
    state["read_from"] = (lens // P * P).to(torch.int32)
    if case["kind"] == "attend":
        # the new tokens are in the cache before they are attended to: the pool holds them already
        del state["k_new"], state["v_new"], state["read_from"]
    return state


def _pools(case, pages, g):
    """Codes and scales of normal values whose spread differs from head to head, block by block."""
    D, H, P = case["head_dim"], case["kv_heads"], case["block"]
    dev, qmax, kind = torch.device("cuda"), QMAX[case["format"]], CODE[case["format"]]
    codes = [torch.empty(pages, H, P, D, dtype=kind, device=dev) for _ in range(2)]
    scale = torch.empty(pages, H, 2, device=dev)
    step = max(1, (1 << 25) // (H * P * D))
    for i, pool in enumerate(codes):
        spread = torch.rand(1, H, 1, 1, generator=g, device=dev) + 0.5
        for a in range(0, pages, step):
            n = min(step, pages - a)
            x = torch.randn(n, H, P, D, generator=g, device=dev) * spread
            s = x.abs().amax(dim=(2, 3)) / qmax
            scale[a:a + n, :, i] = s
            x = (x / s[:, :, None, None]).clamp(-qmax, qmax)
            pool[a:a + n] = (x.round() if case["format"] == "int8" else x).to(kind)
    return codes[0], codes[1], scale


# ---------------------------------------------------------------- the operators


def run(state):
    case = state["case"]
    if own:
        from techjam2026_b200 import ops
        if "cache" not in state:        # the handle that a serving loop makes once and keeps
            state["cache"] = ops.KV8Cache(state["k"], state["v"], state["scale"], state["table"],
                                          state["lens"], state["weight"])
        cache = state["cache"]
        dtype = getattr(torch, case["dtype"])
        if case["kind"] == "append":
            ops.kv8_append(cache, state["k_new"], state["v_new"], counts=state["counts"])
            return ops.kv8_read(cache, case["new"] + case["block"] - 1, start=state["read_from"],
                                counts=state["counts"], dtype=dtype)
        if case["kind"] == "attend":
            out = ops.kv8_attention(state["q"], cache, counts=state["counts"],
                                    causal=case["causal"], track=case["track"])
            return (out, state["weight"]) if case["track"] else out
        kept, short = ops.kv8_evict(cache, state["table_out"], case["budget"], case["recent"])
        k, v = ops.kv8_read(short, case["budget"], dtype=dtype)
        return kept, short.lens, state["weight"][state["table_out"].long()], k, v
    if case["kind"] == "append":
        _append(state)
        return _read(state, state["table"], state["read_from"], state["lens"] + state["counts"],
                     case["new"] + case["block"] - 1)
    if case["kind"] == "attend":
        out = _attend(state)
        return (out, state["weight"]) if case["track"] else out
    return _evict(state)


def _gather(pool, pages):
    """Pages of a pool of any type, the 8-bit ones moved as bytes."""
    return pool.view(torch.uint8)[pages].view(pool.dtype) if pool.element_size() == 1 else pool[pages]


def _scale_of(amax, qmax):
    s = amax * (1.0 / qmax)
    s = torch.where(torch.isfinite(amax), s, torch.full_like(s, float("nan")))
    return torch.where(s < TINY, torch.zeros_like(s), s)


def _inverse(s):
    return torch.where(s > 0, 1.0 / s, torch.zeros_like(s))


def _encode(x, fmt):
    x = torch.nan_to_num(x, nan=0.0).clamp(-QMAX[fmt], QMAX[fmt])
    return (x.round() if fmt == "int8" else x).to(CODE[fmt])


def _append(state):
    case = state["case"]
    B, T, P, fmt = case["batch"], case["new"], case["block"], case["format"]
    lens, counts = state["lens"].long(), state["counts"].long()
    n = (T - 1) // P + 2            # pages that a chunk can reach
    slot = torch.arange(P, device=lens.device)
    block = (lens // P)[:, None] + torch.arange(n, device=lens.device)          # [B, n]
    page = torch.gather(state["table"].long(), 1, block.clamp(max=state["table"].shape[1] - 1))
    pos = block[:, :, None] * P + slot                                           # [B, n, P]
    token = pos - lens[:, None, None]
    is_new = (token >= 0) & (token < counts[:, None, None])
    is_old = token < 0
    touched = is_new.any(dim=2) & (block < state["table"].shape[1])              # [B, n]
    at = token.clamp(0, T - 1)
    b = torch.arange(B, device=lens.device)[:, None, None]
    pages, keep = page[touched], (is_new | is_old)[touched][:, None, :, None]
    fresh = is_new[touched][:, None, :, None]
    held = is_old.any(dim=2)[touched][:, None]
    new_scale = state["scale"][pages].clone()

    def fill(pool, x, which):
        x = x.permute(0, 2, 1, 3)[b, at][touched].permute(0, 2, 1, 3).float()    # [pages, H, P, D]
        x = torch.where(fresh, x, torch.zeros_like(x))
        was = state["scale"][pages][:, :, which]
        was = torch.where(held, was, torch.zeros_like(was))
        s = torch.maximum(was, _scale_of(x.abs().amax(dim=(2, 3)), QMAX[fmt]))
        inv = _inverse(s)
        codes = _gather(pool, pages)
        grown = ((s != was) & held)[:, :, None, None]
        moved = _encode(codes.float() * (was * inv)[:, :, None, None], fmt)
        old = torch.where(grown, moved.view(torch.uint8), codes.view(torch.uint8))
        put = torch.where(fresh, _encode(x * inv[:, :, None, None], fmt).view(torch.uint8), old)
        put = torch.where(keep, put, codes.view(torch.uint8))
        pool.view(torch.uint8)[pages] = put
        new_scale[:, :, which] = s

    fill(state["k"], state["k_new"], 0)
    fill(state["v"], state["v_new"], 1)
    state["scale"][pages] = new_scale


def _read(state, table, start, end, n):
    case = state["case"]
    P, dtype = case["block"], getattr(torch, case["dtype"])
    pos = start.long()[:, None] + torch.arange(n, device=start.device)           # [B, n]
    inside = (pos < end.long()[:, None])[:, :, None, None]
    pos = torch.where(inside[:, :, 0, 0], pos, torch.zeros_like(pos))
    page = torch.gather(table.long(), 1, pos // P)
    s = state["scale"][page]                                                     # [B, n, H, 2]

    def values(pool, which):
        bytes_ = pool.view(torch.uint8)[page, :, pos % P]                        # [B, n, H, D]
        x = bytes_.view(pool.dtype).float() * s[:, :, :, which, None]
        return torch.where(inside, x, torch.zeros_like(x)).permute(0, 2, 1, 3).to(dtype).contiguous()

    return values(state["k"], 0), values(state["v"], 1)


def _attend(state):
    case = state["case"]
    B, T, D, H, Hq, P = (case[k] for k in ("batch", "new", "head_dim", "kv_heads", "heads", "block"))
    G, table = Hq // H, state["table"].long()
    L = table.shape[1] * P
    lens, counts = state["lens"].long(), state["counts"].long()
    key = torch.arange(L, device=lens.device)
    row = torch.arange(T, device=lens.device)
    held = key[None] < (lens + counts)[:, None]                                  # [B, L]
    s = state["scale"][table]                                                    # [B, n, H, 2]

    def values(pool, which):
        x = _gather(pool, table).float() * s[:, :, :, which, None, None]
        x = x.permute(0, 2, 1, 3, 4).reshape(B, H, L, D)
        return torch.where(held[:, None, :, None], x, torch.zeros_like(x))

    q = state["q"].float().reshape(B, H, G, T, D).reshape(B, H, G * T, D) * D ** -0.5
    scores = torch.matmul(q, values(state["k"], 0).transpose(2, 3)).view(B, H, G, T, L)
    seen = held[:, None, :] & (row[None, :] < counts[:, None])[:, :, None]       # [B, T, L]
    if case["causal"]:
        seen = seen & (key[None, None] <= (lens[:, None] + row)[:, :, None])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    p = scores.sub_(torch.where(torch.isinf(top), torch.zeros_like(top), top)).exp_()
    total = p.sum(dim=-1, keepdim=True)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(p.view(B, H, G * T, L), values(state["v"], 1)).view(B, Hq, T, D)
    if case["track"]:
        w = p.sum(dim=(2, 3)).view(B, H, -1, P).permute(0, 2, 1, 3)              # [B, n, H, P]
        state["weight"].index_put_((table,), w, accumulate=True)
    return out.to(getattr(torch, case["dtype"]))


def _evict(state):
    case = state["case"]
    B, D, H, P, fmt = (case[k] for k in ("batch", "head_dim", "kv_heads", "block", "format"))
    budget, table, table_out = case["budget"], state["table"].long(), state["table_out"].long()
    L = table.shape[1] * P
    lens = state["lens"].long()[:, None, None]
    pos = torch.arange(L, device=lens.device)[None, None]
    w = state["weight"][table].permute(0, 2, 1, 3).reshape(B, H, L)
    late = (pos >= lens - case["recent"]) & (pos < lens)
    rank_by = torch.where(late, torch.full_like(w, math.inf), w)
    rank_by = torch.where(pos < lens, rank_by, torch.full_like(w, -1.0))
    order = torch.sort(rank_by, dim=-1, descending=True, stable=True).indices
    rank = torch.empty_like(order).scatter_(2, order, pos.expand(B, H, L).contiguous())
    keep = (rank < budget) & (pos < lens)
    kept = torch.where(keep, pos, torch.full_like(pos, L)).sort(dim=-1).values
    n_out = table_out.shape[1] * P
    pad = max(0, n_out - L)
    kept = torch.nn.functional.pad(kept, (0, pad), value=L)[:, :, :n_out]       # [B, H, n_out]
    slot = torch.arange(n_out, device=lens.device)
    real = (kept < L) & (slot < budget)
    src = torch.where(real, kept, torch.zeros_like(kept))
    page = torch.gather(table[:, None].expand(B, H, -1), 2, src // P)            # [B, H, n_out]
    head = torch.arange(H, device=lens.device)[None, :, None]
    scale = state["scale"][page, head]                                           # [B, H, n_out, 2]
    blocked = (B, H, n_out // P, P)
    real_b = real.view(blocked)

    def move(pool, which):
        x = pool.view(torch.uint8)[page, head, src % P].view(pool.dtype).float()
        x = torch.where(real[..., None], x * scale[..., which, None], torch.zeros_like(x))
        x = x.view(*blocked, D)
        s = _scale_of(x.abs().amax(dim=(3, 4)), QMAX[fmt])                       # [B, H, n]
        codes = _encode(x * _inverse(s)[..., None, None], fmt).view(torch.uint8)
        codes = codes.permute(0, 2, 1, 3, 4)
        live = real_b.permute(0, 2, 1, 3)
        was = pool.view(torch.uint8)[table_out]
        pool.view(torch.uint8)[table_out] = torch.where(live[..., None], codes, was)
        used = live.any(dim=3)
        state["scale"][table_out, :, which] = torch.where(used, s.permute(0, 2, 1),
                                                          state["scale"][table_out][..., which])

    move(state["k"], 0)
    move(state["v"], 1)
    moved = state["weight"][page, head, src % P].view(blocked).permute(0, 2, 1, 3)
    state["weight"][table_out] = torch.where(real_b.permute(0, 2, 1, 3), moved,
                                             state["weight"][table_out])
    new_lens = state["lens"].clamp(max=budget)
    k, v = _read(state, state["table_out"], torch.zeros_like(new_lens), new_lens, budget)
    kept = torch.where(real, kept, torch.full_like(kept, -1))[:, :, :budget].to(torch.int32)
    return kept.contiguous(), new_lens, state["weight"][table_out], k, v


# ---------------------------------------------------------------- in 64 bits


def _round64(x, fmt):
    """The nearest code of each value, ties to even."""
    if fmt == "int8":
        return torch.round(x).clamp(-127, 127)
    x = x.clamp(-448, 448)
    _, e = torch.frexp(x)
    step = torch.ldexp(torch.ones_like(x), (e - 1).clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _values64(state, pool, which, table, b, end):
    """[H, end, D]: what sequence b's first `end` tokens hold."""
    P = state["case"]["block"]
    page = table[b, : -(-end // P)].long()
    x = _gather(pool, page).to(torch.float32).double()
    x = x * state["scale"][page][:, :, which].double()[:, :, None, None]
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :end]


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _append64, "attend": _attend64, "evict": _evict64}[case["kind"]](state)


def _append64(state):
    case = state["case"]
    B, T, P, D, H, fmt = (case[k] for k in ("batch", "new", "block", "head_dim", "kv_heads", "format"))
    n, qmax = T + P - 1, QMAX[fmt]
    outs = []
    for pool, x, which in ((state["k"], state["k_new"], 0), (state["v"], state["v_new"], 1)):
        out = torch.zeros(B, H, n, D, dtype=torch.float64, device=x.device)
        for b in range(B):
            have, count = int(state["lens"][b]), int(state["counts"][b])
            off, page = have % P, state["table"][b].long()
            if count == 0:
                if off:
                    out[b, :, :off] = _values64(state, pool, which, state["table"][b:b + 1], 0,
                                                have)[:, have - off:]
                continue
            new = x[b, :, :count].double()
            codes = _gather(pool, page[have // P]).to(torch.float32).double()[:, :off]
            was = state["scale"][page[have // P], :, which].double() * (1.0 if off else 0.0)
            first = min(P - off, count)
            s = torch.maximum(was, new[:, :first].abs().amax(dim=(1, 2)) / qmax)
            ratio = torch.where(s > 0, was / s, torch.zeros_like(s))[:, None, None]
            old = torch.where((s != was)[:, None, None], _round64(codes * ratio, fmt), codes)
            out[b, :, :off] = old * s[:, None, None]
            inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))[:, None, None]
            out[b, :, off:off + first] = _round64(new[:, :first] * inv, fmt) * s[:, None, None]
            rest = new[:, first:]
            if rest.shape[1]:
                full = -(-rest.shape[1] // P) * P
                y = torch.nn.functional.pad(rest, (0, 0, 0, full - rest.shape[1])).view(H, -1, P, D)
                s = y.abs().amax(dim=(2, 3), keepdim=True) / qmax
                inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
                y = (_round64(y * inv, fmt) * s).view(H, full, D)
                out[b, :, off + first:off + count] = y[:, :rest.shape[1]]
        outs.append(out)
    return tuple(outs)


def _attend64(state):
    case = state["case"]
    B, T, D, H, Hq, P = (case[k] for k in ("batch", "new", "head_dim", "kv_heads", "heads", "block"))
    G, dev = Hq // H, state["lens"].device
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=dev)
    weight = state["weight"].double() if case["track"] else None
    for b in range(B):
        have, count = int(state["lens"][b]), int(state["counts"][b])
        end = have + count
        if not count:
            continue
        k = _values64(state, state["k"], 0, state["table"], b, end)
        v = _values64(state, state["v"], 1, state["table"], b, end)
        for h in range(H):
            q = state["q"][b, h * G:(h + 1) * G, :count].double()                # [G, count, D]
            s = q @ k[h].T / math.sqrt(D)
            if case["causal"]:
                seen = torch.arange(end, device=dev)[None] <= have + torch.arange(count, device=dev)[:, None]
                s.masked_fill_(~seen, -math.inf)
            p = torch.softmax(s, dim=-1)
            out[b, h * G:(h + 1) * G, :count] = p @ v[h]
            if weight is not None:
                w = torch.nn.functional.pad(p.sum(dim=(0, 1)), (0, -end % P)).view(-1, P)
                weight[state["table"][b, :w.shape[0]].long(), h] += w
    return out if weight is None else (out, weight)


def _evict64(state):
    case = state["case"]
    B, D, H, P, fmt = (case[k] for k in ("batch", "head_dim", "kv_heads", "block", "format"))
    budget, dev = case["budget"], state["lens"].device
    n = state["table_out"].shape[1]
    kept = torch.full((B, H, budget), -1, dtype=torch.float64, device=dev)
    weight = state["weight"][state["table_out"].long()].double()                 # [B, n, H, P]
    values = [torch.zeros(B, H, budget, D, dtype=torch.float64, device=dev) for _ in range(2)]
    lens = torch.zeros(B, dtype=torch.float64, device=dev)
    for b in range(B):
        have = int(state["lens"][b])
        m = min(have, budget)
        lens[b] = m
        if not m:
            continue
        page = state["table"][b].long()
        w = state["weight"][page].permute(1, 0, 2).reshape(H, -1)[:, :have].double()
        late = min(case["recent"], have)
        order = torch.argsort(w[:, :have - late], dim=1, descending=True, stable=True)
        order = order[:, :m - late] if m > late else order[:, :0]
        tail = torch.arange(have - min(late, m), have, device=dev).expand(H, -1)
        pick = torch.cat([order, tail], dim=1).sort(dim=1).values                # [H, m]
        kept[b, :, :m] = pick.double()
        moved = torch.gather(w, 1, pick)
        full = torch.nn.functional.pad(moved, (0, n * P - m)).view(H, n, P).permute(1, 0, 2)
        live = (torch.arange(n * P, device=dev) < m).view(n, 1, P)
        weight[b] = torch.where(live, full, weight[b])
        for which, pool in enumerate((state["k"], state["v"])):
            x = _values64(state, pool, which, state["table"], b, have)
            x = torch.gather(x, 1, pick[..., None].expand(H, m, D))
            x = torch.nn.functional.pad(x, (0, 0, 0, -m % P)).view(H, -1, P, D)
            s = x.abs().amax(dim=(2, 3), keepdim=True) / QMAX[fmt]
            inv = torch.where(s > 0, 1 / s, torch.zeros_like(s))
            values[which][b, :, :m] = (_round64(x * inv, fmt) * s).view(H, -1, D)[:, :m]
    return kept, lens, weight, values[0], values[1]
