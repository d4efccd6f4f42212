"""The operators that serve several continuations of one prompt, as cases to be measured.

Sequences of an 8-bit key/value cache (perf/operators.py) that continue one
prompt share its pages. Three kinds of case:

  copy    pages of the layers' pools are copied (kv8_copy): the pages that a
          fork does not share, a compaction, a move into another pool;
  attend  the newest tokens of a batch whose groups share their leading pages
          read the cache, the shared pages once (kv8_attention_shared);
  select  beams and vocabulary give the best continuations (beam_select).

`run` computes them with elementary torch operations where `own` is false, and
calls techjam2026_b200.ops where it is true. `exact` restates them in 64 bits.
"""
import math

import torch

own = False

QMAX = {"int8": 127.0, "fp8": 448.0}
CODE = {"int8": torch.int8, "fp8": torch.float8_e4m3fn}


def listed():
    copy = {"kind": "copy", "layers": 1, "kv_heads": 8, "head_dim": 64, "block": 64,
            "format": "int8", "pages": 0, "pairs": 0, "partial": False, "record": False,
            "other": False}
    attend = {"kind": "attend", "batch": 1, "groups": 1, "even": True, "heads": 8, "kv_heads": 8,
              "head_dim": 64, "block": 64, "format": "int8", "dtype": "float32", "shared_min": 0,
              "shared_max": 0, "own_min": 0, "own_max": 0, "new": 1, "ragged": False,
              "causal": True}
    select = {"kind": "select", "batch": 1, "beams": 4, "vocab": 0, "take": 4,
              "dtype": "float32", "ended": 0.0, "banned": 0.0}

    def case(name, base, **kw):
        return {"name": name, **base, **kw}

    return [
        # a step of beam search forks 8 sequences of a 6-layer stack: their last, half full pages
        case("copy, fork of 8 beams", copy, layers=6, pages=128, pairs=8, partial=True),
        # a pool of a 4-layer stack (12 heads of 64) with its weight records is compacted
        case("copy, compaction", copy, layers=4, kv_heads=12, pages=4000, pairs=1500, record=True),
        # long grouped-head sequences move to another pool
        case("copy, into another pool", copy, layers=2, head_dim=128, block=128, format="fp8",
             pages=2500, pairs=1999, other=True),
        # one token of 4 beams of a short prompt: latency
        case("token, 4 beams", attend, batch=4, shared_min=192, shared_max=448, own_max=63),
        # one token of 64 samples of one prompt (12 heads of 64), fp32 as the stack
        case("token, 64 samples of one prompt", attend, batch=64, heads=12, kv_heads=12,
             shared_min=1536, shared_max=2047, own_max=300),
        # uneven groups of beams on prompts of their own, grouped heads, bf16 over e4m3
        case("token, uneven groups", attend, batch=61, groups=8, even=False, heads=32, head_dim=128,
             format="fp8", dtype="bfloat16", shared_min=2048, shared_max=12000, own_max=700),
        # many samples of one very long document, fp16: the largest
        case("token, long document", attend, batch=64, heads=32, head_dim=128, block=128,
             dtype="float16", shared_min=31000, shared_max=32768, own_max=500),
        # ragged questions about long documents, as chunks, bf16
        case("chunks, questions on two documents", attend, batch=16, groups=2, heads=16,
             kv_heads=16, dtype="bfloat16", shared_min=8000, shared_max=16384, own_max=130,
             new=120, ragged=True),
        # 4 beams of one sequence, an ordinary vocabulary
        case("select, 4 beams", select, vocab=32000),
        # a batch of beams, an odd vocabulary, some beams ended, two candidates a beam
        case("select, batch", select, batch=24, beams=8, vocab=50021, take=16, ended=0.1,
             banned=0.01),
        # a wide batch over a large vocabulary in bf16, where many logits are equal: the largest
        case("select, large vocabulary", select, batch=64, beams=8, vocab=128000, take=16,
             dtype="bfloat16", ended=0.05),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    top = [work(c) for c in listed()]
    most = {k: max(w[k] for w in top) for k in ("bytes", "flops")}
    while True:
        kind = rng.choice(["copy", "attend", "attend", "attend", "select", "select"])
        if kind == "select":
            beams = rng.choice([1, 2, 3, 4, 5, 8, 12, 16])
            c = {"kind": kind, "batch": _log(rng, 1, 64), "beams": beams,
                 "vocab": _log(rng, 500, 200000),
                 "take": rng.choice([beams, 2 * beams, rng.randint(1, 64)]),
                 "dtype": rng.choice(["float32", "bfloat16", "float16"]),
                 "ended": rng.choice([0.0, 0.1, 0.4]), "banned": rng.choice([0.0, 0.02])}
            w = work(c)
            if w["bytes"] <= 1.4e8:
                return c
            continue
        kv = rng.choice([1, 2, 3, 4, 8, 12, 16])
        c = {"kind": kind, "kv_heads": kv, "head_dim": rng.choice([16, 32, 64, 64, 128]),
             "block": rng.choice([16, 32, 64, 128]), "format": rng.choice(["int8", "fp8"])}
        page = 2 * kv * c["head_dim"] * c["block"]
        if kind == "copy":
            pairs = _log(rng, 1, 4000)
            c.update({"layers": rng.randint(1, 8), "pairs": pairs,
                      "pages": 2 * pairs + rng.randint(0, pairs + 20),
                      "partial": rng.random() < 0.5, "record": rng.random() < 0.3,
                      "other": rng.random() < 0.3})
            if page * c["layers"] * c["pages"] <= 2e9:
                return c
            continue
        group = rng.choice([1, 1, 2, 4, 8])
        batch = _log(rng, 1, 64)
        c.update({"batch": batch, "groups": rng.choice([1, 1, max(1, batch // 4), batch]),
                  "even": rng.random() < 0.5, "heads": kv * group,
                  "dtype": rng.choice(["float32", "bfloat16", "float16"]),
                  "shared_max": _log(rng, 20, 33000), "own_max": _log(rng, 1, 2000),
                  "new": rng.choice([1, 1, 1, _log(rng, 1, 300)]), "causal": rng.random() < 0.8})
        c["shared_min"] = int(c["shared_max"] * rng.choice([0.0, 0.5, 0.95]))
        c["own_min"] = int(c["own_max"] * rng.choice([0.0, 0.0, 0.9]))
        c["ragged"] = c["new"] > 1 and rng.random() < 0.5
        w = work(c)
        held = batch * (c["shared_max"] + c["own_max"] + c["new"])
        scores = c["heads"] * c["new"] * held
        pool = (c["groups"] * c["shared_max"] + batch * (c["own_max"] + c["new"] + 3 * c["block"]))
        if (w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and scores <= 1.0e9
                and held * kv * c["head_dim"] <= 2.2e9 and pool * kv * c["head_dim"] <= 4e8):
            return c


def work(case):
    """Bytes and operations of one pass at the expected lengths."""
    if case["kind"] == "select":
        n = 1.0 * case["batch"] * case["beams"] * case["vocab"] * (1 - case["ended"])
        return {"bytes": n * (4 if case["dtype"] == "float32" else 2), "flops": 3 * n}
    H, D, P = case["kv_heads"], case["head_dim"], case["block"]
    if case["kind"] == "copy":
        tokens = (P + 1) / 2 if case["partial"] else P
        page = H * (tokens * (2 * D + (4 if case["record"] else 0)) + 8)
        return {"bytes": 2.0 * case["layers"] * case["pairs"] * page, "flops": 0.0}
    B, T, Hq = case["batch"], case["new"], case["heads"]
    size = 4 if case["dtype"] == "float32" else 2
    common = (case["shared_min"] + case["shared_max"]) / 2
    new = (T + 1) / 2 if case["ragged"] else T
    mine = (case["own_min"] + case["own_max"]) / 2 + new
    pairs = B * new * (common + mine - ((new - 1) / 2 if case["causal"] else 0))
    return {"bytes": 2.0 * H * D * (case["groups"] * common + B * mine) + 2.0 * B * Hq * T * D * size,
            "flops": 4.0 * D * Hq * pairs}


# ---------------------------------------------------------------- inputs


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return {"copy": _prepare_copy, "attend": _prepare_attend,
            "select": _prepare_select}[case["kind"]](case, g)


def _codes(shape, fmt, g):
    """Codes as a block of normal values gives them: their largest is the largest code."""
    out = torch.empty(shape, dtype=CODE[fmt], device="cuda")
    step = max(1, (1 << 25) // math.prod(shape[1:]))
    for a in range(0, shape[0], step):
        n = min(step, shape[0] - a)
        x = torch.randn((n, *shape[1:]), generator=g, device="cuda")
        x = x * (QMAX[fmt] / x.abs().amax(dim=(2, 3), keepdim=True))
        out[a:a + n] = (x.round() if fmt == "int8" else x).to(CODE[fmt])
    return out


def _pool(case, pages, g, record):
    H, P, D = case["kv_heads"], case["block"], case["head_dim"]
    spread = torch.rand(1, H, 2, generator=g, device="cuda") + 0.5
    near = 1 + 0.1 * torch.rand(pages, H, 2, generator=g, device="cuda")
    return {"k": _codes((pages, H, P, D), case["format"], g),
            "v": _codes((pages, H, P, D), case["format"], g),
            "scale": spread * near * 3.5 / QMAX[case["format"]],
            "weight": torch.rand(pages, H, P, generator=g, device="cuda") if record else None}


def _prepare_copy(case, g):
    pages, n = case["pages"], case["pairs"]
    order = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    spare = order[n:2 * n]
    if case["other"]:
        spare = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[:n]
    state = {"case": dict(case), "src": order[:n].contiguous(), "dst": spare.contiguous(),
             "tokens": None,
             "pools": [_pool(case, pages, g, case["record"]) for _ in range(case["layers"])],
             "table": torch.zeros(1, 1, dtype=torch.int32, device="cuda"),
             "lens": torch.zeros(1, dtype=torch.int32, device="cuda")}
    if case["partial"]:
        state["tokens"] = torch.randint(1, case["block"] + 1, (n,), generator=g, device="cuda",
                                        dtype=torch.int32)
    state["into"] = state["pools"]
    if case["other"]:
        state["into"] = [{k: None if t is None else torch.zeros_like(t) for k, t in p.items()}
                         for p in state["pools"]]
    return state


def _prepare_attend(case, g):
    B, N, T, P = case["batch"], case["groups"], case["new"], case["block"]
    D, H, Hq, dev = case["head_dim"], case["kv_heads"], case["heads"], torch.device("cuda")

    def between(lo, hi, n):
        return torch.randint(lo, hi + 1, (n,), generator=g, device=dev, dtype=torch.int32)

    # which sequences make a group: equal shares, or cuts anywhere (some groups may be empty)
    if case["even"]:
        starts = (torch.arange(N + 1, device=dev) * B // N).to(torch.int32)
    else:
        starts = torch.cat([between(0, 0, 1), between(0, B, N - 1).sort().values, between(B, B, 1)])
    group = (torch.arange(B, device=dev)[:, None] >= starts[None, 1:]).sum(dim=1)
    shared = between(case["shared_min"], case["shared_max"], N) // P * P
    lens = (shared[group] + between(case["own_min"], case["own_max"], B)).to(torch.int32)
    counts = between(0, T, B) if case["ragged"] else between(T, T, B)
    front, back = case["shared_max"] // P, (case["own_max"] + T) // P + 1
    order = torch.randperm(N * front + B * back, generator=g, device=dev).to(torch.int32)
    first = torch.cat([order[:N * front].view(N, front),
                       torch.zeros(N, 1, dtype=torch.int32, device=dev)], dim=1)[group]
    rest = order[N * front:].view(B, back)
    at = torch.arange(front + back, device=dev)[None] - (shared[group] // P)[:, None]
    table = torch.where(at < 0, torch.gather(torch.nn.functional.pad(first, (0, back - 1)), 1,
                                             (at + (shared[group] // P)[:, None]).long()),
                        torch.gather(rest, 1, at.clamp(0, back - 1).long()))
    state = {"case": dict(case), **_pool(case, N * front + B * back, g, False),
             "table": table.contiguous(), "lens": lens, "counts": counts,
             "starts": starts.contiguous(), "shared": shared.to(torch.int32)}
    # the query heads of a fused projection [B, T, heads + 2 kv_heads, D], seen as [B, heads, T, D]
    qkv = torch.randn(B, T, Hq + 2 * H, D, generator=g, device=dev).to(getattr(torch, case["dtype"]))
    state["q"] = qkv[:, :, :Hq].permute(0, 2, 1, 3)
    return state


def _prepare_select(case, g):
    B, K, V = case["batch"], case["beams"], case["vocab"]
    dev, dtype = torch.device("cuda"), getattr(torch, case["dtype"])
    logits = torch.empty(B, K, V, dtype=dtype, device=dev)
    ban = torch.rand(V, generator=g, device=dev) < case["banned"]
    # each row with a few likely tokens over a wide rest, more or less peaked
    for b in range(B):
        x = torch.randn(K, V, generator=g, device=dev)
        x *= 1.5 + 2 * torch.rand(K, 1, generator=g, device=dev)
        logits[b] = x.masked_fill(ban, -math.inf).to(dtype)
    scores = -20 * torch.rand(B, 1, generator=g, device=dev) - 3 * torch.rand(B, K, generator=g,
                                                                            device=dev)
    ended = torch.rand(B, K, generator=g, device=dev) < case["ended"]
    return {"case": dict(case), "logits": logits, "scores": scores,
            "ended": ended if case["ended"] else None}


# ---------------------------------------------------------------- the operators


def run(state):
    case = state["case"]
    if own:
        from techjam2026_b200 import ops
        if case["kind"] == "select":
            return ops.beam_select(state["logits"], state["scores"], case["take"],
                                   ended=state["ended"], pad=0)
        if "cache" not in state:        # the handles that a serving loop makes once and keeps
            state["cache"], state["to"] = _handles(state, ops)
        if case["kind"] == "copy":
            ops.kv8_copy(state["cache"], state["src"], state["dst"], tokens=state["tokens"],
                         into=state["to"])
            return _held(state)
        return ops.kv8_attention_shared(
            state["q"], state["cache"], state["starts"], state["shared"], counts=state["counts"],
            causal=case["causal"], max_shared=case["shared_max"],
            max_own=case["own_max"] + case["new"], return_lse=True)
    if case["kind"] == "copy":
        return _copy(state)
    return _attend(state) if case["kind"] == "attend" else _select(state)


def _handles(state, ops):
    if state["case"]["kind"] == "attend":
        return ops.KV8Cache(state["k"], state["v"], state["scale"], state["table"],
                            state["lens"]), None

    def layer(p):
        return ops.KV8Cache(p["k"], p["v"], p["scale"], state["table"], state["lens"], p["weight"])

    cache = [layer(p) for p in state["pools"]]
    return cache, [layer(p) for p in state["into"]] if state["case"]["other"] else None


def _held(state):
    """What the pools hold that were copied into: codes as bytes, scales, records."""
    return [{k: t.view(torch.int8) if k in "kv" else t for k, t in p.items() if t is not None}
            for p in state["into"]]


def _copy(state):
    case = state["case"]
    src, dst, P = state["src"].long(), state["dst"].long(), case["block"]
    if case["partial"]:
        put = (torch.arange(P, device=src.device) < state["tokens"][:, None])[:, None]   # [n, 1, P]

    def move(x, y, token_dims):
        new = x[src]
        if case["partial"] and token_dims:
            keep = put[..., None] if token_dims == 2 else put
            new = torch.where(keep, new, y[dst])
        y[dst] = new

    def layer(p, q):
        for k in "kv":
            move(p[k].view(torch.int8), q[k].view(torch.int8), 2)
        move(p["scale"], q["scale"], 0)
        if case["record"]:
            move(p["weight"], q["weight"], 1)

    list(map(layer, state["pools"], state["into"]))
    return _held(state)


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
        x = pool.view(torch.uint8)[table].view(pool.dtype).float() * s[:, :, :, which, None, None]
        x = x.permute(0, 2, 1, 3, 4).reshape(B, H, L, D)
        return x.masked_fill_(~held[:, None, :, None], 0.0)

    q = state["q"].float().reshape(B, H, G * T, D) * D ** -0.5
    scores = torch.matmul(q, values(state["k"], 0).transpose(2, 3)).view(B, H, G, T, L)
    seen = held[:, None, :] & (row[None, :] < counts[:, None])[:, :, None]       # [B, T, L]
    if case["causal"]:
        seen = seen & (key[None, None] <= (lens[:, None] + row)[:, :, None])
    scores = scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(dim=-1, keepdim=True)
    top = torch.where(torch.isinf(top), torch.zeros_like(top), top)
    p = scores.sub_(top).exp_()
    total = p.sum(dim=-1, keepdim=True)
    lse = (top + total.log()).view(B, Hq, T)
    p = p.div_(torch.where(total > 0, total, torch.ones_like(total)))
    out = torch.matmul(p.view(B, H, G * T, L), values(state["v"], 1)).view(B, Hq, T, D)
    return out.to(getattr(torch, case["dtype"])), lse


def _select(state):
    case = state["case"]
    B, K, V, n = case["batch"], case["beams"], case["vocab"], case["take"]
    # which of two candidates is the better one is decided by small differences: in 64 bits
    x = state["logits"].double()
    top = x.amax(dim=2, keepdim=True)
    lse = top + (x - top).exp_().sum(dim=2, keepdim=True).log()
    c = x.sub_(lse).add_(state["scores"].double()[:, :, None])
    if state["ended"] is not None:
        c.masked_fill_(state["ended"][:, :, None], -math.inf)
        c[:, :, 0] = torch.where(state["ended"], state["scores"].double(), c[:, :, 0])
    best, at = torch.sort(c.view(B, K * V), dim=1, descending=True, stable=True)
    best, at = best[:, :n], at[:, :n]
    some = best > -math.inf
    none = torch.full_like(at, -1)
    return (best.float(), torch.where(some, at // V, none).to(torch.int32),
            torch.where(some, at % V, none).to(torch.int32))


# ---------------------------------------------------------------- in 64 bits


def exact(case, seed):
    state = prepare(case, seed)
    return {"copy": _copy64, "attend": _attend64, "select": _select64}[case["kind"]](state)


def _copy64(state):
    """Page after page, on the host's word."""
    src, dst = state["src"].tolist(), state["dst"].tolist()
    P = state["case"]["block"]
    tokens = [P] * len(src) if state["tokens"] is None else state["tokens"].tolist()
    if len(src) * state["case"]["layers"] > 8000:
        return None
    for p, q in zip(state["pools"], state["into"]):
        for a, b, t in zip(src, dst, tokens):
            q["k"].view(torch.int8)[b, :, :t].copy_(p["k"].view(torch.int8)[a, :, :t])
            q["v"].view(torch.int8)[b, :, :t].copy_(p["v"].view(torch.int8)[a, :, :t])
            q["scale"][b].copy_(p["scale"][a])
            if p["weight"] is not None:
                q["weight"][b, :, :t].copy_(p["weight"][a, :, :t])
    return [{k: (t.view(torch.int8) if k in "kv" else t).double() for k, t in q.items()
             if t is not None} for q in state["into"]]


def _values64(state, pool, which, b, end):
    """[H, end, D]: what sequence b's first `end` tokens hold."""
    P = state["case"]["block"]
    page = state["table"][b, : -(-end // P)].long()
    x = pool.view(torch.uint8)[page].view(pool.dtype).to(torch.float32).double()
    x = x * state["scale"][page][:, :, which].double()[:, :, None, None]
    return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :end]


def _attend64(state):
    case = state["case"]
    B, T, D, H, Hq = (case[k] for k in ("batch", "new", "head_dim", "kv_heads", "heads"))
    G, dev = Hq // H, state["lens"].device
    out = torch.zeros(B, Hq, T, D, dtype=torch.float64, device=dev)
    lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64, device=dev)
    for b, (have, count) in enumerate(zip(state["lens"].tolist(), state["counts"].tolist())):
        end = have + count
        if not count:
            continue
        k = _values64(state, state["k"], 0, b, end)
        v = _values64(state, state["v"], 1, b, end)
        q = state["q"][b, :, :count].double().reshape(H, G * count, D)
        s = (torch.bmm(q, k.transpose(1, 2)) / math.sqrt(D)).view(H, G, count, end)
        if case["causal"]:
            last = have + torch.arange(count, device=dev)
            s = s.masked_fill(torch.arange(end, device=dev)[None] > last[:, None], -math.inf)
        lse[b, :, :count] = torch.logsumexp(s, dim=-1).view(Hq, count)
        p = torch.softmax(s, dim=-1).view(H, G * count, end)
        out[b, :, :count] = torch.bmm(p, v).view(Hq, count, D)
    return out, lse


def _select64(state):
    case = state["case"]
    B, K, V, n = case["batch"], case["beams"], case["vocab"], case["take"]
    outs = [], [], []
    for b in range(B):
        found = []
        for k in range(K):
            score = float(state["scores"][b, k])
            if state["ended"] is not None and bool(state["ended"][b, k]):
                found.append((torch.tensor([score], dtype=torch.float64), [k], [0]))
                continue
            logp = torch.log_softmax(state["logits"][b, k].double(), dim=0) + score
            value, token = torch.sort(logp, descending=True, stable=True)
            keep = (value > -math.inf) & (torch.arange(V, device=value.device) < n)
            m = int(keep.sum())
            found.append((value[:m].cpu(), [k] * m, token[:m].tolist()))
        every = [(-v, k, t) for vs, ks, ts in found for v, k, t in zip(vs.tolist(), ks, ts)]
        every = sorted(every)[:n]
        every += [(math.inf, -1, -1)] * (n - len(every))
        for o, column in zip(outs, zip(*every)):
            o.append(column)
    return (-torch.tensor(outs[0], dtype=torch.float64), torch.tensor(outs[1]),
            torch.tensor(outs[2]))
