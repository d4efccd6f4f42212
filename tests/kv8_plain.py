"""Plain restatements of the 8-bit cache operators for the tests: one sequence
and one head at a time, on the CPU, in float64 except where the operator's own
definition rounds to fp32 (the codes)."""
from __future__ import annotations

import math

import torch

QMAX = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
TINY = 2.0 ** -126


def encode(x, dtype):
    """Codes of fp32 values already divided by their scale."""
    q = QMAX[dtype]
    x = torch.nan_to_num(x, nan=0.0, posinf=q, neginf=-q).clamp(-q, q)
    return (x.round() if dtype == torch.int8 else x).to(dtype)


def scale_of(x, dtype):
    """fp32 scale of a block of fp32 values."""
    a = x.abs().max() if x.numel() else torch.tensor(0.0)
    if not torch.isfinite(a):
        return torch.tensor(math.nan)
    s = a * torch.tensor(1.0 / QMAX[dtype], dtype=torch.float32)
    return torch.where(s < TINY, torch.tensor(0.0), s)


def inverse(s):
    return 1.0 / s if s > 0 else torch.tensor(0.0)


class Plain:
    """A cache on the CPU: codes as float32 [pages, H, P, D], scales, record."""

    def __init__(self, cache):
        self.dtype = cache.k.dtype
        self.code = [cache.k.cpu().to(torch.float32), cache.v.cpu().to(torch.float32)]
        self.scale = cache.scale.cpu().clone()
        self.weight = cache.weight.cpu().clone() if cache.weight is not None else None
        self.table = cache.table.cpu()
        self.lens = cache.lens.cpu()
        self.H, self.P, self.D = self.code[0].shape[1:]

    def spot(self, b, pos):
        return int(self.table[b, pos // self.P]), pos % self.P

    def append(self, k, v, counts):
        for which, x in ((0, k.cpu().float()), (1, v.cpu().float())):
            for b in range(len(self.lens)):
                have, n = int(self.lens[b]), int(counts[b])
                for first in range(have, have + n):
                    page, slot = self.spot(b, first)
                    if first > have and slot:
                        continue                      # its page was written with the one before
                    stop = min(have + n, first - slot + self.P)
                    for h in range(self.H):
                        new = x[b, h, first - have:stop - have]
                        was = self.scale[page, h, which] if slot else torch.tensor(0.0)
                        mine = scale_of(new, self.dtype)
                        s = torch.maximum(was, mine)  # NaN wins
                        inv = inverse(s)
                        code = self.code[which][page, h]
                        if slot and not bool(s == was):
                            code[:slot] = encode(code[:slot] * (was * inv), self.dtype).float()
                        code[slot:slot + stop - first] = encode(new * inv, self.dtype).float()
                        self.scale[page, h, which] = s
                        if self.weight is not None and which == 0:
                            self.weight[page, h, slot:slot + stop - first] = 0

    def values(self, which, b, h, end):
        """fp32 values of the first `end` tokens."""
        rows = [self.spot(b, p) for p in range(end)]
        if not rows:
            return torch.zeros(0, self.D)
        page = torch.tensor([r[0] for r in rows])
        slot = torch.tensor([r[1] for r in rows])
        return self.code[which][page, h, slot] * self.scale[page, h, which][:, None]

    def evict(self, table_out, budget, recent):
        out = table_out.cpu()
        kept = torch.full((len(self.lens), self.H, budget), -1, dtype=torch.int32)
        for b in range(len(self.lens)):
            have = int(self.lens[b])
            n = min(have, budget)
            for h in range(self.H):
                rows = [self.spot(b, p) for p in range(have)]
                w = [float(self.weight[p, h, s]) for p, s in rows]
                late = min(recent, have)
                # the largest first, NaN above infinity, the earliest of equals
                key = [(0, 0.0, i) if math.isnan(x) else (1, -x, i) for i, x in enumerate(w)]
                pick = [i for _, _, i in sorted(key[:have - late])][:n - late]
                pick = sorted(pick + list(range(have - late, have)))[:n] if n < have else \
                    list(range(have))
                kept[b, h, :n] = torch.tensor(pick, dtype=torch.int32)
                vals = [self.values(i, b, h, have)[pick] if n else torch.zeros(0, self.D)
                        for i in (0, 1)]
                old_w = [w[i] for i in pick]
                for j in range(-(-n // self.P)):
                    page, a, z = int(out[b, j]), j * self.P, min(n, (j + 1) * self.P)
                    for i in (0, 1):
                        s = scale_of(vals[i][a:z], self.dtype)
                        self.code[i][page, h, :z - a] = encode(vals[i][a:z] * inverse(s),
                                                               self.dtype).float()
                        self.scale[page, h, i] = s
                    self.weight[page, h, :z - a] = torch.tensor(old_w[a:z])
        return kept

    def attention(self, q, counts, causal, scale, eps_q, eps_p, eps_out):
        """out, lse, weight (float64) and how far each may be off.

        The bounds follow the operator's roundings: q enters with a relative
        error of eps_q, a score's D products are summed in fp32 (with one bit
        to spare), so a score is off by at most `d` (natural units) and a
        weight by a factor of e^d; the sum has the same error, hence 2 d. P is
        rounded to eps_p, and sums over L keys run in fp32."""
        q = q.cpu().double()
        B, Hq, T, D = q.shape
        G = Hq // self.H
        out, tol = torch.zeros(B, Hq, T, D, dtype=torch.float64), torch.zeros(B, Hq, T, D).double()
        lse = torch.full((B, Hq, T), -math.inf, dtype=torch.float64)
        tol_lse = torch.zeros_like(lse)
        weight = self.weight.double() if self.weight is not None else None
        tol_w = torch.zeros_like(weight) if weight is not None else None
        for b in range(B):
            have, n = int(self.lens[b]), int(counts[b])
            end = have + n
            for h in range(self.H):
                k = self.values(0, b, h, end).double()
                v = self.values(1, b, h, end).double()
                for i in range(n):
                    m = min(end, have + i + 1) if causal else end
                    if not m:
                        continue
                    for hq in range(h * G, (h + 1) * G):
                        s = (k[:m] @ q[b, hq, i]) * scale
                        size = (k[:m].abs() @ q[b, hq, i].abs()).max() * scale
                        d = float((eps_q + (D + 4) * 2.0 ** -23) * size) + 2.0 ** -21
                        p = torch.softmax(s, 0)
                        out[b, hq, i] = p @ v[:m]
                        lse[b, hq, i] = torch.logsumexp(s, 0)
                        tol_lse[b, hq, i] = d + 2.0 ** -20 * (1 + abs(float(lse[b, hq, i])))
                        mass = p @ v[:m].abs()
                        # an element of P below 2^-34 of the largest is lost altogether
                        rel = 2 * d + eps_p + (m + 16) * 2.0 ** -23
                        tol[b, hq, i] = mass * rel + out[b, hq, i].abs() * eps_out + 1e-30
                        if eps_p > 2.0 ** -20:
                            tol[b, hq, i] += v[:m].abs().amax(0) * 2.0 ** -30
                        else:
                            tol[b, hq, i] += v[:m].abs().amax(0) * m * 2.0 ** -34
                        if weight is not None:
                            for j in range(m):
                                page, slot = self.spot(b, j)
                                weight[page, h, slot] += p[j]
                                tol_w[page, h, slot] += p[j] * (2 * d + 2.0 ** -20)
        if weight is not None:
            tol_w += weight.abs() * 2.0 ** -22 * 4 + 1e-30
        return out, tol, lse, tol_lse, weight, tol_w
