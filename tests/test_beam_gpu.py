"""beam_select on the GPU against the definition in float64: beams and tokens
exactly, scores within the rounding of the softmax's sum."""
from __future__ import annotations

import math

import pytest
import torch

from techjam2026_b200 import ops

pytestmark = pytest.mark.gpu

F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def plain(logits, scores, n, ended, pad):
    """Scores (float64), beams and tokens, candidate by candidate."""
    x, s = logits.cpu().double(), scores.cpu().double()
    B, K, V = x.shape
    outs = []
    for b in range(B):
        found = []
        for k in range(K):
            if ended is not None and ended[b, k]:
                c = torch.tensor([float(s[b, k])], dtype=torch.float64)
                token = torch.tensor([pad])
            else:
                c = x[b, k] - torch.logsumexp(x[b, k], 0) + s[b, k]
                token = torch.arange(V)
            keep = c > -math.inf                       # NaN is not
            c, token = c[keep], token[keep]
            order = torch.sort(c, descending=True, stable=True).indices[:n]
            found += [(-float(c[i]), k, int(token[i])) for i in order]
        best = sorted(found)[:n]
        outs.append(best + [(math.inf, -1, -1)] * (n - len(best)))
    t = torch.tensor(outs, dtype=torch.float64)
    return -t[..., 0], t[..., 1].int(), t[..., 2].int()


def check(logits, scores, n=None, ended=None, pad=0):
    got = ops.beam_select(logits, scores, n, ended=ended, pad=pad)
    n = logits.shape[1] if n is None else n
    want = plain(logits, scores, n, None if ended is None else ended.cpu(), pad)
    assert torch.equal(got[1].cpu(), want[1])
    assert torch.equal(got[2].cpu(), want[2])
    none = torch.isinf(want[0])
    assert torch.equal(got[0].cpu()[none].double(), want[0][none])
    # The sum of V exponentials in fp32: each off by 2^-22 and by the rounding of
    # its exponent (at most 2^-23 of some 20), added by threads of a 256th of the
    # vocabulary at most; then one rounding of the score to fp32.
    tol = (2 + 20 + logits.shape[2] / 256) * 2.0 ** -23 + want[0].abs() * 2.0 ** -24
    off = (got[0].cpu().double() - want[0]).abs()
    assert (off <= tol)[~none].all(), off[~none].max()
    return got


def rows(B, K, V, kind=F32, seed=0, spread=3.0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(B, K, V, generator=g) * spread).to(kind).cuda()
    return logits, (-5 * torch.rand(B, K, generator=g)).cuda()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("B,K,V", [(1, 1, 1), (1, 1, 7), (2, 3, 100), (1, 4, 2048), (3, 5, 2049),
                                   (2, 8, 5003), (1, 2, 50021), (5, 1, 16384), (40, 16, 777)])
def test_selection(B, K, V, kind):
    logits, scores = rows(B, K, V, kind)
    check(logits, scores)
    for n in (1, 2 * K, 64, 128):
        check(logits, scores, n)


@pytest.mark.parametrize("kind", [F32, BF16])
def test_ended_beams_and_fewer_candidates_than_wanted(kind):
    logits, scores = rows(4, 4, 600, kind, 1)
    ended = torch.tensor([[0, 1, 0, 1], [1, 1, 1, 1], [0, 0, 0, 0], [1, 0, 0, 0]],
                         dtype=torch.bool, device="cuda")
    for n in (2, 4, 9, 100):
        check(logits, scores, n, ended, 17)
    scores[0, 1] = scores[0, 3]           # equal candidates of ended beams: the lower one first
    scores[1] = -1.0
    check(logits, scores, 8, ended, 599)
    check(logits[:, :, :3], scores, 100, ended, 5)


def test_the_first_step_has_one_live_beam():
    logits, scores = rows(2, 6, 1000, F32, 2)
    scores[:, 0] = 0.0
    scores[:, 1:] = -math.inf
    got = check(logits, scores, 6)
    assert not got[1].any()


@pytest.mark.parametrize("kind", [F32, BF16, F16])
def test_equal_candidates_go_by_beam_then_token(kind):
    """All logits equal, all of two values, beams alike, and zeros of both signs."""
    scores = torch.tensor([[-1.0, -1.0, -2.0]], device="cuda")
    for V in (5, 3000, 9000):
        x = torch.full((1, 3, V), 0.25, device="cuda", dtype=kind)
        check(x, scores, 40)
        x[:, :, 1::2] = 1.5
        check(x, scores, 128)
        g = torch.Generator().manual_seed(V)
        x = torch.randint(-2, 3, (1, 1, V), generator=g).to(kind).cuda().expand(1, 3, V)
        check(x, scores, 64)
        x = torch.zeros(1, 3, V, device="cuda", dtype=kind)
        x[:, :, ::3] = -0.0
        check(x, scores, 20)


@pytest.mark.parametrize("n", [1, 128])
@pytest.mark.parametrize("kind", [F32, F16])
def test_logits_that_grow_or_fall_along_the_vocabulary(kind, n):
    """Growing ones replace the best ones found all the way."""
    up = torch.linspace(-8, 8, 40000).to(kind).cuda()
    x = torch.stack([up, up.flip(0), up.abs(), -up.abs()])[None].contiguous()
    check(x, torch.tensor([[-0.5, -0.25, -0.125, 0.0]], device="cuda"), n)


def test_infinities_and_nan():
    logits, scores = rows(6, 3, 5000, F32, 3)
    logits[0, 0, ::2] = -math.inf
    logits[1, 1] = -math.inf                     # a beam of nothing
    logits[2, 2, 4999] = math.nan
    logits[3, 0, 17] = math.inf
    scores[4, 1] = math.nan
    logits[5, :] = -math.inf
    logits[5, :, 3] = 2.0
    check(logits, scores, 7)
    logits[:, :, :] = math.nan
    score, beam, token = ops.beam_select(logits, scores, 4)
    assert (score == -math.inf).all() and (beam == -1).all() and (token == -1).all()


def test_large_magnitudes():
    logits, scores = rows(2, 3, 3000, F32, 4, spread=1e4)
    check(logits, scores * 1e3, 6)
    check(logits * 1e30, scores, 3)


@pytest.mark.parametrize("kind,pad", [(F32, 0), (F32, 1), (BF16, 3), (F16, 8)])
def test_strided_and_unaligned_rows(kind, pad):
    g = torch.Generator().manual_seed(5)
    base = (torch.randn(3, 7, 4000 + 5, generator=g) * 2).to(kind).cuda()
    logits = base[:, 1:5, pad:pad + 3990]
    wide = torch.randn(3, 9, generator=g).cuda()
    ended = torch.zeros(3, 9, dtype=torch.bool, device="cuda")
    ended[1, 3] = True
    check(logits, wide[:, 2:6], 8, ended[:, 1:5], 1)
    check(logits[:, :1].expand(3, 4, 3990), wide[:, 2:6], 8)
    check(base.transpose(0, 1)[:, :2, :3990], wide[:1, :2].expand(7, 2), 3)


def test_graphs_streams_and_two_calls_at_once():
    logits, scores = rows(4, 8, 30000, BF16, 6)
    want = check(logits, scores, 16)
    side = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in side:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(ops.beam_select(logits, scores, 16))
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        one = ops.beam_select(logits, scores, 16)
        two = ops.beam_select(-logits, scores, 5)
    for _ in range(2):
        logits.mul_(-1)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(one, ops.beam_select(logits, scores, 16)))
        assert all(torch.equal(a, b) for a, b in zip(two, ops.beam_select(-logits, scores, 5)))
    assert all(torch.equal(a, b) for a, b in zip(one, want))


def test_an_empty_batch_and_refusals():
    logits, scores = rows(2, 3, 50)
    out = ops.beam_select(logits[:0], scores[:0])
    assert [t.shape for t in out] == [(0, 3)] * 3
    for bad in (0, -1, 129):
        with pytest.raises(ValueError):
            ops.beam_select(logits, scores, bad)
    for x, s, kw in ((logits[0], scores, {}), (logits[:, :, :0], scores, {}),
                     (logits, scores[:, :2], {}), (logits, scores, {"pad": -1}),
                     (logits[:, :, ::2], scores, {}),
                     (logits, scores, {"ended": torch.zeros(2, 2, dtype=torch.bool,
                                                            device="cuda")}),
                     (logits, scores.cpu(), {})):
        with pytest.raises(ValueError):
            ops.beam_select(x, s, **kw)
    for x, s, kw in ((logits.double(), scores, {}), (logits, scores.double(), {}),
                     (logits, scores, {"ended": torch.zeros(2, 3, device="cuda")})):
        with pytest.raises(TypeError):
            ops.beam_select(x, s, **kw)
