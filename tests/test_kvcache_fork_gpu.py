"""CachedStack's forks and beam search on the GPU: sequences that share pages
against sequences of their own that were fed the same tokens in the same chunks,
so the caches hold the same codes and only fp32 roundings differ."""
from __future__ import annotations

import pytest
import torch

from techjam2026_b200 import _lib
from techjam2026_b200.configs import TransformerConfig, init_params_
from techjam2026_b200.kvcache import CachedStack, beam_search, main
from techjam2026_b200.model import LayerStack

pytestmark = pytest.mark.gpu

# One layer: both caches hold the same codes, and the scores' sums run in another
# order (parts of the keys, one or two kernels), 2^-20 relative in each of the few
# products behind an output, on values of order 1.
NEAR = 2e-5
# From the second layer on, K and V differ in their last places, and a value within
# 2e-6 of a border between two codes (1e-4 of them: a step is 1/127 of a page's largest, 4
# standard deviations, so 0.03) takes the other code. One such value of V moves an
# attention output by its weight (1/5 at five keys, less later) times 0.03, 0.006, which
# the output projection spreads; several add in squares. A wrong page or mask moves
# outputs by their own size.
FLIP = 1e-2


def stack_of(d=128, H=4, layers=2, S=200):
    cfg = TransformerConfig(4, S, d, H, 2 * d, layers, True)
    return init_params_(LayerStack(cfg), 5)


def tokens(n, T, d=128, seed=0):
    return torch.randn(n, T, d, generator=torch.Generator().manual_seed(seed)).cuda()


def near(a, b, layers=1):
    bound = NEAR if layers == 1 else FLIP
    return float((a - b).abs().max()) <= bound * max(1.0, float(b.abs().max()))


@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn])
@pytest.mark.parametrize("length", [5, 32, 70])
@pytest.mark.parametrize("layers", [1, 2])
def test_samples_of_one_prompt_are_as_sequences_of_their_own(layers, length, code):
    stack, B = stack_of(layers=layers), 5
    prompt = tokens(1, length)
    model = CachedStack(stack, B, 200, code, block=16)
    first = model(prompt, rows=[0])
    model.fork([0] * B)
    alone = CachedStack(stack, B, 200, code, block=16)
    assert near(first, alone(prompt.expand(B, -1, -1).contiguous())[:1], layers)
    for step in range(20):
        x = tokens(B, 1, seed=step + 1)
        assert near(model(x), alone(x), layers)
    x = tokens(B, 33, seed=99)                       # and a ragged chunk
    counts = [33, 0, 1, 16, 30]
    assert near(model(x, counts=counts), alone(x, counts=counts), layers)
    assert model.lens.tolist() == alone.lens.tolist() == model.held
    assert _lib.lib().kf_device_status(1) == 0


@pytest.mark.parametrize("layers", [1, 2])
def test_forks_of_forks_frees_and_compactions(layers):
    stack, B = stack_of(layers=layers), 4
    model = CachedStack(stack, B, 160, block=16)
    alone = CachedStack(stack, B, 160, block=16)
    fed = [[] for _ in range(B)]                     # what each sequence was fed, chunk by chunk

    def feed(x, counts=None):
        out = model(x, counts=counts)
        for b in range(B):
            n = x.shape[1] if counts is None else counts[b]
            if n:
                fed[b].append(x[b:b + 1, :n])
        return out

    feed(tokens(B, 40, seed=1), [40, 23, 0, 16])
    for step, parents in enumerate(([1, 0, 0, 1], [3, 3, 2, 0], [0, 1, 2, 3], [2, 2, 2, 2])):
        model.fork(parents)
        fed = [list(fed[p]) for p in parents]
        if step == 1:
            model.free([1])
            fed[1] = []
        used = model.compact()
        assert used == sum(n > 0 for n in model.pool.uses)
        assert all(p < used for row in model.pool.rows for p in row)
        out = feed(tokens(B, 3, seed=10 + step))
        out = feed(tokens(B, 1, seed=20 + step))
    for b in range(B):
        alone.free(range(B))
        got = None
        for x in fed[b]:
            got = alone(x, rows=[0])
        assert near(out[b], got[0], layers)
        assert alone.held[0] == model.held[b]
    assert _lib.lib().kf_device_status(1) == 0


def test_a_budget_copies_the_pages_with_their_record():
    stack = stack_of(layers=1)
    model = CachedStack(stack, 3, 96, block=16, budget=64, recent=16)
    model(tokens(1, 50), rows=[0])
    model.fork([0, 0, 0])
    assert max(model.pool.uses) == 1 and model.pool.groups is None
    w = model.caches[0].weight
    rows = [torch.cat([w[p] for p in row], 1)[:, :50] for row in model.pool.rows]
    assert torch.equal(rows[0], rows[1]) and torch.equal(rows[0], rows[2]) and rows[0].any()
    for step in range(30):
        out = model(tokens(3, 1, seed=step).expand(3, 1, 128)[:1].expand(3, 1, 128).contiguous())
        assert max(model.held) <= 64 and torch.isfinite(out).all()
        assert near(out[1], out[0]) and near(out[2], out[0])


@pytest.mark.parametrize("end", [None, 7])
@pytest.mark.parametrize("N,K", [(1, 1), (2, 3), (3, 8)])
def test_beam_search_is_what_hypotheses_of_their_own_give(N, K, end):
    """Against beam search that feeds every hypothesis from its beginning into a
    cache of its own, in the same chunks, with log softmax and sort in float64."""
    d, V, steps = 64, 96, 7
    stack = stack_of(d=d, H=2, layers=1)   # (the same codes: see NEAR)
    g = torch.Generator().manual_seed(K)
    embed = torch.randn(V, d, generator=g).cuda()
    head = (torch.randn(V, d, generator=g) * 0.4).cuda()
    lengths = [17, 5, 32][:N]
    prompts = tokens(N, 32, d, seed=3)
    model = CachedStack(stack, N * K, 64, block=16)
    got, scores = beam_search(model, prompts, lengths, embed, head, K, steps, end)
    one = CachedStack(stack, 1, 64, block=16)

    def logp(n, toks):
        one.free([0])
        out = one(prompts[n:n + 1, :lengths[n]].contiguous())
        for t in toks:
            out = one(embed[t].view(1, 1, d))
        return torch.log_softmax(out[0, -1].double() @ head.double().T, 0)

    for n in range(N):
        beams = [(0.0, [])]
        for _ in range(steps):
            found = []
            for k, (s, toks) in enumerate(beams):
                if end is not None and toks and toks[-1] == end:
                    found.append((-s, k, end))
                    continue
                lp = logp(n, toks) + s
                found += [(-float(lp[v]), k, v) for v in range(V)]
            beams = [(-c, beams[k][1] + [v]) for c, k, v in sorted(found)[:K]]
        assert got[n].tolist() == [toks for _, toks in beams]
        want = torch.tensor([s for s, _ in beams], dtype=torch.float64)
        # logits of order 5 with a relative error of NEAR, over the steps
        assert ((scores[n].cpu().double() - want).abs() <= steps * 20 * NEAR).all()
    assert _lib.lib().kf_device_status(1) == 0


def test_refusals():
    stack = stack_of()
    model = CachedStack(stack, 2, 32, block=16)
    for bad in ([0], [0, 2], [-1, 0]):
        with pytest.raises(ValueError):
            model.fork(bad)
    with pytest.raises(ValueError):
        model.free([2])
    for rows in ([0, 0], [2], [-1]):
        with pytest.raises(ValueError):
            model(tokens(len(rows), 1), rows=rows)
    with pytest.raises(ValueError):
        model(tokens(2, 1), rows=[0])
    embed = torch.zeros(8, 128, device="cuda")
    for args in ((tokens(1, 4), [5], embed, embed, 2, 1), (tokens(1, 4), [0], embed, embed, 2, 1),
                 (tokens(1, 4), [4], embed, embed, 3, 1), (tokens(1, 4), [4], embed, embed, 2, 0)):
        with pytest.raises(ValueError):
            beam_search(model, *args)
    model(tokens(2, 1))
    with pytest.raises(ValueError):
        beam_search(model, tokens(1, 4), [4], embed, embed, 2, 1)


def test_a_search_that_cannot_be_done_is_refused_before_it_begins():
    """Too many beams, no room for the tokens, an end outside the vocabulary: the
    model holds nothing afterwards."""
    stack = stack_of(layers=1)
    embed = torch.randn(8, 128, generator=torch.Generator().manual_seed(0)).cuda()
    many = CachedStack(stack, 129, 32, block=16)
    with pytest.raises(ValueError):
        beam_search(many, tokens(1, 4), [4], embed, embed, 129, 2)
    model = CachedStack(stack, 2, 32, block=16)
    for T, steps, end in ((32, 2, None), (20, 14, None), (4, 2, 8), (4, 2, -1)):
        with pytest.raises(ValueError):
            beam_search(model, tokens(1, T), [T], embed, embed, 2, steps, end)
    for m in (many, model):
        assert not any(m.held) and not m.lens.any() and not any(m.pool.uses)
    out, _ = beam_search(model, tokens(1, 20), [20], embed, embed, 2, 13)    # just fits
    assert out.shape == (1, 2, 13) and max(model.held) == 32


def test_the_example_searches(capsys):
    main(["--config", "c1", "--beams", "3", "--tokens", "4", "--vocab", "100"])
    assert "3 beams" in capsys.readouterr().out
