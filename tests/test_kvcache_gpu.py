"""The layer stack over the 8-bit cache against the CPU oracle. The cache's
own rounding is what separates them: a code step is 1/127 of a block's largest
magnitude (about 4 standard deviations), so int8 K and V carry about 1 %, e4m3
about 2.5 % of relative error, a share of which reaches the outputs."""
from __future__ import annotations

import pytest
import torch

import oracle
from techjam2026_b200 import ops
from techjam2026_b200.configs import TransformerConfig, make_state_dict
from techjam2026_b200.kvcache import CachedStack, main
from techjam2026_b200.model import LayerStack

pytestmark = pytest.mark.gpu


def setup(S, d, H, layers=2, B=3):
    cfg = TransformerConfig(B, S, d, H, 2 * d, layers, True)
    sd = make_state_dict(cfg, 0)
    stack = LayerStack(cfg)
    stack.load_state_dict(sd, strict=True)
    x = torch.randn(B, S, d, generator=torch.Generator().manual_seed(3))
    want = oracle.forward(sd, layers, H, x, torch.ones(B, S, dtype=torch.bool), causal=True)
    return stack, x, want


def rel(a, b):
    return float((a.cpu() - b).norm() / b.norm())


@pytest.mark.parametrize("code,bound", [(torch.int8, 0.02), (torch.float8_e4m3fn, 0.05)])
@pytest.mark.parametrize("d,H", [(128, 4), (256, 4), (256, 2), (64, 4)])
def test_prompt_then_tokens_match_the_whole_sequence(d, H, code, bound):
    stack, x, want = setup(90, d, H)
    model = CachedStack(stack, 3, 90, code, block=16)
    got = [model(x[:, :70].cuda())] + [model(x[:, i:i + 1].cuda()) for i in range(70, 90)]
    assert rel(torch.cat(got, 1), want) < bound
    assert model.lens.tolist() == [90] * 3


def test_ragged_chunks_match_the_whole_sequences():
    stack, x, want = setup(120, 128, 2)
    model = CachedStack(stack, 3, 120, block=32)
    at = [0, 0, 0]
    got = torch.zeros_like(x)
    for counts in ([40, 1, 0], [0, 37, 50], [40, 40, 17], [40, 42, 53]):
        T = max(counts)
        chunk = torch.full((3, T, 128), float("nan"))
        for b, n in enumerate(counts):
            chunk[b, :n] = x[b, at[b]:at[b] + n]
        chunk = chunk.nan_to_num(7.0)            # what stands past a count must not matter
        out = model(chunk.cuda(), counts=counts).cpu()
        for b, n in enumerate(counts):
            got[b, at[b]:at[b] + n] = out[b, :n]
            assert not out[b, n:].any()
            at[b] += n
    assert at == [120] * 3
    assert rel(got, want) < 0.02


def test_a_budget_bounds_the_cache_and_keeps_the_outputs_near():
    stack, x, want = setup(200, 128, 2, layers=1)
    model = CachedStack(stack, 3, 224, block=16, budget=160, recent=32)
    got = [model(x[:, :150].cuda())]
    for i in range(150, 200, 5):
        got.append(model(x[:, i:i + 5].cuda()))
        assert max(model.held) <= 160
        assert model.lens.tolist() == model.held
    used = [p for r in model.pool.rows for p in r]
    assert len(used) == len(set(used)) and not set(used) & set(model.pool.free)
    got = torch.cat(got, 1)
    assert rel(got[:, :160], want[:, :160]) < 0.02       # nothing was cut before
    # a fifth of the tokens are gone: the attention branch moves, the stream less
    assert rel(got, want) < 0.15 and torch.isfinite(got).all()


@pytest.mark.parametrize("code,step", [(torch.int8, 0.011), (torch.float8_e4m3fn, 0.035)])
def test_tokens_past_a_budget_are_evicted_by_the_page_and_keep_their_values(code, step, monkeypatch):
    """200 tokens one by one past a budget of 96 in pages of 16: a sequence is
    cut once a page, only it is moved, and what it still holds is near what was
    appended. A cut rounds anew, independently of the rounding before at worst:
    relative errors of one rounding (`step`) add in squares."""
    from techjam2026_b200 import kvcache
    stack, x, _ = setup(296, 128, 2, layers=1, B=2)
    model = CachedStack(stack, 2, 128, code, block=16, budget=96, recent=16)
    put, cut = kvcache.kv8_append, kvcache.kv8_evict
    told = [[[], []] for _ in range(2)]          # K and V rows of each sequence, by position
    cuts = []

    def append(cache, k, v, counts):
        for b, n in enumerate(counts.tolist()):
            for i in range(n):
                told[b][0].append(k[b, :, i].clone())
                told[b][1].append(v[b, :, i].clone())
        put(cache, k, v, counts=counts)

    def evict(cache, table, budget, recent):
        kept, new = cut(cache, table, budget, recent)
        assert kept.shape[0] == 1                # the other sequence is within its budget
        for which in (0, 1):
            rows = torch.stack(told[0][which], 1)                     # [H, L, D]
            at = kept[0].long()[..., None].expand(-1, -1, rows.shape[2])
            told[0][which] = list(torch.gather(rows, 1, at).unbind(1))
        cuts.append(budget)
        return kept, new

    monkeypatch.setattr(kvcache, "kv8_append", append)
    monkeypatch.setattr(kvcache, "kv8_evict", evict)
    model(x[:, :96].cuda(), counts=[96, 40])
    other = list(model.pool.rows[1])
    for i in range(96, 296):
        model(x[:, i:i + 1].cuda(), counts=[1, 0])
        assert max(model.held) <= 96 and model.lens.tolist() == model.held
    assert cuts == [80] * 12                     # at 97, then every 17 tokens
    assert model.pool.rows[1] == other and model.held[1] == 40
    used = [p for r in model.pool.rows for p in r]
    assert len(used) == len(set(used)) and not set(used) & set(model.pool.free)
    k, v = ops.kv8_read(model.caches[0], 96)
    for b, n in enumerate(model.held):
        for which, got in ((0, k), (1, v)):
            want = torch.stack(told[b][which], 1)
            assert want.shape[1] == n
            bound = step * (1 + (len(cuts) if b == 0 else 0)) ** 0.5
            assert rel(got[b, :, :n], want.cpu()) < bound, (b, which)


def test_refusals():
    stack, x, _ = setup(16, 64, 4, layers=1)
    with pytest.raises(ValueError):
        CachedStack(stack, 3, 16, budget=32)
    model = CachedStack(stack, 3, 16, block=16)
    with pytest.raises(ValueError):
        model(x[:2].cuda())
    with pytest.raises(ValueError):
        model(x.cuda(), counts=[1, 2, 17])
    with pytest.raises(RuntimeError):
        model(torch.cat([x, x], 1).cuda())               # 32 tokens into 16
    assert model.lens.tolist() == [0, 0, 0]
    cfg = TransformerConfig(1, 8, 64, 4, 64, 1, False)
    with pytest.raises(ValueError):
        CachedStack(LayerStack(cfg), 1, 8)


def test_a_slack_needs_a_budget_above_it():
    stack, _, _ = setup(16, 64, 4, layers=1)
    for slack, budget in ((4, None), (-1, 16), (16, 16)):
        with pytest.raises(ValueError):
            CachedStack(stack, 3, 16, budget=budget, slack=slack)
    assert CachedStack(stack, 3, 64, block=16, budget=32, recent=32).keep == 24
    assert CachedStack(stack, 3, 64, block=16, budget=32, slack=0).keep == 32


@pytest.mark.parametrize("recent", [8, 32])
def test_a_budget_that_fills_the_rows_is_served_past(recent):
    """budget == max_tokens, a multiple of the page: the token that finds no
    room cuts its sequence first. A chunk that fits in no case is refused and
    cuts nothing."""
    stack, x, _ = setup(80, 64, 4, layers=2, B=2)
    model = CachedStack(stack, 2, 32, block=16, budget=32, recent=recent)
    model(x[:, :32].cuda(), counts=[32, 5])
    for i in range(32, 80):
        out = model(x[:, i:i + 1].cuda(), counts=[1, 0])
        assert torch.isfinite(out).all() and out[0].any()
        assert model.lens.tolist() == model.held and max(model.held) <= 32 and model.held[1] == 5
    held = list(model.held)
    with pytest.raises(RuntimeError):
        model(x[:, :30].cuda(), counts=[30, 0])
    assert model.held == held and model.lens.tolist() == held
    with pytest.raises(ValueError):
        CachedStack(stack, 2, 32, block=16, budget=32, slack=0)


@pytest.mark.parametrize("tokens", [1, 2, 5])
def test_the_example_runs(tokens, capsys):
    main(["--config", "c1", "--tokens", str(tokens)])
    said = capsys.readouterr().out
    assert f"{tokens} single ones" in said and "ms a token" in said
    assert float(said.split("forward ")[1].split(",")[0]) < 0.02
