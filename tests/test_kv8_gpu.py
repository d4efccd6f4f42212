"""The 8-bit key/value cache on the GPU against plain restatements: codes and
kept tokens exactly, attention against float64 within the bounds that its own
roundings give (kv8_plain.Plain.attention)."""
from __future__ import annotations

import math

import pytest
import torch

from kv8_plain import Plain
from techjam2026_b200 import _lib, ops

pytestmark = pytest.mark.gpu

I8, F8 = torch.int8, torch.float8_e4m3fn
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
EPS_Q = {F32: 2.0 ** -21, BF16: 2.0 ** -23, F16: 2.0 ** -23}
EPS_P = {F32: 2.0 ** -21, BF16: 2.0 ** -11, F16: 2.0 ** -11}
EPS_OUT = {F32: 2.0 ** -23, BF16: 2.0 ** -8, F16: 2.0 ** -11}


def make(lens, heads=2, dim=64, block=16, dtype=I8, room=64, weight=False, spare=0, seed=0):
    """A cache whose sequences hold `lens` tokens, its pages scattered over the
    pool, every slot and scale filled with junk (NaN among it) first."""
    g = torch.Generator().manual_seed(seed)
    B = len(lens)
    blocks = -(-(max(lens) + room) // block)
    pages = B * blocks + spare + 3
    order = torch.randperm(pages, generator=g).to(torch.int32)
    table = order[:B * blocks].view(B, blocks).cuda()
    cache = ops.KV8Cache.empty(pages, heads, block, dim, table,
                               torch.zeros(B, dtype=torch.int32, device="cuda"), dtype, weight)
    cache.k.view(torch.uint8).fill_(0xFF)
    cache.v.view(torch.uint8).fill_(0x7F)
    cache.scale.fill_(math.nan)
    if weight:
        cache.weight.fill_(math.nan)
    longest = max(lens)
    if longest:
        x = torch.randn(2, B, heads, longest, dim, generator=g).cuda()
        counts = torch.tensor(lens, dtype=torch.int32, device="cuda")
        ops.kv8_append(cache, x[0], x[1], counts=counts)
        cache.lens += counts
    return cache, order[B * blocks:B * blocks + spare].cuda(), g


def same_codes(cache, plain, b_end):
    """Every token below b_end[b], bit for bit, and its page's scale."""
    k, v = cache.k.cpu().float(), cache.v.cpu().float()
    scale = cache.scale.cpu()
    for b, end in enumerate(b_end):
        for pos in range(int(end)):
            page, slot = plain.spot(b, pos)
            assert torch.equal(k[page, :, slot], plain.code[0][page, :, slot]), (b, pos)
            assert torch.equal(v[page, :, slot], plain.code[1][page, :, slot]), (b, pos)
            assert torch.equal(scale[page].nan_to_num(-1), plain.scale[page].nan_to_num(-1))


def clean():
    assert _lib.lib().kf_device_status(1) == 0


# ---------------------------------------------------------------- append, read


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("dim,block", [(16, 16), (32, 128), (64, 64), (128, 32), (128, 128)])
def test_append_gives_the_defined_codes(dim, block, kind, dtype):
    lens = [0, 1, block - 1, block, block + 1, 5]
    cache, _, g = make(lens, dim=dim, block=block, dtype=dtype, weight=True, room=2 * block + 9)
    T = block + 7
    k = (torch.randn(6, 2, T, dim, generator=g) * 2).to(kind).cuda()
    v = (torch.randn(6, 2, T, dim, generator=g) * 0.3).to(kind).cuda()
    counts = torch.tensor([T, 3, T - 1, 1, 0, T], dtype=torch.int32, device="cuda")
    plain = Plain(cache)
    ops.kv8_append(cache, k, v, counts=counts)
    plain.append(k, v, counts)
    ends = [a + int(n) for a, n in zip(lens, counts)]
    same_codes(cache, plain, ends)
    # read-back: codes * scales exactly, zeros past the end, any start
    start = torch.tensor([0, 1, 0, block, 2, 4], dtype=torch.int32, device="cuda")
    n = T + block
    for out in (F32, kind):
        rk, rv = ops.kv8_read(cache, n, start=start, counts=counts, dtype=out)
        for b in range(6):
            for h in range(2):
                for which, r in ((0, rk), (1, rv)):
                    want = plain.values(which, b, h, ends[b])[int(start[b]):][:n]
                    assert torch.equal(r[b, h, :len(want)].cpu(), want.to(out))
                    assert not r[b, h, len(want):].any()
    # the new tokens start with no recorded weight, the old ones keep theirs
    w = cache.weight.cpu()
    for b, end in enumerate(ends):
        for pos in range(end):
            page, slot = plain.spot(b, pos)
            assert torch.equal(w[page, :, slot], torch.zeros(2))
    clean()


@pytest.mark.parametrize("dtype,half_step", [(I8, 0.5), (F8, None)])
def test_append_error_is_half_a_step(dtype, half_step):
    """Against float64: a value is off by at most half a code step of its
    page, and a code in the largest binade is at least half full scale."""
    cache, _, g = make([0], heads=3, dim=64, block=64, dtype=dtype, room=640)
    x = torch.randn(1, 3, 600, 64, generator=g) * torch.logspace(-3, 3, 600).view(1, 1, -1, 1)
    ops.kv8_append(cache, x.cuda(), x.cuda())
    cache.lens += 600
    k, _ = ops.kv8_read(cache, 600)
    x = torch.nn.functional.pad(x.double(), (0, 0, 0, 40)).view(3, 10, 64, 64)
    k = torch.nn.functional.pad(k.cpu().double(), (0, 0, 0, 40)).view(3, 10, 64, 64)
    s = x.abs().amax(dim=(2, 3), keepdim=True) / (127 if dtype == I8 else 448)
    step = s if dtype == I8 else torch.maximum(
        torch.exp2(torch.floor(torch.log2((x / s).abs().clamp(min=2.0 ** -6)))) / 8, x * 0) * s
    assert ((k - x).abs() <= step * (0.5 + 2.0 ** -14)).all()


@pytest.mark.parametrize("dtype", [I8, F8])
def test_tokens_one_by_one_rescale_their_page(dtype):
    """Growing magnitudes: every token raises its page's scale, zeros and the
    smallest numbers among them."""
    cache, _, g = make([3, 0], heads=1, dim=32, block=16, dtype=dtype, room=64)
    plain = Plain(cache)
    one = torch.ones(2, dtype=torch.int32, device="cuda")
    for i in range(20):
        mag = [0.0, 1e-42, 1e-38, 1e-30][i] if i < 4 else 1.7 ** i
        x = torch.randn(2, 1, 1, 32, generator=g).cuda() * mag
        plain.lens = cache.lens.cpu()
        plain.append(x, -x, one)
        ops.kv8_append(cache, x, -x)
        cache.lens += 1
    same_codes(cache, plain, cache.lens.cpu())
    clean()


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_a_bad_value_spoils_its_page_only(bad, dtype):
    cache, _, g = make([4, 20], heads=2, dim=64, block=16, dtype=dtype)
    x = torch.randn(2, 2, 1, 64, generator=g).cuda()
    y = x.clone()
    y[1, 1, 0, 7] = bad
    ops.kv8_append(cache, y, x)          # K of sequence 1, head 1, its second page
    cache.lens += 1
    k, v = ops.kv8_read(cache, 21)
    assert torch.isfinite(v).all() and torch.isfinite(k[0]).all() and torch.isfinite(k[1, 0]).all()
    assert torch.isfinite(k[1, 1, :16]).all() and k[1, 1, 16:].isnan().all()
    cache.lens -= 1
    q = torch.randn(2, 4, 1, 64, generator=g).cuda()
    out = ops.kv8_attention(q, cache)
    assert torch.isfinite(out[0]).all() and torch.isfinite(out[1, :2]).all()
    assert out[1, 2:].isnan().all()
    # values past a sequence's count are never looked at
    ops.kv8_append(cache, y * math.nan, y * math.nan,
                   counts=torch.zeros(2, dtype=torch.int32, device="cuda"))
    assert torch.isfinite(ops.kv8_read(cache, 20)[1]).all()
    clean()


# ---------------------------------------------------------------- attention


def attend(cache, q, counts, causal=True, scale=None, track=False, **kw):
    plain = Plain(cache)
    if not track:
        plain.weight = None
    n = counts.cpu() if counts is not None else torch.full((q.shape[0],), q.shape[2])
    out, lse = ops.kv8_attention(q, cache, counts=counts, causal=causal, sm_scale=scale,
                                 track=track, return_lse=True, **kw)
    ref, tol, ref_lse, tol_lse, w, tol_w = plain.attention(
        q, n, causal, scale if scale is not None else q.shape[3] ** -0.5,
        EPS_Q[q.dtype], EPS_P[q.dtype], EPS_OUT[q.dtype])
    diff = (out.cpu().double() - ref).abs()
    assert (diff <= tol).all(), (diff / tol).max()
    empty = torch.isinf(ref_lse)
    assert torch.equal(torch.isinf(lse.cpu()), empty)
    d = torch.where(empty, torch.zeros_like(ref_lse), (lse.cpu().double() - ref_lse).abs())
    assert (d <= tol_lse).all()
    if track:
        got = cache.weight.cpu().double()
        ok = torch.isnan(w) & torch.isnan(got) | ((got - w).abs() <= tol_w)
        assert ok.all(), float((got - w).abs().nan_to_num().max())
    clean()
    return out


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("dim,block,group", [(16, 16, 1), (32, 32, 3), (64, 64, 1), (64, 16, 8),
                                             (128, 128, 4), (128, 16, 16)])
def test_single_tokens(dim, block, group, kind, dtype):
    lens = [0, 1, 15, 16, 17, 63, 64, 300]
    cache, _, g = make(lens, dim=dim, block=block, dtype=dtype, weight=True)
    cache.weight.zero_()
    x = torch.randn(8, 2, 1, dim, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    q = torch.randn(8, 2 * group, 1, dim, generator=g).to(kind).cuda()
    attend(cache, q, None, track=True)


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("track", [True, False])
@pytest.mark.parametrize("kind,dtype", [(F32, I8), (BF16, F8), (F16, I8)])
@pytest.mark.parametrize("T,group,dim", [(2, 1, 32), (5, 3, 64), (17, 1, 128), (40, 2, 64),
                                         (129, 1, 64), (70, 4, 128)])
def test_chunks(T, group, dim, kind, dtype, track, causal):
    lens = [0, 1, 33, 130]
    cache, _, g = make(lens, heads=2, dim=dim, block=32, dtype=dtype, weight=True, room=T)
    cache.weight.zero_()
    x = torch.randn(4, 2, T, dim, generator=g).cuda()
    counts = torch.tensor([T, T - 1, 0, (T + 1) // 2], dtype=torch.int32, device="cuda")
    ops.kv8_append(cache, x, x, counts=counts)
    q = torch.randn(4, 2 * group, T, dim, generator=g).to(kind).cuda()
    attend(cache, q, counts, causal=causal, track=track)


@pytest.mark.parametrize("track", [True, False])
@pytest.mark.parametrize("kind,dtype", [(F32, F8), (BF16, I8)])
@pytest.mark.parametrize("T,group,dim,block", [(100, 1, 16, 16), (45, 2, 32, 128), (50, 1, 32, 64),
                                               (31, 2, 16, 32), (11, 12, 128, 64)])
def test_chunks_of_other_widths(T, group, dim, block, kind, dtype, track):
    """Both kernels (up to and above 64 query rows of a kv head) at the small
    head widths, and pages as wide as a step."""
    lens = [3, 0, 140]
    cache, _, g = make(lens, heads=1, dim=dim, block=block, dtype=dtype, weight=True, room=T)
    cache.weight.zero_()
    x = torch.randn(3, 1, T, dim, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    q = torch.randn(3, group, T, dim, generator=g).to(kind).cuda()
    attend(cache, q, None, track=track)


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("kind,T", [(F32, 80), (BF16, 80), (BF16, 20), (F32, 7)])
@pytest.mark.parametrize("which", ["k", "v"])
def test_a_spoiled_page_reaches_the_rows_that_see_it(which, kind, T, dtype):
    """A page whose scale is NaN: rows that see a token of it are NaN, the
    others are as if it were not there (it shares a step with good pages)."""
    cache, _, g = make([40 + 80 - T], heads=1, dim=64, block=16, dtype=dtype, room=96)
    x = torch.randn(1, 1, T, 64, generator=g).cuda()
    y = x.clone()
    y[0, 0, T - 5, 3] = math.inf                     # position 115: page 7 (112 to 127)
    ops.kv8_append(cache, y if which == "k" else x, y if which == "v" else x)
    q = torch.randn(1, 2, T, 64, generator=g).to(kind).cuda()
    out = ops.kv8_attention(q, cache).cpu()
    plain = Plain(cache)
    plain.weight = None
    ref, tol, *_ = plain.attention(q, [T], True, 0.125, EPS_Q[kind], EPS_P[kind], EPS_OUT[kind])
    # the first of the rows from position 112 on sees the page
    seen = torch.arange(T) + 120 - T >= 112
    assert out[:, :, seen].isnan().all() and ref[:, :, seen].isnan().all()
    good = ~seen
    assert ((out.double() - ref).abs()[:, :, good] <= tol[:, :, good]).all()
    clean()


@pytest.mark.parametrize("T", [80, 20])
def test_a_refused_page_hides_its_tokens_from_a_chunk(T):
    """A table entry outside the pool in the middle of a step: the rows attend
    to the other tokens; the same with the hidden keys' weights."""
    cache, _, g = make([60], heads=1, dim=64, block=16, room=96, weight=True)
    cache.weight.zero_()
    x = torch.randn(1, 1, T, 64, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    q = torch.randn(1, 1, T, 64, generator=g).cuda()
    keep = int(cache.table[0, 2])
    cache.table[0, 2] = 1 << 20
    out = ops.kv8_attention(q, cache, track=True).cpu()
    assert _lib.lib().kf_device_status(1) == 6
    weight = cache.weight.cpu()
    cache.table[0, 2] = keep
    plain = Plain(cache)
    k = plain.values(0, 0, 0, 60 + T).double()
    v = plain.values(1, 0, 0, 60 + T).double()
    s = (q.cpu().double()[0, 0] @ k.T) / 8
    pos = torch.arange(60 + T)
    hidden = (pos >= 32) & (pos < 48)
    s.masked_fill_(hidden[None] | (pos[None] > 60 + torch.arange(T)[:, None]), -math.inf)
    p = torch.softmax(s, -1)
    assert ((out[0, 0].double() - p @ v).abs() <= 1e-4).all()
    got = torch.cat([weight[int(cache.table[0, i]), 0] for i in range(-(-(60 + T) // 16))])
    want = p.sum(0)
    assert ((got[:60 + T].double() - want).abs()[~hidden] <= 1e-4).all()
    assert not weight[keep].any()


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("T,group", [(1, 1), (1, 12), (20, 1), (31, 2), (80, 1)])
def test_a_refused_page_is_as_if_its_tokens_were_not_there(T, group, kind, dtype):
    """The same when every page that is not in the table holds codes and scales
    that are no numbers (0x7F and 0xFF are e4m3 NaN): nothing of them may enter.
    Without the block of the refused page, queries and keys stand 16 earlier."""
    blocks = -(-(60 + T) // 16)
    table = torch.arange(2, 2 + 2 * blocks, dtype=torch.int32, device="cuda").view(2, blocks)
    lens = torch.tensor([60, 52], dtype=torch.int32, device="cuda")
    cache = ops.KV8Cache.empty(2 * blocks + 4, 2, 16, 64, table, torch.zeros_like(lens), dtype)
    cache.k.view(torch.uint8).fill_(0xFF)
    cache.v.view(torch.uint8).fill_(0x7F)
    cache.scale.fill_(math.nan)
    g = torch.Generator().manual_seed(T)
    x = torch.randn(2, 2, 2, 60 + T, 64, generator=g).cuda()
    ops.kv8_append(cache, x[0], x[1], counts=lens + T)
    cache.lens.copy_(lens)
    q = torch.randn(2, 2 * group, T, 64, generator=g).to(kind).cuda()
    plain = Plain(cache)
    plain.weight = None
    plain.table = torch.cat([plain.table[:, :2], plain.table[:, 3:]], 1)
    plain.lens = plain.lens - 16
    ref, tol, *_ = plain.attention(q, [T, T], True, 0.125, EPS_Q[kind], EPS_P[kind], EPS_OUT[kind])
    for wrong in (-1, 2 * blocks + 4, 1 << 30):
        cache.table[:, 2] = wrong
        out = ops.kv8_attention(q, cache).cpu().double()
        assert _lib.lib().kf_device_status(1) == 6
        assert ((out - ref).abs() <= tol).all(), (out - ref).abs().max()


@pytest.mark.parametrize("lens", [[4000], [1, 5000, 300]])
def test_long_caches_are_split_and_joined(lens):
    cache, _, g = make(lens, heads=1, dim=64, block=64, dtype=I8, weight=True)
    cache.weight.zero_()
    x = torch.randn(len(lens), 1, 2, 64, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    q = (torch.randn(len(lens), 2, 2, 64, generator=g) * 3).cuda()
    attend(cache, q, None, track=True)


@pytest.mark.parametrize("dim,dtype", [(64, I8), (128, F8)])
@pytest.mark.parametrize("batch,heads,group,T", [(16, 20, 1, 1), (16, 20, 12, 1), (16, 10, 2, 20),
                                                 (4, 4, 1, 200)])
@pytest.mark.parametrize("mean", [0.0, 1.0])
def test_fp32_keeps_its_precision_over_thousands_of_keys(mean, batch, heads, group, T, dim, dtype):
    """Heads enough that a CTA takes 4096 keys in one part, and V with and
    without a mean (its sums then grow key by key). The relative error has
    2e-7 from q (22 bits), 4e-7 from the scores (8 products of 16, each with
    its last place lost), 1.5e-7 from P and 4e-7 from the sums of 256 products
    in fp32: 1.2e-6. A lost second plane of q or P would be 1e-4."""
    L = 4090 - T
    cache, _, g = make([0] * batch, heads=heads, dim=dim, block=64, dtype=dtype, room=4090)
    x = torch.randn(2, batch, heads, 4090, dim, generator=torch.Generator("cuda").manual_seed(7),
                    device="cuda")
    x[1] += mean
    ops.kv8_append(cache, x[0] * 1.5, x[1])
    cache.lens += L
    q = torch.randn(batch, heads * group, T, dim, generator=g).cuda()
    out = ops.kv8_attention(q, cache)
    count = torch.full((batch,), T, dtype=torch.int32, device="cuda")
    k, v = ops.kv8_read(cache, 4090, counts=count)
    off = size = 0.0
    hidden = torch.arange(4090, device="cuda") > L + torch.arange(T, device="cuda")[:, None]
    for b in range(batch):
        s = q[b].double().view(heads, group, T, dim) @ k[b].double().transpose(1, 2)[:, None]
        p = torch.softmax((s * dim ** -0.5).masked_fill(hidden, -math.inf), -1)
        want = (p @ v[b].double()[:, None]).view(heads * group, T, dim)
        off += float((out[b].double() - want).square().sum())
        size += float(want.square().sum())
    assert math.sqrt(off / size) <= 1.2e-6
    clean()


@pytest.mark.parametrize("dim,dtype", [(32, I8), (64, F8), (128, I8)])
@pytest.mark.parametrize("group,T", [(1, 1), (12, 1), (1, 20), (3, 20), (1, 300)])
@pytest.mark.parametrize("kind", [F16, BF16])
def test_16_bit_outputs_are_as_near_as_their_own_rounding(kind, group, T, dim, dtype):
    """Against float64, relative to the error of rounding the float64 result to
    the type. fp16 (2.1e-4): q and two planes of P leave less than 2e-6, which
    does not show. bf16 (1.65e-3): P rounded to fp16 is off by at most 2.9e-4
    (2^-11 of a value over the square root of 3), which adds in squares: 1.016."""
    cache, _, g = make([2000, 1500], heads=3, dim=dim, block=32, dtype=dtype, room=T)
    x = torch.randn(2, 2, 3, T, dim, generator=g).cuda()
    ops.kv8_append(cache, x[0], x[1])
    q = torch.randn(2, 3 * group, T, dim, generator=g).to(kind).cuda()
    out = ops.kv8_attention(q, cache)
    count = torch.full((2,), T, dtype=torch.int32, device="cuda")
    k, v = ops.kv8_read(cache, 2000 + T, counts=count)
    off = own = 0.0
    for b, have in enumerate((2000, 1500)):
        pos = torch.arange(2000 + T, device="cuda")
        hidden = pos > have + torch.arange(T, device="cuda")[:, None]
        s = q[b].double().view(3, group, T, dim) @ k[b].double().transpose(1, 2)[:, None]
        p = torch.softmax((s * dim ** -0.5).masked_fill(hidden, -math.inf), -1)
        want = (p @ v[b].double()[:, None]).view(3 * group, T, dim)
        off += float((out[b].double() - want).square().sum())
        own += float((want.to(kind).double() - want).square().sum())
    assert math.sqrt(off / own) <= 1.03
    clean()


def test_scores_that_grow_along_the_cache():
    """Each page's scores exceed the last one's by far, then fall: the running
    reference moves often, and early weights vanish against late ones."""
    cache, _, g = make([0], heads=1, dim=64, block=16, room=400)
    ramp = torch.cat([torch.linspace(0, 60, 200), torch.linspace(60, -60, 200)])
    k = ramp.view(1, 1, -1, 1) / 64 + torch.randn(1, 1, 400, 64, generator=g) * 0.01
    v = torch.randn(1, 1, 400, 64, generator=g)
    ops.kv8_append(cache, k.cuda(), v.cuda())
    cache.lens += 399
    for kind in (F32, BF16, F16):
        attend(cache, torch.full((1, 3, 1, 64), 1.0, device="cuda").to(kind), None, scale=1.0)


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("mag", [1e-30, 1e-5, 1e4])
def test_rows_of_any_magnitude(kind, mag):
    """q rows are scaled by powers of two before they are rounded to fp16."""
    if kind == F16 and mag < 1e-20:
        pytest.skip("not an fp16 number")
    cache, _, g = make([70], heads=1, dim=64, block=16)
    x = torch.randn(1, 1, 20, 64, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    q = (torch.randn(1, 1, 20, 64, generator=g) * mag).to(kind).cuda()
    attend(cache, q, None, scale=1.0 / (8 * mag))


def test_v_blocks_of_very_different_scales():
    cache, _, g = make([0], heads=1, dim=64, block=16, room=160)
    k = torch.randn(1, 1, 160, 64, generator=g)
    v = torch.randn(1, 1, 160, 64, generator=g) * torch.logspace(-4, 0, 160).view(1, 1, -1, 1)
    ops.kv8_append(cache, k.cuda(), v.cuda())
    cache.lens += 130
    for kind in (F32, BF16):
        q = torch.randn(1, 2, 30, 64, generator=g).to(kind).cuda()
        attend(cache, q, None)


def test_strided_views_offsets_and_out():
    """q, k and v as views of one fused projection, out as a merged-head view,
    rows that are only element aligned."""
    cache, _, g = make([40, 7], heads=2, dim=64, block=16, room=32)
    for kind in (F32, BF16):
        for shift in (0, 1):
            raw = torch.randn(2 * 9 * 6 * 64 + shift, generator=g).to(kind).cuda()
            qkv = raw[shift:].view(2, 9, 6, 64).permute(0, 2, 1, 3)
            ops.kv8_append(cache, qkv[:, 2:4], qkv[:, 4:])
            out = torch.full((2, 9, 2, 64), math.nan, dtype=kind, device="cuda").permute(0, 2, 1, 3)
            got = attend(cache, qkv[:, :2], None, out=out)
            assert got.data_ptr() == out.data_ptr()


@pytest.mark.parametrize("kind", [F32, BF16])
def test_few_rows_under_a_table_of_a_million_tokens(kind):
    """16 rows of a kv head with weights recorded: kept scores would take 8 GB,
    so the kernel for many rows serves the call; with max_len the other one."""
    table = torch.zeros(16, 1 << 14, dtype=torch.int32, device="cuda")
    table[:, 0] = torch.arange(1, 17, device="cuda")
    g = torch.Generator().manual_seed(2)
    lens = torch.randint(0, 40, (16,), generator=g).int().cuda()
    cache = ops.KV8Cache.empty(17, 8, 64, 64, table, torch.zeros_like(lens), I8, weight=True)
    x = torch.randn(2, 16, 8, 40, 64, generator=g).cuda()
    ops.kv8_append(cache, x[0], x[1], counts=lens + 1)
    cache.lens.copy_(lens)
    q = torch.randn(16, 128, 1, 64, generator=g).to(kind).cuda()
    attend(cache, q, None, track=True)
    attend(cache, q, None, track=True, max_len=64)


def test_max_len_cuts_the_work_not_the_result():
    cache, _, g = make([100, 37], heads=2, dim=64, block=16, room=4000)
    x = torch.randn(2, 2, 1, 64, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    q = torch.randn(2, 4, 1, 64, generator=g).cuda()
    attend(cache, q, None, max_len=101)
    ops.kv8_attention(q, cache, max_len=64)      # a broken promise is recorded, not followed
    assert _lib.lib().kf_device_status(1) == 6


def test_bad_pages_and_lengths_are_refused_on_the_device():
    """A page number outside the pool hides its tokens, a length beyond the
    table is cut; both are recorded, and the next call is clean."""
    cache, _, g = make([40, 7], heads=2, dim=64, block=16, weight=True)
    cache.weight.zero_()
    q = torch.randn(2, 2, 1, 64, generator=g).cuda()
    x = torch.randn(2, 2, 1, 64, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    good = ops.kv8_attention(q, cache)
    keep = int(cache.table[0, 1])
    for wrong in (-1, 1 << 30):
        cache.table[0, 1] = wrong
        out = ops.kv8_attention(q, cache, track=True)
        ops.kv8_read(cache, 64)
        assert _lib.lib().kf_device_status(1) == 6
        assert torch.equal(out[1], good[1]) and torch.isfinite(out).all()
        assert not torch.equal(out[0], good[0])
    cache.table[0, 1] = keep
    cache.lens[1] = 1 << 29
    ops.kv8_append(cache, x, x)
    ops.kv8_attention(q, cache)
    ops.kv8_read(cache, 64)
    assert _lib.lib().kf_device_status(1) == 6
    cache.lens[1] = -5
    ops.kv8_attention(q, cache)
    assert _lib.lib().kf_device_status(1) == 6
    cache.lens[1] = 7
    assert torch.equal(ops.kv8_attention(q, cache)[0], good[0])
    clean()


@pytest.mark.parametrize("T", [1, 5, 80])
def test_a_negative_length_holds_nothing_and_takes_nothing(T):
    """Its new tokens are not written (they would fall on tokens that are valid
    once the length is), its queries see no key, an eviction keeps none."""
    cache, spare, g = make([40, 7], heads=2, dim=64, block=16, room=96, weight=True, spare=4)
    cache.weight.zero_()
    held = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8),
                                cache.scale, cache.weight)]
    x = (torch.randn(2, 2, T, 64, generator=g) * 9).cuda()
    q = torch.randn(2, 4, T, 64, generator=g).cuda()
    cache.lens[1] = -5
    for counts in (None, torch.full((2,), T, dtype=torch.int32, device="cuda")):
        cache.lens[0] = 40
        ops.kv8_append(cache, x, x, counts=counts)
        assert _lib.lib().kf_device_status(1) == 6
        own = cache.table[1].long()
        for was, t in zip(held, (cache.k.view(torch.uint8), cache.v.view(torch.uint8),
                                 cache.scale, cache.weight)):
            assert torch.equal(t[own].nan_to_num(-1), was[own].nan_to_num(-1))
        out, lse = ops.kv8_attention(q, cache, counts=counts, track=True, return_lse=True)
        assert _lib.lib().kf_device_status(1) == 6
        assert not out[1].any() and torch.isinf(lse[1]).all() and out[0].any()
        assert not cache.weight[own].any()
        k, v = ops.kv8_read(cache, 64, counts=counts)
        assert _lib.lib().kf_device_status(1) == 6
        assert not k[1].any() and not v[1].any() and k[0].any()
        kept, new = ops.kv8_evict(cache, spare.view(2, 2), 20, 3)
        assert _lib.lib().kf_device_status(1) == 6
        assert (kept[1] == -1).all() and new.lens.tolist() == [20, 0]


def test_nothing_to_do():
    cache, _, _ = make([0, 0], heads=2, dim=64, block=16)
    q = torch.randn(2, 2, 0, 64, device="cuda")
    assert ops.kv8_attention(q, cache).shape == (2, 2, 0, 64)
    ops.kv8_append(cache, q, q)
    k, v = ops.kv8_read(cache, 0)
    assert k.numel() == 0
    zero = torch.zeros(2, dtype=torch.int32, device="cuda")
    q = torch.randn(2, 2, 3, 64, device="cuda")
    out, lse = ops.kv8_attention(q, cache, counts=zero, return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    clean()


@pytest.mark.parametrize("T", [1, 70])
@pytest.mark.parametrize("batch,blocks,pages", [(0, 4, 8), (2, 0, 8), (2, 4, 0), (0, 0, 0)])
def test_no_sequence_no_page_no_table(batch, blocks, pages, T):
    table = torch.zeros(batch, blocks, dtype=torch.int32, device="cuda")
    lens = torch.zeros(batch, dtype=torch.int32, device="cuda")
    cache = ops.KV8Cache.empty(pages, 2, 16, 64, table, lens, weight=True)
    held = cache.k.clone()
    x = torch.randn(batch, 2, T, 64, device="cuda")
    none = torch.zeros_like(lens)
    ops.kv8_append(cache, x, x, counts=none)
    out, lse = ops.kv8_attention(x, cache, counts=none, track=True, return_lse=True)
    assert out.shape == x.shape and not out.any() and torch.isinf(lse).all()
    k, v = ops.kv8_read(cache, 5)
    assert k.shape == (batch, 2, 5, 64) and not k.any() and not v.any()
    kept, new = ops.kv8_evict(cache, torch.zeros(batch, 2, dtype=torch.int32, device="cuda"), 20)
    assert kept.shape == (batch, 2, 20) and (kept == -1).all() and not new.lens.any()
    clean()
    ops.kv8_append(cache, x, x)                       # no place: recorded where there is a batch
    ops.kv8_attention(x, cache)
    assert _lib.lib().kf_device_status(1) == (6 if batch and not (blocks and pages) else 0)
    assert torch.equal(cache.k, held)


def test_repeated_calls_give_the_same_bits():
    cache, _, g = make([3000, 900], heads=2, dim=64, block=64, weight=True)
    for T in (1, 60):
        x = torch.randn(2, 2, T, 64, generator=g).cuda()
        ops.kv8_append(cache, x, x)
        q = torch.randn(2, 8, T, 64, generator=g).cuda()
        runs = []
        for _ in range(3):
            cache.weight.zero_()
            runs.append((ops.kv8_attention(q, cache, track=True), cache.weight.clone()))
        for out, w in runs[1:]:
            assert torch.equal(out, runs[0][0]) and torch.equal(w, runs[0][1])


def test_a_step_in_a_graph_and_on_another_stream():
    """append, attention and the lengths' advance captured once and replayed,
    against the same steps run eagerly on a side stream."""
    def build():
        return make([30, 3], heads=2, dim=64, block=16, weight=True, seed=5)[0]

    g = torch.Generator().manual_seed(9)
    xs = torch.randn(6, 2, 6, 1, 64, generator=g).cuda()
    x = xs[0].clone()
    a, b = build(), build()
    for c in (a, b):
        c.weight.zero_()

    def step(cache, x):
        ops.kv8_append(cache, x[:, 2:4], x[:, 4:])
        out = ops.kv8_attention(x[:, :2], cache, track=True)
        cache.lens += 1
        return out

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    eager = []
    with torch.cuda.stream(side):
        for i in range(6):
            eager.append(step(a, xs[i]))
    torch.cuda.current_stream().wait_stream(side)
    lens = b.lens.clone()
    step(b, x)                       # warm up, then back to where it began
    fresh = build()
    for t, u in ((b.k, fresh.k), (b.v, fresh.v), (b.scale, fresh.scale)):
        t.view(torch.uint8).copy_(u.view(torch.uint8))
    b.weight.zero_()
    b.lens.copy_(lens)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(b, x)
    b.lens.copy_(lens)
    for i in range(6):
        x.copy_(xs[i])
        graph.replay()
        assert torch.equal(out, eager[i]), i
    assert torch.equal(a.weight.nan_to_num(-1), b.weight.nan_to_num(-1))


@pytest.mark.parametrize("track", [False, True])
@pytest.mark.parametrize("kind,dim", [(BF16, 64), (BF16, 32), (F16, 64), (BF16, 128), (F32, 64),
                                      (F32, 128)])
def test_waits_that_run_out_end_the_call_and_the_next_is_right(kind, dim, track):
    """Under a limit of one cycle the waits of the prompt kernels give up where
    what they wait for is not there at once (which at head_dim <= 64 and bf16
    it never is: products are issued as their inputs come). Every role leaves,
    the call returns, the status word tells, the next call is as before."""
    L = _lib.lib()
    cache, _, g = make([700, 90], heads=2, dim=dim, block=32, dtype=F8, weight=True, room=200)
    x = torch.randn(2, 2, 200, dim, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    q = torch.randn(2, 4, 200, dim, generator=g).to(kind).cuda()
    cache.weight.zero_()
    good = ops.kv8_attention(q, cache, track=track)
    weight = cache.weight.clone()
    clean()
    _lib.check(L.kf_set_wait_limit(1), "kf_set_wait_limit")
    try:
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        ops.kv8_attention(q, cache, track=track)
        end.record()
        torch.cuda.synchronize()
        status = L.kf_device_status(1)
    finally:
        L.kf_set_wait_limit(0)
    assert begin.elapsed_time(end) < 1000
    assert status in ((1, 2, 4) if kind == BF16 and dim <= 64 else (0, 1, 2, 4))
    cache.weight.zero_()
    assert torch.equal(ops.kv8_attention(q, cache, track=track), good)
    assert torch.equal(cache.weight, weight)
    clean()


# ---------------------------------------------------------------- evict


@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("dim,block,budget,recent", [(64, 16, 20, 5), (16, 128, 200, 0),
                                                     (128, 32, 33, 33), (32, 64, 1, 0),
                                                     (64, 128, 129, 1)])
def test_evict_keeps_the_heaviest_and_the_latest(dim, block, budget, recent, dtype):
    lens = [0, 1, budget - 1, budget, budget + 1, 3 * budget + 40, 700]
    cols = -(-budget // block)
    cache, spare, g = make(lens, heads=3, dim=dim, block=block, dtype=dtype, weight=True,
                           spare=len(lens) * cols, seed=budget)
    # few distinct weights, so ties decide; zeros of both signs, infinities, NaN
    w = torch.randint(0, 6, cache.weight.shape, generator=g).float() / 4
    w[torch.rand(w.shape, generator=g) < 0.02] = math.inf
    w[torch.rand(w.shape, generator=g) < 0.02] = -0.0
    w[torch.rand(w.shape, generator=g) < 0.01] = math.nan
    cache.weight.copy_(w)
    table_out = spare.view(len(lens), cols)
    plain = Plain(cache)
    before = [t.clone() for t in (cache.k.view(torch.uint8), cache.scale)]
    kept, new = ops.kv8_evict(cache, table_out, budget, recent)
    want = plain.evict(table_out, budget, recent)
    assert torch.equal(kept.cpu(), want)
    assert new.lens.tolist() == [min(n, budget) for n in lens]
    plain.table, plain.lens = table_out.cpu(), new.lens.cpu()
    same_codes(new, plain, new.lens)
    got = cache.weight.cpu()
    for b, n in enumerate(new.lens.tolist()):
        for pos in range(n):
            page, slot = plain.spot(b, pos)
            assert torch.equal(got[page, :, slot].nan_to_num(-7),
                               plain.weight[page, :, slot].nan_to_num(-7))
    # the old pages are as they were
    old = cache.table.flatten().long()
    assert torch.equal(cache.k.view(torch.uint8)[old], before[0][old])
    assert torch.equal(cache.scale[old].nan_to_num(-1), before[1][old].nan_to_num(-1))
    clean()


def test_evict_long_rows():
    """Rows longer than the selection's tile, weights of every magnitude."""
    cache, spare, g = make([9000, 4097], heads=2, dim=16, block=128, weight=True, spare=2 * 16)
    w = torch.exp(torch.randn(cache.weight.shape, generator=g) * 20)
    cache.weight.copy_(w)
    kept, new = ops.kv8_evict(cache, spare.view(2, 16), 2000, 100)
    for b, n in enumerate((9000, 4097)):
        for h in range(2):
            row = torch.cat([w[int(p), h] for p in cache.table[b]])[:n]
            order = torch.sort(row[:n - 100], descending=True, stable=True).indices[:1900]
            want = torch.cat([order.sort().values, torch.arange(n - 100, n)])
            assert torch.equal(kept[b, h].cpu().long(), want)
    clean()


def test_evict_rows_beyond_what_shared_memory_holds():
    """More candidates than the selection keeps as keys on the chip."""
    n = 56000
    cache, spare, g = make([n], heads=1, dim=16, block=128, weight=True, spare=40)
    w = torch.randint(0, 40, cache.weight.shape, generator=g).float()
    cache.weight.copy_(w)
    kept, _ = ops.kv8_evict(cache, spare.view(1, 40), 5000, 7)
    row = torch.cat([w[int(p), 0] for p in cache.table[0]])[:n]
    order = torch.sort(row[:n - 7], descending=True, stable=True).indices[:4993]
    want = torch.cat([order.sort().values, torch.arange(n - 7, n)])
    assert torch.equal(kept[0, 0].cpu().long(), want)
    clean()


def test_evicted_cache_serves_on():
    """Decode, evict, decode: the next token attends to what was kept."""
    cache, spare, g = make([90, 12], heads=2, dim=64, block=16, weight=True, spare=2 * 5)
    cache.weight.zero_()
    x = torch.randn(2, 2, 1, 64, generator=g).cuda()
    ops.kv8_append(cache, x, x)
    attend(cache, torch.randn(2, 4, 1, 64, generator=g).cuda(), None, track=True)
    cache.lens += 1
    kept, new = ops.kv8_evict(cache, spare.view(2, 5), 64, 16)
    assert kept[0, 0].tolist()[-16:] == list(range(75, 91))
    ops.kv8_append(new, x, -x)
    attend(new, torch.randn(2, 4, 1, 64, generator=g).cuda(), None, track=True)


# ---------------------------------------------------------------- refusals


def test_refusals():
    cache, spare, g = make([40, 7], heads=2, dim=64, block=16, weight=True, spare=4)
    q = torch.randn(2, 4, 1, 64, device="cuda")
    for bad in (q[:1], q[:, :3], q[..., :32], q.transpose(2, 3)):
        with pytest.raises(ValueError):
            ops.kv8_attention(bad, cache)
    with pytest.raises(TypeError):
        ops.kv8_attention(q.double(), cache)
    with pytest.raises(ValueError):
        ops.kv8_attention(q.cpu(), cache)
    with pytest.raises(ValueError):
        ops.kv8_attention(q, cache, counts=torch.zeros(2, device="cuda"))
    with pytest.raises(ValueError):
        ops.kv8_attention(q, cache, out=torch.empty_like(q, dtype=F16))
    with pytest.raises(ValueError):
        ops.kv8_append(cache, q, q)                      # 4 heads into a cache of 2
    with pytest.raises(TypeError):
        ops.kv8_append(cache, q[:, :2], q[:, 2:].half())
    with pytest.raises(TypeError):
        ops.kv8_read(cache, 4, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.kv8_read(cache, 4, start=torch.zeros(1, dtype=torch.int32, device="cuda"))
    out = spare.view(2, 2)
    for budget, recent in ((0, 0), (8, 9), (8, -1), (33, 0)):
        with pytest.raises(ValueError):
            ops.kv8_evict(cache, out, budget, recent)
    bare = ops.KV8Cache(cache.k, cache.v, cache.scale, cache.table, cache.lens)
    with pytest.raises(ValueError):
        ops.kv8_evict(bare, out, 8)
    with pytest.raises(ValueError):
        ops.kv8_attention(q, bare, track=True)
    with pytest.raises(ValueError):
        ops.KV8Cache(cache.k, cache.v[:1], cache.scale, cache.table, cache.lens)
    with pytest.raises(TypeError):
        ops.KV8Cache(cache.k, cache.v, cache.scale, cache.table.long(), cache.lens)
    with pytest.raises(TypeError):
        ops.KV8Cache(cache.k, cache.v, cache.scale, cache.table, cache.lens.long())
    with pytest.raises(AttributeError):
        cache.lens = cache.lens + 1                      # the C side would not see it
    cache.lens += 0
    clean()
