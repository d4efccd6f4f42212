"""kv8_attention_shared and kv8_copy on the GPU: attention against float64 within
the bounds of its roundings, copies bit for bit."""
from __future__ import annotations

import math

import pytest
import torch

from shared_plain import attention64, make_groups
from techjam2026_b200 import _lib, ops

pytestmark = pytest.mark.gpu

I8, F8 = torch.int8, torch.float8_e4m3fn
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def status():
    return _lib.lib().kf_device_status(1)


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def check(cache, starts, shared, q, counts=None, causal=True, scale=None, **kw):
    out, lse = ops.kv8_attention_shared(q, cache, starts, shared, counts=counts, causal=causal,
                                        sm_scale=scale, return_lse=True, **kw)
    want, tol, want_lse, tol_lse = attention64(
        q, cache, counts, causal, cache.head_dim ** -0.5 if scale is None else scale)
    off = (out.double() - want).abs()
    assert (off <= tol).all(), (off - tol).max()
    none = torch.isinf(want_lse)
    assert torch.equal(torch.isinf(lse), none)
    off = (lse.double() - want_lse).abs()[~none]
    assert (off <= tol_lse[~none]).all(), off.max()
    assert status() == 0
    return out


def queries(cache, group, T, kind=F32, seed=1):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(cache.batch, cache.kv_heads * group, T, cache.head_dim,
                       generator=g).to(kind).cuda()


def append(cache, T, counts=None, seed=2):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(2, cache.batch, cache.kv_heads, T, cache.head_dim, generator=g).cuda()
    ops.kv8_append(cache, x[0], x[1], counts=counts)


# ---------------------------------------------------------------- attention


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("dtype", [I8, F8])
@pytest.mark.parametrize("dim,block", [(16, 16), (32, 128), (64, 64), (128, 32)])
@pytest.mark.parametrize("group", [1, 3])
def test_single_tokens(group, dim, block, dtype, kind):
    """Groups of one, of several and of none, sequences in no group, nothing of
    their own, nothing shared."""
    cache, starts, shared = make_groups([1, 5, 0, 3], [2 * block, 5 * block, block, 0],
                                        [0, 0, 1, block - 1, block, 7, 40, 0, 1, 9, 0], dim=dim,
                                        block=block, dtype=dtype, rest=2)
    append(cache, 1)
    check(cache, starts, shared, queries(cache, group, 1, kind))


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("dim,dtype", [(16, I8), (32, F8), (64, I8), (64, F8), (128, I8), (128, F8)])
@pytest.mark.parametrize("members,group,keys", [(70, 1, 640), (20, 8, 320), (33, 4, 1664)])
def test_many_rows_of_a_group(members, group, keys, dim, dtype, kind):
    """More rows than a tile of 128, and a tile that ends between groups."""
    cache, starts, shared = make_groups([members, 3, members // 2], [keys, 64, keys - 64],
                                        [(5 * b) % 23 for b in range(members + 3 + members // 2)],
                                        dim=dim, block=64, dtype=dtype, heads=2)
    append(cache, 1)
    check(cache, starts, shared, queries(cache, group, 1, kind))


@pytest.mark.parametrize("kind", [F32, BF16, F16])
@pytest.mark.parametrize("dim,block,dtype", [(64, 16, I8), (128, 64, F8), (32, 32, F8)])
@pytest.mark.parametrize("T,group", [(2, 1), (5, 4), (40, 1), (37, 3), (130, 2)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(causal, T, group, dim, block, dtype, kind):
    """Ragged chunks over shared pages: counts of 0, 1 and all."""
    cache, starts, shared = make_groups([4, 1, 2], [6 * block, block, 0],
                                        [3, 0, block, 2 * block + 1, 5, 0, 11], dim=dim,
                                        block=block, dtype=dtype, room=T)
    counts = ints([T, 0, 1, T - 1, T, max(1, T // 2), T])
    append(cache, T, counts)
    check(cache, starts, shared, queries(cache, group, T, kind), counts, causal)


@pytest.mark.parametrize("kind", [F32, BF16])
@pytest.mark.parametrize("members,T,group", [(3, 1, 1), (40, 1, 4), (6, 30, 2)])
def test_long_shared_prefixes_are_split_and_joined(members, T, group, kind):
    cache, starts, shared = make_groups([members, 2], [9024, 4160], [17] * (members + 2), heads=1,
                                        dim=64, block=64, room=T)
    append(cache, T)
    check(cache, starts, shared, queries(cache, group, T, kind) * 3)


@pytest.mark.parametrize("kind,dim,dtype", [(F32, 32, I8), (BF16, 64, F8), (F16, 128, I8),
                                            (F32, 128, F8), (BF16, 16, F8)])
@pytest.mark.parametrize("T", [1, 9])
def test_more_tiles_than_processors(T, kind, dim, dtype):
    """Many tiles of unequal lengths: a CTA ends one and begins others, and some
    groups share nothing or have one sequence."""
    sizes = [70, 1, 40, 0, 55, 64]
    cache, starts, shared = make_groups(sizes, [640, 576, 64, 128, 0, 1280],
                                        [b % 19 for b in range(sum(sizes) + 1)], dim=dim, block=64,
                                        dtype=dtype, heads=16, room=T, rest=1)
    counts = None if T == 1 else ints([b % (T + 1) for b in range(sum(sizes) + 1)])
    append(cache, T, counts)
    check(cache, starts, shared, queries(cache, 8 if T == 1 else 2, T, kind), counts)


@pytest.mark.parametrize("T,group", [(1, 1), (70, 1)])
def test_more_groups_than_one_list_holds(T, group):
    cache, starts, shared = make_groups([1] * 1100, [16 * (n % 4) for n in range(1100)],
                                        [n % 3 for n in range(1100)], dim=16, block=16, heads=1,
                                        room=T)
    append(cache, T)
    check(cache, starts, shared, queries(cache, group, T, BF16))


@pytest.mark.parametrize("kind,dim", [(BF16, 64), (BF16, 32), (F16, 64), (BF16, 128), (F32, 64),
                                      (F32, 128)])
@pytest.mark.parametrize("members,T", [(40, 1), (90, 1), (6, 100)])
def test_waits_that_run_out_end_the_call_and_the_next_is_right(members, T, kind, dim):
    """Under a limit of one cycle the waits of the tensor-memory kernel give up where
    what they wait for is not there at once. Every role leaves, the call returns, the
    next one is as before."""
    L = _lib.lib()
    cache, starts, shared = make_groups([members, 3], [1216, 640], [20] * (members + 3), dim=dim,
                                        block=32, dtype=F8, heads=3, room=T)
    append(cache, T)
    q = queries(cache, 2, T, kind)
    good = check(cache, starts, shared, q)
    _lib.check(L.kf_set_wait_limit(1), "kf_set_wait_limit")
    try:
        begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
        begin.record()
        ops.kv8_attention_shared(q, cache, starts, shared)
        end.record()
        torch.cuda.synchronize()
        got = status()
    finally:
        L.kf_set_wait_limit(0)
    assert begin.elapsed_time(end) < 1000
    assert got in (0, 1, 2, 4)
    assert torch.equal(ops.kv8_attention_shared(q, cache, starts, shared), good)
    assert status() == 0


@pytest.mark.parametrize("kind,dim", [(BF16, 64), (BF16, 128), (F16, 32), (F16, 128), (F32, 64),
                                      (F32, 128)])
@pytest.mark.parametrize("sizes,T", [([80, 3], 1), ([150, 3], 1), ([6, 3], 100),
                                     ([70, 1, 40, 0, 55, 64], 4)])
def test_waits_that_run_out_are_recorded(sizes, T, kind, dim):
    """With a limit of one cycle some wait gives up in every configuration of the
    tensor-memory kernel (more than 64 rows a group on average, of one tile, of two,
    of ragged chunks); with longer ones it is one of a later step, or of a later
    stretch of a CTA that has several (the last sizes: 16 heads of 230 sequences are
    more tiles than processors). The next call is right."""
    L = _lib.lib()
    many = len(sizes) > 2
    shared = [640, 576, 64, 128, 64, 1280] if many else [1216, 640]
    B = sum(sizes)
    cache, starts, shared = make_groups(sizes, shared, [b % 19 for b in range(B)], dim=dim, block=64,
                                        dtype=F8, heads=16 if many else 3, room=T)
    append(cache, T)
    q = queries(cache, 2, T, kind)
    good = ops.kv8_attention_shared(q, cache, starts, shared)
    assert status() == 0
    seen = {}
    try:
        for limit in (1, 1, 1, 500, 3000, 10000, 40000):
            _lib.check(L.kf_set_wait_limit(limit), "kf_set_wait_limit")
            begin, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            begin.record()
            ops.kv8_attention_shared(q, cache, starts, shared)
            end.record()
            torch.cuda.synchronize()
            assert begin.elapsed_time(end) < 1000
            seen.setdefault(limit, set()).add(status())
    finally:
        L.kf_set_wait_limit(0)
    assert all(codes <= {0, 1, 2, 4} for codes in seen.values()), seen
    assert seen[1] & {1, 2, 4}, seen
    assert torch.equal(ops.kv8_attention_shared(q, cache, starts, shared), good)
    assert status() == 0


def test_what_counts_as_shared_is_cut():
    """shared is cut to whole pages, to the shortest of the group's lens and to
    max_shared; the result is that of kv8_attention whatever it says."""
    cache, starts, _ = make_groups([3, 2], [64, 48], [20, 0, 40, 0, 33], block=16)
    append(cache, 1)
    q = queries(cache, 2, 1)
    for shared in ([64, 48], [79, 50], [64 + 16, 48], [1 << 30, 1 << 30], [63, 47], [-5, 0]):
        # (a value beyond what is common is cut by the sequence that holds no more)
        check(cache, starts, ints(shared), q)
    for max_shared in (1, 16, 40, 63, 64, 1 << 20):
        check(cache, starts, ints([64, 48]), q, max_shared=max_shared)
    check(cache, starts, ints([64, 48]), q, max_shared=64, max_own=41)


def test_own_tokens_beyond_their_bound_are_cut_and_recorded():
    cache, starts, shared = make_groups([2], [32], [10, 200], block=16)
    append(cache, 1)
    q = queries(cache, 1, 1)
    whole = ops.kv8_attention(q, cache)
    out = ops.kv8_attention_shared(q, cache, starts, shared, max_own=128)
    assert status() == 6
    assert (out[0] - whole[0]).abs().max() <= 1e-5 * whole[0].abs().max()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("starts", [[0, 3, 1, 4], [0, -1, 2, 4], [0, 2, 9, 4], [5, 1 << 30, -9, 2]])
def test_starts_out_of_order_are_recorded_and_fault_nothing(starts):
    cache, _, _ = make_groups([4], [64], [3, 4, 5, 6], block=16)
    append(cache, 1)
    ops.kv8_attention_shared(queries(cache, 2, 1), cache, ints(starts), ints([64, 64, 64]))
    assert status() == 7


@pytest.mark.parametrize("members", [4, 40])
def test_a_refused_page_hides_its_tokens_from_the_group(members):
    cache, starts, shared = make_groups([members], [96], [9] * members, block=16, heads=1)
    append(cache, 1)
    q = queries(cache, 4, 1)
    table = cache.table.clone()
    for wrong in (-1, cache.k.shape[0], 1 << 30):
        cache.table[:, 2] = wrong
        out = ops.kv8_attention_shared(q, cache, starts, shared)
        assert status() == 6
        # without the block of the refused page, everything stands 16 earlier
        cut = ops.KV8Cache(cache.k, cache.v, cache.scale,
                           torch.cat([table[:, :2], table[:, 3:]], 1).contiguous(), cache.lens - 16)
        want, tol, _, _ = attention64(q, cut, None, True, 0.125)
        assert ((out.double() - want).abs() <= tol).all()


@pytest.mark.parametrize("which", [0, 1])
@pytest.mark.parametrize("members", [3, 40])
def test_a_spoiled_page_reaches_the_rows_that_see_it(members, which):
    """A page whose scale is NaN: a shared one spoils its group, a sequence's own
    one that sequence; others are as without it."""
    cache, starts, shared = make_groups([members, 2], [64, 32], [20] * (members + 2), block=16,
                                        heads=1)
    append(cache, 1)
    q = queries(cache, 4, 1)
    fine = ops.kv8_attention_shared(q, cache, starts, shared)
    page = int(cache.table[0, 1])
    keep = cache.scale[page].clone()
    cache.scale[page, :, which] = math.nan
    out = ops.kv8_attention_shared(q, cache, starts, shared)
    assert torch.isnan(out[:members]).all()
    assert torch.equal(out[members:], fine[members:])
    cache.scale[page] = keep
    cache.scale[int(cache.table[1, 4]), :, which] = math.nan
    out = ops.kv8_attention_shared(q, cache, starts, shared)
    assert torch.isnan(out[1]).all()
    rest = [b for b in range(members + 2) if b != 1]
    assert torch.equal(out[rest], fine[rest])
    status()


def test_a_sequence_of_a_negative_length_holds_nothing():
    cache, starts, shared = make_groups([2, 3], [32, 48], [5, 6, 7, 8, 9], block=16)
    append(cache, 1)
    q = queries(cache, 1, 1)
    cache.lens[3] = -4
    out, lse = ops.kv8_attention_shared(q, cache, starts, shared, return_lse=True)
    assert status() == 6
    assert not out[3].any() and torch.isinf(lse[3]).all()
    cache.lens[3] = 0       # (nothing is shared then: the shortest holds none)
    want, tol, _, _ = attention64(q, cache, ints([1, 1, 1, 0, 1]), True, 0.125)
    assert ((out.double() - want).abs() <= tol)[[0, 1, 2, 4]].all()


@pytest.mark.parametrize("kind,dim", [(F32, 32), (BF16, 64), (F16, 128)])
@pytest.mark.parametrize("members,T", [(5, 1), (40, 1), (6, 9), (12, 9), (4, 100)])
@pytest.mark.parametrize("idle", [[0], [2], [0, 1, 3]])
def test_members_without_a_new_token_take_nothing_from_the_others(idle, members, T, kind, dim):
    """Idle members of a group: of length 0, of a negative one, with more tokens of
    their own than the bound and a table row that names no page. The others have what
    they share, under bounds that just hold."""
    own = [(7 * b) % 20 for b in range(members + 3)]
    for i in idle:
        own[i] = 90
    cache, starts, shared = make_groups([members, 3], [320, 64], own, dim=dim, block=16, room=T)
    counts = [1 + (5 * b) % T for b in range(members + 3)]
    for i in idle:
        counts[i] = 0
    counts = ints(counts)
    append(cache, T, counts)
    bounds = dict(max_shared=320, max_own=19 + T)
    q = queries(cache, 4, T, kind)
    check(cache, starts, shared, q, counts, **bounds)
    cache.table[idle] = -1
    check(cache, starts, shared, q, counts, **bounds)
    cache.lens[idle] = 0
    want = check(cache, starts, shared, q, counts, **bounds)
    cache.lens[idle] = -3
    out = ops.kv8_attention_shared(q, cache, starts, shared, counts=counts, **bounds)
    assert status() == 6
    assert torch.equal(out, want) and not out[idle].any()


def test_a_group_of_idle_members_only():
    cache, starts, shared = make_groups([3, 2], [160, 64], [200, 100, 3, 4, 5], block=16)
    counts = ints([0, 0, 0, 1, 1])
    append(cache, 1, counts)
    check(cache, starts, shared, queries(cache, 2, 1), counts, max_shared=160, max_own=6)


def test_strided_views_and_out():
    cache, starts, shared = make_groups([3], [80], [3, 0, 30], heads=2, dim=32, block=16, room=9)
    append(cache, 7)
    for kind, pad in ((F32, 0), (BF16, 3), (F16, 1)):
        base = torch.randn(3, 7, 4, 32 + pad, device="cuda").to(kind)
        q = base[..., pad:].permute(0, 2, 1, 3)
        want = check(cache, starts, shared, q)
        room = torch.full((3, 7, 5, 32 + pad), 7.0, device="cuda", dtype=kind)
        out = room[:, :, :4, pad:].permute(0, 2, 1, 3)
        assert ops.kv8_attention_shared(q, cache, starts, shared, out=out) is out
        assert torch.equal(out, want)
        assert (room[:, :, 4] == 7).all() and (room[..., :pad] == 7).all()


def test_nothing_to_do():
    cache, starts, shared = make_groups([3], [32], [1, 2, 3], block=16)
    q = queries(cache, 1, 1)
    assert ops.kv8_attention_shared(q[:, :, :0], cache, starts, shared).shape == (3, 2, 0, 64)
    append(cache, 1)
    # no group at all, and groups of no sequence
    none = torch.zeros(0, dtype=torch.int32, device="cuda")
    check(cache, ints([0]), none, q)
    check(cache, ints([0, 0, 0]), ints([64, 64]), q)
    check(cache, ints([3, 3]), ints([64]), q)
    # no new token of any sequence
    out, lse = ops.kv8_attention_shared(q, cache, starts, shared, counts=ints([0, 0, 0]),
                                        return_lse=True)
    assert not out.any() and torch.isinf(lse).all()
    empty = cache.with_table(cache.table[:0], cache.lens[:0])
    assert ops.kv8_attention_shared(q[:0], empty, ints([0, 0]), ints([16])).shape == (0, 2, 1, 64)
    assert status() == 0


@pytest.mark.parametrize("members,T", [(5, 1), (40, 2), (3, 50)])
def test_repeated_calls_graphs_and_streams_give_the_same_bits(members, T):
    cache, starts, shared = make_groups([members, 4], [1024, 64], [30] * (members + 4), block=64,
                                        room=T)
    append(cache, T)
    q = queries(cache, 4, T, BF16)
    want = check(cache, starts, shared, q)
    for _ in range(3):
        assert torch.equal(ops.kv8_attention_shared(q, cache, starts, shared), want)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = ops.kv8_attention_shared(q, cache, starts, shared)
    side.synchronize()
    assert torch.equal(again, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.kv8_attention_shared(q, cache, starts, shared)
        two = ops.kv8_attention_shared(q * 2, cache, starts, shared)
    q0 = q.clone()
    for x in (q0, q0 * 3, q0):
        q.copy_(x)
        graph.replay()
        assert torch.equal(got, ops.kv8_attention_shared(q, cache, starts, shared))
        assert torch.equal(two, ops.kv8_attention_shared(q * 2, cache, starts, shared))
    assert torch.equal(got, want)
    # the groups are read on the device: a replay goes by what they hold then
    starts.copy_(ints([0, 2, members + 4]))
    shared.copy_(ints([512, 64]))
    cache.table[2:, :1] = cache.table[members:members + 1, :1]
    graph.replay()
    assert torch.equal(got, ops.kv8_attention_shared(q, cache, starts, shared))
    assert status() == 0


@pytest.mark.parametrize("members,T,group", [(5, 1, 1), (5, 3, 8), (40, 1, 4), (40, 2, 2), (3, 50, 2)])
def test_what_is_written_just_before_a_call_is_read_by_all_of_its_kernels(members, T, group):
    """q, lengths, counts, table, scales and groups change between calls that nothing
    waits between; each is as the same call alone."""
    cache, starts, shared = make_groups([members, 4], [640, 64], [30 + b % 9 for b in range(members + 4)],
                                        block=16, room=T)
    append(cache, T)
    B = members + 4
    g = torch.Generator().manual_seed(7)
    own = cache.table[:, 40:].clone()
    counts = ints([T] * B)
    q = queries(cache, group, T, BF16)
    held = [t.clone() for t in (q, cache.lens, cache.table, cache.scale)]
    states = []
    for i in range(12):
        lens = cache.lens - torch.randint(0, 25, (B,), generator=g, dtype=torch.int32).cuda()
        table = cache.table.clone()
        order = torch.randperm(members, generator=g).cuda()
        table[:members, 40:] = own[order]
        scale = cache.scale * (0.5 + torch.rand(cache.scale.shape, generator=g).cuda())
        cut = int(torch.randint(0, members + 1, (1,), generator=g))
        states.append((q * (1 + i % 3), lens, table, scale,
                       torch.randint(0, T + 1, (B,), generator=g, dtype=torch.int32).cuda(),
                       ints([0, cut, B if i % 2 else members]), ints([640, 64 if i % 2 else 320])))
    live = (q, cache.lens, cache.table, cache.scale, counts, starts, shared)

    def call(state):
        for to, x in zip(live, state):
            to.copy_(x)
        return ops.kv8_attention_shared(q, cache, starts, shared, counts=counts, return_lse=True)

    alone = []
    for state in states:
        torch.cuda.synchronize()
        alone.append([t.clone() for t in call(state)])
        torch.cuda.synchronize()
    for _ in range(3):
        got = [call(state) for state in states]
        for (out, lse), (want, want_lse) in zip(got, alone):
            # (bits, since a row of the table may name a page that was never written, NaN)
            assert torch.equal(out.view(torch.int16), want.view(torch.int16))
            assert torch.equal(lse.view(torch.int32), want_lse.view(torch.int32))
    for to, x in zip(live, held):
        to.copy_(x)
    assert status() == 0


def test_refusals():
    cache, starts, shared = make_groups([2], [16], [1, 2], block=16, heads=2)
    q = queries(cache, 1, 1)
    call = ops.kv8_attention_shared
    with pytest.raises(ValueError):
        call(q[:1], cache, starts, shared)
    with pytest.raises(ValueError):
        call(q[:, :1], cache, starts, shared)
    with pytest.raises(TypeError):
        call(q.double(), cache, starts, shared)
    with pytest.raises(ValueError):
        call(q.transpose(2, 3).contiguous().transpose(2, 3).expand(2, 2, 1, 64)[..., ::2], cache,
             starts, shared)
    for bad in (starts.long(), starts.cpu(), starts[:1], starts.view(1, 2),
                torch.zeros(4, dtype=torch.int32, device="cuda")[::2]):
        with pytest.raises(ValueError):
            call(q, cache, bad, shared)
    for bad in (shared.float(), shared.cpu(), torch.cat([shared, shared])):
        with pytest.raises(ValueError):
            call(q, cache, starts, bad)
    for kw in (dict(counts=ints([1])), dict(out=torch.empty_like(q, dtype=BF16))):
        with pytest.raises(ValueError):
            call(q, cache, starts, shared, **kw)
    for kw in (dict(sm_scale=-1.0), dict(sm_scale=math.nan), dict(max_own=-1), dict(max_shared=-1)):
        with pytest.raises(_lib.KernelError):
            call(q, cache, starts, shared, **kw)


# ---------------------------------------------------------------- copies


def pools(layers, pages, heads, block, dim, dtype, weight, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    table = torch.zeros(1, 1, dtype=torch.int32, device="cuda")
    lens = torch.zeros(1, dtype=torch.int32, device="cuda")
    made = []
    for _ in range(layers):
        c = ops.KV8Cache.empty(pages, heads, block, dim, table, lens, dtype, weight)
        for t in (c.k, c.v):
            t.view(torch.uint8).copy_(torch.randint(0, 256, t.shape, generator=g, device="cuda"))
        c.scale.copy_(torch.randn(c.scale.shape, generator=g, device="cuda"))
        if weight:
            c.weight.copy_(torch.randn(c.weight.shape, generator=g, device="cuda"))
        made.append(c)
    return made


def held(caches):
    return [[t.view(torch.uint8).cpu().clone() for t in (c.k, c.v, c.scale, c.weight)
             if t is not None] for c in caches]


def copied(from_, into, src, dst, tokens, same):
    """What the pools hold afterwards, and whether a pair was refused."""
    a, b = held(from_), held(into)
    P = from_[0].block
    pages, pages_to = from_[0].k.shape[0], into[0].k.shape[0]
    tokens = [P] * len(src) if tokens is None else tokens
    valid = [0 <= s < pages and 0 <= d < pages_to for s, d in zip(src, dst)]
    live = [v and t > 0 and not (same and s == d)
            for v, s, d, t in zip(valid, src, dst, tokens)]
    writes, reads = {}, set()
    for s, d, on in zip(src, dst, live):
        if on:
            writes[d] = writes.get(d, 0) + 1
            reads.add(s)
    refused = not all(valid)
    for s, d, t, on in zip(src, dst, tokens, live):
        if not on:
            continue
        if writes[d] > 1 or (same and d in reads):
            refused = True
            continue
        t = min(t, P)
        for x, y in zip(a, b):
            for i, (u, v) in enumerate(zip(x, y)):
                if i < 2:
                    v[d, :, :t] = u[s, :, :t]
                elif i == 2:
                    v[d] = u[s]
                else:
                    v[d, :, :4 * t] = u[s, :, :4 * t]
    return b, refused


def check_copy(from_, into, src, dst, tokens=None):
    same = into is None
    want, refused = copied(from_, from_ if same else into, src, dst, tokens, same)
    ops.kv8_copy(from_, ints(src), ints(dst), tokens=None if tokens is None else ints(tokens),
                 into=into)
    for x, y in zip(held(from_ if same else into), want):
        assert all(torch.equal(u, v) for u, v in zip(x, y))
    assert status() == (6 if refused else 0)


@pytest.mark.parametrize("dtype,weight", [(I8, False), (F8, True)])
@pytest.mark.parametrize("heads,block,dim", [(1, 16, 16), (3, 32, 64), (2, 128, 128), (12, 64, 32)])
@pytest.mark.parametrize("layers", [1, 5])
def test_copies_of_pages(layers, heads, block, dim, dtype, weight):
    from_ = pools(layers, 40, heads, block, dim, dtype, weight)
    order = torch.randperm(40, generator=torch.Generator().manual_seed(3)).tolist()
    check_copy(from_, None, order[:15], order[15:30])
    check_copy(from_, None, [order[0]] * 9, order[20:29],
               [1, 2, block - 1, block, block + 5, 0, -3, block // 2, 1])
    into = pools(layers, 33, heads, block, dim, dtype, weight, seed=9)
    check_copy(from_, into, list(range(33)), list(range(32, -1, -1)))
    check_copy(from_, into, [7] * 20, list(range(20)), [i % (block + 2) for i in range(20)])


@pytest.mark.parametrize("n", [1, 2, 511, 513, 2000])
def test_copies_of_any_number(n):
    from_ = pools(2, 2 * n + 3, 2, 16, 16, I8, True)
    order = torch.randperm(2 * n + 3, generator=torch.Generator().manual_seed(n)).tolist()
    check_copy(from_, None, order[:n], order[n:2 * n])


def test_more_layers_than_a_launch_takes():
    from_ = pools(71, 6, 1, 16, 32, I8, False)
    check_copy(from_, None, [0, 1], [4, 5])


@pytest.mark.parametrize("extra", [0, 600])
def test_pairs_that_name_a_page_twice_are_refused(extra):
    """With few pairs and with many: a page written twice, a page that is read
    and written, chains and cycles; pairs that copy nothing name nothing."""
    pages = 40 + 2 * extra
    from_ = pools(1, pages, 2, 16, 32, I8, True)
    into = pools(1, pages, 2, 16, 32, I8, True, seed=5)
    src = [0, 1, 2, 3, 4, 5, 6, 7, 8, 9, 30, 31, 32]
    dst = [20, 20, 3, 21, 5, 4, 6, 22, 22, 23, 24, 25, 24]
    tok = [16, 16, 16, 16, 16, 16, 16, 3, 0, 16, 4, 16, -1]
    src += list(range(40, 40 + extra))
    dst += list(range(40 + extra, 40 + 2 * extra))
    tok += [16] * extra
    check_copy(from_, None, src, dst, tok)
    check_copy(from_, into, src, dst, tok)
    check_copy(from_, None, [3, 3, 3], [10, 10, 11])
    check_copy(from_, None, [3, 4], [3, 4])            # a page onto itself is no copy
    check_copy(from_, None, [3, 4], [3, 3])            # and reads nothing


def test_entries_outside_the_pool_are_refused():
    from_ = pools(2, 12, 2, 32, 64, F8, False)
    into = pools(2, 5, 2, 32, 64, F8, False, seed=2)
    bad = [-1, 12, 1 << 30, -(1 << 31)]
    check_copy(from_, None, bad + [1], [3, 4, 5, 6, 7])
    check_copy(from_, None, [1, 2, 3, 4, 8], bad + [7])
    check_copy(from_, into, [6, 7, 8, 11], [4, 5, 3, 11])


def test_copies_of_nothing_and_refusals():
    from_ = pools(2, 8, 2, 16, 32, I8, True)
    other = pools(2, 8, 2, 16, 64, I8, True)
    check_copy(from_, None, [], [])
    ops.kv8_copy([], ints([0]), ints([1]))
    for into in (other, pools(2, 8, 3, 16, 32, I8, True), pools(2, 8, 2, 32, 32, I8, True),
                 pools(2, 8, 2, 16, 32, F8, True), pools(1, 8, 2, 16, 32, I8, True)):
        with pytest.raises(ValueError):
            ops.kv8_copy(from_, ints([0]), ints([1]), into=into)
    with pytest.raises(ValueError):
        ops.kv8_copy([from_[0], other[0]], ints([0]), ints([1]))
    for src, dst, tok in ((ints([0]).long(), ints([1]), None), (ints([0, 1]), ints([2]), None),
                          (ints([0]).cpu(), ints([1]), None), (ints([[0]]), ints([[1]]), None),
                          (ints([0, 9, 1])[::2], ints([2, 3]), None),
                          (ints([0]), ints([1]), ints([4, 4]))):
        with pytest.raises(ValueError):
            ops.kv8_copy(from_, src, dst, tokens=tok)
    # layers of several sizes, and two pools that have a tensor in common
    mixed = [from_[0], pools(1, 9, 2, 16, 32, I8, True)[0]]
    with pytest.raises(_lib.KernelError):
        ops.kv8_copy(mixed, ints([0]), ints([1]))
    half = ops.KV8Cache(from_[0].k, other[0].v.new_empty(from_[0].v.shape), from_[0].scale,
                        from_[0].table, from_[0].lens, from_[0].weight)
    with pytest.raises(_lib.KernelError):
        ops.kv8_copy(from_[0], ints([0]), ints([1]), into=half)


def test_pools_that_lie_side_by_side_or_are_read_twice():
    """Views of one allocation, one cache read for two layers, and a record that only
    one side keeps: nothing that is written is written or read elsewhere."""
    whole = pools(1, 30, 2, 16, 32, I8, True)[0]

    def part(a, z, weight=True):
        return ops.KV8Cache(whole.k[a:z], whole.v[a:z], whole.scale[a:z], whole.table, whole.lens,
                            whole.weight[a:z] if weight else None)

    check_copy([part(0, 10)], [part(10, 20)], [3, 4], [0, 9])
    check_copy([part(0, 10), part(0, 10)], [part(10, 20), part(20, 30)], [1, 2], [5, 6], [16, 7])
    one = ops.KV8Cache(whole.k[:10], whole.v[:10], whole.scale[:10], whole.table, whole.lens)
    two = ops.KV8Cache(whole.k[10:20], whole.v[10:20], whole.scale[10:20], whole.table, whole.lens,
                       whole.weight[:10])
    record = whole.weight.clone()
    ops.kv8_copy(one, ints([7]), ints([2]), into=two)
    assert torch.equal(whole.k[12], whole.k[7]) and torch.equal(whole.weight, record)
    assert status() == 0
    for from_, into in (([part(0, 10)], [part(9, 19)]), ([part(0, 10)] * 2, [part(10, 20)] * 2),
                        ([part(0, 10), part(10, 20)], [part(10, 20), part(0, 10)]),
                        ([part(0, 10)] * 2, None)):
        with pytest.raises(_lib.KernelError):
            ops.kv8_copy(from_, ints([1]), ints([2]), into=into)
    assert status() == 0


def test_copies_in_a_graph_and_without_a_record():
    from_ = pools(3, 30, 2, 32, 32, I8, True)
    into = pools(3, 30, 2, 32, 32, I8, False, seed=4)
    check_copy(from_, None, [1], [2])
    src, dst = ints([1, 2, 3]), ints([20, 21, 22])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.kv8_copy(from_, src, dst)
    for a, b in (([1, 2, 3], [20, 21, 22]), ([4, 4, 9], [0, 11, 9])):
        src.copy_(ints(a))
        dst.copy_(ints(b))
        want, _ = copied(from_, from_, a, b, None, True)
        graph.replay()
        for x, y in zip(held(from_), want):
            assert all(torch.equal(u, v) for u, v in zip(x, y))
    want = held(from_)
    ops.kv8_copy(from_, ints([5]), ints([6]), into=into)
    for x, y in zip(held(into), want):
        assert torch.equal(x[0][6], y[0][5]) and torch.equal(x[2][6], y[2][5])
    assert status() == 0
