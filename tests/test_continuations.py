"""Host-side checks of kf_kv8_attention_shared, kf_kv8_copy and kf_beam_select: bad
arguments are refused before any CUDA call. CPU only."""
from __future__ import annotations

import ctypes

import pytest
import torch

from techjam2026_b200 import _lib, build, ops

FAKE = 0x10000     # never dereferenced


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def struct(**kw):
    f = dict(k=FAKE, v=FAKE, scale=FAKE, weight=FAKE, table=FAKE, lens=FAKE, pages=8, ld_table=4,
             blocks=4, batch=2, kv_heads=2, head_dim=64, block=16, format=_lib.KF_KV8_INT8)
    f.update(kw)
    return _lib.KV8CacheStruct(*(f[n] for n, _ in _lib.KV8CacheStruct._fields_))


def shared(lib, c, q=FAKE, dtype=0, T=1, heads=2, starts=FAKE, lens=FAKE, groups=1, max_shared=0,
           max_own=0, flags=0, work=None, size=0, scale=1.0):
    return lib.kf_kv8_attention_shared(ctypes.byref(c), q, 1, 1, 1, FAKE, 1, 1, 1, dtype, None, T,
                                       heads, starts, lens, groups, max_shared, max_own, scale,
                                       flags, None, work, size, None)


def need(lib, c, dtype=0, T=1, heads=2, groups=1, max_shared=0, max_own=0, flags=0):
    return lib.kf_kv8_attention_shared_workspace_bytes(ctypes.byref(c), dtype, T, heads, groups,
                                                       max_shared, max_own, flags)


@pytest.mark.parametrize("field,value,code", [
    ("k", None, _lib.KF_E_INVALID), ("table", None, _lib.KF_E_INVALID),
    ("pages", -1, _lib.KF_E_INVALID), ("head_dim", 8, _lib.KF_E_UNSUPPORTED),
    ("block", 48, _lib.KF_E_UNSUPPORTED), ("batch", 40000, _lib.KF_E_UNSUPPORTED)])
def test_a_bad_cache_is_refused(lib, field, value, code):
    c = struct(**{field: value})
    assert shared(lib, c) == code
    assert need(lib, c) == -1
    refs = (ctypes.POINTER(_lib.KV8CacheStruct) * 1)(ctypes.pointer(c))
    assert lib.kf_kv8_copy(refs, refs, 1, FAKE, FAKE, None, 1, None, 0, None) == code
    assert lib.kf_kv8_copy_workspace_bytes(ctypes.byref(c), ctypes.byref(c), 1) == -1


def test_shared_attention_refuses_bad_arguments(lib):
    bad = _lib.KF_E_INVALID
    c = struct()
    for kw in (dict(q=None), dict(starts=None), dict(lens=None), dict(dtype=5), dict(heads=3),
               dict(heads=0), dict(T=-1), dict(groups=-1), dict(groups=40000), dict(max_shared=-1),
               dict(max_own=-1), dict(flags=4), dict(scale=-1.0), dict(scale=float("nan")),
               dict(scale=float("inf")), {}, dict(work=FAKE, size=8), dict(work=FAKE + 8, size=1 << 30)):
        assert shared(lib, c, **kw) == bad, kw
    assert shared(lib, c, flags=_lib.KF_KV8_TRACK) == _lib.KF_E_UNSUPPORTED
    assert b"weight record" in lib.kf_last_error()
    wide = struct(batch=32767)
    assert shared(lib, wide, T=1 << 16) == _lib.KF_E_UNSUPPORTED
    assert need(lib, wide, T=1 << 16) == -1


def test_shared_attention_workspace(lib):
    c = struct(blocks=4096, ld_table=4096, pages=10000)
    assert need(lib, c) > 0
    assert need(lib, c, T=0) == 0 and need(lib, struct(batch=0)) == 0
    assert need(lib, c, max_shared=256, max_own=256) < need(lib, c)
    assert need(lib, c, groups=0, max_own=64) == 0            # the plain call, in one part
    for kw in (dict(max_shared=-1), dict(groups=-1), dict(heads=3), dict(dtype=9)):
        assert need(lib, c, **kw) == -1


@pytest.mark.parametrize("T,heads", [(1, 64), (8, 64), (64, 64)])
@pytest.mark.parametrize("groups", [1, 64])
def test_shared_attention_workspace_is_bounded(lib, groups, T, heads):
    """64 sequences, 8 kv heads of 128, tables that reach 131k tokens. Each part of a
    row is 128 sums, its reference and its sum. The shared tokens' parts take 256 MB,
    or 8 parts a row where that is more, and two for the ends of a tile; the own ones
    are at most 64."""
    c = struct(blocks=2048, ld_table=2048, block=64, batch=64, kv_heads=8, head_dim=128,
               pages=1 << 20)
    rows = 64 * heads * T
    for dtype in (0, 1):
        most = (1 << 28) * 130 // 128 + rows * (10 + 64) * 130 * 4 + (1 << 20)
        assert 0 < need(lib, c, dtype, T, heads, groups) <= most


def test_copy_refuses_bad_arguments(lib):
    bad = _lib.KF_E_INVALID
    kind = ctypes.POINTER(_lib.KV8CacheStruct)

    def call(a, b, src=FAKE, dst=FAKE, n=1, layers=None, work=None, size=0):
        x = (kind * len(a))(*map(ctypes.pointer, a))
        y = (kind * len(b))(*map(ctypes.pointer, b))
        return lib.kf_kv8_copy(x, y, len(a) if layers is None else layers, src, dst, None, n, work,
                               size, None)

    one, two = struct(), struct(k=2 * FAKE, v=2 * FAKE, scale=2 * FAKE, weight=None, pages=9)
    assert call([one], [one], src=None) == bad
    assert call([one], [one], dst=None) == bad
    assert call([one], [one], n=-1) == bad
    assert call([one], [one], n=1 << 40) == bad
    assert call([one], [one], layers=-1) == bad
    assert call([one], [one], layers=257) == bad
    assert lib.kf_kv8_copy(None, None, 1, FAKE, FAKE, None, 1, None, 0, None) == bad
    for other in (struct(kv_heads=3), struct(head_dim=32), struct(block=32),
                  struct(format=_lib.KF_KV8_E4M3)):
        other.k = other.v = other.scale = 2 * FAKE
        assert call([one], [other]) == bad
    assert call([one, two], [one, two]) == bad                     # pools of several sizes
    assert call([one], [struct(v=2 * FAKE)]) == bad                # half in common
    assert call([one], [struct(pages=9)]) == bad
    assert call([one], [one], n=1000) == bad                       # many pairs need a workspace
    assert b"workspace" in lib.kf_last_error()
    size = lib.kf_kv8_copy_workspace_bytes(ctypes.byref(one), ctypes.byref(two), 1000)
    assert size == 9 * 4
    assert call([one], [two], n=1000, work=FAKE, size=size - 1) == bad
    assert call([one], [two], n=1000, work=FAKE + 4, size=size) == bad
    assert lib.kf_kv8_copy_workspace_bytes(ctypes.byref(one), ctypes.byref(two), 10) == 0
    assert call([], []) == 0 and call([one], [one], n=0) == 0


def test_copy_refuses_tensors_that_it_would_write_twice_or_read_as_well(lib):
    """8 pages of 2 heads of 16 x 64 codes: 16384 bytes of K and of V, 128 of scales,
    1024 of the record."""
    kind = ctypes.POINTER(_lib.KV8CacheStruct)

    def pool(n, **kw):
        base = (n + 1) << 20
        f = dict(k=base, v=base + 0x10000, scale=base + 0x20000, weight=base + 0x30000)
        f.update(kw)
        return struct(**f)

    def refused(a, b):
        x = (kind * len(a))(*map(ctypes.pointer, a))
        y = (kind * len(b))(*map(ctypes.pointer, b))
        rc = lib.kf_kv8_copy(x, y, len(a), FAKE, FAKE, None, 1, None, 0, None)
        return rc == _lib.KF_E_INVALID

    p = [pool(n) for n in range(4)]
    assert refused([p[0], p[1]], [p[1], p[0]])                   # layers the other way round
    assert refused([p[0], p[1]], [p[1], p[2]])                   # read by another layer
    assert refused([p[0], p[1]], [p[2], p[2]])                   # written twice
    assert refused([p[0], p[0]], [p[0], p[0]])
    far = [pool(n) for n in range(40)]
    assert refused(far[:20] + [p[0]], far[20:] + [far[39]])      # (the list may be long)
    for name, size in (("k", 16384), ("v", 16384), ("scale", 128), ("weight", 1024)):
        at = getattr(p[0], name)
        # one tensor in common, or the end of one and the beginning of another
        for where in (at, at + size - 16, at - size + 16):
            assert refused([p[0]], [pool(3, **{name: where})]), name
            assert refused([p[1], p[2]], [p[0], pool(3, **{name: where})]), name
    # the record of one pool over the codes of the other
    assert refused([p[0]], [pool(3, weight=p[0].k)])
    assert refused([pool(3, weight=p[0].k)], [p[0]])


def test_beam_select_refuses_bad_arguments(lib):
    def call(logits=FAKE, dtype=0, scores=FAKE, batch=1, beams=2, vocab=10, n=2, pad=0, out=FAKE,
             work=FAKE, size=1 << 20):
        return lib.kf_beam_select(logits, 20, 10, dtype, scores, 2, None, 0, batch, beams, vocab, n,
                                  pad, out, FAKE, FAKE, work, size, None)

    bad, far = _lib.KF_E_INVALID, _lib.KF_E_UNSUPPORTED
    for kw, code in ((dict(logits=None), bad), (dict(scores=None), bad), (dict(out=None), bad),
                     (dict(dtype=3), bad), (dict(batch=-1), bad), (dict(beams=0), bad),
                     (dict(vocab=0), bad), (dict(n=0), bad), (dict(pad=-1), bad),
                     (dict(n=129), far), (dict(beams=1025), far), (dict(vocab=1 << 31), far),
                     (dict(batch=70000), far), (dict(work=None), bad), (dict(size=8), bad),
                     (dict(work=FAKE + 4), bad)):
        assert call(**kw) == code, kw
    assert call(batch=0) == 0
    size = lib.kf_beam_select_workspace_bytes
    assert size(1, 2, 10, 2) > 0 and size(0, 2, 10, 2) == 0
    for a in ((-1, 2, 10, 2), (1, 0, 10, 2), (1, 2, 0, 2), (1, 2, 10, 0), (1, 2, 10, 129)):
        assert size(*a) == -1


def test_python_refuses_tensors_of_the_cpu():
    with pytest.raises(RuntimeError):
        ops.beam_select(torch.zeros(1, 2, 3), torch.zeros(1, 2))
