"""Host-side checks of the 8-bit cache entry points: bad arguments are refused
before any CUDA call (this runs without a GPU). CPU only."""
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


def cache(**kw):
    f = dict(k=FAKE, v=FAKE, scale=FAKE, weight=FAKE, table=FAKE, lens=FAKE, pages=8, ld_table=4,
             blocks=4, batch=2, kv_heads=2, head_dim=64, block=16, format=_lib.KF_KV8_INT8)
    f.update(kw)
    return ctypes.byref(_lib.KV8CacheStruct(*(f[n] for n, _ in _lib.KV8CacheStruct._fields_)))


def append(lib, c, k=FAKE, dtype=0, T=1):
    return lib.kf_kv8_append(c, k, 1, 1, 1, FAKE, 1, 1, 1, dtype, None, T, None)


def attention(lib, c, q=FAKE, dtype=0, T=1, heads=2, flags=0, work=None, size=0, max_len=0,
              scale=1.0):
    return lib.kf_kv8_attention(c, q, 1, 1, 1, FAKE, 1, 1, 1, dtype, None, T, heads, max_len, scale,
                                flags, None, work, size, None)


@pytest.mark.parametrize("field,value,code", [
    ("k", None, _lib.KF_E_INVALID), ("scale", None, _lib.KF_E_INVALID),
    ("table", None, _lib.KF_E_INVALID), ("lens", None, _lib.KF_E_INVALID),
    ("pages", -1, _lib.KF_E_INVALID), ("kv_heads", 0, _lib.KF_E_INVALID),
    ("ld_table", 3, _lib.KF_E_INVALID), ("format", 2, _lib.KF_E_INVALID),
    ("head_dim", 8, _lib.KF_E_UNSUPPORTED), ("head_dim", 256, _lib.KF_E_UNSUPPORTED),
    ("block", 8, _lib.KF_E_UNSUPPORTED), ("block", 48, _lib.KF_E_UNSUPPORTED),
    ("k", FAKE + 8, _lib.KF_E_UNSUPPORTED), ("scale", FAKE + 4, _lib.KF_E_UNSUPPORTED),
    ("batch", 40000, _lib.KF_E_UNSUPPORTED), ("pages", 1 << 40, _lib.KF_E_UNSUPPORTED)])
def test_a_bad_cache_is_refused_by_every_entry(lib, field, value, code):
    c = cache(**{field: value})
    assert append(lib, c) == code
    assert attention(lib, c) == code
    assert lib.kf_kv8_read(c, None, None, 1, FAKE, FAKE, 0, None) == code
    assert lib.kf_kv8_evict(c, FAKE, 4, 8, 0, FAKE, FAKE + 64, None) == code
    assert lib.kf_kv8_attention_workspace_bytes(c, 0, 1, 2, 0, 0) == -1
    assert b"kf_kv8" in lib.kf_last_error()


def test_bad_arguments_are_refused(lib):
    bad = _lib.KF_E_INVALID
    assert append(lib, None) == bad
    assert append(lib, cache(), k=None) == bad
    assert append(lib, cache(), dtype=3) == bad
    assert append(lib, cache(), T=-1) == bad
    assert attention(lib, cache(), q=None) == bad
    assert attention(lib, cache(), dtype=7) == bad
    assert attention(lib, cache(), heads=3) == bad
    assert attention(lib, cache(), heads=0) == bad
    assert attention(lib, cache(), flags=4) == bad
    assert attention(lib, cache(), max_len=-1) == bad
    for scale in (-0.125, float("nan"), float("inf")):
        assert attention(lib, cache(), scale=scale) == bad
        assert b"sm_scale" in lib.kf_last_error()
    assert attention(lib, cache(weight=None), flags=_lib.KF_KV8_TRACK) == bad
    assert attention(lib, cache(), flags=_lib.KF_KV8_TRACK) == bad        # no workspace
    assert b"workspace" in lib.kf_last_error()
    assert lib.kf_kv8_read(cache(), None, None, -1, FAKE, FAKE, 0, None) == bad
    assert lib.kf_kv8_read(cache(), None, None, 1, None, FAKE, 0, None) == bad
    assert lib.kf_kv8_read(cache(), None, None, 1, FAKE + 8, FAKE, 0, None) == \
        _lib.KF_E_UNSUPPORTED
    other = FAKE + 64
    assert lib.kf_kv8_evict(cache(), None, 4, 8, 0, FAKE, other, None) == bad
    assert lib.kf_kv8_evict(cache(), FAKE, 4, 0, 0, FAKE, other, None) == bad
    assert lib.kf_kv8_evict(cache(), FAKE, 4, 8, 9, FAKE, other, None) == bad
    assert lib.kf_kv8_evict(cache(), FAKE, 4, 65, 0, FAKE, other, None) == bad
    assert lib.kf_kv8_evict(cache(), FAKE, 4, 8, 0, FAKE, FAKE, None) == bad   # lens in place
    assert lib.kf_kv8_evict(cache(weight=None), FAKE, 4, 8, 0, FAKE, other, None) == bad


def test_empty_calls_are_no_ops(lib):
    assert append(lib, cache(), T=0) == 0
    assert append(lib, cache(batch=0)) == 0
    assert attention(lib, cache(), T=0) == 0
    assert lib.kf_kv8_read(cache(), None, None, 0, FAKE, FAKE, 0, None) == 0


def test_empty_tensors_have_no_address(lib):
    """A batch, a table or a pool of size 0 comes with null pointers."""
    none = cache(batch=0, table=None, lens=None)
    assert append(lib, none, k=None) == 0
    assert attention(lib, none, q=None) == 0
    assert lib.kf_kv8_read(none, None, None, 1, None, None, 0, None) == 0
    assert lib.kf_kv8_evict(none, None, 4, 8, 0, None, None, None) == 0
    assert lib.kf_kv8_evict(none, None, 4, 8, 9, None, None, None) == _lib.KF_E_INVALID
    pool = dict(pages=0, k=None, v=None, scale=None, weight=None)
    for c in (cache(**pool), cache(blocks=0, ld_table=0, table=None)):
        assert lib.kf_kv8_attention_workspace_bytes(c, 0, 1, 2, 0, 0) == 0
        assert append(lib, c, T=0) == 0
        assert append(lib, c, k=None) == _lib.KF_E_INVALID


def test_workspace_grows_with_the_work(lib):
    size = lambda c, **kw: lib.kf_kv8_attention_workspace_bytes(   # noqa: E731
        c, 0, kw.get("T", 1), kw.get("heads", 2), kw.get("max_len", 0), kw.get("flags", 0))
    short = cache(blocks=4, ld_table=4)
    long = cache(blocks=4096, ld_table=4096, pages=10000)
    assert size(short) == 0                           # one part: nothing to join
    assert size(long) > 0
    assert size(long, max_len=64) == 0
    assert size(long, T=0) == 0 and size(cache(batch=0)) == 0
    assert size(long, flags=_lib.KF_KV8_TRACK) > size(long)


@pytest.mark.parametrize("T,heads", [(1, 8), (1, 64), (2, 64), (4, 64), (8, 64), (64, 64)])
@pytest.mark.parametrize("blocks", [128, 2048, 16384])
def test_recorded_weights_take_a_bounded_workspace(lib, blocks, T, heads):
    """A table may reach far beyond what its sequences hold: 64 sequences, 8 kv
    heads of 128, up to a million tokens a row. Scores that are kept for the last
    pass stay within 4 GiB; parts and planes are under half a gigabyte."""
    c = cache(blocks=blocks, ld_table=blocks, block=64, batch=64, kv_heads=8, head_dim=128,
              pages=1 << 20)
    for dtype in (0, 1):
        need = lib.kf_kv8_attention_workspace_bytes(c, dtype, T, heads, 0, _lib.KF_KV8_TRACK)
        assert 0 <= need <= 9 << 29


def test_python_refuses_what_is_no_cache():
    k = torch.zeros(3, 2, 16, 64, dtype=torch.int8)
    scale, lens = torch.zeros(3, 2, 2), torch.zeros(1, dtype=torch.int32)
    table = torch.zeros(1, 3, dtype=torch.int32)
    with pytest.raises(TypeError):
        ops.KV8Cache(k.float(), k, scale, table, lens)
    with pytest.raises(ValueError):
        ops.KV8Cache(k[0], k, scale, table, lens)
    with pytest.raises(ValueError):
        ops.KV8Cache(k[..., :24], k, scale, table, lens)
    with pytest.raises(TypeError):
        ops.KV8Cache(k, k, scale, table, lens)        # CPU tensors
