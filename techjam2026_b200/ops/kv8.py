"""An 8-bit key/value cache: writing, reading, attention and eviction.

A layer's cache (`KV8Cache`) holds K and V of B sequences in pages of `block`
tokens as int8 or e4m3 codes, with one fp32 scale for each page and head and
for K and V apart. Pages of one pool are handed to sequences through a page
table, so sequences grow and shrink without copies.

  kv8_append     quantises a chunk of new tokens into the cache;
  kv8_attention  attention of the newest tokens over the cache, any number of
                 query heads per kv head, optionally recording how much weight
                 every cached token received;
  kv8_evict      cuts each head's tokens to a budget: the most recent and, of
                 the others, the ones with the most recorded weight;
  kv8_read       values of a range of tokens;
  kv8_attention_shared  kv8_attention for sequences that share leading pages,
                 which are read once for all of them;
  kv8_copy       copies of pages, of all layers at once.

A step over one layer: `kv8_append(cache, k, v)`, `kv8_attention(q, cache)`;
after the last layer, `cache.lens += T` (all layers of a model may share one
`lens` and one `table`). `techjam2026_b200.kvcache` does this for the layer
stack. Runs csrc/kv8_cache_sm100.cu, csrc/kv8_attn_sm100.cu,
csrc/kv8_prompt_sm100.cu, csrc/kv8_group_sm100.cu and csrc/kv8_copy_sm100.cu.
The reference has no cache: it recomputes the whole sequence
(kernelforge/optimized.py:397-458).

Calls are stream-ordered on the current stream, launch a fixed number of
kernels for given shapes and read lengths on the device, so a step may be
captured in a CUDA graph. A length beyond the table or a page number outside
the pool is never used as an index: it is recorded in the device status word
(code 6) and the tokens count as absent. A sequence of a negative length holds
no token and takes none. Groups of sequences out of order are recorded as code 7.
"""
from __future__ import annotations

import ctypes
from typing import Optional, Sequence, Tuple, Union

import torch

from .. import _lib

HEAD_DIMS = (16, 32, 64, 128)
BLOCKS = (16, 32, 64, 128)
CODE_DTYPES = {torch.int8: _lib.KF_KV8_INT8, torch.float8_e4m3fn: _lib.KF_KV8_E4M3}
VALUE_DTYPES = {torch.float32: _lib.KF_DT_F32, torch.bfloat16: _lib.KF_DT_BF16,
                torch.float16: _lib.KF_DT_F16}


def _want(t, name, dtype, shape=None):
    if t.dtype != dtype:
        raise TypeError(f"KV8Cache: {name} must be {dtype}, got {t.dtype}")
    if not t.is_cuda:
        raise RuntimeError(f"KV8Cache: {name} must be a CUDA tensor (no CPU path)")
    if not t.is_contiguous():
        raise ValueError(f"KV8Cache: {name} must be contiguous")
    if shape is not None and tuple(t.shape) != shape:
        raise ValueError(f"KV8Cache: {name} must have shape {shape}, got {tuple(t.shape)}")


class KV8Cache:
    """One layer's cache: a view of tensors that the caller owns.

    k, v     [pages, kv_heads, block, head_dim] int8 or float8_e4m3fn codes
    scale    [pages, kv_heads, 2] float32, of K and of V
    table    [B, blocks] int32: page of each block of a sequence (rows may be
             strided)
    lens     [B] int32: tokens held
    weight   [pages, kv_heads, block] float32, or None: attention weight each
             token has received (needed by `track` and kv8_evict)
    """

    __slots__ = ("k", "v", "scale", "table", "lens", "weight", "struct", "batch", "kv_heads",
                 "head_dim", "block", "device", "_ref", "_ptr", "_kind", "_work")
    _TENSORS = frozenset(("k", "v", "scale", "table", "lens", "weight"))

    def __init__(self, k: torch.Tensor, v: torch.Tensor, scale: torch.Tensor, table: torch.Tensor,
                 lens: torch.Tensor, weight: Optional[torch.Tensor] = None):
        if k.dtype not in CODE_DTYPES:
            raise TypeError(f"KV8Cache: codes must be int8 or float8_e4m3fn, got {k.dtype}")
        if k.dim() != 4:
            raise ValueError("KV8Cache: k must be [pages, kv_heads, block, head_dim]")
        pages, heads, block, head_dim = k.shape
        if head_dim not in HEAD_DIMS or block not in BLOCKS:
            raise ValueError(f"KV8Cache: head_dim must be one of {HEAD_DIMS} and block one of "
                             f"{BLOCKS}, got {head_dim} and {block}")
        if table.dim() != 2 or table.dtype != torch.int32 or not table.is_cuda:
            raise TypeError("KV8Cache: table must be an int32 CUDA tensor [B, blocks]")
        if table.shape[1] > 1 and table.stride(1) != 1:
            raise ValueError("KV8Cache: table needs unit stride along its blocks")
        _want(k, "k", k.dtype)
        _want(v, "v", k.dtype, (pages, heads, block, head_dim))
        _want(scale, "scale", torch.float32, (pages, heads, 2))
        _want(lens, "lens", torch.int32, (table.shape[0],))
        if weight is not None:
            _want(weight, "weight", torch.float32, (pages, heads, block))
        for t in (v, scale, table, lens, weight):
            if t is not None and t.device != k.device:
                raise ValueError("KV8Cache: all tensors must be on one device")
        self.k, self.v, self.scale, self.table, self.lens = k, v, scale, table, lens
        self.weight = weight
        self.struct = _lib.KV8CacheStruct(
            k.data_ptr(), v.data_ptr(), scale.data_ptr(),
            weight.data_ptr() if weight is not None else None, table.data_ptr(), lens.data_ptr(),
            pages, table.stride(0) if table.shape[0] > 1 else table.shape[1], table.shape[1],
            table.shape[0], heads, head_dim, block, CODE_DTYPES[k.dtype])
        self._ref = ctypes.byref(self.struct)
        self._ptr = ctypes.pointer(self.struct)
        self._kind = (k.dtype, heads, block, head_dim, k.get_device())
        self.batch, self.kv_heads, self.block, self.head_dim = table.shape[0], heads, block, head_dim
        self.device = k.device
        self._work = {}              # workspace bytes by (type, T, heads, max_len, flags)

    def __setattr__(self, name, value):
        # The C side holds the tensors' addresses: `cache.lens += n` updates in
        # place, but another tensor would go unseen.
        if name in KV8Cache._TENSORS and getattr(self, "_ref", None) is not None \
                and value is not getattr(self, name):
            raise AttributeError(f"KV8Cache: {name} is fixed; update the tensor in place")
        object.__setattr__(self, name, value)

    def with_table(self, table: torch.Tensor, lens: torch.Tensor) -> "KV8Cache":
        """The same pool under another table [B, blocks] and other lengths [B]."""
        if table.dim() != 2 or table.dtype != torch.int32 or table.device != self.device \
                or (table.shape[1] > 1 and table.stride(1) != 1):
            raise ValueError(f"KV8Cache: table must be an int32 tensor [B, blocks] on {self.device} "
                             "with unit stride along its blocks")
        batch, blocks = table.shape
        if lens.dtype != torch.int32 or tuple(lens.shape) != (batch,) \
                or lens.device != self.device or not lens.is_contiguous():
            raise ValueError(f"KV8Cache: lens must be a contiguous int32 tensor [{batch}] on "
                             f"{self.device}")
        struct = _lib.KV8CacheStruct.from_buffer_copy(self.struct)
        struct.table, struct.lens = table.data_ptr(), lens.data_ptr()
        struct.ld_table = table.stride(0) if batch > 1 else blocks
        struct.blocks, struct.batch = blocks, batch
        new = object.__new__(KV8Cache)
        put = object.__setattr__
        for name in ("k", "v", "scale", "weight", "kv_heads", "block", "head_dim", "device",
                     "_kind"):
            put(new, name, getattr(self, name))
        put(new, "table", table)
        put(new, "lens", lens)
        put(new, "batch", batch)
        put(new, "_work", {})
        put(new, "struct", struct)
        put(new, "_ref", ctypes.byref(struct))
        put(new, "_ptr", ctypes.pointer(struct))
        return new

    @classmethod
    def empty(cls, pages: int, kv_heads: int, block: int, head_dim: int, table: torch.Tensor,
              lens: torch.Tensor, dtype: torch.dtype = torch.int8, weight: bool = False):
        """A cache over a new pool on `table`'s device."""
        dev = table.device
        k = torch.empty((pages, kv_heads, block, head_dim), dtype=dtype, device=dev)
        return cls(k, torch.empty_like(k),
                   torch.zeros((pages, kv_heads, 2), dtype=torch.float32, device=dev), table, lens,
                   torch.zeros((pages, kv_heads, block), dtype=torch.float32, device=dev)
                   if weight else None)


def _dtype_code(t: torch.Tensor, what: str) -> int:
    code = VALUE_DTYPES.get(t.dtype)
    if code is None:
        raise TypeError(f"{what} must be float32, bfloat16 or float16, got {t.dtype}")
    return code


def _check_call(what: str, cache: KV8Cache, counts: Optional[torch.Tensor], *tensors) -> int:
    """Checks that a call's tensors are where the cache is; its stream."""
    index = cache.device.index
    for t in tensors:
        if t.get_device() != index:
            raise ValueError(f"{what}: tensors must be on the cache's device {cache.device}, "
                             f"got {t.device}")
    if index != torch.cuda.current_device():
        raise RuntimeError(f"{what}: the cache is on {cache.device}, which is not the current "
                           "device")
    if counts is not None:
        _check_index(what, "counts", counts, cache)
    return torch._C._cuda_getCurrentRawStream(index)


def _check_index(what: str, name: str, t: torch.Tensor, cache: KV8Cache) -> None:
    if t.dtype is not torch.int32 or t.shape != cache.lens.shape or not t.is_contiguous() \
            or t.get_device() != cache.device.index:
        raise ValueError(f"{what}: {name} must be a contiguous int32 tensor [{cache.batch}] on "
                         f"{cache.device}")


def kv8_append(cache: KV8Cache, k: torch.Tensor, v: torch.Tensor,
               counts: Optional[torch.Tensor] = None) -> None:
    """Quantise new tokens into the cache at positions lens[b], lens[b] + 1, ...

    k, v    [B, kv_heads, T, head_dim] float32, bfloat16 or float16, any
            strides with unit stride along head_dim (e.g. views of a fused
            projection)
    counts  int32 [B], how many of the T tokens each sequence takes (default
            all); the others are not read

    A page's scale is its largest magnitude / 127 (int8) or / 448 (e4m3). A
    token that raises it rescales the earlier codes of its page. An infinity or
    NaN makes the page's scale NaN, and what reads the page NaN. The pages must
    be in the table already; `lens` is not changed (the layers of a model share
    it). The record of the new tokens' weights is set to 0."""
    what = "kv8_append"
    B, H, T, D = k.shape
    if v.shape != k.shape or (B, H, D) != (cache.batch, cache.kv_heads, cache.head_dim):
        raise ValueError(f"{what}: k and v must be [{cache.batch}, {cache.kv_heads}, T, "
                         f"{cache.head_dim}], got {tuple(k.shape)} and {tuple(v.shape)}")
    code = _dtype_code(k, f"{what}: k")
    if v.dtype != k.dtype:
        raise TypeError(f"{what}: k and v must have one type")
    if k.stride(3) != 1 or v.stride(3) != 1:
        raise ValueError(f"{what}: k and v need unit stride along head_dim")
    stream = _check_call(what, cache, counts, k, v)
    rc = _lib.lib().kf_kv8_append(
        cache._ref, k.data_ptr(), *k.stride()[:3], v.data_ptr(), *v.stride()[:3], code,
        counts.data_ptr() if counts is not None else None, T, stream)
    _lib.check(rc, "kf_kv8_append")


def kv8_read(cache: KV8Cache, n: int, start: Optional[torch.Tensor] = None,
             counts: Optional[torch.Tensor] = None,
             dtype: torch.dtype = torch.float32) -> Tuple[torch.Tensor, torch.Tensor]:
    """Values (code * scale) of n tokens of each sequence from position
    start[b] (default 0), as K and V [B, kv_heads, n, head_dim] of `dtype`.
    Positions past lens[b] + counts[b] (default lens[b]) read 0."""
    what = "kv8_read"
    if n < 0:
        raise ValueError(f"{what}: n must not be negative")
    if dtype not in VALUE_DTYPES:
        raise TypeError(f"{what}: dtype must be float32, bfloat16 or float16, got {dtype}")
    stream = _check_call(what, cache, counts)
    if start is not None:
        _check_index(what, "start", start, cache)
    shape = (cache.batch, cache.kv_heads, n, cache.head_dim)
    k = torch.empty(shape, dtype=dtype, device=cache.device)
    v = torch.empty(shape, dtype=dtype, device=cache.device)
    rc = _lib.lib().kf_kv8_read(
        cache._ref, start.data_ptr() if start is not None else None,
        counts.data_ptr() if counts is not None else None, n, k.data_ptr(), v.data_ptr(),
        VALUE_DTYPES[dtype], stream)
    _lib.check(rc, "kf_kv8_read")
    return k, v


def kv8_attention(q: torch.Tensor, cache: KV8Cache, counts: Optional[torch.Tensor] = None,
                  causal: bool = True, sm_scale: Optional[float] = None, track: bool = False,
                  max_len: int = 0, out: Optional[torch.Tensor] = None,
                  return_lse: bool = False
                  ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """Attention of the newest tokens over the cache that holds them already.

    q         [B, heads, T, head_dim] float32, bfloat16 or float16, unit stride
              along head_dim; heads is a multiple of the cache's kv_heads, and
              head h reads kv head h // (heads // kv_heads). Query i stands at
              position lens[b] + i
    counts    int32 [B], how many of the T queries are real (default all); the
              sequence's keys are the positions below lens[b] + counts[b]
    causal    query i sees positions up to its own; otherwise all keys
    sm_scale  default head_dim ** -0.5; finite, not negative
    track     add to cache.weight each key's weight, summed over the queries
              and over the heads that read it
    max_len   an upper bound of lens + counts known to the caller (0: what the
              table can hold); a smaller one saves work and, with track,
              workspace (4 * B * heads * T * max_len bytes up to 64 query rows
              of a kv head, at most 4 GB)

    Returns out [B, heads, T, head_dim] of q's type (with return_lse also the
    float32 log of each softmax's sum [B, heads, T]). Rows that see no key, and
    rows from counts[b] on, are 0 (lse -inf). fp16 and fp32 outputs are as near
    to float64 as elementary fp32 torch; for chunks bf16 is up to 1.8 times as
    fast as fp16."""
    what = "kv8_attention"
    B, Hq, T, D = q.shape
    if B != cache.batch or D != cache.head_dim or Hq % cache.kv_heads:
        raise ValueError(f"{what}: q must be [{cache.batch}, a multiple of {cache.kv_heads}, T, "
                         f"{cache.head_dim}], got {tuple(q.shape)}")
    code = _dtype_code(q, f"{what}: q")
    if q.stride(3) != 1:
        raise ValueError(f"{what}: q needs unit stride along head_dim")
    if track and cache.weight is None:
        raise ValueError(f"{what}: track needs a cache with a weight record")
    if out is None:
        out = torch.empty((B, Hq, T, D), dtype=q.dtype, device=q.device)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(3) != 1:
        raise ValueError(f"{what}: out must have q's shape and type and unit stride along "
                         "head_dim")
    stream = _check_call(what, cache, counts, q, out)
    lse = torch.empty((B, Hq, T), dtype=torch.float32, device=q.device) if return_lse else None
    flags = (_lib.KF_KV8_CAUSAL if causal else 0) | (_lib.KF_KV8_TRACK if track else 0)
    L = _lib.lib()
    key = (code, T, Hq, max_len, flags)
    need = cache._work.get(key)
    if need is None:
        need = L.kf_kv8_attention_workspace_bytes(cache._ref, *key)
        if need < 0:
            raise _lib.KernelError(f"{what}: {L.kf_last_error().decode(errors='replace')}")
        if len(cache._work) >= 256:      # a max_len of its own every step
            cache._work.clear()
        cache._work[key] = need
    work = torch.empty(need, dtype=torch.uint8, device=q.device) if need else None
    rc = L.kf_kv8_attention(
        cache._ref, q.data_ptr(), *q.stride()[:3], out.data_ptr(), *out.stride()[:3], code,
        counts.data_ptr() if counts is not None else None, T, Hq, max_len,
        float(sm_scale) if sm_scale is not None else D ** -0.5, flags,
        lse.data_ptr() if lse is not None else None,
        work.data_ptr() if work is not None else None, need, stream)
    _lib.check(rc, "kf_kv8_attention")
    return (out, lse) if return_lse else out


def kv8_evict(cache: KV8Cache, table_out: torch.Tensor, budget: int, recent: int = 0
              ) -> Tuple[torch.Tensor, KV8Cache]:
    """Cut every sequence to `budget` tokens, each kv head by its own record:
    the last `recent` tokens stay and, of the others, those with the most
    recorded weight (ties: the earliest), in their order. A sequence within
    the budget keeps everything.

    table_out  int32 [B, ceil(budget / block)]: pages of the same pool that no
               sequence of `cache` uses; the kept tokens are requantised into
               them by blocks and their weights moved along

    Returns (kept, new): kept int32 [B, kv_heads, budget], the kept positions
    in order and then -1; `new` is the cache of the same pool with `table_out`
    and new lengths. The old pages are not changed and may be reused once work
    on this stream has read them."""
    what = "kv8_evict"
    if cache.weight is None:
        raise ValueError(f"{what}: the cache keeps no weight record")
    if budget <= 0 or not 0 <= recent <= budget:
        raise ValueError(f"{what}: needs budget > 0 and 0 <= recent <= budget")
    new = cache.with_table(table_out, torch.empty_like(cache.lens))
    if new.batch != cache.batch or table_out.shape[1] * cache.block < budget:
        raise ValueError(f"{what}: table_out must be [{cache.batch}, at least "
                         f"{-(-budget // cache.block)}]")
    stream = _check_call(what, cache, None)
    kept = torch.empty((cache.batch, cache.kv_heads, budget), dtype=torch.int32,
                       device=cache.device)
    rc = _lib.lib().kf_kv8_evict(cache._ref, table_out.data_ptr(), new.struct.ld_table, budget,
                                 recent, kept.data_ptr(), new.lens.data_ptr(), stream)
    _lib.check(rc, "kf_kv8_evict")
    return kept, new


def kv8_attention_shared(q: torch.Tensor, cache: KV8Cache, starts: torch.Tensor,
                         shared: torch.Tensor, counts: Optional[torch.Tensor] = None,
                         causal: bool = True, sm_scale: Optional[float] = None,
                         max_shared: int = 0, max_own: int = 0,
                         out: Optional[torch.Tensor] = None, return_lse: bool = False
                         ) -> Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]:
    """kv8_attention for a batch whose groups share their leading pages: samples
    or beams of one prompt, questions about one document. What a group shares is
    read once for all of its rows; the result is kv8_attention's, but for
    rounding.

    starts      int32 [N + 1], ascending: group n is the sequences starts[n] to
                starts[n + 1] - 1. A sequence in no group shares nothing
    shared      int32 [N]: how many leading tokens of its sequences lie on pages
                that their table rows name alike. Cut to whole pages, and to the
                shortest of the group's lens (new tokens are not shared). A
                sequence without a new token does not count: it may hold anything
    max_shared  an upper bound of shared known to the caller (0: what the table
                can hold); what is beyond it is read sequence by sequence
    max_own     an upper bound of the tokens of a sequence that has a new one, new
                ones among them, besides those (0: what the table can hold). A
                sequence with more is cut there and recorded in the device status
                word

    The other arguments, what is returned and which rows are 0 as for
    kv8_attention. There is no weight record to add to: it belongs to the pages,
    which here are several sequences'."""
    what = "kv8_attention_shared"
    B, Hq, T, D = q.shape
    if B != cache.batch or D != cache.head_dim or Hq % cache.kv_heads:
        raise ValueError(f"{what}: q must be [{cache.batch}, a multiple of {cache.kv_heads}, T, "
                         f"{cache.head_dim}], got {tuple(q.shape)}")
    code = _dtype_code(q, f"{what}: q")
    if q.stride(3) != 1:
        raise ValueError(f"{what}: q needs unit stride along head_dim")
    if out is None:
        out = q.new_empty((B, Hq, T, D))   # (half the host time of torch.empty)
    elif out.shape != q.shape or out.dtype != q.dtype or out.stride(3) != 1:
        raise ValueError(f"{what}: out must have q's shape and type and unit stride along "
                         "head_dim")
    stream = _check_call(what, cache, counts, q, out)
    groups = shared.shape[0] if shared.dim() == 1 else -1
    index = q.get_device()
    if starts.dtype is not torch.int32 or shared.dtype is not torch.int32 \
            or starts.shape != (groups + 1,) or not starts.is_contiguous() \
            or not shared.is_contiguous() or starts.get_device() != index \
            or shared.get_device() != index:
        raise ValueError(f"{what}: starts and shared must be contiguous int32 tensors [N + 1] and [N] "
                         f"on {cache.device}, got {starts.dtype} {tuple(starts.shape)} on "
                         f"{starts.device} and {shared.dtype} {tuple(shared.shape)} on "
                         f"{shared.device}")
    lse = q.new_empty((B, Hq, T), dtype=torch.float32) if return_lse else None
    flags = _lib.KF_KV8_CAUSAL if causal else 0
    L = _lib.lib()
    key = (code, T, Hq, groups, max_shared, max_own, flags)
    need = cache._work.get(key)
    if need is None:
        need = L.kf_kv8_attention_shared_workspace_bytes(cache._ref, *key)
        if need < 0:
            raise _lib.KernelError(f"{what}: {L.kf_last_error().decode(errors='replace')}")
        if len(cache._work) >= 256:      # bounds of its own every step
            cache._work.clear()
        cache._work[key] = need
    work = q.new_empty(need, dtype=torch.uint8) if need else None
    rc = L.kf_kv8_attention_shared(
        cache._ref, q.data_ptr(), *q.stride()[:3], out.data_ptr(), *out.stride()[:3], code,
        counts.data_ptr() if counts is not None else None, T, Hq, starts.data_ptr(),
        shared.data_ptr(), groups, max_shared, max_own,
        float(sm_scale) if sm_scale is not None else D ** -0.5, flags,
        lse.data_ptr() if lse is not None else None,
        work.data_ptr() if work is not None else None, need, stream)
    _lib.check(rc, "kf_kv8_attention_shared")
    return (out, lse) if return_lse else out


Caches = Union[KV8Cache, Sequence[KV8Cache]]


def _refs(caches: Sequence[KV8Cache]):
    return (ctypes.POINTER(_lib.KV8CacheStruct) * len(caches))(*[c._ptr for c in caches])


def kv8_copy(cache: Caches, src: torch.Tensor, dst: torch.Tensor,
             tokens: Optional[torch.Tensor] = None, into: Optional[Caches] = None) -> None:
    """Copy pages: page dst[i] becomes page src[i], for all kv heads, codes and
    scales, and the weight record where both caches keep one.

    cache     the cache, or the layers' caches (of one geometry), copied in one
              call
    src, dst  int32 [n]; a pair of the same page is no copy
    tokens    int32 [n] (default whole pages): only the first tokens[i] slots
              are copied, with the scales; the others stay as they are
    into      the caches whose pages dst are (default: the same ones); another
              pool, of any number of pages. A tensor that is written may not
              occur twice in a call, nor be read by it (but for copies within a
              pool)

    A pair is not done, and recorded in the device status word (code 6), if an
    entry is no page of its pool, or if another pair writes the same page or,
    within one pool, reads it. The caches' tables and lens are not used."""
    what = "kv8_copy"
    caches = [cache] if isinstance(cache, KV8Cache) else list(cache)
    to = caches if into is None else [into] if isinstance(into, KV8Cache) else list(into)
    if not caches:
        return
    if len(to) != len(caches):
        raise ValueError(f"{what}: {len(caches)} caches into {len(to)}")
    first = caches[0]
    kind, index = first._kind, first._kind[4]
    for c in caches if into is None else caches + to:
        if c._kind != kind:
            raise ValueError(f"{what}: all caches must have the codes, heads, block, head_dim and "
                             "device of the first")
    stream = _check_call(what, first, None)
    shape = src.shape
    for t in (src, dst) if tokens is None else (src, dst, tokens):
        if t.dtype is not torch.int32 or t.shape != shape or len(shape) != 1 \
                or not t.is_contiguous() or t.get_device() != index:
            raise ValueError(f"{what}: src, dst and tokens must be contiguous int32 tensors [n] on "
                             f"{first.device}, got {t.dtype} {tuple(t.shape)} on {t.device}")
    n = shape[0]
    L = _lib.lib()
    need = 0
    if n > 256:                  # few pairs need no workspace
        need = L.kf_kv8_copy_workspace_bytes(first._ref, to[0]._ref, n)
        if need < 0:
            raise _lib.KernelError(f"{what}: {L.kf_last_error().decode(errors='replace')}")
    work = src.new_empty(need, dtype=torch.uint8) if need else None
    refs = _refs(caches)
    rc = L.kf_kv8_copy(refs, refs if into is None else _refs(to), len(caches), src.data_ptr(),
                       dst.data_ptr(), tokens.data_ptr() if tokens is not None else None, n,
                       work.data_ptr() if work is not None else None, need, stream)
    _lib.check(rc, "kf_kv8_copy")
