"""Beam search's selection: which beams go on, and with which tokens.

`beam_select` takes the logits of every beam and the beams' scores and returns
the n best continuations of each batch row. With `kv8_copy` (the pages of the
beams that go on) and `kv8_attention_shared` (beams share their prompt) it makes
a step of beam search over the 8-bit cache; `techjam2026_b200.kvcache` does this
for the layer stack. Runs csrc/beam_sm100.cu: one pass over the logits. The
reference generates nothing, so it has no counterpart.

Calls are stream-ordered on the current stream and may be captured in a CUDA
graph.
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from .. import _lib
from .kv8 import VALUE_DTYPES

MAX_TAKE = 128
MAX_BEAMS = 1024


def beam_select(logits: torch.Tensor, scores: torch.Tensor, n: Optional[int] = None,
                ended: Optional[torch.Tensor] = None, pad: int = 0
                ) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The n best of the candidates scores[b, k] + log softmax(logits[b, k])[v].

    logits  [B, K, V] float32, bfloat16 or float16, any strides with unit
            stride along V
    scores  [B, K] float32, unit stride along K: log probability of each beam so
            far; a beam of -inf has no candidates
    n       how many to take, 1 to 128 (default K)
    ended   [B, K] bool or None: an ended beam has one candidate, its score
            unchanged, with the token `pad`

    Returns (scores [B, n] float32, beams [B, n] int32, tokens [B, n] int32),
    best first; of equal candidates the one of the lowest beam, then token. They
    are compared in 64 bits (the softmax's sum is one of float32 values). Which
    tokens of a beam are among its n best is decided by their logits: of two that
    differ but give equal candidates, the larger logit comes first there.
    Candidates that are -inf or NaN are none; a logit of +inf or NaN leaves its beam
    without candidates. Where there are fewer than n, the rest is (-inf, -1, -1)."""
    what = "beam_select"
    if logits.dim() != 3:
        raise ValueError(f"{what}: logits must be [B, K, V], got {tuple(logits.shape)}")
    B, K, V = logits.shape
    code = VALUE_DTYPES.get(logits.dtype)
    if code is None:
        raise TypeError(f"{what}: logits must be float32, bfloat16 or float16, got {logits.dtype}")
    if scores.dtype is not torch.float32:
        raise TypeError(f"{what}: scores must be float32, got {scores.dtype}")
    if not logits.is_cuda:
        raise RuntimeError(f"{what}: CUDA tensors required (no CPU path)")
    n = K if n is None else n
    if not 0 < n <= MAX_TAKE or not 0 < K <= MAX_BEAMS or V == 0:
        raise ValueError(f"{what}: needs 1 to {MAX_BEAMS} beams, a vocabulary, and n from 1 to "
                         f"{MAX_TAKE}, got {K}, {V} and {n}")
    if not 0 <= pad < 2 ** 31:
        raise ValueError(f"{what}: pad must be a token, got {pad}")
    index = logits.get_device()
    for t in (scores,) if ended is None else (scores, ended):
        if t.shape != (B, K) or (K > 1 and t.stride(1) != 1) or t.get_device() != index:
            raise ValueError(f"{what}: scores and ended must be [{B}, {K}] with unit stride along the "
                             f"beams, on {logits.device}; got {tuple(t.shape)}, strides {t.stride()}, "
                             f"on {t.device}")
    if V > 1 and logits.stride(2) != 1:
        raise ValueError(f"{what}: logits need unit stride along the vocabulary")
    if ended is not None and ended.dtype is not torch.bool:
        raise TypeError(f"{what}: ended must be bool, got {ended.dtype}")
    if index != torch.cuda.current_device():
        raise RuntimeError(f"{what}: logits are on {logits.device}, which is not the current device")
    score = scores.new_empty((B, n))
    beam = scores.new_empty((B, n), dtype=torch.int32)
    token = torch.empty_like(beam)
    L = _lib.lib()
    need = L.kf_beam_select_workspace_bytes(B, K, V, n)
    if need < 0:
        raise _lib.KernelError(f"{what}: {L.kf_last_error().decode(errors='replace')}")
    work = scores.new_empty(need, dtype=torch.uint8) if need else None
    sb, sk, _ = logits.stride()
    rc = L.kf_beam_select(
        logits.data_ptr(), sb, sk, code, scores.data_ptr(), scores.stride(0),
        ended.data_ptr() if ended is not None else None,
        ended.stride(0) if ended is not None else 0, B, K, V, n, pad, score.data_ptr(),
        beam.data_ptr(), token.data_ptr(), work.data_ptr() if work is not None else None, need,
        torch._C._cuda_getCurrentRawStream(index))
    _lib.check(rc, "kf_beam_select")
    return score, beam, token
