"""
Beam search's choice among the continuations of its beams (`V3Cache.beam_step` and `PagedV3Cache.beam_step` choose by it and let the cache follow).
"""
from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _native

MAX_BEST, MAX_BEAMS = 64, 1024


def beam_select(logits: torch.Tensor, scores: torch.Tensor, best: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Of the continuations of every sequence's beams the `best` (default: as many as there are beams) with the largest sums scores + log_softmax(logits).
    logits [batch, beams, vocabulary] (float32, float16 or bfloat16), scores [batch, beams] -> sums (float32), tokens and beams they continue (int64),
    each [batch, best], in falling order, equal ones by beam and then token.  Sums are formed and compared in 64 bits, from sums of exponentials in 32 (a beam's sums can be off by some 2^-22,
    all by the same); beams of equal logits and scores have equal sums, wherever in memory they lie.
    A beam whose sums are no numbers (a NaN or +infinity among its logits, nothing but -infinity, a score that is not finite: a beam that has ended or not begun) counts with sums of
    -infinity.  At most 64 are chosen, of at most 1024 beams.  Not differentiable."""
    n = logits.shape[1] if best is None and logits.dim() > 1 else best
    if logits.is_cuda and not torch.compiler.is_compiling():
        chosen = _native.fast().beam_select(logits, scores, n)
        if chosen is not None:
            if type(chosen) is int:
                _native.check(chosen, "tq_beam_select")
            return chosen
    return _select(logits, scores, n)


@torch.compiler.disable
@torch.no_grad()
def _select(logits: torch.Tensor, scores: torch.Tensor, best: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """beam_select for logits and scores of any layout, with every check."""
    _native._require_gpu(logits, "logits")
    if logits.dim() != 3 or tuple(scores.shape) != tuple(logits.shape[:2]):
        raise ValueError(f"beam_select takes logits [batch, beams, vocabulary] and scores [batch, beams]; got {tuple(logits.shape)} and {tuple(scores.shape)}")
    code = _native.dtype_code(logits.dtype)
    if scores.device != logits.device:
        raise _native.TqError(f"scores on {scores.device}, logits on {logits.device}")
    if not scores.dtype.is_floating_point:
        raise ValueError(f"scores must be floats, got {scores.dtype}")
    batch, beams, vocab = logits.shape
    n = best
    if isinstance(n, bool) or int(n) != n or not 0 <= n <= MAX_BEST or (batch and n > beams * vocab):
        raise ValueError(f"best must be a whole number from 0 to {min(MAX_BEST, beams * vocab)}, got {n!r}")
    n = int(n)
    if beams > MAX_BEAMS or beams * vocab > 0x7fffffff:
        raise ValueError(f"at most {MAX_BEAMS} beams and 2^31 - 1 continuations a sequence; got {beams} x {vocab}")
    scores = scores.float().contiguous()
    if vocab > 1 and logits.stride(2) != 1:
        logits = logits.contiguous()
    dev = logits.device
    with _native._on(dev):
        values = torch.empty((batch, n), dtype=torch.float32, device=dev)
        tokens = torch.empty((batch, n), dtype=torch.int64, device=dev)
        parents = torch.empty_like(tokens)
        if values.numel():
            size = int(_native.lib().tq_beam_scratch(batch, beams, vocab, n))
            if size < 0:
                _native.check(size, "tq_beam_scratch")
            scratch = torch.empty(size, dtype=torch.uint8, device=dev)
            _native.check(_native.lib().tq_beam_select(logits.data_ptr(), code, batch, beams, vocab, logits.stride(0), logits.stride(1), scores.data_ptr(), scores.stride(0), n,
                                                       values.data_ptr(), tokens.data_ptr(), parents.data_ptr(), scratch.data_ptr(), size, _native._stream_handle(dev)), "tq_beam_select")
    return values, tokens, parents
