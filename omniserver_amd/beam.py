"""Beam search's choice over the beams of a request and the vocabulary.

A step of beam search scores the next token of every beam in one forward; ``select`` then keeps the
best continuations, and ``PagedKVCache.reorder`` makes the cache's rows go on from the beams that
these continue.
"""

from __future__ import annotations

from functools import lru_cache
from typing import NamedTuple

import torch

from ._lib import call, lib, ptr, require_here, stream
from .hostio import to_device
from .speculative import _DTYPES, _is

MAX_BEAMS, MAX_K, MAX_VOCAB = 32, 64, 64 * 8192


class Selected(NamedTuple):
    """Per request its k best continuations, the best first."""
    scores: torch.Tensor     # fp32 [n, k]: sums of log-probabilities, -inf where there is none
    parents: torch.Tensor    # int32 [n, k]: the beams they continue, or -1
    tokens: torch.Tensor     # int64 [n, k]: by which token, or -1
    done: torch.Tensor       # bool [n, k]: finished (or none)


@lru_cache(maxsize=256)
def _work(n: int, W: int, V: int, k: int) -> int:
    work = lib().omni_beam_select_work(n, W, V, k)
    if work < 0:
        raise ValueError(f"{n} requests of {W} beams over a vocabulary of {V}: too large")
    return work


def select(logits: torch.Tensor, scores: torch.Tensor, k: int | None = None,
           done: torch.Tensor | None = None, stop=None, pad: int = 0) -> Selected:
    """The k best continuations (default W, at most 64) of n requests with W <= 32 beams each.

    logits [n, W, V] (fp16, bf16 or fp32, columns contiguous); scores fp32 [n, W]: the beams' sums of
    log-probabilities.  Going on with token v is worth scores + logits[v] - log sum exp logits; a beam
    whose score is not finite is not in use (so a request's first step has one beam in use).  ``done``
    bool [n, W]: a finished beam goes on only as itself, with token ``pad`` at its score, whatever its
    logits.  ``stop``: tokens that finish a beam, a list, or int64 [m] or [n, m] on the
    device (-1: none).

    Ties go to the lower beam, then to the lower token.  A NaN logit counts as -inf, infinite ones
    share all the weight; tokens at -inf, or whose sum is too low for fp32, are no continuations, and
    where a request has fewer than k the rest is -inf, -1, -1, finished.  Values are compared in 64
    bits, those within a beam by their logits; the same inputs give the same choice.  The scores given
    out are fp32, and where no other beam's value stood close they have the logarithm of a sum in 32 bits
    in them: off by 4e-6 at most beside their rounding.  A list of stop tokens is uploaded, which a
    capture refuses."""
    if logits.dim() != 3:
        raise ValueError(f"logits of shape {tuple(logits.shape)}: expected [n, beams, vocab]")
    n, W, V = logits.shape
    k = W if k is None else int(k)
    if not 1 <= W <= MAX_BEAMS or not 1 <= k <= MAX_K or not 1 <= V <= MAX_VOCAB:
        raise ValueError(f"{k} of {W} beams over a vocabulary of {V}: 1 to {MAX_K}, 1 to {MAX_BEAMS}, "
                         f"1 to {MAX_VOCAB}")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits are fp16, bf16 or fp32 (got {logits.dtype})")
    if logits.stride(2) != 1 and V > 1:
        raise ValueError("the logits' columns have to be contiguous")
    dev = logits.device
    if stop is not None and not isinstance(stop, torch.Tensor):
        stop = to_device([int(t) for t in stop], torch.int64, dev)
    _is(scores, (n, W), torch.float32, "scores")
    _is(done, (n, W), torch.bool, "done")
    m = 0
    if stop is not None:
        m = stop.shape[-1] if stop.dim() else 0
        _is(stop, (m,) if stop.dim() == 1 else (n, m), torch.int64, "stop")
    require_here(logits, scores, done, stop)
    out = Selected(torch.empty(n, k, device=dev, dtype=torch.float32),
                   torch.empty(n, k, device=dev, dtype=torch.int32),
                   torch.empty(n, k, device=dev, dtype=torch.int64),
                   torch.empty(n, k, device=dev, dtype=torch.bool))
    work = _work(n, W, V, k)
    ws = torch.empty(work, device=dev, dtype=torch.float64)
    call("omni_beam_select", logits.data_ptr(), _DTYPES[logits.dtype], logits.stride(0),
         logits.stride(1), scores.data_ptr(), ptr(done), ptr(stop), m,
         m if stop is not None and stop.dim() == 2 else 0, int(pad), n, W, V, k,
         out.scores.data_ptr(), out.parents.data_ptr(), out.tokens.data_ptr(), out.done.data_ptr(),
         ws.data_ptr(), work, stream())
    return out
