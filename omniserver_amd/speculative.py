"""Verification of drafted tokens against the target model's probabilities.

A step of speculative decoding scores the nodes of a drafted tree in one forward
(``PreallocatedKVCache.tree_cache``); ``verify`` then walks each tree from its root and decides,
from random numbers the caller gives, which drafted tokens stand and which token follows them,
such that the emitted tokens are distributed as if the target had been sampled one by one;
``TreeCache.accept`` makes the accepted nodes the end of the cached sequence.
"""

from __future__ import annotations

from typing import NamedTuple

import torch

from ._lib import call, lib, ptr, require_here, stream
from .kv_cache import TREE_MAX_NODES as MAX_NODES

_DTYPES = {torch.float16: 0, torch.bfloat16: 1, torch.float32: 2}


class Verified(NamedTuple):
    """Per sequence the accepted nodes and the tokens they emit."""
    path: torch.Tensor       # int32 [n, T]: 0, then the accepted nodes, -1 after them
    tokens: torch.Tensor     # int64 [n, T]: the accepted nodes' tokens and the next one, then -1
    emitted: torch.Tensor    # int32 [n]: how many of each (0 for a sequence without nodes)


def chain_parents(n: int, nodes: int, device) -> torch.Tensor:
    """Parents of n chains: every node the child of the one before it."""
    return torch.arange(-1, nodes - 1, device=device, dtype=torch.int32).repeat(n, 1)


def verify(logits: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor | None = None,
           temperature=0.0, parents: torch.Tensor | None = None,
           draft_logits: torch.Tensor | None = None,
           counts: torch.Tensor | None = None) -> Verified:
    """Accept drafted tokens and draw the next one, for n sequences of T <= 64 nodes.

    logits [n, T, V] (fp16, bf16 or fp32, columns contiguous): the target's after each node;
    tokens int64 [n, T]: the nodes' tokens (node 0's is not read).  With p = softmax(logits /
    temperature) at a node:

    * ``parents`` int32 [n, T]: trees of proposed tokens.  A node's children are tried in index
      order; child x with random number u stands if u * (1 - p(siblings tried before)) < p(x).  A
      token that a sibling has tried, or outside [0, V), never stands.  If no child stands the
      next token comes from p without the tried tokens.
    * neither ``parents`` nor ``draft_logits``: chains of proposed tokens (node i + 1 below node i).
    * ``draft_logits`` [n, T - 1, V], logits' type: chains drawn from q = softmax(draft_logits /
      temperature), row i the distribution of node i + 1.  x stands if u * q(x) < p(x); at the first
      that does not, the next token comes from max(p - q, 0), after the last from p.

    uniforms fp32 [n, T] in [0, 1): node i's is tried against its parent's distribution, node 0's
    draws the next token: the first v whose running sum of weights exceeds u * their total (p itself
    where the remaining weights are all zero).  temperature: a number, or fp32 [n]; 0 (in a tensor
    also what is not above 0) puts all mass on the first maximum, and needs no random numbers.
    counts int32 [n]: nodes in use (default T).

    A NaN logit counts as -inf; where no token is above -inf the next token is -1.  The same
    inputs give the same tokens: those of 64-bit weights and sums, which the 32-bit sums of the rows
    stand for only where they cannot change what is decided."""
    draft, work = _check(logits, tokens, uniforms, temperature, parents, draft_logits, counts)
    n, T, V = logits.shape
    dev = logits.device
    out = Verified(torch.empty(n, T, device=dev, dtype=torch.int32),
                   torch.empty(n, T, device=dev, dtype=torch.int64),
                   torch.empty(n, device=dev, dtype=torch.int32))
    ws = torch.empty(work, device=dev, dtype=torch.float64)
    per_row = isinstance(temperature, torch.Tensor)
    s0, s1, _ = logits.stride()
    d0, d1, _ = (0, 0, 1) if draft is None else draft.stride()
    call("omni_spec_verify", logits.data_ptr(), _DTYPES[logits.dtype], s0, s1, ptr(draft), d0, d1,
         tokens.data_ptr(), ptr(parents), ptr(counts), ptr(uniforms),
         temperature.data_ptr() if per_row else None, 0.0 if per_row else float(temperature), n, T,
         V, out.path.data_ptr(), out.tokens.data_ptr(), out.emitted.data_ptr(), ws.data_ptr(), work,
         stream())
    return out


def _check(logits, tokens, uniforms, temperature, parents, draft_logits, counts) -> tuple:
    """Refuse what the kernels do not take; (draft logits or None, doubles of workspace)."""
    if logits.dim() != 3:
        raise ValueError(f"logits of shape {tuple(logits.shape)}: expected [n, nodes, vocab]")
    n, T, V = logits.shape
    if not 1 <= T <= MAX_NODES or V < 1:
        raise ValueError(f"{T} nodes over a vocabulary of {V}: 1 to {MAX_NODES} nodes")
    if logits.dtype not in _DTYPES:
        raise TypeError(f"logits are fp16, bf16 or fp32 (got {logits.dtype})")
    if logits.stride(2) != 1 and V > 1:
        raise ValueError("the logits' columns have to be contiguous")
    if draft_logits is not None:
        if parents is not None:
            raise ValueError("draft_logits are for chains: give parents or draft_logits")
        if tuple(draft_logits.shape) != (n, T - 1, V) or draft_logits.dtype != logits.dtype:
            raise ValueError(f"draft_logits {tuple(draft_logits.shape)} {draft_logits.dtype}: "
                             f"expected [{n}, {T - 1}, {V}] {logits.dtype}")
        if draft_logits.stride(2) != 1 and V > 1:
            raise ValueError("the draft logits' columns have to be contiguous")
    per_row = isinstance(temperature, torch.Tensor)
    if not per_row and not 0.0 <= float(temperature) < float("inf"):
        raise ValueError(f"temperature {temperature}: zero or above, finite")
    if uniforms is None and (per_row or temperature > 0):
        raise ValueError("sampling needs random numbers: uniforms [n, nodes]")
    _is(tokens, (n, T), torch.int64, "tokens")
    _is(uniforms, (n, T), torch.float32, "uniforms")
    _is(parents, (n, T), torch.int32, "parents")
    _is(counts, (n,), torch.int32, "counts")
    if per_row:
        _is(temperature, (n,), torch.float32, "temperature")
        require_here(temperature)
    require_here(logits, draft_logits, tokens, uniforms, parents, counts)
    if T == 1:
        draft_logits = None
    work = lib().omni_spec_verify_work(n, T, V, int(draft_logits is not None))
    if work < 0:
        raise ValueError(f"{n} sequences of {T} nodes over a vocabulary of {V}: too large")
    return draft_logits, work


def _is(t, shape, dtype, name: str) -> None:
    if t is None:
        return
    if t.dtype != dtype:
        raise TypeError(f"{name}: expected {dtype}, got {t.dtype}")
    if t.shape != shape or not t.is_contiguous():
        raise ValueError(f"{name} of shape {tuple(t.shape)}: expected a contiguous {list(shape)}")
