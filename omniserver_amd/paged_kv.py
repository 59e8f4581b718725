"""Paged KV cache: keys and values in pages of a few dozen tokens, named by a block table per sequence.

Beside ``PreallocatedKVCache`` (a row of ``max_len`` tokens for every sequence) this one gives each
sequence the pages that its tokens need, anywhere in the pool, and lets sequences share them: beams
of one prompt hold its pages together.  A table and a length are all the state there is.  A page is
free where no sequence's table names it within its length; nothing is counted or returned.

A step asks for room first (``reserve``, or the adapters for a model's forward: ``prefill_cache``,
``decode_cache``), writes and attends, and moves the lengths last (``finish``).  ``reorder`` makes
rows go on from their parents' tables after a beam search's choice (``beam.select``).  All of it
runs on the device from device tensors, without a host synchronisation, and can be captured in a
graph: omni_page_reserve, omni_paged_attention, omni_page_reorder.  Lists in their place are uploaded,
which a capture refuses.
"""

from __future__ import annotations

from typing import List, Sequence

import torch

from ._lib import call, ptr, require_here, stream
from .attention import num_cus, prefill_attention_pool
from .hostio import to_device
from .kv_cache import PreallocatedKVCache, _head_rows, _ints

MAX_PAGES = 1 << 19
MAX_SEQS = 2048
MAX_TOKENS = 1 << 28               # packed rows of a reservation
PAGE_SIZES = (16, 32, 64, 128, 256, 512, 1024)
UNIT = 128                         # keys of a workgroup's step in omni_paged_attention
_DTYPES = {torch.float16: 0, torch.bfloat16: 1}


def attention_columns(n: int, nh: int, nkv: int, max_len: int, cus: int) -> int:
    """Columns of workgroups that n sequences' keys are cut over: two workgroups a CU, as many as fit
    at once, and no column without a step.  us of attention and merge with one, two and four a CU: 32
    sequences at 2048 tokens of 2 KV heads 18.2 / 19.2 / 21.8, 8 at 100-8000 14.8 / 11.2 / 11.3, 32 x 4
    beams at 4096 37.1 / 32.7 / 37.8, 32 at 4096 of 8 KV heads 98.6 / 102.5 / 104.3."""
    per = nkv * -(-(nh // nkv) // 32)
    return max(1, min(2 * cus // per, n * -(-max_len // UNIT)))


def attention_group(nh: int, nkv: int) -> int:
    """How many sequences a workgroup takes together where they share pages: 32 queries in all, two
    matrix operands' columns, whose outputs fill a wave's registers."""
    return 32 // (nh // nkv) if nh // nkv <= 16 else 1


class PagedKVCache:
    """``num_pages`` pages of ``page_size`` tokens (a power of two from 16 to 1024) for up to
    ``max_seqs`` sequences of up to ``max_len`` tokens.

    storage [n_layers, 2, num_pages, page_size, n_kv_heads, head_dim] fp16 or bf16 (``k[l]`` and
    ``v[l]`` are views of it), head_dim 64 or 128; tables int32 [max_seqs, pages of max_len]; lengths
    int64 [max_seqs].  Token t of sequence r is in page tables[r, t // page_size], place t %
    page_size.  Entries behind a sequence's length mean nothing.  The tables and lengths may be read
    and written between steps; no two sequences may hold a page of which only a part is filled."""

    def __init__(self, n_layers: int, num_pages: int, n_kv_heads: int, page_size: int, head_dim: int,
                 device, max_seqs: int, max_len: int, dtype=torch.float16,
                 n_heads: int | None = None):
        n_heads = 6 * n_kv_heads if n_heads is None else n_heads
        if dtype not in _DTYPES:
            raise ValueError(f"the pages are fp16 or bf16 (got {dtype})")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"pages of {page_size} tokens: one of {PAGE_SIZES}")
        if head_dim not in (64, 128):
            raise ValueError(f"head_dim {head_dim}: 64 or 128")
        if n_layers < 1 or n_kv_heads < 1 or n_heads < 1 or n_heads % n_kv_heads:
            raise ValueError(f"{n_layers} layers, {n_heads} heads over {n_kv_heads} KV heads")
        if not 1 <= num_pages <= MAX_PAGES or not 1 <= max_seqs <= MAX_SEQS:
            raise ValueError(f"{num_pages} pages, {max_seqs} sequences: 1 to {MAX_PAGES} and 1 to "
                             f"{MAX_SEQS}")
        if not 1 <= max_len <= 1 << 30:
            raise ValueError(f"max_len {max_len}: 1 to {1 << 30}")
        self.n_layers, self.num_pages, self.page_size = n_layers, num_pages, page_size
        self.n_heads, self.n_kv_heads, self.head_dim = n_heads, n_kv_heads, head_dim
        self.max_seqs, self.max_len = max_seqs, max_len
        self.device = torch.device(device)
        self.storage = torch.zeros(n_layers, 2, num_pages, page_size, n_kv_heads, head_dim,
                                   device=device, dtype=dtype)
        self.k: List[torch.Tensor] = [self.storage[l, 0] for l in range(n_layers)]
        self.v: List[torch.Tensor] = [self.storage[l, 1] for l in range(n_layers)]
        self.tables = torch.zeros(max_seqs, -(-max_len // page_size), device=device,
                                  dtype=torch.int32)
        self.lengths = torch.zeros(max_seqs, device=device, dtype=torch.int64)
        self._step = 0             # counts what may give pages away
        self._plans = {}

    def _geometry(self) -> tuple:
        return (self.tables.data_ptr(), self.lengths.data_ptr(), self.max_seqs,
                self.tables.shape[1], self.num_pages, self.page_size, self.max_len)

    def _attention_plan(self, n: int) -> tuple:
        """(columns, rows taken together, floats of split states) for n sequences."""
        plan = self._plans.get(n)
        if plan is None:
            columns = attention_columns(n, self.n_heads, self.n_kv_heads, self.max_len,
                                        num_cus(self.device))
            most = attention_group(self.n_heads, self.n_kv_heads)
            states = columns + n + (columns * most + n if most > 1 else 0)
            plan = self._plans[n] = (columns, most, states * self.n_heads * (self.head_dim + 4))
        return plan

    # ---- room for new tokens ---------------------------------------------------------
    def reserve(self, counts, rows: Sequence[int] | None = None,
                tokens: int | None = None) -> "PageSlots":
        """Room for counts[i] new tokens behind sequence rows[i] (default: i), packed one request
        after another: see PageSlots.  counts int32 [n] on the device, with ``tokens`` the number of
        packed rows, or a list."""
        return PageSlots(self, counts, rows, tokens)

    def prefill_cache(self, rows: Sequence[int], seg_lengths: Sequence[int]) -> "PagedPrefill":
        """Adapter for one forward over packed prompts, which become sequences ``rows``."""
        return PagedPrefill(self, rows, seg_lengths)

    def decode_cache(self, n: int, counts=None, rope_delta: torch.Tensor | None = None) -> "PagedDecode":
        """Adapter for one forward over one new token for each of sequences [0, n): see
        PagedDecode."""
        return PagedDecode(self, n, counts, rope_delta)

    def free(self, rows: Sequence[int]) -> None:
        """Forget the sequences ``rows``; pages that no other one holds are free."""
        rows = self._checked_rows(rows)
        self._step += 1
        if rows:
            self.lengths.index_fill_(0, to_device(rows, torch.int64, self.device), 0)

    def _checked_rows(self, rows) -> List[int]:
        rows = [int(r) for r in rows]
        if any(not 0 <= r < self.max_seqs for r in rows) or len(set(rows)) != len(rows):
            raise ValueError(f"rows {rows}: all different, within the {self.max_seqs} sequences")
        return rows

    # ---- beams -----------------------------------------------------------------------
    def reorder(self, parents) -> None:
        """Make beams go on from others: parents int32 [n, W] (on the device, or a list); row s * W +
        w of the first n * W takes the place of row s * W + parents[s, w] as it was, table, length
        and K/V.  Whole pages are shared.  A page that is filled in part stays with its parent's first
        child, every other child gets the lowest free page and a copy of the tokens in it, in every
        layer.  Rows whose parent is outside [0, W), or for which no page is free, are empty."""
        if not isinstance(parents, torch.Tensor):
            parents = [[int(p) for p in row] for row in parents]
            W = len(parents[0]) if parents else 0
            if any(len(row) != W or any(not -1 <= p < W for p in row) for row in parents):
                raise ValueError(f"parents {parents}: a beam of the same request each, or -1")
            parents = to_device(parents, torch.int32, self.device)
        if parents.dim() != 2 or not 1 <= parents.numel() <= self.max_seqs:
            raise ValueError(f"parents of shape {tuple(parents.shape)}: [n, beams], 1 to "
                             f"{self.max_seqs} in all")
        n, W = parents.shape
        parents = _ints(parents, (n, W), torch.int32, self.device, "parents")
        require_here(self.storage, parents)
        work = torch.empty(4 * n * W, device=self.device, dtype=torch.int32)
        self._step += 1
        call("omni_page_reorder", self.storage.data_ptr(), self.n_layers,
             self.n_kv_heads * self.head_dim, *self._geometry(), parents.data_ptr(), n, W,
             work.data_ptr(), 4 * n * W, stream())


class PageSlots:
    """Where the tokens of a step go.

    Request i brings counts[i] tokens (less than one: none) to sequence rows[i].  It is granted all
    of them or none: none where they run past max_len or the packed rows, or where the pages that they
    need are not free.  New pages are the lowest free ones, request by request; one that goes
    without leaves those it asked for unused, and one that needs no page never goes without.

    The tables name the new pages at once; the lengths, read when this is made, move with
    ``finish``.  Until then the pages are only asked for: the next reservation, or reordering, may
    give them to others, and this one then refuses to be used any further.  (A captured graph's
    steps are not seen by that check: finish before replaying one.)  The buffers belong to this
    object, so two captured graphs never share them."""

    def __init__(self, pool: PagedKVCache, counts, rows=None, tokens=None, dense: bool = False,
                 n: int | None = None, rope_delta=None, columns: int = 0, most: int = 0,
                 floats: int = 0):
        dev = pool.device
        if rows is not None:
            rows = pool._checked_rows(rows)
        if counts is not None and not isinstance(counts, torch.Tensor):
            counts = [int(c) for c in counts]
            if any(not 0 <= c <= pool.max_len for c in counts):
                raise ValueError(f"counts {counts}: new tokens, 0 to {pool.max_len}")
            if tokens is None:
                tokens = sum(counts)
        if n is None:
            if counts is None or tokens is None:
                raise ValueError("counts on the device need the number of packed rows: tokens")
            n = len(counts)
        if not 1 <= n <= pool.max_seqs or (rows is not None and len(rows) != n):
            raise ValueError(f"{n} requests for {pool.max_seqs if rows is None else len(rows)} "
                             f"sequences")
        T = n if dense else int(tokens)
        if not 0 <= T <= MAX_TOKENS:
            raise ValueError(f"{T} packed rows: 0 to {MAX_TOKENS}")
        self.counts = _ints(counts, (n,), torch.int32, dev, "counts")
        self.rows = _ints(rows, (n,), torch.int64, dev, "rows")
        rope_delta = _ints(rope_delta, None, torch.int64, dev, "rope_delta")
        if rope_delta is not None and rope_delta.numel() < pool.max_seqs:
            raise ValueError(f"rope_delta holds one value per sequence ({pool.max_seqs})")
        require_here(pool.lengths, self.counts, rope_delta)
        self.pool, self.n, self.T = pool, n, T
        self._axes = axes = 3 if dense else 1
        # int64: starts, lengths after, pages, places, positions; int32: granted, sums of rows; on
        # 16-byte boundaries the attention's schedule, int32, and its split states, fp32 (for all layers:
        # launches on one stream are ordered)
        words = 2 * n + (2 + axes) * T
        ints = 2 * n + 1 + (-(2 * words + 2 * n + 1) % 4)
        more = 8 * n + 4 * columns if columns else 0
        self._plan = torch.empty(words + (ints + more + floats + 1) // 2, device=dev,
                                 dtype=torch.int64)
        p = self._plan.data_ptr()
        self._granted = p + 8 * words
        self._schedule = self._granted + 4 * ints if columns else None
        self._states = self._granted + 4 * (ints + more)
        self._page, self._place = p + 16 * n, p + 16 * n + 8 * T
        pool._step += 1
        self._step = pool._step
        call("omni_page_reserve", *pool._geometry(), ptr(self.counts), ptr(self.rows),
             ptr(rope_delta), n, T, int(dense), axes, p, p + 8 * n, self._page, self._place,
             p + 16 * (n + T), self._granted, self._granted + 4 * n, self._schedule, columns,
             most, stream())

    @property
    def starts(self) -> torch.Tensor:
        """int64 [n]: the sequences' lengths before."""
        return self._plan[:self.n]

    @property
    def after(self) -> torch.Tensor:
        """int64 [n]: and with what is granted."""
        return self._plan[self.n:2 * self.n]

    @property
    def token_page(self) -> torch.Tensor:
        """int64 [T]: the packed tokens' pages, -1 where a row has none."""
        return self._plan[2 * self.n:2 * self.n + self.T]

    token_slot = token_page          # as the pool's adapters call it

    @property
    def token_pos(self) -> torch.Tensor:
        """int64 [T]: their places in the pages, or -1."""
        return self._plan[2 * self.n + self.T:2 * (self.n + self.T)]

    @property
    def positions(self) -> torch.Tensor:
        """int64 [T]: their positions in the sequences, or -1."""
        return self._plan[2 * (self.n + self.T):2 * self.n + 3 * self.T]

    @property
    def granted(self) -> torch.Tensor:
        """int32 [n]: tokens granted, counts[i] or 0."""
        ints = self._plan.view(torch.int32)
        at = 2 * (2 * self.n + (2 + self._axes) * self.T)
        return ints[at:at + self.n]

    def _current(self) -> None:
        if self._step != self.pool._step:
            raise RuntimeError("a later reservation, reordering or freeing of sequences may have given "
                               "these pages away")

    def write(self, k: torch.Tensor, v: torch.Tensor, layer_idx: int) -> None:
        """K/V rows [T, n_kv_heads, head_dim] of the packed tokens to their places."""
        pool = self.pool
        shape = (self.T, pool.n_kv_heads, pool.head_dim)
        if k.shape != shape or v.shape != shape:
            raise ValueError(f"k {tuple(k.shape)}, v {tuple(v.shape)}: expected {list(shape)}")
        if not k.dtype == v.dtype == pool.storage.dtype:
            raise TypeError(f"the pages are {pool.storage.dtype} (got {k.dtype}, {v.dtype})")
        self._current()
        require_here(pool.storage, k, v)
        if not self.T:
            return
        (k, ks), (v, vs) = _head_rows(k), _head_rows(v)
        call("omni_kv_write_rows", k.data_ptr(), ks, v.data_ptr(), vs,
             pool.k[layer_idx].data_ptr(), pool.v[layer_idx].data_ptr(), self._page, self._place,
             pool.num_pages, pool.page_size, pool.n_kv_heads * pool.head_dim, self.T, stream())

    def finish(self) -> None:
        """The granted tokens are part of their sequences: lengths move."""
        self._current()
        if self.rows is None:
            self.pool.lengths[:self.n].copy_(self.after)
        else:
            self.pool.lengths.index_copy_(0, self.rows, self.after)

    # ---- the adapters' protocol ------------------------------------------------------
    def _check_rows(self, qkv: torch.Tensor, heads: int, out: torch.Tensor | None = None) -> None:
        """Rows of a projection with the first ``heads`` heads, and a place for the attention's."""
        pool = self.pool
        width = heads * pool.head_dim
        if qkv.dim() != 2 or qkv.shape[0] != self.T or qkv.shape[1] < width or qkv.stride(1) != 1:
            raise ValueError(f"rows of shape {tuple(qkv.shape)}: expected [{self.T}, >= {width}] with "
                             f"contiguous columns")
        if qkv.dtype != pool.storage.dtype or (out is not None and out.dtype != qkv.dtype):
            raise TypeError(f"the pages are {pool.storage.dtype} (got {qkv.dtype}"
                            f"{'' if out is None else f' -> {out.dtype}'})")
        if out is not None and (out.numel() != self.T * width or not out.is_contiguous()):
            raise ValueError(f"attention output of shape {tuple(out.shape)}: expected a contiguous "
                             f"[{self.T}, {heads}, {pool.head_dim}]")

    def _check_heads(self, q: torch.Tensor) -> None:
        pool = self.pool
        if q.shape != (self.T, pool.n_heads, pool.head_dim) or q.dtype != pool.storage.dtype:
            raise ValueError(f"q {tuple(q.shape)} {q.dtype}: expected [{self.T}, {pool.n_heads}, "
                             f"{pool.head_dim}] {pool.storage.dtype}")
        require_here(pool.storage, q)

    def bind(self, T: int) -> None:
        if T != self.T:
            raise ValueError(f"the forward brings {T} tokens, the adapter was made for {self.T}")

    def rope_and_write(self, qkv: torch.Tensor, layer_idx: int, positions: torch.Tensor, cos_tab,
                       sin_tab, mrope_section, parts=None) -> None:
        """M-RoPE on q/k (in place in the qkv rows) and the K/V rows' write, as
        PackedPrefillWriter.rope_and_write."""
        pool = self.pool
        self._current()
        if pool.storage.dtype != torch.float16 or pool.head_dim != 128:
            raise ValueError("rotary embedding is for fp16 pages of head_dim 128")
        self._check_rows(qkv, pool.n_heads + 2 * pool.n_kv_heads)
        if positions.numel() != 3 * self.T or positions.dtype != torch.int64 or \
                not positions.is_contiguous():
            raise ValueError(f"positions {tuple(positions.shape)} {positions.dtype}: expected a "
                             f"contiguous int64 [3, {self.T}]")
        require_here(pool.storage, qkv, positions)
        if parts is None:
            fn, extra = "omni_mrope_kv_write", ()
        else:
            pbuf, S, bias, bar = parts
            fn, extra = "omni_mrope_kv_write_partials", (ptr(pbuf), S, ptr(bias), int(bar))
        call(fn, ptr(qkv), qkv.stride(0), *extra, ptr(positions), None, None, ptr(cos_tab),
             ptr(sin_tab), cos_tab.shape[0], pool.k[layer_idx].data_ptr(),
             pool.v[layer_idx].data_ptr(), self._page, self._place, pool.num_pages, pool.page_size,
             self.T, pool.n_heads, pool.n_kv_heads, pool.head_dim, *mrope_section, stream())


class PagedPrefill(PageSlots):
    """Packed prompts that become sequences ``rows`` (whatever those held is forgotten): causal
    attention within each.  It runs over a copy of the layer's K/V in rows of one prompt each, all as
    long as the longest, by the pool's prefill kernels.  A call that is refused leaves the rows as they
    were.  fp16, head_dim 128."""

    leaves_rows = False

    def __init__(self, pool: PagedKVCache, rows: Sequence[int], seg_lengths: Sequence[int]):
        if pool.storage.dtype != torch.float16 or pool.head_dim != 128:
            raise ValueError("prompts are for fp16 pages of head_dim 128")
        rows, seg = pool._checked_rows(rows), [int(L) for L in seg_lengths]
        if not seg or len(seg) != len(rows) or any(not 1 <= L <= pool.max_len for L in seg):
            raise ValueError(f"prompts of {seg} tokens for rows {rows}: 1 to {pool.max_len} each")
        if sum(seg) > MAX_TOKENS:
            raise ValueError(f"prompts of {sum(seg)} tokens: up to {MAX_TOKENS} in all")
        require_here(pool.storage)
        # all that may be refused before the rows' sequences are forgotten
        one = PreallocatedKVCache(1, len(seg), pool.n_kv_heads, max(seg), 128, pool.device,
                                  n_heads=pool.n_heads)
        self._prompt = one.packed_prefill_cache(range(len(seg)), seg)
        pool.free(rows)
        super().__init__(pool, seg, rows)

    def rope_and_write(self, qkv, layer_idx, positions, cos_tab, sin_tab, mrope_section,
                       parts=None) -> None:
        super().rope_and_write(qkv, layer_idx, positions, cos_tab, sin_tab, mrope_section, parts)
        nh, nkv = self.pool.n_heads, self.pool.n_kv_heads
        at = qkv.data_ptr() + 2 * nh * 128
        self._copy(at, qkv.stride(0), at + 2 * nkv * 128, qkv.stride(0))

    def _copy(self, k: int, k_stride: int, v: int, v_stride: int) -> None:
        w, one = self._prompt, self._prompt.pool
        call("omni_kv_write_rows", k, k_stride, v, v_stride, one.k[0].data_ptr(),
             one.v[0].data_ptr(), w.token_slot.data_ptr(), w.token_pos.data_ptr(), one.max_batch,
             one.max_len, one.n_kv_heads * 128, self.T, stream())

    def attend_qkv(self, qkv: torch.Tensor, layer_idx: int, scale: float,
                   out: torch.Tensor) -> torch.Tensor:
        """As PackedPrefillWriter.attend_qkv."""
        self._check_rows(qkv, self.pool.n_heads, out)
        require_here(self.pool.storage, qkv, out)
        return prefill_attention_pool(self._prompt, qkv, 0, scale, out)

    def flash_prefill(self, q, k, v, layer_idx, scale):
        """The adapters' protocol on rotated tensors: q [T, nh, hd], k / v [T, nkv, hd]; lengths on
        the last layer."""
        pool = self.pool
        self.bind(q.shape[0])
        self._check_heads(q)
        self.write(k, v, layer_idx)
        (k, ks), (v, vs) = _head_rows(k), _head_rows(v)
        self._copy(k.data_ptr(), ks, v.data_ptr(), vs)
        q = q.contiguous()
        out = torch.empty_like(q)
        prefill_attention_pool(self._prompt, q, 0, scale, out, q_stride=q.shape[1] * q.shape[2])
        if layer_idx == pool.n_layers - 1:
            self.finish()
        return out


class PagedDecode(PageSlots):
    """One new token for each of sequences [0, n) (counts[i] less than one: none), row i of the
    forward the token of sequence i.  Rotary positions are length + rope_delta (int64 per sequence):
    ``positions`` [3, n].  A row attends to its sequence and itself; a row without a token, or without
    a page for it, gets zeros.

    The sequences' keys stand in one line that is cut into equal stretches for the attention's
    workgroups, so that one long sequence among short ones takes no longer than its share; the pages
    that the tables of neighbours begin with alike (beams of one prompt) stand there, and are read,
    once for a group of up to 32 queries a KV head.  What a group shares is the least that two neighbours
    in it do: keep rows that share most next to each other.  The split states are the adapter's own, one
    for all layers: its calls go to one stream at a time."""

    leaves_rows = False

    def __init__(self, pool: PagedKVCache, n: int, counts=None, rope_delta=None):
        if not 1 <= n <= pool.max_seqs:
            raise ValueError(f"{n} sequences, the cache has {pool.max_seqs}")
        self._columns, self._most, self._floats = pool._attention_plan(n)
        super().__init__(pool, counts, dense=True, n=n, rope_delta=rope_delta, columns=self._columns,
                         most=self._most, floats=self._floats)

    @property
    def positions(self) -> torch.Tensor:
        """int64 [3, n]: rotary positions, -1 for a row without a token."""
        return self._plan[4 * self.n:7 * self.n].view(3, self.n)

    def attend_qkv(self, qkv: torch.Tensor, layer_idx: int, scale: float,
                   out: torch.Tensor) -> torch.Tensor:
        """out [n, nh, hd] (contiguous): attention of the rows whose queries are the first nh * hd
        columns of the rows qkv; their K/V is in the pages (rope_and_write)."""
        pool = self.pool
        self._check_rows(qkv, pool.n_heads, out)
        self._current()
        require_here(pool.storage, qkv, out)
        width = pool.n_heads * pool.head_dim
        stride = qkv.stride(0) if self.n > 1 else width
        return self._attend(qkv.data_ptr(), stride, layer_idx, scale, out)

    def _attend(self, q: int, q_stride: int, layer_idx: int, scale: float, out):
        pool = self.pool
        nh, hd = pool.n_heads, pool.head_dim
        call("omni_paged_attention", q, q_stride, pool.k[layer_idx].data_ptr(),
             pool.v[layer_idx].data_ptr(), _DTYPES[pool.storage.dtype], pool.num_pages,
             pool.page_size, pool.tables.data_ptr(), pool.tables.shape[1], self.n, self._schedule,
             self._columns, self._most, out.data_ptr(), nh * hd, nh, pool.n_kv_heads, hd, float(scale),
             self._states, self._floats, stream())
        return out

    def flash_decode(self, q, key, value, layer_idx, scale):
        """The decode views' protocol on rotated tensors: q [n, nh, hd], key / value [n, nkv, hd].
        Writes the K/V rows, attends; lengths on the last layer."""
        pool = self.pool
        self._check_heads(q)
        self.write(key, value, layer_idx)
        q, qs = _head_rows(q)
        out = torch.empty(q.shape, device=q.device, dtype=q.dtype)
        self._attend(q.data_ptr(), qs, layer_idx, scale, out)
        if layer_idx == pool.n_layers - 1:
            self.finish()
        return out
