"""Model runners: the drop-in boundary the engine/scheduler call every iteration.

``ModelRunner`` (omniserve/runners/base.py:26-57) is the abstract interface;
``StubRunner`` (:60-91) the no-GPU control-plane double; ``MultimodalRunner``
(runners/multimodal.py:19-379) the model-agnostic runner over the preallocated KV
pool; ``NativeQwenVLRunner`` (runners/qwen_vl_native.py:14-20) keeps the
reference's entry-point name and constructor signature.

Decode (multimodal.py:286-357): sequences sorted by slot must occupy slots [0, n);
one step advances each by one token.  With ``use_graph=True`` the whole step -
embedding gather + 28 layers + final norm + lm_head/argmax + length advance - is one
HIP-graph replay per batch size (captured lazily, static buffers kept alive; a batch with
non-greedy rows replays a second graph that also writes the fp16 logits, from which the
host samples, multimodal.py:306-313, 342-357).  The
host does at most one small H2D (token ids, only when the batch composition
changed) and one D2H (the new ids) per step.  While the batch can go on unchanged
(nobody has finished, every row has room) the next step's replay is enqueued before the
current step is waited for - its input ids are the current step's outputs, left on the
device by the graph - so the GPU never waits for the host's per-step bookkeeping.  Any
other call on the runner (a different batch, prefill, free, chunked prefill) first takes
that step back with ``settle()``: its length advance is undone and the K/V row it wrote
lies past the valid length, to be overwritten.

Chunked prefill and mixed batching (multimodal.py:200-284): a long text prompt is
prefilled chunk by chunk into the reserve slot (pool row ``max_running``), each chunk
attending to the chunks before it; ``mixed_step`` runs the running sequences' decode
tokens and one chunk in a single forward.  After the last chunk the prompt's KV prefix
is copied into the next decode slot.

Speculative decoding: ``speculate`` takes a drafted tree of tokens per running sequence (from
any draft: prompt lookup, extra heads, a smaller model), scores all of them in one forward and
advances every sequence by the drafted tokens that stand and one more.

Beam search: ``beam_search`` finds the best continuations of prompts, in a paged cache beside the
pool.
"""

from __future__ import annotations

import abc
from typing import Dict, List, NamedTuple

import numpy as np
import torch

from .beam import MAX_BEAMS, select
from .hostio import to_device
from .kv_cache import PreallocatedKVCache
from .linear import weights_epoch
from .paged_kv import MAX_SEQS, PAGE_SIZES, PagedKVCache
from .request import Sequence, Status
from .speculative import MAX_NODES, verify


class Beam(NamedTuple):
    """A continuation that beam search has found."""
    tokens: List[int]      # with its stop token, if it ended with one
    logprob: float         # sum of the tokens' log-probabilities
    score: float           # logprob / len(tokens) ** length_penalty


def _beams_of(tokens, parents, scores, length_penalty: float) -> List[List[Beam]]:
    """Each request's beams, the best first, from every step's choices [t][request][beam]."""
    out = []
    for s, row in enumerate(scores):
        found = []
        for w, logprob in enumerate(row):
            if logprob == -float("inf"):
                continue
            line, b = [], w
            for t in range(len(tokens) - 1, -1, -1):
                line.append(tokens[t][s][b])
                b = parents[t][s][b]
            line = [x for x in reversed(line) if x >= 0]          # a finished beam goes on with -1
            found.append(Beam(line, logprob, logprob / len(line) ** length_penalty))
        found.sort(key=lambda b: -b.score)
        out.append(found)
    return out


class ModelRunner(abc.ABC):
    @abc.abstractmethod
    def tokenize(self, seq: Sequence) -> None:
        """Fill seq.prompt_token_ids from the request prompt."""

    @abc.abstractmethod
    def prefill(self, seqs: List[Sequence]) -> None:
        """Prefill each sequence's prompt; append the first generated token."""

    @abc.abstractmethod
    def decode(self, seqs: List[Sequence]) -> None:
        """Advance every running sequence by exactly one token."""

    def chunk_prefill(self, seq: Sequence) -> None:
        raise NotImplementedError("this runner does not support chunked prefill")

    def mixed_step(self, chunk_seq: Sequence, decode_seqs: List[Sequence]) -> None:
        self.chunk_prefill(chunk_seq)
        self.decode(decode_seqs)

    @abc.abstractmethod
    def detokenize(self, seq: Sequence, new_token_ids: List[int]) -> str:
        """Render new token ids as text for streaming."""

    def free(self, seq: Sequence) -> None:
        """Release a finished sequence's resources (default: nothing)."""


class StubRunner(ModelRunner):
    """Deterministic no-GPU runner for exercising a scheduler/engine."""

    def __init__(self, reply: str = "ok " * 8):
        self._reply_tokens = reply.split()

    def tokenize(self, seq: Sequence) -> None:
        p = seq.request.prompt
        n = len(p.split()) if isinstance(p, str) else len(p)
        seq.prompt_token_ids = list(range(max(1, n)))

    def prefill(self, seqs: List[Sequence]) -> None:
        for seq in seqs:
            seq.kv_handle = {"len": seq.num_prompt_tokens}
            seq.append_token(0)
            seq.maybe_finish()

    def decode(self, seqs: List[Sequence]) -> None:
        for seq in seqs:
            seq.append_token(seq.num_output_tokens)
            seq.kv_handle["len"] += 1
            seq.maybe_finish()

    def detokenize(self, seq: Sequence, new_token_ids: List[int]) -> str:
        return " ".join(self._reply_tokens[t % len(self._reply_tokens)] for t in new_token_ids) + " "


class MultimodalRunner(ModelRunner):
    def __init__(self, adapter, max_running: int = 32, max_len: int = 1024, prefix_cache=None,
                 use_graph: bool = False):
        if prefix_cache is not None:
            raise NotImplementedError("prefix caching is not part of this build")
        self.adapter = adapter
        self.device = adapter.device
        self.max_running = max_running
        self.image_token_id = adapter.image_token_id
        self.eos_ids = adapter.eos_ids
        self._use_graph = use_graph
        self._reserve_slot = max_running       # kept for layout parity (multimodal.py:32-37)
        self._pool = PreallocatedKVCache(
            n_layers=adapter.num_layers, max_batch=max_running + 1,
            n_kv_heads=adapter.num_kv_heads, max_len=max_len, head_dim=adapter.head_dim,
            device=self.device, dtype=torch.float16, n_heads=adapter.num_heads)
        self._rope_delta = torch.zeros(max_running + 1, dtype=torch.int64, device=self.device)
        self._slot_seq: List[Sequence] = []
        self._kv_len: List[int] = []          # host mirror of pool.lengths for active slots
        self._graphs: Dict[int, tuple] = {}
        self._prefill_graphs: Dict[tuple, dict] = {}
        self._prefill_epoch = weights_epoch()
        self._graphs_sampled: Dict[int, tuple] = {}
        self._spec_graphs: Dict[tuple, dict] = {}
        self._eager: Dict[int, dict] = {}
        self._dev_ids_for = None              # batch whose next ids already sit on device
        self._pinned_ids = torch.zeros(max_running + 1, dtype=torch.int64).pin_memory()
        # new ids come back through two pinned buffers (the step being collected and the
        # one enqueued ahead of it), each with its event
        self._pinned_out = [torch.zeros(max_running + 1, dtype=torch.int64).pin_memory()
                            for _ in range(2)]
        self._out_ready = [torch.cuda.Event() for _ in range(2)] if torch.cuda.is_available() else None
        self._pin_next = 0
        self._ahead = None                    # (batch key, n, buffer) of a step enqueued ahead

    @property
    def pool(self) -> PreallocatedKVCache:
        return self._pool

    # ---- ModelRunner interface -----------------------------------------------------
    def tokenize(self, seq: Sequence) -> None:
        if not seq.prompt_token_ids:
            seq.prompt_token_ids = self.adapter.encode_prompt(seq.request.prompt)
        sp = seq.request.sampling
        for e in self.eos_ids:
            if e not in sp.stop_token_ids:
                sp.stop_token_ids.append(e)

    # ---- the decode step enqueued ahead --------------------------------------------
    def steps_ahead(self) -> int:
        """1 while a decode step for the last batch has been enqueued ahead of the caller."""
        return 0 if self._ahead is None else 1

    def settle(self) -> None:
        """Take back a decode step enqueued ahead: undo its length advance and drop its
        ids (its K/V rows sit at the first position past each valid length)."""
        if self._ahead is None:
            return
        _, n, _ = self._ahead
        self._ahead = None
        self._pool.lengths[:n] -= 1
        self._dev_ids_for = None

    def _pack_prompts(self, seqs: List[Sequence]):
        """(embeddings [1, T, H], positions [3, 1, T], prompt lengths, rope deltas, the deltas on
        the device) of the sequences' prompts, one after another."""
        dev = self.device
        # The packed prompt's host-side inputs are gathered as numpy arrays and uploaded in
        # one pinned copy (ids, image row indices, positions, rope deltas): the GPU is idle
        # until the host has issued them, so per-token Python work and per-input uploads
        # would add to every prefill's latency.
        ids_l, pos_l, seg_lens, deltas, img_rows, vis = [], [], [], [], [], []
        T = 0
        for seq in seqs:
            if not seq.prompt_token_ids:
                self.tokenize(seq)
            ids = np.asarray(seq.prompt_token_ids, dtype=np.int64)
            L = int(ids.shape[0])
            if L == 0 or L >= self._pool.max_len:
                raise ValueError(f"prompt length {L} outside [1, max_len={self._pool.max_len})")
            images = seq.request.images
            grids = [im.grid for im in images] if images else None
            if images:
                # the image rows located on the host: a mask on the device would make the
                # host wait for the queue (its count, its nonzero rows)
                rows = np.flatnonzero(ids == self.image_token_id)
                v = self.adapter.vision_embed(images)
                if rows.shape[0] != v.shape[0]:
                    raise ValueError("image token count does not match the vision rows")
                img_rows.append(rows + T)
                vis.append(v)
            pos, delta = self.adapter.prefill_positions(ids, grids)
            ids_l.append(ids)
            pos_l.append(pos.numpy() if isinstance(pos, torch.Tensor) else np.asarray(pos))
            seg_lens.append(L)
            deltas.append(int(delta))
            T += L
        nr = sum(int(r.shape[0]) for r in img_rows)
        host = np.concatenate(ids_l + img_rows + [np.concatenate(pos_l, axis=1).reshape(-1),
                                                  np.asarray(deltas, dtype=np.int64)])
        up = to_device(torch.from_numpy(host), torch.int64, dev)
        emb = self.adapter.embed_tokens(up[:T])
        if img_rows:
            emb.index_copy_(0, up[T:T + nr], torch.cat(vis, 0).to(emb.dtype))
        packed = emb.unsqueeze(0)
        pos = up[T + nr:T + nr + 3 * T].view(3, 1, T)                           # [3, 1, T]
        return packed, pos, seg_lens, deltas, up[T + nr + 3 * T:]

    @torch.inference_mode()
    def prefill(self, seqs: List[Sequence]) -> None:
        """Packed prefill, compute branch (multimodal.py:116-144): every prompt in one
        forward, causal within its segment, K/V written to its slot, logits only at
        segment ends."""
        if not seqs:
            return
        self.settle()
        base = len(self._slot_seq)
        if base + len(seqs) > self.max_running:
            raise RuntimeError(f"KV pool full: {base} running + {len(seqs)} new > "
                               f"{self.max_running}")
        packed, pos, seg_lens, deltas, delta_rows = self._pack_prompts(seqs)
        slots = [base + i for i in range(len(seqs))]
        if self._use_graph and self.prefill_graph_layouts > 0:
            logits = self._prefill_graphed(packed, pos, slots, seg_lens)
        else:
            last = torch.tensor(seg_lens).cumsum(0) - 1
            cache = self._pool.packed_prefill_cache(slots, seg_lens)
            logits = self.adapter.llm(packed, pos, None, cache, logits_indices=last.tolist())[0]
        self._rope_delta[base:base + len(seqs)].copy_(delta_rows)
        toks = self._sample_rows(logits, seqs)
        for i, seq in enumerate(seqs):
            slot = slots[i]
            self._slot_seq.append(seq)
            self._kv_len.append(seg_lens[i])
            seq.kv_handle = {"slot": slot, "rope_delta": deltas[i]}
            seq.append_token(toks[i])
            seq.maybe_finish()
        self._dev_ids_for = None

    # Packed prefills run as HIP graphs keyed by their segment lengths (with use_graph): the
    # first prefill of a layout runs eagerly on the layout's static input buffers and is then
    # captured; a later prefill of the same layout copies its embeddings, positions and slots
    # into those buffers and replays.  Token positions, query blocks and new lengths depend
    # only on the layout; the slot of every token is rewritten on the device before a replay.
    # Up to this many layouts are kept (least recently used dropped); 0 disables.
    prefill_graph_layouts = 4

    def drop_prefill_graphs(self) -> None:
        """Forget the captured prefill graphs.  They launch on the device addresses of the
        weights they were captured with, so call this after replacing weight tensors (a
        GPTQ linear's release_f16 is noticed by itself: see _prefill_graphed)."""
        self._prefill_graphs.clear()
        self._spec_graphs.clear()

    def _prefill_graphed(self, packed, pos, slots, seg_lens):
        key = tuple(int(L) for L in seg_lens)
        graphs = self._prefill_graphs
        epoch = weights_epoch()
        if epoch != self._prefill_epoch:         # a resident fp16 expansion was released
            self.drop_prefill_graphs()
            self._prefill_epoch = epoch
        ent = graphs.pop(key, None)
        dev = self.device
        if ent is not None:
            graphs[key] = ent                                     # most recently used last
            ent["x"].copy_(packed)
            ent["pos"].copy_(pos)
            if ent["slots"] != slots:
                writer = ent["writer"]
                tok = [s for s, L in zip(slots, key) for _ in range(L)]
                new = to_device(tok + list(slots), torch.int64, dev)
                writer.token_slot.copy_(new[:len(tok)])
                writer._fin_slots.copy_(new[len(tok):])
                writer.slots = list(slots)
                ent["slots"] = list(slots)
            ent["graph"].replay()
            self._pool._active = max(self._pool._active, max(slots) + 1)
            return ent["out"]
        # first prefill of this layout: run it on static buffers, then capture (outside
        # inference mode, as the decode graphs are: a capture made inside it would leave the
        # generator's graph state as inference tensors that later captures cannot update)
        with torch.inference_mode(False):
            last = torch.tensor(key).cumsum(0) - 1
            ent = {"x": packed.clone(), "pos": pos.clone(), "slots": list(slots),
                   "idx": to_device(last, torch.int64, dev),
                   "writer": self._pool.packed_prefill_cache(slots, list(key))}
            run = lambda: self.adapter.llm(ent["x"], ent["pos"], None, ent["writer"],
                                           logits_indices=ent["idx"])[0]
            logits = run().clone()
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g):
                ent["out"] = run()
            ent["graph"] = g
        graphs[key] = ent
        while len(graphs) > self.prefill_graph_layouts:
            graphs.pop(next(iter(graphs)))
        return logits

    def attach_prefilled(self, seqs: List[Sequence], lengths: List[int],
                         rope_deltas: List[int] | None = None) -> List[int]:
        """Seat sequences whose KV prefix the caller already wrote into the pool (the
        set_slot_prefix contract, cache/kv_prealloc.py:43-49): each takes the next slot
        with lengths[slot] = L and decodes from there.  Returns the slots."""
        self.settle()
        base = len(self._slot_seq)
        if base + len(seqs) > self.max_running:
            raise RuntimeError("KV pool full")
        slots = []
        for i, (seq, L) in enumerate(zip(seqs, lengths)):
            if not 0 < L < self._pool.max_len:
                raise ValueError(f"length {L} outside (0, max_len)")
            slot = base + i
            d = 0 if rope_deltas is None else int(rope_deltas[i])
            self._pool.lengths[slot] = L
            self._rope_delta[slot] = d
            self._slot_seq.append(seq)
            self._kv_len.append(int(L))
            seq.kv_handle = {"slot": slot, "rope_delta": d}
            slots.append(slot)
        self._dev_ids_for = None
        return slots

    # ---- chunked prefill / mixed batching (multimodal.py:200-284) -------------------
    def _chunk_bounds(self, seq: Sequence):
        self.settle()
        if not seq.prompt_token_ids:
            self.tokenize(seq)
        P = len(seq.prompt_token_ids)
        start, L = seq.num_prefilled, seq.prefill_chunk
        if P == 0 or P >= self._pool.max_len:
            raise ValueError(f"prompt length {P} outside [1, max_len={self._pool.max_len})")
        if L < 1 or start < 0 or start + L > P:
            raise ValueError(f"chunk [{start}, {start + L}) outside the {P}-token prompt")
        if start == 0:
            # positions of the whole prompt once, sliced by later chunks (:212-216)
            if seq.request.images:
                raise AssertionError("chunked prefill supports text-only prompts (no images)")
            pos_full, delta = self.adapter.prefill_positions(seq.prompt_token_ids, None)
            seq.kv_handle = {"slot": self._reserve_slot, "rope_delta": int(delta),
                             "pos_full": pos_full}
        elif not seq.kv_handle or "pos_full" not in seq.kv_handle:
            raise ValueError("a later chunk of a prompt whose first chunk was not run")
        return start, L, start + L, P

    def _seat_prefilled(self, seq: Sequence, length: int, logits_row: torch.Tensor) -> None:
        """Last chunk done: move the reserve slot's KV into the decode region (valid prefix
        only) and emit the first token (:229-235)."""
        slot = len(self._slot_seq)
        if slot >= self.max_running:
            raise RuntimeError(f"KV pool full: {slot} running")
        delta = seq.kv_handle["rope_delta"]
        self._pool.copy_slot_kv(self._reserve_slot, slot, length)
        self._rope_delta[slot] = delta
        seq.kv_handle = {"slot": slot, "rope_delta": delta}
        self._slot_seq.append(seq)
        self._kv_len.append(length)
        seq.append_token(self._sample_rows(logits_row, [seq])[0])
        seq.maybe_finish()
        self._dev_ids_for = None

    def chunk_prefill(self, seq: Sequence) -> None:
        """One chunk [num_prefilled, num_prefilled + prefill_chunk) of a long text prompt
        (multimodal.py:200-235): appended to the reserve slot, attending to the chunks
        before it; after the last chunk the sequence joins the decode slots and emits its
        first token."""
        with torch.inference_mode():
            start, L, end, P = self._chunk_bounds(seq)
            dev = self.device
            ids = to_device(seq.prompt_token_ids[start:end], torch.int64, dev)
            emb = self.adapter.embed_tokens(ids).unsqueeze(0)                 # [1, L, H]
            pos = to_device(seq.kv_handle["pos_full"][:, start:end], torch.int64,
                            dev).unsqueeze(1)                                 # [3, 1, L]
            cache = self._pool.chunked_prefill_cache(self._reserve_slot, start)
            logits = self.adapter.llm(emb, pos, None, cache, logits_indices=[L - 1])[0]
            seq.num_prefilled = end
            if end == P:
                self._seat_prefilled(seq, end, logits[0:1])

    def mixed_step(self, chunk_seq: Sequence, decode_seqs: List[Sequence]) -> None:
        """Mixed batching (multimodal.py:237-284): the running sequences' decode tokens and
        one prefill chunk in a single forward - decode tokens first, the chunk after; each
        segment appends to its own slot and attends to its own KV."""
        with torch.inference_mode():
            decode_seqs = sorted(decode_seqs, key=lambda s: s.kv_handle["slot"])
            n = len(decode_seqs)
            if [s.kv_handle["slot"] for s in decode_seqs] != list(range(n)):
                raise AssertionError("mixed_step expects the running sequences in slots [0, n)")
            for b in range(n):
                if self._kv_len[b] >= self._pool.max_len:
                    raise RuntimeError(f"sequence in slot {b} reached max_len={self._pool.max_len}")
            start, L, end, P = self._chunk_bounds(chunk_seq)
            dev = self.device
            dec_len = [int(v) for v in self._kv_len[:n]]        # write positions = KV lengths
            ids = [s.last_token_id() for s in decode_seqs] + chunk_seq.prompt_token_ids[start:end]
            emb = self.adapter.embed_tokens(
                to_device(ids, torch.int64, dev)).unsqueeze(0)                   # [1, n+L, H]
            dec_pos = torch.tensor([dec_len[b] + int(s.kv_handle["rope_delta"])
                                    for b, s in enumerate(decode_seqs)], dtype=torch.int64)
            pos = torch.cat([dec_pos.view(1, n).expand(3, n),
                             chunk_seq.kv_handle["pos_full"][:, start:end].to(torch.int64)], 1)
            pos = to_device(pos, torch.int64, dev).unsqueeze(1)                   # [3, 1, n+L]
            cache = self._pool.mixed_cache(list(range(n)) + [self._reserve_slot],
                                           [1] * n + [L], dec_len + [start])
            final = end == P
            idx = list(range(n)) + ([n + L - 1] if final else [])
            logits = self.adapter.llm(emb, pos, None, cache, logits_indices=idx)[0]
            self._dev_ids_for = None
            if n:
                self._emit(decode_seqs, self._sample_rows(logits[:n], decode_seqs))
            chunk_seq.num_prefilled = end
            if final:
                self._seat_prefilled(chunk_seq, end, logits[n:n + 1])

    def decode(self, seqs: List[Sequence]) -> None:
        seqs = sorted(seqs, key=lambda s: s.kv_handle["slot"])
        n = len(seqs)
        if n == 0:
            return
        if [s.kv_handle["slot"] for s in seqs] != list(range(n)):
            raise AssertionError("decode expects the running sequences in slots [0, n)")
        for b in range(n):
            if self._kv_len[b] >= self._pool.max_len:
                raise RuntimeError(f"sequence in slot {b} reached max_len={self._pool.max_len}")
        greedy = all(s.request.sampling.greedy for s in seqs)
        fused = self.adapter.model.fused_decode_ready()
        if self._use_graph and fused:
            if greedy:
                self._decode_graph(seqs, n)
            else:
                self._decode_graph_sampled(seqs, n)
        else:
            self.settle()
            with torch.inference_mode():
                if fused:
                    self._decode_eager(seqs, n, greedy)
                else:
                    self._decode_forward(seqs, n)

    # ---- speculative decoding --------------------------------------------------------
    # Steps run as HIP graphs (with use_graph) keyed by the number of sequences, the nodes of a
    # tree and the kind of verification: up to this many are kept, each with its activations and
    # logits (0 disables).
    spec_graph_layouts = 4

    @torch.inference_mode()
    def speculate(self, seqs: List[Sequence], drafts, draft_logits=None) -> List[int]:
        """Advance every running sequence by the drafted tokens that stand and one more.

        ``drafts``: per sequence (in the order of ``seqs``) either a list of tokens to follow one
        another, or (tokens, parents) with each token's parent in that list (-1: the sequence's
        last token), parents first; at most 63.  ``draft_logits`` fp16 [n, D, V] on the device (D =
        the most tokens of a draft): row j of a sequence the logits its token j was drawn from, at
        the sequence's temperature, for chains alone; without them the tokens are proposals.  Greedy
        sequences keep the tokens that decode() would have produced, up to near ties (the forward
        over a tree rounds otherwise than decode's), sampled ones are distributed as its.
        Returns the number of tokens each sequence has gained (a stop token or the length limit
        ends a sequence early).  Where nothing is left to draw a sequence's next token from (all
        of its logits NaN or -inf) every other one advances as ever, that one by the drafted tokens
        that stand, and a RuntimeError names its slot."""
        self.settle()
        n = len(seqs)
        if len(drafts) != n:
            raise ValueError(f"{len(drafts)} drafts for {n} sequences")
        if n == 0:
            return []
        order = sorted(range(n), key=lambda i: seqs[i].kv_handle["slot"])
        if [seqs[i].kv_handle["slot"] for i in order] != list(range(n)):
            raise AssertionError("speculate expects the running sequences in slots [0, n)")
        trees = [self._draft_tree(drafts[i], draft_logits is not None) for i in order]
        T = 1 + max(len(t) for t, _ in trees)
        if T > MAX_NODES:
            raise ValueError(f"a draft of {T - 1} tokens: at most {MAX_NODES - 1}")
        vocab = self.adapter.model.cfg.vocab_size
        if draft_logits is not None and tuple(draft_logits.shape) != (n, T - 1, vocab):
            raise ValueError(f"draft_logits {tuple(draft_logits.shape)}: expected "
                             f"{(n, T - 1, vocab)}")
        if draft_logits is not None and draft_logits.dtype != torch.float16:
            # (rounded to the logits' type they would no longer be what the tokens were drawn from)
            raise TypeError(f"draft_logits are fp16, as the logits (got {draft_logits.dtype})")
        ids, parents, counts, temps = [], [], [], []
        for slot, i in enumerate(order):
            tokens, ups = trees[slot]
            if any(not 0 <= t < vocab for t in tokens):
                raise ValueError(f"drafted tokens {tokens}: outside the vocabulary of {vocab}")
            room = self._pool.max_len - self._kv_len[slot]
            if room < 1:
                raise RuntimeError(f"sequence in slot {slot} reached max_len={self._pool.max_len}")
            pad = T - 1 - len(tokens)
            # padding nodes are scored like others (no row of the forward is left undefined) and
            # never stand: counts ends before them, and before nodes that the pool cannot hold
            ids += [seqs[i].last_token_id()] + tokens + [0] * pad
            parents += [-1] + [p + 1 for p in ups] + [0] * pad
            counts.append(min(1 + len(tokens), room))
            temps.append(float(seqs[i].request.sampling.temperature))
        dev = self.device
        host = to_device(ids + parents + counts, torch.int64, dev)
        step = {"ids": host[:n * T].view(n, T),
                "parents": host[n * T:2 * n * T].view(n, T).to(torch.int32),
                "counts": host[2 * n * T:].to(torch.int32)}
        if any(t != 0.0 for t in temps):
            step["temps"] = to_device(temps, torch.float32, dev)
            step["uniforms"] = torch.rand(n, T, device=dev)
            if draft_logits is not None and T > 1:
                step["draft"] = draft_logits.index_select(0, to_device(order, torch.int64, dev))
        run = self._spec_graphed if self._use_graph and self.spec_graph_layouts else self._spec_step
        try:
            v = run(step)
            out = torch.cat([v.tokens, v.emitted.to(torch.int64).unsqueeze(1)], 1).tolist()
        except BaseException:
            # acceptance may have moved the lengths already (a capture behind the eager step that
            # fails): without its tokens the step has not been
            self._pool.lengths[:n].copy_(to_device(self._kv_len[:n], torch.int64, dev))
            raise
        self._dev_ids_for = None
        gained, dry = [0] * n, []
        for slot, i in enumerate(order):
            seq, new = seqs[i], out[slot][:out[slot][T]]
            if -1 in new:
                # nothing to draw the next token from: the sequence keeps the drafted tokens that
                # stand, the last of them still to be scored
                new = new[:new.index(-1)]
                dry.append(slot)
            self._kv_len[slot] += len(new)
            for t in new:
                seq.append_token(t)
                gained[i] += 1
                if seq.maybe_finish():
                    break
        if dry:
            self._pool.lengths[:n].copy_(to_device(self._kv_len[:n], torch.int64, dev))
            raise RuntimeError(f"no token is left to draw for the sequences in slots {dry} (the others "
                               f"have advanced)")
        return gained

    @staticmethod
    def _draft_tree(draft, chain: bool):
        """(tokens, parents within them) of a draft."""
        tokens, up = draft if isinstance(draft, tuple) else (draft, None)
        tokens = [int(t) for t in tokens]
        if up is None:
            return tokens, list(range(-1, len(tokens) - 1))
        up = [int(p) for p in up]
        if len(up) != len(tokens) or any(not -1 <= p < i for i, p in enumerate(up)):
            raise ValueError(f"parents {up} of {len(tokens)} drafted tokens: one each, before it")
        if chain and up != list(range(-1, len(tokens) - 1)):
            raise ValueError("draft_logits are for chains")
        return tokens, up

    def _spec_step(self, step: dict):
        """The step on device tensors: forward over the trees, verification, acceptance."""
        n, T = step["ids"].shape
        emb = self.adapter.embed_tokens(step["ids"].reshape(-1)).unsqueeze(0)
        cache = self._pool.tree_cache(step["parents"], rope_delta=self._rope_delta)
        logits = self.adapter.llm(emb, cache.positions.view(3, 1, n * T), None, cache)[0]
        tree = ({"draft_logits": step["draft"]} if "draft" in step
                else {"parents": step["parents"]})
        v = verify(logits.view(n, T, -1), step["ids"], step.get("uniforms"),
                   step.get("temps", 0.0), counts=step["counts"], **tree)
        cache.accept(v.path, v.emitted)
        return v

    def _spec_graphed(self, step: dict):
        """_spec_step as a graph per layout: the first call runs eagerly and is captured after."""
        epoch = weights_epoch()
        if epoch != self._prefill_epoch:
            self.drop_prefill_graphs()
            self._prefill_epoch = epoch
        key = (*step["ids"].shape, *sorted(step))
        ent = self._spec_graphs.pop(key, None)
        if ent is not None:
            self._spec_graphs[key] = ent                          # most recently used last
            for name, t in step.items():
                ent["in"][name].copy_(t)
            ent["graph"].replay()
            return ent["out"]
        with torch.inference_mode(False):
            ent = {"in": {name: t.clone() for name, t in step.items()}}
            v = self._spec_step(ent["in"])
            ent["graph"] = torch.cuda.CUDAGraph()
            with torch.cuda.graph(ent["graph"]):
                ent["out"] = self._spec_step(ent["in"])
        self._spec_graphs[key] = ent
        while len(self._spec_graphs) > self.spec_graph_layouts:
            self._spec_graphs.pop(next(iter(self._spec_graphs)))
        return v

    # ---- beam search -----------------------------------------------------------------
    @torch.inference_mode()
    def beam_search(self, seqs: List[Sequence], beams: int = 4, length_penalty: float = 1.0,
                    page_size: int = 32) -> List[List["Beam"]]:
        """The best continuations of each prompt, ``beams`` of them, the best first.

        Every step keeps the ``beams`` continuations of a request with the largest sums of
        log-probabilities, over all of its beams and the vocabulary (``beam.select``); a beam ends with
        one of the request's stop tokens, after max_new_tokens, or at the runner's max_len, and holds
        its place from then on.  They are ranked by sum / tokens ** length_penalty.  The sequences'
        prompts are read, nothing else of them is changed, and running sequences go on as ever: the
        beams live in a paged cache of their own, in which those of a request share its prompt's pages.
        With ``use_graph=True`` the steps of a call behind its first are one captured graph.  Cache and
        graph are made in every call.  28 layers of int4 weights: 1 x 4 beams behind 500 tokens 1.64 ms a
        step, 32 x 4 behind 400 3.76, behind 2000 4.09."""
        if not seqs:
            return []
        if not 1 <= beams <= MAX_BEAMS or len(seqs) * beams > MAX_SEQS:
            raise ValueError(f"{len(seqs)} x {beams} beams: 1 to {MAX_BEAMS} each, {MAX_SEQS} in all")
        if any(not s.request.sampling.greedy for s in seqs):
            raise ValueError("beam search draws nothing: temperature has to be 0")
        if page_size not in PAGE_SIZES:
            raise ValueError(f"pages of {page_size} tokens: one of {PAGE_SIZES}")
        self.settle()
        n, W, dev = len(seqs), beams, self.device
        packed, pos, lens, _, deltas = self._pack_prompts(seqs)
        limits = [min(max(s.request.sampling.max_new_tokens, 1), self._pool.max_len - L)
                  for s, L in zip(seqs, lens)]
        steps = max(limits)
        # whole pages of the prompts are shared; behind them every beam has its own
        held = lambda tokens: -(-tokens // page_size)
        own = W * (held(steps) + 1)
        pool = self._pool
        with torch.inference_mode(False):                         # (captured outside of it)
            cache = PagedKVCache(pool.n_layers, sum(held(L) + own for L in lens), pool.n_kv_heads,
                                 page_size, pool.head_dim, dev, max_seqs=n * W,
                                 max_len=max(lens) + steps, n_heads=pool.n_heads)
        last = torch.tensor(lens).cumsum(0) - 1
        logits = self.adapter.llm(packed, pos, None, cache.prefill_cache(range(0, n * W, W), lens),
                                  logits_indices=last.tolist())[0]
        stops = [list(s.request.sampling.stop_token_ids) for s in seqs]
        most = max(1, max(map(len, stops)))
        st = {"stop": to_device([t + [-1] * (most - len(t)) for t in stops], torch.int64, dev),
              "delta": deltas.repeat_interleave(W)}
        scores = torch.full((n, W), -float("inf"), device=dev)
        scores[:, 0] = 0.0                      # one beam to begin with
        first = select(logits.view(n, 1, -1).expand(n, W, -1), scores, stop=st["stop"], pad=-1)
        cache.reorder(first.parents)
        limit = to_device(limits, torch.int64, dev).unsqueeze(1)
        st.update(scores=first.scores, tokens=first.tokens, parents=first.parents,
                  done=first.done | (limit <= 1))
        tokens = torch.empty(steps, n, W, device=dev, dtype=torch.int64)
        parents = torch.empty(steps, n, W, device=dev, dtype=torch.int32)
        graph, t = None, 0
        while True:
            tokens[t].copy_(st["tokens"])
            parents[t].copy_(st["parents"])
            t += 1
            if t == steps or bool(st["done"].all()):
                break
            if graph is not None:
                graph.replay()
            else:
                self._beam_step(cache, st)
                if self._use_graph and t == 1 and steps > 4:
                    with torch.inference_mode(False):
                        st = {name: v.clone() for name, v in st.items()}
                        graph = torch.cuda.CUDAGraph()
                        with torch.cuda.graph(graph):
                            self._beam_step(cache, st)
            st["done"].logical_or_(limit <= t + 1)
        return _beams_of(tokens[:t].tolist(), parents[:t].tolist(), st["scores"].tolist(),
                         length_penalty)

    def _beam_step(self, cache: PagedKVCache, st: dict) -> None:
        """One token for every beam, on device tensors: forward, choice, the cache after it."""
        n, W = st["tokens"].shape
        emb = self.adapter.embed_tokens(st["tokens"].reshape(-1).clamp(min=0)).unsqueeze(0)
        step = cache.decode_cache(n * W, rope_delta=st["delta"])
        logits = self.adapter.llm(emb, step.positions.view(3, 1, n * W), None, step)[0]
        b = select(logits.view(n, W, -1), st["scores"], done=st["done"], stop=st["stop"], pad=-1)
        cache.reorder(b.parents)
        for name, v in zip(("scores", "parents", "tokens", "done"), b):
            st[name].copy_(v)

    # ---- decode paths ----------------------------------------------------------------
    def _load_ids(self, seqs, n, dst: torch.Tensor) -> None:
        key = tuple(id(s) for s in seqs)
        if self._dev_ids_for == key:
            return                      # dst already holds the last step's outputs
        for b, s in enumerate(seqs):
            self._pinned_ids[b] = s.last_token_id()
        dst.copy_(self._pinned_ids[:n], non_blocking=True)

    def _decode_eager(self, seqs, n, greedy: bool):
        model = self.adapter.model
        if n not in self._eager:
            self._eager[n] = {
                "ids": torch.zeros(n, dtype=torch.int64, device=self.device),
                "out": torch.zeros(n, dtype=torch.int64, device=self.device),
                "logits": torch.empty(n, model.cfg.vocab_size, device=self.device,
                                      dtype=torch.float16),
            }
        b = self._eager[n]
        self._dev_ids_for = None
        self._load_ids(seqs, n, b["ids"])
        view = self._pool.view(n, self._rope_delta)
        model.decode_greedy(b["ids"], view, b["out"], None if greedy else b["logits"],
                            lengths=self._pool.lengths)
        if greedy:
            self._emit(seqs, b["out"].tolist())
        else:
            self._emit(seqs, self._sample_rows(b["logits"], seqs))

    def _decode_forward(self, seqs, n):
        """Decode through the model's forward (multimodal.py:286-313, eager): for linears
        the fused step cannot run (FP8 W8A8 modules, an fp8_out norm), the reference's
        per-op route - one token per row appended at its length, logits, then sampling."""
        model = self.adapter.model
        self._dev_ids_for = None
        ids = to_device([s.last_token_id() for s in seqs], torch.int64, self.device)
        emb = model.embed_tokens(ids).unsqueeze(1)                       # [n, 1, H]
        view = self._pool.view(n, self._rope_delta)
        pos = self.adapter.decode_positions(self._pool.lengths[:n], self._rope_delta[:n])
        logits = self.adapter.llm(emb, pos, None, view)[:, -1, :]
        self._emit(seqs, self._sample_rows(logits, seqs))

    def _capture_graph(self, n, sampled: bool = False):
        """Capture the step for rows [0, n).  Greedy: the final launch advances lengths[:n]
        and leaves the new ids in bufs["ids"] as the next step's input.  ``sampled``: the
        step also writes the fp16 logits to bufs["logits"] (the host samples from them and
        loads the next ids itself)."""
        model = self.adapter.model
        bufs = {"ids": torch.zeros(n, dtype=torch.int64, device=self.device),
                "out": torch.zeros(n, dtype=torch.int64, device=self.device)}
        if sampled:
            bufs["logits"] = torch.empty(n, model.cfg.vocab_size, device=self.device,
                                         dtype=torch.float16)
        view = self._pool.view(n, self._rope_delta)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(3):   # warm-up: writes K/V at the (not yet valid) next position only
                model.decode_greedy(bufs["ids"], view, bufs["out"], bufs.get("logits"))
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            model.decode_greedy(bufs["ids"], view, bufs["out"], bufs.get("logits"),
                                next_ids=None if sampled else bufs["ids"],
                                lengths=self._pool.lengths)
        # the view and buffers are referenced by the graph: keep them alive with it
        (self._graphs_sampled if sampled else self._graphs)[n] = (g, bufs, view)

    def _decode_graph_sampled(self, seqs, n):
        """A batch with non-greedy rows in graph mode (multimodal.py:306-313, 342-357):
        replay the step graph that also captures the logits, then sample every row from
        them on the host side of the step (greedy rows take the argmax, as _sample_rows
        does for the eager paths)."""
        self.settle()
        if n not in self._graphs_sampled:
            self._capture_graph(n, sampled=True)
        g, bufs, _view = self._graphs_sampled[n]
        self._dev_ids_for = None               # the next ids come from the host
        self._load_ids(seqs, n, bufs["ids"])
        g.replay()
        self._emit(seqs, self._sample_rows(bufs["logits"], seqs))

    def _launch(self, n: int) -> int:
        """Replay the step graph for rows [0, n) (inputs: bufs["ids"]) and start the new
        ids' copy to a pinned buffer; returns the buffer index."""
        g, bufs, _view = self._graphs[n]
        g.replay()
        i = self._pin_next
        self._pin_next ^= 1
        self._pinned_out[i][:n].copy_(bufs["out"], non_blocking=True)
        self._out_ready[i].record()
        return i

    def _decode_graph(self, seqs, n):
        key = tuple(id(s) for s in seqs)
        if self._ahead is not None and self._ahead[0] == key:
            cur = self._ahead[2]               # enqueued by the previous call
            self._ahead = None
        else:
            self.settle()
            if n not in self._graphs:
                self._capture_graph(n)
            self._load_ids(seqs, n, self._graphs[n][1]["ids"])
            cur = self._launch(n)
        # The next step goes out before this one is waited for, when the batch will decode
        # again as is unless this step finishes someone (nobody has finished, every row has
        # room): its inputs are this step's ids, which the graph leaves on the device.  If
        # this step does finish a sequence, the caller's free() takes the next one back.
        if (all(s.status not in (Status.FINISHED, Status.ABORTED) for s in seqs)
                and all(self._kv_len[b] + 1 < self._pool.max_len for b in range(n))):
            self._ahead = (key, n, self._launch(n))
        self._out_ready[cur].synchronize()
        toks = self._pinned_out[cur][:n].tolist()
        self._emit(seqs, toks)
        self._dev_ids_for = key

    def _emit(self, seqs, toks):
        for b, seq in enumerate(seqs):
            self._kv_len[b] += 1
            seq.append_token(int(toks[b]))
            seq.maybe_finish()

    def _sample_rows(self, logits: torch.Tensor, seqs) -> List[int]:
        """Greedy = argmax of the fp16 logits (multimodal.py:374-377); else temperature
        sampling."""
        out = []
        greedy_rows = logits.argmax(-1).tolist()      # first maximum, as on the fp32 copy
        for i, seq in enumerate(seqs):
            sp = seq.request.sampling
            if sp.greedy:
                out.append(int(greedy_rows[i]))
            else:
                probs = torch.softmax(logits[i].float() / sp.temperature, dim=-1)
                out.append(int(torch.multinomial(probs, 1).item()))
        return out

    # ---- release ----------------------------------------------------------------------
    def free(self, seq: Sequence) -> None:
        """Swap-compact the pool (multimodal.py:359-369): the last slot's sequence moves
        into the freed slot; only its valid KV prefix is copied."""
        self.settle()
        h = seq.kv_handle or {}
        slot = h.get("slot")
        if slot is None:
            return
        last = len(self._slot_seq) - 1
        if slot != last:
            L = self._kv_len[last]
            self._pool.copy_slot_kv(last, slot, L)
            self._rope_delta[slot] = self._rope_delta[last]
            moved = self._slot_seq[last]
            moved.kv_handle["slot"] = slot
            self._slot_seq[slot] = moved
            self._kv_len[slot] = L
        self._slot_seq.pop()
        self._kv_len.pop()
        self._dev_ids_for = None

    def detokenize(self, seq: Sequence, new_token_ids: List[int]) -> str:
        return self.adapter.detokenize(new_token_ids)


class NativeQwenVLRunner(MultimodalRunner):
    """Entry point with the reference's constructor (runners/qwen_vl_native.py:14-20).
    Extra keyword arguments go to the adapter (weights=, seed=, num_layers=, ...)."""

    def __init__(self, model_dir: str = None, max_running: int = 32, max_len: int = 1024,
                 prefix_cache=None, quant: str = None, gptq_dir: str = None,
                 use_graph: bool = False, **adapter_kwargs):
        from .adapter import Qwen2VLAdapter
        adapter = Qwen2VLAdapter(model_dir=model_dir, quant=quant, gptq_dir=gptq_dir,
                                 max_pos=max(8192, 2 * max_len), **adapter_kwargs)
        super().__init__(adapter, max_running=max_running, max_len=max_len,
                         prefix_cache=prefix_cache, use_graph=use_graph)
