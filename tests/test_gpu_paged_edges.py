"""The paged cache's operators and beam search where terms cancel, counts overflow, rows are many or have
no more room, and what a runner's own sequences keep of a search beside them."""

import math
import random

import pytest
import torch

from oracle import paged_ref as ref
from tests import test_gpu_paged as paged
from tests.test_gpu_paged import check_rows, fill_pages, i32, make_cache, say

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,parts", [(torch.float16, 2.0 ** -22), (torch.bfloat16, 2.0 ** -24)])
def test_decode_attention_cancelling_terms(gpu, dtype, parts):
    """Two keys of nearly the same weight and opposite V: the output is their weights' difference, which
    a weight held in fewer bits than fp32 would show."""
    say(f"paged attention of cancelling terms {dtype}")
    n, nh, nkv, hd = 64, 12, 2, 128
    rng, g = random.Random(4), torch.Generator().manual_seed(5)
    cache, tables, lengths = make_cache(gpu, [2] * n, 16, rng, nkv, nh, hd, 1, dtype, spare=1, max_len=16)
    # scores x + y 2^-13 and x + z 2^-13 of the two keys, exact in fp32, and 0 of the new one, the largest
    k, v = torch.zeros(n, 3, nkv, hd), torch.zeros(n, 3, nkv, hd)
    x = -0.25 - 0.5 * torch.rand(n, nkv, generator=g)
    k[:, 0, :, 0] = k[:, 1, :, 0] = x
    k[:, :2, :, 1] = torch.rand(n, 2, nkv, generator=g)
    v[:, 0], v[:, 1] = 1.0, -1.0
    q = torch.zeros(n, nh, hd)
    q[:, :, 0], q[:, :, 1] = 1.0, 2.0 ** -13
    k, v, q = k.to(dtype), v.to(dtype), q.to(dtype)
    for i, row in enumerate(tables):
        cache.storage[0, 0, row[0], :2] = k[i, :2].to(gpu)
        cache.storage[0, 1, row[0], :2] = v[i, :2].to(gpu)
    step = cache.decode_cache(n)
    step.write(k[:, 2].contiguous().to(gpu), v[:, 2].contiguous().to(gpu), 0)
    out = step.attend_qkv(q.view(n, -1).to(gpu), 0, 1.0, torch.empty(n, nh, hd, device=gpu, dtype=dtype))
    s = k[:, :, :, 0].double() + k[:, :, :, 1].double() * 2.0 ** -13          # [n, 3, nkv]
    p = torch.exp(s - s.amax(1, keepdim=True))
    L = p.sum(1)
    exact = ((p[:, 0] - p[:, 1]) / L).repeat_interleave(nh // nkv, 1)[..., None].expand(n, nh, hd)
    # a weight: its exponent, below 1.45, off by log2 e's rounding and the product's, 2^-24 of it each, ln 2 of
    # that relative; 2^-23 for the exponential; and the parts.  Six products added up, sums below 1, are off
    # by 2^-24 each.  All over L; then the output's rounding, and L's and its reciprocal's
    weight = 2 * 1.45 * math.log(2) * 2.0 ** -24 + 2.0 ** -23 + parts
    bound = (((p[:, 0] + p[:, 1]) * weight + 6 * 2.0 ** -24) / L).repeat_interleave(nh // nkv, 1)[..., None]
    low = 2.0 ** -25 if dtype == torch.float16 else 0.0
    bound = bound + exact.abs() * (torch.finfo(dtype).eps / 2 + 2.0 ** -20) + low
    err = ((out.cpu().double() - exact).abs() / bound).max().item()
    say(f"  worst error {err:.2f} of the bound")
    assert err <= 1.0


@pytest.mark.parametrize("rows,length", [(1, 60), (3, 3000), (1, 40000), (2, 65000)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_attention_small_weights(gpu, rows, length, dtype):
    """One key far above all others, whose weights are 2^-20 to 2^-35 of its own: they count with their V, however
    small a type's smallest number leaves them."""
    say(f"paged attention of small weights, {rows} x {length} {dtype}")
    page, nh, nkv, hd = 64, 4, 1, 64
    rng, g = random.Random(length), torch.Generator().manual_seed(length)
    cache, tables, lengths = make_cache(gpu, [length] * rows, page, rng, nkv, nh, hd, 1, dtype, spare=rows,
                                        max_len=length + 1, shared=rows)
    k = torch.zeros(rows, length, nkv, hd)
    # scores of whole sixteenths, exact; those of a shared page are the same rows'
    k[..., 0] = -14 - torch.randint(0, 160, (1, length, 1), generator=g) / 16.0
    k[:, 0] = 0.0
    v = torch.rand(1, length, nkv, hd, generator=g).expand(rows, -1, -1, -1).clone()
    v[:, 0] = 0.0
    k, v = k.to(dtype), v.to(dtype)
    for r, row in enumerate(tables):
        pages = torch.tensor(row[:ref.pages_of(length, page)], device=gpu)
        for i, x in enumerate((k, v)):
            full = torch.zeros(len(pages) * page, nkv, hd, dtype=dtype)
            full[:length] = x[r]
            cache.storage[0, i, pages] = full.view(-1, page, nkv, hd).to(gpu)
    q = torch.zeros(rows, nh, hd, dtype=dtype)
    q[..., 0] = 1.0
    new = torch.zeros(rows, nkv, hd, dtype=dtype)
    low = new.clone()
    low[..., 0] = -18.0
    step = cache.decode_cache(rows)
    step.write(low.to(gpu), (new + 1).to(gpu), 0)
    out = step.attend_qkv(q.view(rows, -1).to(gpu), 0, 1.0, torch.empty(rows, nh, hd, device=gpu, dtype=dtype)).cpu()
    for r in range(rows):
        want, mag = ref.attention(q[r], torch.cat([k[r], low[r:r + 1]]), torch.cat([v[r], new[r:r + 1] + 1]), 1.0)
        # the output's rounding; fp32 scores, sums and exponentials, 2^-13 of the weights; and a weight 2^-40 of
        # the largest away from what it is: fp16's step of 2^-24, halved, where the largest weight is 2^15
        bound = want.abs() * torch.finfo(dtype).eps / 2 + mag * 2.0 ** -13 + (length + 1) * 2.0 ** -40 + 2.0 ** -25
        err = ((out[r].double() - want).abs() / bound).max().item()
        say(f"  row {r}: output {float(want[0, 0]):.2e}, error {err:.2f} of the bound")
        assert err <= 1.0


@pytest.mark.parametrize("kind", ["packed", "rows", "dense"])
@pytest.mark.parametrize("n,tokens,where", [(3, 8, (0, 1)), (8, 64, (0, 1, 4, 5)), (8, 64, (2,)), (200, 1500, (60, 61, 62, 130)),
                                            (200, 4000, (3, 199)), (200, 4000, (150, 151, 152)),
                                            (1500, 5000, (1100, 1101, 1499)), (1500, 1500, (0, 63, 64, 1030))])
def test_reserve_counts_beyond_all_sums(gpu, n, tokens, where, kind):
    """Counts on the device that no sum in 32 bits holds: those requests and the ones behind them in the packed
    rows go without, whatever the sums, and no row behind them has a place."""
    say(f"reserve {n} requests, {tokens} rows, counts of 2^30 and more at {where} {kind}")
    rng = random.Random(n + tokens)
    lengths = [rng.randint(0, 60) for _ in range(n)]
    cache, tables, lengths = make_cache(gpu, lengths, 16, rng, spare=3 * n, max_len=128)
    counts = [rng.randint(0, 5) for _ in range(n)]
    counts[-1] = 15
    for j, i in enumerate(where):
        counts[i] = [(1 << 31) - 1, 1 << 30, (1 << 30) + 5][j % 3]
    rows = rng.sample(range(n), n) if kind == "rows" else list(range(n))
    tokens = n if kind == "dense" else tokens
    new_tables, granted, starts, after, slots = ref.reserve(tables, lengths, counts, rows, cache.num_pages, 16, 128,
                                                            tokens, kind == "dense")
    if kind == "dense":
        got = cache.decode_cache(n, i32(counts, gpu))
    else:
        got = cache.reserve(i32(counts, gpu), rows if kind == "rows" else None, tokens)
    assert got.granted.tolist() == granted
    assert got.starts.tolist() == starts and got.after.tolist() == after
    assert got.token_page.tolist() == [s[0] for s in slots]
    assert got.token_pos.tolist() == [s[1] for s in slots]
    positions = [s[2] for s in slots]
    assert got.positions.tolist() == ([positions] * 3 if kind == "dense" else positions)
    assert cache.tables.tolist() == new_tables


def test_lists_are_refused_in_captured_steps(gpu):
    """A captured upload would read its staging memory at every replay, when other values are there: lists
    are refused while a graph is captured, device tensors in their place are not."""
    from omniserver_amd.beam import select
    from omniserver_amd.hostio import to_device
    say("lists while a graph is captured")
    rng = random.Random(3)
    cache, tables, lengths = make_cache(gpu, [20, 7, 9, 3], 16, rng, spare=8, max_len=64)
    logits = torch.randn(2, 2, 50, generator=torch.Generator().manual_seed(1)).half().to(gpu)
    scores = torch.zeros(2, 2, device=gpu)
    listed = [lambda: cache.reserve([1, 1]), lambda: cache.reserve(i_counts, rows=[1, 0], tokens=2),
              lambda: cache.decode_cache(4, [1, 0, 1, 1]), lambda: cache.reorder([[0, 0], [1, 0]]),
              lambda: cache.free([1]), lambda: cache.prefill_cache([0], [5]),
              lambda: select(logits, scores, stop=[3]), lambda: to_device([1, 2], torch.int64, gpu)]
    i_counts, parents, stop = i32([1, 1], gpu), i32([[0, 0], [1, 0]], gpu), torch.tensor([3], device=gpu)
    select(logits, scores, stop=stop)
    keep = cache.tables.clone(), cache.lengths.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        for call in listed:
            with pytest.raises(RuntimeError, match="captured"):
                call()
        got = select(logits, scores, stop=stop)
        slots = cache.reserve(i_counts, tokens=2)
        cache.reorder(parents)
    assert torch.equal(cache.tables, keep[0]) and torch.equal(cache.lengths, keep[1])
    want = select(logits, scores, stop=[3])
    new_tables, granted, _, _, places = ref.reserve(tables, lengths, [1, 1], [0, 1], cache.num_pages, 16, 64, 2)
    for turn in range(3):
        cache.tables.copy_(keep[0])
        cache.lengths.copy_(keep[1])
        [to_device([90 + turn] * 8, torch.int64, gpu) for _ in range(4)]
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), turn
        assert slots.token_page.tolist() == [p[0] for p in places], turn
        after, m, _ = ref.reorder(new_tables, lengths, [[0, 0], [1, 0]], cache.num_pages, 16)
        assert cache.lengths.tolist() == m, turn
        for r in range(4):
            held = ref.pages_of(m[r], 16)
            assert cache.tables[r, :held].tolist() == after[r][:held], (turn, r)


def tables_cache(gpu, tables, lengths, pages, page, nkv, nh, hd, dtype, max_len):
    """A cache that holds these tables (lists as long as the rows' pages) and lengths."""
    from omniserver_amd.paged_kv import PagedKVCache
    cache = PagedKVCache(1, pages, nkv, page, hd, gpu, max_seqs=len(tables), max_len=max_len, dtype=dtype,
                         n_heads=nh)
    width = cache.tables.shape[1]
    cache.tables.copy_(torch.tensor([row + [0] * (width - len(row)) for row in tables], dtype=torch.int32))
    cache.lengths.copy_(torch.tensor(lengths))
    return cache


def common_prompt_rows(layout, page, order):
    """Tables and lengths of requests (own prompt, beams, new tokens) behind one common prompt."""
    system, requests = layout
    first = [order.pop() for _ in range(system // page)]
    tables, lengths = [], []
    for prompt, beams, new in requests:
        shared = first + [order.pop() for _ in range(prompt // page)]
        for w in range(beams):
            m = len(shared) * page + new + w
            tables.append(shared + [order.pop() for _ in range(ref.pages_of(m, page) - len(shared))])
            lengths.append(m)
    return tables, lengths


COMMON = [
    # (tokens of the common prompt, (a request's own prompt, beams, new tokens behind it)), heads
    (512, ((3500, 2, 3), (0, 1, 88), (3500, 2, 3)), 12, 2, 128),
    (512, tuple((900, 4, 5) for _ in range(6)), 12, 2, 128),
    (256, tuple((0, 3, 1 + 7 * i) for i in range(9)), 8, 1, 64),
    (1024, ((128, 5, 0), (2000, 1, 9), (0, 4, 127), (128, 16, 1)), 4, 2, 64),
]


@pytest.mark.parametrize("system,requests,nh,nkv,hd", COMMON)
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_attention_common_prompt(gpu, system, requests, nh, nkv, hd, dtype):
    """Requests that share a common prompt's pages, and each request's beams its own prompt's behind them: groups
    of rows go over the requests' borders.  And the same rows with copies of all pages to themselves."""
    say(f"shared pages: common prompt {system}, {len(requests)} requests, heads {nh}/{nkv} x {hd} {dtype}")
    page, rng, g = 32, random.Random(system + nh), torch.Generator().manual_seed(system)
    held = sum((system + p + 200) // page * b for p, b, _ in requests) + 8
    order = list(range(held))
    rng.shuffle(order)
    tables, lengths = common_prompt_rows((system, requests), page, order)
    n, max_len = len(tables), max(lengths) + 1
    cache = tables_cache(gpu, tables, lengths, held, page, nkv, nh, hd, dtype, max_len)
    host = fill_pages(cache, cache.tables.tolist(), lengths, g)
    own = list(range(sum(map(len, tables)) + n))
    rng.shuffle(own)
    apart = [[own.pop() for _ in row] for row in tables]
    alone = tables_cache(gpu, apart, lengths, len(own) + sum(map(len, tables)), page, nkv, nh, hd, dtype, max_len)
    for row, copy in zip(tables, apart):
        alone.storage[:, :, copy] = host[:, :, row].to(gpu)
    qkv = torch.randn(n, (nh + 2 * nkv) * hd, generator=g).to(dtype).to(gpu)
    q, k, v = qkv.view(n, nh + 2 * nkv, hd).split((nh, nkv, nkv), 1)
    for c in (cache, alone):
        step = c.decode_cache(n)
        step.write(k, v, 0)
        out = step.attend_qkv(qkv, 0, hd ** -0.5, torch.full((n, nh, hd), 7.0, device=gpu, dtype=dtype))
        check_rows(out, q, c.storage.cpu(), 0, c.tables.tolist(), [m + 1 for m in lengths], page, hd ** -0.5)


def test_decode_attention_many_rows(gpu):
    """More rows than the scheduling workgroup has threads, in groups, some over its turns' borders."""
    paged.test_decode_attention_shared(gpu, 260, 5, 300, (0, 40), 16, 6, 1, 64, torch.float16)


@pytest.mark.parametrize("rows,length", [(1, 40000), (2, 40001), (3, 65400)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decode_attention_many_states(gpu, rows, length, dtype):
    """More states of a row than the merge takes at once: one KV head and a sequence of more than 32768 tokens,
    alone, and several that share all whole pages."""
    say(f"{rows} rows of {length} tokens {dtype}")
    page, nh, nkv, hd = 64, 4, 1, 64
    shared = length // page
    order = list(range(shared + rows * 3))
    random.Random(length).shuffle(order)
    first = [order.pop() for _ in range(shared)]
    tables = [first + [order.pop() for _ in range(ref.pages_of(length, page) - shared)] for _ in range(rows)]
    cache = tables_cache(gpu, tables, [length] * rows, shared + rows * 3, page, nkv, nh, hd, dtype, length + 1)
    g = torch.Generator().manual_seed(length)
    fill_pages(cache, cache.tables.tolist(), [length] * rows, g)
    step = cache.decode_cache(rows)
    assert step._columns > 256
    qkv = (2 * torch.randn(rows, (nh + 2 * nkv) * hd, generator=g)).to(dtype).to(gpu)
    q, k, v = qkv.view(rows, nh + 2 * nkv, hd).split((nh, nkv, nkv), 1)
    step.write(k, v, 0)
    out = step.attend_qkv(qkv, 0, hd ** -0.5, torch.full((rows, nh, hd), 7.0, device=gpu, dtype=dtype))
    check_rows(out, q, cache.storage.cpu(), 0, cache.tables.tolist(), [length + 1] * rows, page, hd ** -0.5)


def test_select_stop_lists(gpu):
    """More stop tokens than a workgroup keeps at hand, the same for all requests or each its own; none."""
    from omniserver_amd.beam import select
    g = torch.Generator().manual_seed(6)
    n, W, V = 3, 3, 400
    logits = torch.randn(n, W, V, generator=g).half() * 3
    scores = -torch.rand(n, W, generator=g)
    stops = torch.stack([torch.randperm(V, generator=g)[:150] for _ in range(n)])
    for stop in ([], stops[0].tolist(), stops):
        want = ref.select(logits, scores, 8, None, stop.tolist() if torch.is_tensor(stop) else stop or None)
        got = select(logits.to(gpu), scores.to(gpu), 8, stop=stop.to(gpu) if torch.is_tensor(stop) else stop)
        for name, i in (("parents", 1), ("tokens", 2), ("done", 3)):
            assert getattr(got, name).tolist() == [[r[i] for r in q] for q in want], (name, len(stop))


# ----------------------------------------------------------------------------- the runner
def runner_of(shape, w, quant, use_graph, running=2):
    from omniserver_amd.runner import NativeQwenVLRunner
    return NativeQwenVLRunner(max_running=running, max_len=160, use_graph=use_graph, weights=w, quant=quant)


def sequence(prompt, steps, images=None):
    from omniserver_amd.request import Request, SamplingParams, Sequence
    return Sequence(Request(prompt=list(prompt), sampling=SamplingParams(max_new_tokens=steps), images=images))


@pytest.mark.parametrize("quant,use_graph", [(None, False), (None, True), ("gptq", False), ("gptq", True)])
def test_beam_search_leaves_running_sequences(gpu, quant, use_graph):
    """Two runners of the same weights decode the same sequences; one of them searches beams in between (with
    graphs behind a step that is enqueued ahead): the same tokens, lengths and K/V rows."""
    from omniserver_amd import synth
    say(f"beam search beside running sequences quant={quant} use_graph={use_graph}")
    shape = synth.DecoderShape()
    w = (synth.gptq_decoder if quant else synth.fp16_decoder)(shape, seed=7, num_layers=2)
    prompts = [synth.random_ids(L, shape.vocab_size, 7, f"p{L}").tolist() for L in (33, 50, 20)]
    runners = [runner_of(shape, w, quant, use_graph) for _ in range(2)]
    running = [[sequence(p, 60) for p in prompts[:2]] for _ in runners]
    for r, seqs in zip(runners, running):
        r.prefill(seqs)
    for turn in range(4):
        for i, (r, seqs) in enumerate(zip(runners, running)):
            for _ in range(3):
                r.decode(seqs)
            if i == 0 and turn < 3:
                assert len(r.beam_search([sequence(p, 7 + turn) for p in prompts[turn:]], beams=3,
                                         page_size=16)) == 3 - turn
    for r in runners:
        r.settle()
    torch.cuda.synchronize()
    assert [s.output_token_ids for s in running[0]] == [s.output_token_ids for s in running[1]]
    assert len(running[0][0].output_token_ids) == 13
    a, b = (r.pool for r in runners)
    lengths = a.lengths.tolist()
    assert lengths[:2] == [33 + 12, 50 + 12] and lengths[:2] == b.lengths.tolist()[:2]
    for slot in range(2):
        assert torch.equal(a.storage[:, :, slot, :lengths[slot]].view(torch.int16),
                           b.storage[:, :, slot, :lengths[slot]].view(torch.int16))


@pytest.mark.parametrize("quant,use_graph", [(None, True), ("gptq", False)])
def test_one_beam_is_the_greedy_stream(gpu, quant, use_graph):
    """One beam takes, at every step, the token that the oracle's logits behind the same tokens put first, wherever
    their margin is larger than what logits may be off."""
    from omniserver_amd import synth
    from tests.helpers import check_stream, oracle_from_fp16, oracle_from_gptq, oracle_stream_logits
    say(f"one beam quant={quant} use_graph={use_graph}")
    shape = synth.DecoderShape()
    w = (synth.gptq_decoder if quant else synth.fp16_decoder)(shape, seed=7, num_layers=2)
    orc = oracle_from_gptq(w, shape) if quant else oracle_from_fp16(w, shape)
    r = runner_of(shape, w, quant, use_graph)
    prompts = [synth.random_ids(L, shape.vocab_size, 7, f"p{L}").tolist() for L in (31, 12)]
    found = r.beam_search([sequence(p, 8) for p in prompts], beams=1)
    for p, (beam,) in zip(prompts, found):
        rows = torch.as_tensor(oracle_stream_logits(orc, p, beam.tokens, 256))
        # logits within 2e-2 of the oracle's: two of them within twice that of each other
        check_stream(beam.tokens, rows, 2 * 2e-2, 4, "beam")


def test_beam_search_with_images(gpu):
    """Prompts with images, whose rotary positions do not follow their lengths: every step's positions are those of
    the prompt's continuation, and the beams' log-probabilities those of one forward over prompt and beam."""
    from omniserver_amd import synth
    from omniserver_amd.kv_cache import PreallocatedKVCache
    from omniserver_amd.positions import IMAGE_TOKEN_ID, VISION_START_TOKEN_ID
    from omniserver_amd.request import VisionInput
    say("beam search with images")
    shape = synth.DecoderShape()
    r = runner_of(shape, synth.fp16_decoder(shape, seed=9, num_layers=2), None, False)
    images = [VisionInput(synth.randn16((16, shape.hidden_size), 1.0, 9, "img").to(gpu), (1, 8, 8))]
    prompts = [synth.random_ids(L, shape.vocab_size, 9, f"p{L}").tolist() for L in (45, 30)]
    prompts[0][10:27] = [VISION_START_TOKEN_ID] + [IMAGE_TOKEN_ID] * 16
    W, steps = 3, 6
    seqs = [sequence(prompts[0], steps, images), sequence(prompts[1], steps)]
    seen, llm = [], r.adapter.llm

    def watched(emb, pos, *rest, **kw):
        seen.append(pos.cpu())
        return llm(emb, pos, *rest, **kw)

    r.adapter.llm = watched
    try:
        found = r.beam_search(seqs, beams=W, page_size=16)
    finally:
        r.adapter.llm = llm
    assert len(seen) == steps
    deltas = [r.adapter.prefill_positions(torch.tensor(s.prompt_token_ids).numpy(),
                                          [im.grid for im in s.request.images] if s.request.images else None)[1]
              for s in seqs]
    assert int(deltas[0]) < 0 == int(deltas[1])
    for t, pos in enumerate(seen[1:]):
        want = [len(p) + t + int(d) for p, d in zip(prompts, deltas) for _ in range(W)]
        assert pos.view(3, -1).tolist() == [want] * 3, t
    for s, beams in zip(seqs, found):
        L = len(s.prompt_token_ids)
        for b in beams:
            line = sequence(list(s.prompt_token_ids) + b.tokens[:-1], 1, s.request.images)
            with torch.inference_mode():
                packed, pos, lens, _, _ = r._pack_prompts([line])
                pool = PreallocatedKVCache(2, 1, 2, lens[0], 128, gpu, n_heads=12)
                rows = llm(packed, pos, None, pool.packed_prefill_cache([0], lens),
                           logits_indices=list(range(L - 1, lens[0])))[0]
            lp = torch.log_softmax(rows.double(), -1).cpu()
            exact = sum(float(lp[i, t]) for i, t in enumerate(b.tokens))
            # two routes of the model, logits within 2e-2 each: log-probabilities within four times that
            assert abs(b.logprob - exact) <= 4 * 2e-2 * len(b.tokens)
