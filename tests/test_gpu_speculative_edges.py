"""Speculative decoding on the GPU at its edges: attention maxima that grow from tile to tile, steps
that fail or have nothing to draw from, padded trees and FP8 linears, draws and tests on a border."""

import math
import random

import numpy as np
import pytest
import torch

from oracle import speculative_ref as ref
from tests.test_gpu_speculative import HD, check_verify, i32, say, trees

pytestmark = pytest.mark.gpu

LOG2E = 1.0 / math.log(2.0)

GROWING = [
    # n, T, start, capacity, the plan's (rows, groups), cut or not: two to four tiles a key group
    (2, 5, 490, 512, (32, 8, False)),
    (20, 33, 470, 512, (64, 4, False)),
    (32, 64, 448, 512, (128, 2, False)),
    (33, 2, 1500, 4096, (32, 8, True)),
    (32, 8, 2000, 4096, (64, 4, True)),
    (9, 40, 1800, 4096, (128, 2, True)),
]


def growing_pool(gpu, n, T, start, capacity):
    from omniserver_amd.kv_cache import PreallocatedKVCache
    pool = PreallocatedKVCache(1, n, 2, capacity, HD, gpu, n_heads=12)
    pool.storage.zero_()
    pool.lengths.fill_(start)
    g = torch.Generator().manual_seed(n + T + start)
    return pool, g, trees(random.Random(n + T), n, T, "tree")


@pytest.mark.parametrize("rise", [2.75, 6.1, 7.9, 8.1, 20.0])
@pytest.mark.parametrize("n,T,start,capacity,form", GROWING)
def test_tree_attention_growing_maximum(gpu, n, T, start, capacity, form, rise):
    """One key in 32 lies `rise` to 1.5 `rise` (row by row) powers of two above the one 32 before
    it, the others far below; every key of a (sequence, KV head) has the same V row, so each output
    is that row.

    Exactly: a row's largest probability rounds to 1; the next are some 2^-2.75, 2^-5.5, .. of it
    (k[0]'s own rounding moves a rise by 0.13 at most, where rises are small), 0.2 together, each off
    by at most 2^-11 of itself in fp16, 2^-13.3 of the sum.  A score of up to 2^11 in log2 units is
    off by 2^-13 at most against the sum's, in fp32, 2^-13.5 of the largest probability.  Together
    under 2^-12, half a step of any fp16 value at least."""
    say(f"growing maximum: n={n} T={T} start={start} capacity={capacity} rise={rise}")
    pool, g, parents = growing_pool(gpu, n, T, start, capacity)
    scale = HD ** -0.5
    # dims 0 and 1 carry the score: 16 (1 + r) k[0] - 64 k[1]
    steps = torch.arange(start, device=gpu) // 32
    on = torch.arange(start, device=gpu) % 32 == 5
    k = pool.k[0]
    k[:, :, :, 1] = 60.0                                  # off: far below
    k[:, :start, :, 1] = torch.where(on, 0.0, 60.0).half()[None, :, None]
    unit = rise / (16.0 * scale * LOG2E)
    k[:, :start, :, 0] = torch.where(on, steps * unit, torch.zeros(())).half()[None, :, None]
    v = torch.randn(n, 1, 2, HD, generator=g).half().to(gpu)
    pool.v[0].copy_(v.expand_as(pool.v[0]))
    q = torch.zeros(n, T, 12, HD)
    q[..., 0] = 16.0 * (1.0 + 0.5 * torch.rand(n, T, 12, generator=g))
    q[..., 1] = -64.0
    q = q.half().to(gpu)
    cache = pool.tree_cache(i32(parents, gpu))
    assert (*cache.form[:2], cache.form[3] > 0) == form
    out = torch.zeros(n * T, 12, HD, device=gpu, dtype=torch.float16)
    cache.attend_qkv(q.view(n * T, 12 * HD), 0, scale, out)
    want = v.repeat_interleave(6, 2).expand(n, T, 12, HD)
    off = (out.view(n, T, 12, HD) != want).sum().item()
    say(f"  {off} of {out.numel()} outputs differ")
    assert off == 0


@pytest.mark.parametrize("n,T,start,capacity,form", GROWING)
def test_tree_attention_wide_scores(gpu, n, T, start, capacity, form):
    """Scores of some 8 standard deviations, keys boosted late in the context for some sequences:
    maxima grow in most tiles, by less and by more than 2^8.  The bound is the oracle's and, twice
    (numerator and denominator), that of a score's fp32 products and sums: 128 roundings of at
    most sum |q k|."""
    say(f"wide scores: n={n} T={T} start={start} capacity={capacity}")
    pool, g, parents = growing_pool(gpu, n, T, start, capacity)
    scale = HD ** -0.5
    most = start + T
    pool.storage[:, :, :, :most] = torch.randn(1, 2, n, most, 2, HD, generator=g).half().to(gpu)
    pool.k[0][::2, start - 40:start - 20] *= 2.0
    q = (8 * torch.randn(n, T, 12, HD, generator=g)).half()
    few = sorted(random.Random(n).sample(range(n), min(n, 4)))
    cache = pool.tree_cache(i32(parents, gpu))
    assert (*cache.form[:2], cache.form[3] > 0) == form
    out = torch.zeros(n * T, 12, HD, device=gpu, dtype=torch.float16)
    cache.attend_qkv(q.to(gpu).view(n * T, 12 * HD), 0, scale, out)
    out = out.view(n, T, 12, HD)[few].cpu().double()
    assert out.isfinite().all()
    k, v = pool.k[0][few].cpu(), pool.v[0][few].cpu()
    want, mag, seen = ref.tree_attention(q[few], k, v, [start] * len(few), [parents[s] for s in few],
                                         [T] * len(few), list(range(len(few))), scale)
    products = (q[few].float().abs().view(len(few), T, 2, 6, HD).permute(0, 2, 1, 3, 4)
                .reshape(len(few), 2, T * 6, HD)
                @ k[:, :most].float().abs().permute(0, 2, 3, 1).contiguous()).amax().item()
    score = 128 * 2.0 ** -24 * products * scale
    bound = ref.attention_bound(want, mag, seen, v.float().abs().max().item()) + 2 * score * mag
    worst = ((out - want).abs() / bound).max().item()
    say(f"  worst error {worst:.2f} of the bound")
    assert worst <= 1.0


# ----------------------------------------------------------------------------- the runner
def started(shape, w, prompts, **kw):
    from omniserver_amd.request import Request, SamplingParams, Sequence
    from omniserver_amd.runner import NativeQwenVLRunner
    r = NativeQwenVLRunner(max_running=len(prompts), max_len=128, weights=w, **kw)
    seqs = [Sequence(Request(prompt=list(p), sampling=SamplingParams(max_new_tokens=40)))
            for p in prompts]
    for s in seqs:
        r.tokenize(s)
    r.prefill(seqs)
    return r, seqs


def test_runner_speculate_others_go_on(gpu, monkeypatch):
    """The rows of one sequence NaN, at its last token or behind drafted ones that stand: it keeps
    those, the others gain what they gain without it, and all decode on from there."""
    from omniserver_amd import runner as runner_mod
    from omniserver_amd import synth
    shape = synth.DecoderShape()
    w = synth.fp16_decoder(shape, seed=9, num_layers=2)
    prompts = [synth.random_ids(L, shape.vocab_size, 9, f"o{L}").tolist() for L in (9, 21, 33)]
    r, seqs = started(shape, w, prompts)
    for _ in range(4):
        r.decode(seqs)
    drafts = [s.output_token_ids[1:4] for s in seqs]
    verify = runner_mod.verify

    def run(node):
        r, seqs = started(shape, w, prompts)
        first = seqs[1].output_token_ids[0]

        def tainted(logits, *a, **kw):
            logits[1, torch.arange(3), torch.tensor(drafts[1])] = 60000.0    # the draft stands
            if node is not None:
                logits[1, node:] = math.nan
            return verify(logits, *a, **kw)

        monkeypatch.setattr(runner_mod, "verify", tainted)
        if node is None:
            r.speculate(seqs, drafts)
        else:
            with pytest.raises(RuntimeError, match=r"\[1\]"):
                r.speculate(seqs, drafts)
            assert seqs[1].output_token_ids == [first] + drafts[1][:node]
        monkeypatch.setattr(runner_mod, "verify", verify)
        for _ in range(2):
            assert r._kv_len == [s.total_len - 1 for s in seqs]
            assert r.pool.lengths[:3].tolist() == r._kv_len
            r.decode(seqs)
        return [list(s.output_token_ids) for s in seqs]

    want = run(None)
    for node in (0, 1, 3):
        say(f"rows of one sequence NaN from node {node} on")
        got = run(node)
        assert got[0] == want[0] and got[2] == want[2]


def test_runner_speculate_capture_that_fails(gpu):
    """The first step of a layout runs, its capture fails: the call can be made again and gives
    what it gives without the failure."""
    from omniserver_amd import synth
    shape = synth.DecoderShape()
    w = synth.fp16_decoder(shape, seed=10, num_layers=1)
    prompts = [synth.random_ids(L, shape.vocab_size, 10, f"c{L}").tolist() for L in (9, 21)]
    results = []
    for fails in (False, True):
        r, seqs = started(shape, w, prompts, use_graph=True)
        if fails:
            real, calls = r._spec_step, []

            def step(s):
                calls.append(0)
                if len(calls) == 2:
                    raise MemoryError("no room for the graph")
                return real(s)

            r._spec_step = step
            before = r.pool.lengths.tolist()
            with pytest.raises(MemoryError):
                r.speculate(seqs, [[1, 2], [3]])
            assert r.pool.lengths.tolist() == before and r._kv_len == before[:2]
            assert [s.num_output_tokens for s in seqs] == [1, 1]
        for _ in range(3):
            r.speculate(seqs, [[1, 2], [3]])
            assert r.pool.lengths[:2].tolist() == r._kv_len == [s.total_len - 1 for s in seqs]
        results.append([list(s.output_token_ids) for s in seqs])
    assert results[0] == results[1]


def test_runner_speculate_draft_logits_of_another_type(gpu):
    """Refused alike before a layout's first step, between that and a replay, and after."""
    from omniserver_amd import synth
    shape = synth.DecoderShape()
    w = synth.fp16_decoder(shape, seed=10, num_layers=1)
    prompts = [synth.random_ids(L, shape.vocab_size, 10, f"c{L}").tolist() for L in (9, 21)]
    r, seqs = started(shape, w, prompts, use_graph=True)
    for s in seqs:
        s.request.sampling.temperature = 0.9
    draft = torch.randn(2, 2, shape.vocab_size, device=gpu)
    for _ in range(3):
        before = [list(s.output_token_ids) for s in seqs]
        for other in (draft, draft.bfloat16()):
            with pytest.raises(TypeError):
                r.speculate(seqs, [[1, 2], [3, 4]], draft_logits=other)
        assert [s.output_token_ids for s in seqs] == before
        r.speculate(seqs, [[1, 2], [3, 4]], draft_logits=draft.half())


@pytest.mark.parametrize("quant", ["fp16", "fp8"])
@pytest.mark.parametrize("n,T", [(3, 7), (9, 12)])
def test_model_over_padded_trees(gpu, monkeypatch, quant, n, T):
    """Padding nodes (counts=) take no part in what the others get: the used rows' logits do not
    depend on what fresh memory holds, also behind linears that take one scale from all rows."""
    from omniserver_amd import synth
    from omniserver_amd.kv_cache import PreallocatedKVCache
    from omniserver_amd.mixed_precision import apply_mixed
    from omniserver_amd.qwen2_llm import Qwen2LLM
    say(f"model over padded trees, {quant}, n={n} T={T}")
    shape = synth.DecoderShape()
    w = synth.fp16_decoder(shape, seed=12, num_layers=2)
    model = Qwen2LLM.from_fp16(w, shape, gpu, max_pos=512)
    if quant == "fp8":
        apply_mixed(model, {"qkv": "fp8", "o": "fp8", "gate_up": "fp8", "down": "fp8"})
    rng = random.Random(n)
    parents = i32(trees(rng, n, T, "tree"), gpu)
    counts = i32([rng.randint(1, T - 1) for _ in range(n)], gpu)
    ids = synth.random_ids(n * T, shape.vocab_size, 12, "pad").to(gpu)
    pool = PreallocatedKVCache(2, n, 2, 128, HD, gpu, n_heads=12)
    prefix = torch.randn(pool.storage.shape, device=gpu).half()
    empty = torch.empty
    got = []
    for fill in (0.0, 3e4, math.nan):
        def filled(*a, **kw):
            t = empty(*a, **kw)
            return t.fill_(fill) if t.dtype in (torch.float16, torch.float32) and t.is_cuda else t

        pool.storage.copy_(prefix)
        pool.lengths.fill_(40)
        cache = pool.tree_cache(parents, counts=counts)
        monkeypatch.setattr(torch, "empty", filled)
        out = model(model.embed_tokens(ids).unsqueeze(0), cache.positions.view(3, 1, n * T), None,
                    cache)[0]
        monkeypatch.setattr(torch, "empty", empty)
        used = torch.arange(T, device=gpu) < counts[:, None]
        got.append(out.view(n, T, -1)[used])
    assert got[0].isfinite().all()
    assert torch.equal(got[0], got[1]) and torch.equal(got[0], got[2])


def test_runner_speculates_with_fp8_linears(gpu):
    """A decoder on FP8 linears, which decodes op by op: speculative steps, eager and as graphs,
    give the same tokens, and decode() goes on from there."""
    from omniserver_amd import synth
    from omniserver_amd.mixed_precision import apply_mixed
    say("runner speculates on FP8 linears")
    shape = synth.DecoderShape()
    w = synth.fp16_decoder(shape, seed=13, num_layers=2)
    prompts = [synth.random_ids(L, shape.vocab_size, 13, f"q{L}").tolist() for L in (19, 30)]
    streams = []
    for use_graph in (False, True):
        r, seqs = started(shape, w, prompts, use_graph=use_graph)
        apply_mixed(r.adapter.model, {"qkv": "fp8", "o": "fp8", "gate_up": "fp8", "down": "fp8"})
        r.drop_prefill_graphs()
        assert not r.adapter.model.fused_decode_ready()
        rng = random.Random(2)
        for _ in range(4):
            ids = [rng.randrange(shape.vocab_size) for _ in range(5)]
            r.speculate(seqs, [ids[:3], (ids[3:], [-1, -1])])
            r.decode(seqs)
            assert r.pool.lengths[:2].tolist() == r._kv_len == [s.total_len - 1 for s in seqs]
        streams.append([list(s.output_token_ids) for s in seqs])
    assert streams[0] == streams[1]


# ----------------------------------------------------------------------------- verification
def test_verify_draws_with_64_bit_weights(gpu):
    """Two tokens of weights 1 and w = exp(-x), random numbers 2e-14 to 4e-13 (relative) from the
    border 1 / (1 + w): what 64-bit weights draw.  Their roundings come to some 1e-15."""
    from omniserver_amd.speculative import verify
    rng = np.random.default_rng(3)
    rows, us, want = [], [], []
    for _ in range(8):
        x = rng.uniform(0.01, 3.0, 1 << 21).astype(np.float32)
        total = 1.0 + np.exp(-x.astype(np.float64))
        u = (1.0 / total).astype(np.float32)
        gap = u.astype(np.float64) * total - 1.0
        near = (np.abs(gap) > 2e-14) & (np.abs(gap) < 4e-13)
        rows.append(-x[near])
        us.append(u[near])
        want.append(gap[near] >= 0)
    x, u, want = (torch.from_numpy(np.concatenate(a)) for a in (rows, us, want))
    n = x.numel()
    say(f"{n} draws by the border")
    assert n > 100
    logits = torch.stack([torch.zeros(n), x], 1).view(n, 1, 2)
    got = verify(logits.to(gpu), torch.zeros(n, 1, dtype=torch.int64, device=gpu),
                 u.view(n, 1).to(gpu), 1.0)
    off = (got.tokens[:, 0].cpu() != want.long()).sum().item()
    say(f"  {off} differ")
    assert off == 0


@pytest.mark.parametrize("V,noise", [(9001, 1e-6), (40000, 1e-6), (40000, 3e-7), (40000, 1e-4),
                                     (40000, 0.0)])
def test_verify_draft_next_to_the_target(gpu, V, noise):
    """Drafts that are the target but for `noise` and one token of little mass that they overrate:
    max(p - q, 0) comes to some 10^-6 of p, and its terms' signs hang on the totals' ratio in 64
    bits.  The order of 64-bit sums moves a border by some 10^-10 of that total, one draw in 10^5."""
    from omniserver_amd.speculative import verify
    say(f"draft next to the target: V={V} noise={noise}")
    g = torch.Generator().manual_seed(5)
    m, draws = 24, 64
    target = torch.randn(m, V, generator=g) * 2
    target.scatter_add_(1, torch.randint(0, V, (m, 6), generator=g), torch.full((m, 6), 9.0))
    draft = target + noise * torch.randn(m, V, generator=g)
    p = torch.softmax(target.double(), -1)
    x = (p - 1e-8).abs().argmin(-1)
    draft[torch.arange(m), x] += 3.0
    us = (torch.arange(draws) + 0.5) / draws
    assert (0.9 * torch.softmax(draft.double(), -1)[torch.arange(m), x] > p[torch.arange(m), x]).all()
    want = []
    for t, d in zip(target, draft):
        left = (ref.weights(t, 1.0) - ref.weights(d, 1.0)).clamp(min=0.0)
        run = left.cumsum(0)
        want += torch.searchsorted(run, us.double() * run[-1], right=True).tolist()
    each = lambda y: y.to(gpu).repeat_interleave(draws, 0)  # noqa: E731
    u = torch.stack([us.repeat(m), torch.full((m * draws,), 0.9)], 1).to(gpu)
    tokens = torch.stack([torch.zeros_like(x), x], 1)
    got = verify(each(torch.stack([target, target], 1)), each(tokens), u, 1.0,
                 draft_logits=each(draft[:, None]))
    off = (got.tokens[:, 0].cpu() != torch.tensor(want)).sum().item()
    say(f"  {off} of {len(want)} draws differ")
    assert got.emitted.eq(1).all() and off == 0


def test_verify_open_tests_over_a_floor(gpu):
    """One token against 151935 that together weigh as much: all of the 32-bit sums' error is there,
    the same in every weight.  Random numbers on the test's border and beside it."""
    g = torch.Generator().manual_seed(6)
    n, V = 36, 151936
    temps = (0.3 + torch.rand(n, generator=g) * 1.2).tolist()
    temps = torch.tensor(temps, dtype=torch.float32)
    floor = -11.9 * temps[:, None, None] + 0.02 * torch.randn(n, 2, V, generator=g)
    floor[:, :, 777] = 0.01 * torch.randn(n, 2, generator=g)
    p = torch.softmax(floor[:, 0].double() / temps.double()[:, None], -1)[:, 777]
    assert 0.3 < p.min() and p.max() < 0.7
    near = p.float()
    step = torch.tensor([-1.0, 0.0, 1.0])[torch.arange(n) % 3]
    u = torch.rand(n, 2, generator=g)
    u[:, 1] = torch.where(step == 0, near, torch.nextafter(near, near + step))
    say("tests on a border over a floor of equal tokens")
    total = check_verify(gpu, floor, [[0, 777]] * n, u, temps.tolist(), parents=[[-1, 0]] * n)
    assert 0 < (total == 2).sum() < n


def test_verify_draft_next_to_the_target_replayed(gpu):
    """The draw that sums what is left anew, in a graph: every replay as the eager call, also with
    other numbers and ordinary drafts in between."""
    from omniserver_amd.speculative import verify
    g = torch.Generator().manual_seed(8)
    n, V = 16, 20011
    target = torch.randn(n, 2, V, generator=g) * 2
    near, far = (target[:, :1] + noise * torch.randn(n, 1, V, generator=g) for noise in (1e-6, 0.5))
    x = (torch.softmax(target[:, 0].double(), -1) - 1e-8).abs().argmin(-1)
    for d in (near, far):
        d[torch.arange(n), 0, x] = target[torch.arange(n), 0, x] + 3.0
    tokens = torch.stack([torch.zeros_like(x), x], 1).to(gpu)
    sets = [(d.to(gpu), torch.stack([torch.rand(n, generator=g), torch.full((n,), 0.97)], 1).to(gpu))
            for d in (near, far, near)]
    target = target.to(gpu)
    want = [[t.clone() for t in verify(target, tokens, u, 1.0, draft_logits=d)] for d, u in sets]
    draft, u = sets[0][0].clone(), sets[0][1].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = verify(target, tokens, u, 1.0, draft_logits=draft)
    for turn in range(3):
        for (d, uu), w in zip(sets, want):
            draft.copy_(d)
            u.copy_(uu)
            graph.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(out, w)), turn
            verify(target, tokens, uu, 1.0, draft_logits=d)
