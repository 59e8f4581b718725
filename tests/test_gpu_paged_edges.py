"""The paged cache's operators and beam search where terms cancel, counts overflow, rows are many or have
no more room, and what a runner's own sequences keep of a search beside them."""

import math
import random

import pytest
import torch

from oracle import paged_ref as ref
from tests.test_gpu_paged import i32, make_cache, say

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
