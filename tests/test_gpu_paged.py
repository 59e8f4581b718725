"""The paged cache's operators and beam search's choice on the GPU against plain forms in 64 bits:
room for new tokens, attention of one new token per sequence, beams that take over their parents'
pages, the best continuations."""

import math
import random

import pytest
import torch

from oracle import paged_ref as ref

pytestmark = pytest.mark.gpu


def say(msg):
    print(f"[gpu-test] {msg}", flush=True)


def i32(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def make_cache(gpu, lengths, page, rng, nkv=2, nh=12, hd=128, layers=1, dtype=torch.float16, spare=0,
               max_len=None, shared=1, seqs=None, room=0):
    """A cache whose sequences hold `lengths` tokens in pages anywhere; groups of `shared` rows hold
    their whole pages together.  Entries behind a sequence's length are anything at all."""
    from omniserver_amd.paged_kv import PagedKVCache
    seqs = len(lengths) if seqs is None else seqs
    lengths = list(lengths) + [0] * (seqs - len(lengths))
    held = sum(ref.pages_of(m, page) for m in lengths)
    pages = held + spare
    max_len = max(max(lengths) + room, 1) if max_len is None else max_len
    cache = PagedKVCache(layers, max(pages, 1), nkv, page, hd, gpu, max_seqs=seqs, max_len=max_len,
                         dtype=dtype, n_heads=nh)
    order = list(range(cache.num_pages))
    rng.shuffle(order)
    width = cache.tables.shape[1]
    tables = [[rng.choice([-1, -7, 1 << 30, rng.randrange(max(pages, 1))]) for _ in range(width)]
              for _ in range(seqs)]
    for r, m in enumerate(lengths):
        keep = 0
        if shared > 1 and r % shared and lengths[r - 1] == m:
            keep = m // page
            tables[r][:keep] = tables[r - 1][:keep]
        for j in range(keep, ref.pages_of(m, page)):
            tables[r][j] = order.pop()
    cache.tables.copy_(torch.tensor(tables, dtype=torch.int32))
    cache.lengths.copy_(torch.tensor(lengths))
    return cache, tables, lengths


RESERVE = [
    # sequences, asking, page, lengths, new tokens, spare pages, max_len
    (1, 1, 16, (0, 0), (1, 1), 1, 1),
    (1, 1, 16, (15, 15), (1, 1), 0, 16),
    (1, 1, 16, (16, 16), (1, 1), 0, 64),              # no page left
    (3, 3, 16, (0, 40), (1, 1), 3, 64),
    (5, 4, 32, (0, 100), (0, 70), 9, 256),
    (33, 33, 16, (0, 300), (-2, 3), 12, 400),
    (64, 60, 16, (0, 90), (0, 40), 60, 100),          # too few pages, some past max_len
    (100, 100, 256, (0, 2000), (1, 1), 20, 2048),
    (300, 300, 16, (0, 64), (0, 30), 200, 80),        # more token rows than one workgroup writes
    (1500, 1400, 16, (0, 50), (0, 2), 300, 64),       # more requests than a workgroup has threads
    (2, 2, 1024, (1000, 1030), (1, 3000), 5, 8192),
    (40, 40, 16, (2000, 4000), (1, 1), 40, 5000),
]


@pytest.mark.parametrize("seqs,n,page,span,new,spare,max_len", RESERVE)
@pytest.mark.parametrize("kind", ["packed", "rows", "dense"])
def test_reserve(gpu, seqs, n, page, span, new, spare, max_len, kind):
    say(f"reserve {n} of {seqs} sequences, pages of {page}, lengths {span}, new {new} {kind}")
    rng = random.Random(seqs * 31 + page)
    lengths = [rng.randint(*span) for _ in range(seqs)]
    cache, tables, lengths = make_cache(gpu, lengths, page, rng, spare=spare, max_len=max_len)
    counts = [rng.randint(*new) for _ in range(n)]
    rows = rng.sample(range(seqs), n) if kind == "rows" else list(range(n))
    tokens = n if kind == "dense" else sum(max(c, 0) for c in counts)
    if kind == "packed" and tokens > 8:
        tokens -= 3                                     # not enough rows for the last ones
    want = ref.reserve(tables, lengths, counts, rows, cache.num_pages, page, max_len, tokens,
                       kind == "dense")
    delta = torch.arange(seqs, device=gpu) * 7 if kind == "dense" else None
    for turn in range(2):                               # the second finds what the first has written
        if kind == "dense":
            got = cache.decode_cache(n, i32(counts, gpu), delta)
        else:
            got = cache.reserve(i32(counts, gpu), rows if kind == "rows" else None, tokens)
        new_tables, granted, starts, after, slots = want
        assert got.granted.tolist() == granted
        assert got.starts.tolist() == starts and got.after.tolist() == after
        assert got.token_page.tolist() == [s[0] for s in slots]
        assert got.token_pos.tolist() == [s[1] for s in slots]
        if kind == "dense":
            pos = [s[2] + 7 * i if s[2] >= 0 else -1 for i, s in enumerate(slots)]
            assert got.positions.tolist() == [pos] * 3
        else:
            assert got.positions.tolist() == [s[2] for s in slots]
        assert cache.tables.tolist() == new_tables
    assert cache.lengths.tolist() == lengths            # they move in finish
    got.finish()
    for r, m in zip(rows, after):
        lengths[r] = m
    assert cache.lengths.tolist() == lengths
    if kind == "rows":
        cache.free(rows[:2])
        for r in rows[:2]:
            lengths[r] = 0
        assert cache.lengths.tolist() == lengths


def fill_pages(cache, tables, lengths, g):
    """Random K/V where tokens are, NaN and infinities everywhere else; per sequence its K and V."""
    page, dev = cache.page_size, cache.storage.device
    cache.storage.fill_(math.nan)
    cache.storage[:, :, ::2] = math.inf
    content = torch.randn(cache.storage.shape, generator=g).to(cache.storage.dtype)
    host = cache.storage.cpu()
    for row, m in zip(tables, lengths):
        for j in range(ref.pages_of(m, page)):
            some = min(page, m - j * page)
            host[:, :, row[j], :some] = content[:, :, row[j], :some]
    cache.storage.copy_(host)
    return host


def tokens_of(host, layer, row, m, page):
    """K and V [m, nkv, hd] of a sequence."""
    pages = torch.tensor(row[:ref.pages_of(m, page)], dtype=torch.long)
    return tuple(host[layer, i][pages].reshape(-1, *host.shape[4:])[:m] for i in (0, 1))


def check_rows(out, q, host, layer, tables, keys, page, scale):
    """out [n, nh, hd] against the plain form over keys[i] tokens of table i."""
    worst = 0.0
    out = out.cpu()
    for i, m in enumerate(keys):
        if m == 0:
            assert (out[i] == 0).all(), f"row {i} has no keys"
            continue
        k, v = tokens_of(host, layer, tables[i], m, page)
        want, mag = ref.attention(q[i].cpu(), k, v, scale)
        bound = ref.attention_bound(want, mag, m, v.float().abs().max().item(), out.dtype)
        err = ((out[i].double() - want).abs() / bound).max().item()
        assert err <= 1.0, f"row {i} of {m} keys: {err:.2f} of the bound"
        worst = max(worst, err)
    say(f"  worst error {worst:.2f} of the bound")


ATTENTION = [
    # n, lengths, page, nh, nkv, hd, dtype, max_len
    (1, (0, 0), 16, 12, 2, 128, torch.float16, None),
    (2, (1, 15), 16, 12, 2, 128, torch.float16, None),
    (3, (16, 32), 32, 12, 2, 128, torch.float16, None),
    (4, (100, 130), 16, 12, 2, 128, torch.float16, None),
    (5, (120, 140), 64, 12, 2, 128, torch.bfloat16, None),
    (7, (0, 700), 16, 12, 2, 128, torch.float16, 4096),
    (3, (0, 300), 128, 16, 16, 64, torch.bfloat16, None),
    (4, (30, 400), 16, 8, 1, 64, torch.float16, 1000),
    (2, (500, 600), 256, 28, 4, 128, torch.float16, None),
    (3, (60, 70), 16, 40, 2, 128, torch.float16, None),       # 20 heads a KV head: two groups
    (2, (128, 130), 32, 64, 1, 64, torch.bfloat16, None),     # four
    (33, (0, 300), 16, 12, 2, 128, torch.float16, 8192),
    (1, (5000, 5000), 64, 12, 2, 128, torch.float16, None),   # every column a piece of one row
    (300, (0, 40), 16, 4, 2, 64, torch.float16, None),        # more rows than columns
    (6, (127, 129), 1024, 6, 1, 128, torch.float16, None),
    (9, (0, 1500), 16, 1, 1, 128, torch.bfloat16, 2000),
]


@pytest.mark.parametrize("n,span,page,nh,nkv,hd,dtype,max_len", ATTENTION)
def test_decode_attention(gpu, n, span, page, nh, nkv, hd, dtype, max_len):
    say(f"paged attention n={n} lengths {span} page {page} heads {nh}/{nkv} x {hd} {dtype}")
    rng = random.Random(n * 131 + page)
    lengths = [rng.randint(*span) for _ in range(n)]
    lengths[0], lengths[-1] = span[1], span[0]
    cache, tables, lengths = make_cache(gpu, lengths, page, rng, nkv, nh, hd, 2, dtype, spare=n,
                                        max_len=max_len or max(lengths) + 1)
    g = torch.Generator().manual_seed(n)
    fill_pages(cache, tables, lengths, g)
    counts = [1] * n if n < 4 else [int(rng.random() < 0.8) for _ in range(n)]
    step = cache.decode_cache(n, counts)
    tables = cache.tables.tolist()
    rows = torch.randn(n, (nh + 2 * nkv) * hd, generator=g).to(dtype).to(gpu)
    q, k, v = rows.view(n, nh + 2 * nkv, hd).split((nh, nkv, nkv), 1)
    step.write(k, v, 1)
    host = cache.storage.cpu()
    keys = [m + 1 if c else 0 for m, c in zip(lengths, counts)]
    for i, m in enumerate(keys):
        if m:
            assert torch.equal(host[1, 0, tables[i][(m - 1) // page], (m - 1) % page], k[i].cpu())
    out = torch.full((n, nh, hd), 7.0, device=gpu, dtype=dtype)
    assert step.attend_qkv(rows, 1, hd ** -0.5, out) is out
    check_rows(out, q, host, 1, tables, keys, page, hd ** -0.5)
    again = torch.full_like(out, 3.0)
    step.attend_qkv(rows, 1, hd ** -0.5, again)
    assert torch.equal(out, again)
    # the protocol on separate tensors: the same rows, lengths move with the last layer
    step = cache.decode_cache(n, i32(counts, gpu))
    assert torch.equal(step.flash_decode(q, k, v, 1, hd ** -0.5), out)
    assert cache.lengths.tolist() == [m + c for m, c in zip(lengths, counts)]


SHARED = [
    # requests, beams, prompt, own tokens, page, nh, nkv, hd, dtype
    (1, 4, 500, (1, 40), 16, 12, 2, 128, torch.float16),
    (3, 4, 1000, (1, 200), 32, 12, 2, 128, torch.float16),
    (2, 16, 700, (0, 30), 64, 12, 2, 128, torch.bfloat16),     # groups of five, the last of one
    (5, 3, 300, (0, 300), 16, 8, 1, 64, torch.float16),
    (2, 32, 400, (1, 9), 16, 4, 4, 128, torch.float16),        # 32 queries of 32 rows
    (4, 2, 2000, (1, 20), 128, 16, 1, 128, torch.float16),     # two rows of sixteen heads
    (2, 4, 600, (1, 20), 16, 34, 2, 64, torch.bfloat16),       # seventeen heads: none together
    (40, 5, 260, (0, 300), 16, 6, 1, 64, torch.float16),
]


@pytest.mark.parametrize("n,W,prompt,own,page,nh,nkv,hd,dtype", SHARED)
def test_decode_attention_shared(gpu, n, W, prompt, own, page, nh, nkv, hd, dtype):
    """Beams that hold their prompt's pages together, some requests' prompts almost all of it, others
    hardly any, some rows idle; and what a row gets does not depend on its neighbours."""
    from omniserver_amd.paged_kv import PagedKVCache
    say(f"shared pages: {n} x {W} beams, prompt {prompt}, heads {nh}/{nkv} x {hd} {dtype}")
    rng = random.Random(n * 17 + W)
    rows, g = n * W, torch.Generator().manual_seed(prompt)
    most = prompt + own[1] + 2
    pages = rows * ref.pages_of(most, page) + 4
    cache = PagedKVCache(1, pages, nkv, page, hd, gpu, max_seqs=rows, max_len=most, dtype=dtype,
                         n_heads=nh)
    order = list(range(pages))
    rng.shuffle(order)
    tables, lengths = [], []
    for s in range(n):
        shared = prompt // rng.choice([1, 1, 1, 3]) // page
        common = [order.pop() for _ in range(shared)]
        for w in range(W):
            m = max(0, prompt + rng.randint(*own) - (prompt if rng.random() < 0.05 else 0))
            held = ref.pages_of(m, page)
            keep = common[:min(held, shared) if held > shared or m % page == 0 else max(held - 1, 0)]
            row = keep + [order.pop() for _ in range(held - len(keep))]
            tables.append(row + [0] * (cache.tables.shape[1] - held))
            lengths.append(m)
    cache.tables.copy_(torch.tensor(tables, dtype=torch.int32))
    cache.lengths.copy_(torch.tensor(lengths))
    fill_pages(cache, tables, lengths, g)
    counts = [int(rng.random() < 0.95) for _ in range(rows)]
    step = cache.decode_cache(rows, counts)
    tables = cache.tables.tolist()
    qkv = torch.randn(rows, (nh + 2 * nkv) * hd, generator=g).to(dtype).to(gpu)
    q, k, v = qkv.view(rows, nh + 2 * nkv, hd).split((nh, nkv, nkv), 1)
    step.write(k, v, 0)
    out = torch.full((rows, nh, hd), 7.0, device=gpu, dtype=dtype)
    step.attend_qkv(qkv, 0, hd ** -0.5, out)
    keys = [m + 1 if c else 0 for m, c in zip(lengths, counts)]
    check_rows(out, q, cache.storage.cpu(), 0, tables, keys, page, hd ** -0.5)
    again = torch.full_like(out, 3.0)
    step.attend_qkv(qkv, 0, hd ** -0.5, again)
    assert torch.equal(out, again)


def test_decode_attention_bad_pages(gpu):
    """Table entries outside the pool: their tokens are not there, the others' attention is."""
    rng = random.Random(5)
    cache, tables, lengths = make_cache(gpu, [100, 70, 40], 16, rng, spare=3, max_len=128)
    g = torch.Generator().manual_seed(1)
    host = fill_pages(cache, tables, lengths, g)
    cache.tables[0, 2], cache.tables[0, 3], cache.tables[2, 0] = -1, cache.num_pages, 1 << 30
    cache.tables[2, 1:3] = -5
    step = cache.decode_cache(3)
    q = torch.randn(3, 12 * 128, generator=g).half().to(gpu)
    rows = torch.randn(3, 2, 2, 128, generator=g).half().to(gpu)
    step.write(rows[:, 0], rows[:, 1], 0)
    host = cache.storage.cpu()
    out = step.attend_qkv(q, 0, 128 ** -0.5, torch.empty(3, 12, 128, device=gpu, dtype=torch.float16))
    tables, q = cache.tables.tolist(), q.view(3, 12, 128).cpu()
    # sequence 0 without its pages 2 and 3
    left = [t for j, t in enumerate(tables[0][:7]) if j not in (2, 3)]
    k, v = tokens_of(host, 0, left, 101 - 32, 16)
    want, mag = ref.attention(q[0], k, v, 128 ** -0.5)
    bound = ref.attention_bound(want, mag, 101, 8.0, torch.float16)
    assert ((out[0].cpu().double() - want).abs() <= bound).all()
    check_rows(out[1:2], q[1:2], host, 0, tables[1:2], [71], 16, 128 ** -0.5)
    assert (out[2] == 0).all()


def test_reserve_in_a_bad_page(gpu):
    """A sequence whose last, partly filled page is an entry outside the pool: its new tokens have no
    place until a page of their own begins."""
    rng = random.Random(6)
    cache, tables, lengths = make_cache(gpu, [20, 30, 5], 16, rng, spare=3, max_len=64)
    cache.tables[0, 1], cache.tables[1, 1] = -7, cache.num_pages
    free = sorted(set(range(cache.num_pages)) - {tables[0][0], tables[1][0], tables[2][0]})
    got = cache.reserve([14, 1, 1])
    assert got.granted.tolist() == [14, 1, 1]
    assert got.token_page.tolist() == [-1] * 12 + [free[0]] * 2 + [-1, tables[2][0]]
    assert got.token_pos.tolist() == [-1] * 12 + [0, 1, -1, 5]
    assert got.positions.tolist() == [-1] * 12 + [32, 33, -1, 5]
    got = cache.decode_cache(3)
    assert got.token_page.tolist() == [-1, -1, tables[2][0]]
    assert got.positions.tolist() == [[-1, -1, 5]] * 3


def test_decode_attention_far_pages(gpu):
    """K and V of more than 2^31 elements each."""
    from omniserver_amd.paged_kv import PagedKVCache
    pages = (1 << 31) // (64 * 2 * 128) + 40
    cache = PagedKVCache(1, pages, 2, 64, 128, gpu, max_seqs=2, max_len=200)
    g = torch.Generator().manual_seed(3)
    table = [[pages - 1, 3, pages - 3], [pages - 2, pages - 4, 0]]
    used = [p for row in table for p in row]
    cache.storage[:, :, used] = torch.randn(1, 2, 6, 64, 2, 128, generator=g).half().to(gpu)
    cache.tables[:, :3] = i32(table, gpu)
    cache.lengths.copy_(torch.tensor([150, 180]))
    step = cache.decode_cache(2)
    q = torch.randn(2, 12 * 128, generator=g).half().to(gpu)
    out = step.attend_qkv(q, 0, 0.1, torch.empty(2, 12, 128, device=gpu, dtype=torch.float16))
    host = cache.storage[:, :, used].cpu()
    check_rows(out, q.view(2, 12, 128), host, 0, [[0, 1, 2], [3, 4, 5]], [151, 181], 64, 0.1)


REORDER = [
    # requests, beams, page, lengths, spare pages, layers
    (1, 1, 16, (5, 5), 0, 1),
    (1, 4, 16, (33, 33), 4, 2),
    (1, 4, 16, (32, 32), 0, 2),               # nothing in part
    (3, 3, 32, (0, 70), 5, 3),
    (2, 5, 16, (1, 200), 1, 2),               # too few pages
    (8, 4, 64, (50, 300), 32, 1),
    (100, 7, 16, (0, 30), 500, 1),
    (300, 5, 16, (0, 20), 900, 1),            # more rows than a workgroup has threads
    (2, 32, 128, (100, 500), 64, 1),
]


@pytest.mark.parametrize("n,W,page,span,spare,layers", REORDER)
@pytest.mark.parametrize("shared", [False, True])
def test_reorder(gpu, n, W, page, span, spare, layers, shared):
    say(f"reorder {n} x {W} beams, pages of {page}, lengths {span}, shared={shared}")
    rng = random.Random(n * 7 + W)
    lengths = [rng.randint(*span) for _ in range(n) for _ in range(W)]
    if shared:
        lengths = [lengths[r - r % W] for r in range(n * W)]
    cache, tables, lengths = make_cache(gpu, lengths, page, rng, nkv=1, nh=2, hd=64, layers=layers,
                                        spare=spare, max_len=span[1] + 40, seqs=n * W + 3,
                                        shared=W if shared else 1)
    g = torch.Generator().manual_seed(W)
    cache.storage.copy_(torch.randn(cache.storage.shape, generator=g))
    for turn in range(3):
        parents = [[rng.choice([-1, rng.randrange(W), rng.randrange(W), 0]) for _ in range(W)]
                   for _ in range(n)]
        if turn == 0:
            parents[0][-1] = 0
        before = cache.storage.clone()
        new_tables, new_lengths, copies = ref.reorder(tables, lengths, parents, cache.num_pages, page)
        if turn == 1:
            cache.reorder(parents)
        else:
            given = i32(parents, gpu)
            given[given < 0] = rng.choice([-1, -100, W, 1 << 30])
            cache.reorder(given)
        assert cache.lengths.tolist() == new_lengths
        got = cache.tables.tolist()
        for r, m in enumerate(new_lengths):
            held = ref.pages_of(m, page)
            assert got[r][:held] == new_tables[r][:held], f"row {r}"
        for a, b, m in copies:
            before[:, :, b, :m] = before[:, :, a, :m].clone()
        assert torch.equal(cache.storage, before)
        tables, lengths = got, new_lengths


SELECT = [
    # requests, beams, k, vocab, dtype, kind
    (1, 1, 1, 1, torch.float32, "normal"),
    (1, 1, 1, 7, torch.float16, "normal"),
    (2, 3, 5, 2, torch.float16, "normal"),            # k near everything there is
    (1, 4, 64, 5, torch.bfloat16, "normal"),          # fewer continuations than k
    (3, 4, 4, 1000, torch.float16, "normal"),
    (3, 4, 8, 1000, torch.float16, "ties"),
    (2, 5, 10, 4097, torch.float32, "normal"),
    (2, 5, 10, 8191, torch.bfloat16, "ties"),
    (2, 4, 64, 20000, torch.float16, "sorted"),       # all of the best in one block
    (2, 4, 64, 20000, torch.float32, "constant"),
    (4, 32, 32, 3001, torch.float16, "ended"),
    (5, 6, 12, 9999, torch.float32, "ended"),
    (3, 4, 8, 5000, torch.float16, "odd"),            # NaN, infinities, empty rows
    (3, 4, 8, 5000, torch.float32, "odd"),
    (3, 4, 8, 5000, torch.bfloat16, "odd"),
    (1, 4, 4, 151936, torch.float16, "normal"),
    (40, 2, 4, 33333, torch.float16, "normal"),       # blocks of 8192
    (1, 2, 16, 524288, torch.float16, "normal"),
    (7, 16, 32, 32003, torch.bfloat16, "normal"),
]


def select_case(n, W, V, dtype, kind, g, rng):
    logits = torch.randn(n, W, V, generator=g) * 3
    if kind == "ties":
        logits = (logits * 2).round() / 2
    elif kind == "sorted":
        logits = logits.sort(-1, descending=rng.random() < 0.5).values
    elif kind == "constant":
        logits = torch.full((n, W, V), 1.5)
    scores = -torch.rand(n, W, generator=g) * 5
    done = torch.zeros(n, W, dtype=torch.bool)
    if kind == "ended":
        done = torch.rand(n, W, generator=g) < 0.4
        scores[torch.rand(n, W, generator=g) < 0.3] = -math.inf
        scores[0] = -math.inf
        scores[1, 0], done[1, 0] = -0.25, True
        scores[2, :3] = torch.tensor([math.nan, math.inf, -1.0])
    if kind == "odd":
        logits[torch.rand(logits.shape, generator=g) < 0.5] = -math.inf
        logits[torch.rand(logits.shape, generator=g) < 0.1] = math.nan
        logits[0, 1] = -math.inf
        logits[0, 2] = math.nan
        logits[0, 3, 3:] = -math.inf
        logits[0, 3, :3] = torch.tensor([math.nan, -2.0, -3.0])
        logits[1, 0, [7, 90, 4000]] = math.inf
        logits[2] = -math.inf
        logits[2, 1, 4999] = -60000.0
        logits[2, 3, 17] = 0.0
        logits[2, 3, 16] = -0.0
    return logits.to(dtype), scores, done


@pytest.mark.parametrize("n,W,k,V,dtype,kind", SELECT)
def test_select(gpu, n, W, k, V, dtype, kind):
    from omniserver_amd.beam import select
    say(f"select {k} of {n} x {W} beams over {V} {dtype} {kind}")
    rng, g = random.Random(n + V), torch.Generator().manual_seed(V + k)
    logits, scores, done = select_case(n, W, V, dtype, kind, g, rng)
    stop = [[rng.randrange(V), -1, int(logits[s, 0].nan_to_num(nan=-9e4).argmax())] for s in range(n)]
    want = ref.select(logits, scores, k, done, stop, pad=11)
    got = select(logits.to(gpu), scores.to(gpu), k, done.to(gpu),
                 torch.tensor(stop, device=gpu), pad=11)
    pick = lambda i: [[row[i] for row in request] for request in want]
    assert got.parents.tolist() == pick(1)
    assert got.tokens.tolist() == pick(2)
    assert got.done.tolist() == pick(3)
    exact = torch.tensor(pick(0), dtype=torch.float64)
    have = got.scores.cpu().double()
    assert torch.equal(have == -math.inf, exact == -math.inf)
    fine = exact > -math.inf
    # one rounding to fp32, and the logarithm of a sum in 32 bits: a weight 2^-t is off by 2 t ln 2
    # 2^-24 (the difference's and the exponent's roundings) and 2^-23 (the exponential), which the
    # largest weight's 1 bounds at t = 30 for 2^19 tokens; a lane's 8 additions in each of 4 sums, 2
    # of those, 6 over the wave are off by 2^-24 each
    bound = (2 * 30 * math.log(2) + 2 + 16) * 2.0 ** -24
    assert ((have - exact).abs() <= exact.abs() * 2.0 ** -24 + bound)[fine].all()
    again = select(logits.to(gpu), scores.to(gpu), k, done.to(gpu), torch.tensor(stop, device=gpu), 11)
    assert all(torch.equal(a, b) for a, b in zip(got, again))


@pytest.mark.parametrize("V,dtype", [(300001, torch.float16), (300001, torch.bfloat16), (270000, torch.float32),
                                     (140003, torch.float16), (9001, torch.float16)])
def test_select_level_rows(gpu, V, dtype):
    """Rows of one value with a few above it, in blocks of every size: more equal logits than a block ranks,
    so that its best are taken out one after another."""
    from omniserver_amd.beam import select
    say(f"select level rows {V} {dtype}")
    g = torch.Generator().manual_seed(V)
    logits = torch.full((1, 3, V), -0.75)
    for b, few in enumerate((2, 7, 30)):
        at = torch.randperm(V, generator=g)[:few]
        logits[0, b, at] = torch.randint(0, 4, (few,), generator=g).float()
    logits[0, 2, 5:50] = -math.inf
    logits[0, 1, 3] = math.nan
    logits, scores = logits.to(dtype), torch.tensor([[-1.0, -2.5, -0.5]])
    for k in (3, 40):
        want = ref.select(logits, scores, k)
        got = select(logits.to(gpu), scores.to(gpu), k)
        assert got.parents.tolist() == [[r[1] for r in q] for q in want], k
        assert got.tokens.tolist() == [[r[2] for r in q] for q in want], k


def test_select_defaults_and_strides(gpu):
    """k defaults to the beams; rows that are views of wider ones; one list of stop tokens; nothing
    finished."""
    from omniserver_amd.beam import select
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(4, 3, 2, 1009, generator=g).half()
    logits = wide[1:, :, 1, 5:1004]
    scores = -torch.rand(3, 3, generator=g)
    want = ref.select(logits, scores, 3, None, [4, 990])
    got = select(wide.to(gpu)[1:, :, 1, 5:1004], scores.to(gpu), stop=[4, 990])
    assert got.parents.tolist() == [[r[1] for r in q] for q in want]
    assert got.tokens.tolist() == [[r[2] for r in q] for q in want]
    assert got.done.tolist() == [[r[3] for r in q] for q in want]
    one = select(logits[:1, :1].expand(2, 3, 999).to(gpu), torch.zeros(2, 3, device=gpu))
    assert one.parents.tolist() == [[0, 1, 2]] * 2      # all alike: the lower beam first


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_select_close_values(gpu, dtype):
    """Beams whose continuations differ by less than 32-bit sums resolve: the order is that of 64-bit
    values, and of the lower beam where these are equal."""
    from omniserver_amd.beam import select
    say(f"select close values {dtype}")
    g = torch.Generator().manual_seed(8)
    V, W, n = 20011, 5, 6
    row = (torch.randn(1, 1, V, generator=g) * 3).to(dtype)
    logits = row.expand(n, W, V).contiguous()
    # the same logits; scores a rounding step or two apart, or equal
    steps = torch.tensor([[0, 1, 2, 3, 4], [4, 3, 2, 1, 0], [1, 1, 0, 0, 1], [0] * 5, [2, 0, 2, 1, 0],
                          [3, 3, 3, 0, 3]])
    scores = (-1.0 - steps * 2.0 ** -23).float()
    # rows that differ by one small logit: sums apart by 1e-9 of themselves and less
    for s in (3, 4):
        for b in range(W):
            logits[s, b, 100 + b] = (-14.0 - 0.01 * ((b * 3) % 5))
    done = torch.zeros(n, W, dtype=torch.bool)
    done[5, 1] = True
    for k in (5, 12, 40):
        want = ref.select(logits, scores, k, done)
        got = select(logits.to(gpu), scores.to(gpu), k, done.to(gpu))
        assert got.parents.tolist() == [[r[1] for r in q] for q in want], k
        assert got.tokens.tolist() == [[r[2] for r in q] for q in want], k


def test_select_lowest_values(gpu):
    """Logits masked by the type's lowest number are continuations while their sums fit fp32; a sum
    that does not is none: no parent, no token, finished."""
    from omniserver_amd.beam import select
    low = torch.finfo(torch.float32).min
    logits = torch.full((1, 2, 40), low)
    logits[0, :, 7] = 1.0
    got = select(logits.to(gpu), torch.tensor([[0.0, low]], device=gpu), 5)
    # beam 0: token 7 at 0, the others at low - 1, which is low in 64 bits too; beam 1: token 7 at low,
    # behind those, the others at 2 low
    assert got.scores.tolist() == [[0.0] + [low] * 4]
    assert got.parents.tolist() == [[0] * 5] and got.tokens.tolist() == [[7, 0, 1, 2, 3]]
    assert got.done.tolist() == [[False] * 5]
    for W in (1, 2):                                  # one unfinished row; many values in question
        scores = torch.full((1, 2), low)[:, :W].contiguous().to(gpu)
        for k in (3, 50):
            got = select(logits[:, :W].contiguous().to(gpu), scores, k)
            none = k - W
            assert got.scores.tolist() == [[low] * W + [-math.inf] * none]
            assert got.parents.tolist() == [[0, 1][:W] + [-1] * none]
            assert got.tokens.tolist() == [[7] * W + [-1] * none]
            assert got.done.tolist() == [[False] * W + [True] * none]


def test_select_vector_of_values(gpu):
    """More beams times continuations than lanes, close ones among them."""
    from omniserver_amd.beam import select
    g = torch.Generator().manual_seed(9)
    n, W, V = 3, 24, 5003
    row = (torch.randn(n, 1, V, generator=g) * 3).half()
    logits = row.expand(n, W, V).contiguous()
    logits[:, 12:] = (torch.randn(n, 12, V, generator=g) * 3).half()
    scores = (-2.0 - torch.randint(0, 3, (n, W), generator=g) * 2.0 ** -22).float()
    for k in (8, 48):
        want = ref.select(logits, scores, k)
        got = select(logits.to(gpu), scores.to(gpu), k)
        assert got.parents.tolist() == [[r[1] for r in q] for q in want], k
        assert got.tokens.tolist() == [[r[2] for r in q] for q in want], k


# ----------------------------------------------------------------------------- as a step runs them
def beam_step(cache, x, n, W, nh, nkv, hd):
    """One step of beam search on the operators alone: x holds the tensors that a model would give."""
    from omniserver_amd.beam import select
    rows = n * W
    step = cache.decode_cache(rows)
    q, k, v = x["qkv"].view(rows, nh + 2 * nkv, hd).split((nh, nkv, nkv), 1)
    for layer in range(cache.n_layers):
        step.write(k, v, layer)
        step.attend_qkv(x["qkv"], layer, hd ** -0.5, x["out"][layer])
    step.finish()
    b = select(x["logits"], x["scores"], done=x["done"], stop=x["stop"], pad=-1)
    cache.reorder(b.parents)
    x["scores"].copy_(b.scores)
    x["done"].copy_(b.done)
    return b


def beam_inputs(rng, g, n, W, nh, nkv, hd, layers, V, gpu):
    x = {"qkv": torch.randn(n * W, (nh + 2 * nkv) * hd, generator=g).half(),
         "logits": torch.randn(n, W, V, generator=g).half() * 3,
         "stop": torch.tensor([rng.randrange(V)])}
    return x


def test_beam_steps_follow_their_tokens(gpu):
    """Ten steps of beam search on random K/V: what every beam holds is what a list of its tokens' K/V
    rows holds, and its attention that of the list."""
    from omniserver_amd.paged_kv import PagedKVCache
    say("beam steps against lists")
    n, W, nh, nkv, hd, layers, page, V = 3, 4, 6, 2, 64, 2, 16, 700
    rng, g = random.Random(3), torch.Generator().manual_seed(4)
    prompts = [37, 16, 5]
    cache = PagedKVCache(layers, 60, nkv, page, hd, gpu, max_seqs=n * W, max_len=80, n_heads=nh)
    slots = cache.reserve(prompts, rows=range(0, n * W, W))
    kv = torch.randn(layers, 2, sum(prompts), nkv, hd, generator=g).half()
    for layer in range(layers):
        slots.write(kv[layer, 0].to(gpu), kv[layer, 1].to(gpu), layer)
    slots.finish()
    held, at = [], 0
    for L in prompts:
        held.append([kv[:, :, at:at + L]] + [kv[:, :, :0]] * (W - 1))
        at += L
    state = {"scores": torch.full((n, W), -math.inf), "done": torch.zeros(n, W, dtype=torch.bool),
             "out": torch.zeros(layers, n * W, nh, hd).half()}
    state["scores"][:, 0] = 0.0
    state = {name: v.to(gpu) for name, v in state.items()}
    for turn in range(10):
        x = beam_inputs(rng, g, n, W, nh, nkv, hd, layers, V, gpu)
        want = ref.select(x["logits"], state["scores"].cpu(), W, state["done"].cpu(), x["stop"].tolist(), -1)
        rows = x["qkv"].view(n * W, nh + 2 * nkv, hd)
        state.update({name: v.to(gpu) for name, v in x.items()})
        b = beam_step(cache, state, n, W, nh, nkv, hd)
        for s in range(n):
            for w in range(W):
                r = s * W + w
                new = rows[r, nh:].reshape(2, 1, nkv, hd)
                held[s][w] = torch.cat([held[s][w], new.expand(layers, 2, 1, nkv, hd)], 2)
                for layer in range(layers):
                    k, v = held[s][w][layer]
                    exact, mag = ref.attention(rows[r, :nh], k, v, hd ** -0.5)
                    bound = ref.attention_bound(exact, mag, k.shape[0], v.float().abs().max().item(),
                                                torch.float16)
                    err = (state["out"][layer, r].cpu().double() - exact).abs()
                    assert (err <= bound).all(), (turn, s, w, layer)
        assert b.parents.tolist() == [[e[1] for e in q] for q in want], turn
        assert b.tokens.tolist() == [[e[2] for e in q] for q in want], turn
        assert b.done.tolist() == [[e[3] for e in q] for q in want], turn
        held = [[held[s][e[1]] if e[1] >= 0 else kv[:, :, :0] for e in q] for s, q in enumerate(want)]
        tables, host = cache.tables.tolist(), cache.storage.cpu()
        assert cache.lengths.tolist() == [h.shape[2] for q in held for h in q], turn
        for r, h in enumerate(h for q in held for h in q):
            for layer in range(layers):
                k, v = tokens_of(host, layer, tables[r], h.shape[2], page)
                assert torch.equal(k, h[layer, 0]) and torch.equal(v, h[layer, 1]), (turn, r)


def test_beam_step_in_graphs(gpu):
    """A step captured on one cache, and another on a second one, replayed in turn with eager work
    between: each does what an eager twin does."""
    from omniserver_amd.paged_kv import PagedKVCache
    say("beam steps in two graphs")
    n, W, nh, nkv, hd, layers, page, V = 2, 3, 12, 2, 128, 1, 16, 3001
    rng, g = random.Random(5), torch.Generator().manual_seed(6)

    def start():
        cache = PagedKVCache(layers, 40, nkv, page, hd, gpu, max_seqs=n * W, max_len=96, n_heads=nh)
        cache.storage.copy_(torch.randn(cache.storage.shape, generator=torch.Generator().manual_seed(1)))
        for s, L in enumerate((30, 47)):
            cache.reserve([L], rows=[s * W]).finish()
        x = {"scores": torch.full((n, W), -math.inf, device=gpu),
             "done": torch.zeros(n, W, dtype=torch.bool, device=gpu),
             "out": torch.zeros(layers, n * W, nh, hd, device=gpu, dtype=torch.float16),
             "qkv": torch.zeros(n * W, (nh + 2 * nkv) * hd, device=gpu, dtype=torch.float16),
             "logits": torch.zeros(n, W, V, device=gpu, dtype=torch.float16),
             "stop": torch.tensor([5], device=gpu)}
        x["scores"][:, 0] = 0.0
        return cache, x

    twins = [(start(), start()) for _ in range(2)]
    graphs = []
    for (cache, x), _ in twins:
        keep = {name: t.clone() for name, t in
                list(x.items()) + [("l", cache.lengths), ("t", cache.tables), ("s", cache.storage)]}
        beam_step(cache, x, n, W, nh, nkv, hd)                 # warm
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            b = beam_step(cache, x, n, W, nh, nkv, hd)
        for name, t in list(x.items()) + [("l", cache.lengths), ("t", cache.tables), ("s", cache.storage)]:
            t.copy_(keep[name])
        graphs.append((graph, b))
    for turn in range(8):
        which = turn % 2
        (cache, x), (twin, y) = twins[which]
        new = beam_inputs(rng, g, n, W, nh, nkv, hd, layers, V, gpu)
        for name, v in new.items():
            x[name].copy_(v)
            y[name].copy_(v)
        graphs[which][0].replay()
        want = beam_step(twin, y, n, W, nh, nkv, hd)
        torch.cuda.synchronize()
        for a, b in zip(graphs[which][1], want):
            assert torch.equal(a, b), turn
        for name in x:
            assert torch.equal(x[name], y[name]), (turn, name)
        assert torch.equal(cache.tables, twin.tables) and torch.equal(cache.lengths, twin.lengths)
        assert torch.equal(cache.storage, twin.storage), turn


def test_another_stream(gpu):
    """Launches go to the current stream: a step on a side stream behind a long kernel of its own."""
    rng = random.Random(7)
    cache, tables, lengths = make_cache(gpu, [90, 33], 16, rng, spare=4, max_len=128)
    g = torch.Generator().manual_seed(2)
    host = fill_pages(cache, tables, lengths, g)
    rows = torch.randn(2, 16 * 128, generator=g).half()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        x = torch.randn(3000, 3000, device=gpu)
        for _ in range(5):
            x = x @ x / 3000
        qkv = rows.to(gpu)
        step = cache.decode_cache(2)
        q, k, v = qkv.view(2, 16, 128).split((12, 2, 2), 1)
        out = step.flash_decode(q, k, v, 0, 0.1)
    side.synchronize()
    check_rows(out, rows.view(2, 16, 128)[:, :12], cache.storage.cpu(), 0, cache.tables.tolist(),
               [91, 34], 16, 0.1)


def test_superseded_reservations(gpu):
    """A later reservation or reordering may give the same pages away: the older one says so."""
    rng = random.Random(8)
    cache, _, _ = make_cache(gpu, [20, 7, 9], 16, rng, spare=6, max_len=128)
    first = cache.decode_cache(3)
    second = cache.reserve([1, 2], rows=[2, 0])
    k = torch.zeros(3, 2, 128, device=gpu, dtype=torch.float16)
    out = torch.empty(3, 12, 128, device=gpu, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="later"):
        first.write(k, k, 0)
    with pytest.raises(RuntimeError, match="later"):
        first.attend_qkv(torch.zeros(3, 1536, device=gpu).half(), 0, 0.1, out)
    with pytest.raises(RuntimeError, match="later"):
        first.finish()
    second.finish()
    assert cache.lengths.tolist() == [22, 7, 10]
    third = cache.reserve([3])
    cache.reorder([[0, 0, 2]])
    with pytest.raises(RuntimeError, match="later"):
        third.finish()
    assert cache.lengths.tolist() == [22, 22, 10]
    fourth = cache.decode_cache(3)
    cache.free([1])
    with pytest.raises(RuntimeError, match="later"):
        fourth.finish()
    assert cache.lengths.tolist() == [22, 0, 10]


def test_prompts_short_of_pages(gpu):
    """Prompts whose pages are not there are attended to like the others and leave nothing behind; rows
    that held something before are begun anew; more packed rows than tokens."""
    from omniserver_amd.kv_cache import PreallocatedKVCache
    from omniserver_amd.paged_kv import PagedKVCache
    cache = PagedKVCache(1, 4, 2, 16, 128, gpu, max_seqs=5, max_len=40, n_heads=12)
    cache.reserve([40, 3], rows=[1, 4]).finish()                 # all four pages
    assert cache.lengths.tolist() == [0, 40, 0, 0, 3]
    pool = PreallocatedKVCache(1, 3, 2, 40, 128, gpu, n_heads=12)
    g = torch.Generator().manual_seed(3)
    lens, T = [20, 30, 10], 60
    q, k, v = (torch.randn(T, h, 128, generator=g).half().to(gpu) for h in (12, 2, 2))
    want = pool.packed_prefill_cache(range(3), lens).flash_prefill(q, k, v, 0, 0.1)
    prompts = cache.prefill_cache([1, 0, 3], lens)               # row 1's three pages are free for it
    assert prompts.granted.tolist() == [20, 0, 0]
    assert torch.equal(prompts.flash_prefill(q, k, v, 0, 0.1), want)
    assert cache.lengths.tolist() == [0, 20, 0, 0, 3]
    kk, vv = tokens_of(cache.storage.cpu(), 0, cache.tables[1].tolist(), 20, 16)
    assert torch.equal(kk, k[:20].cpu()) and torch.equal(vv, v[:20].cpu())
    more = cache.reserve([2, 1], rows=[1, 4], tokens=6)
    assert more.token_pos.tolist() == [4, 5, 3, -1, -1, -1] and more.granted.tolist() == [2, 1]


# ----------------------------------------------------------------------------- the model
@pytest.mark.parametrize("quant", [None, "gptq"])
def test_model_over_pages(gpu, quant):
    """The decoder's forward over a paged cache against the same over the preallocated pool: packed
    prompts, then single tokens, for which the pool's view runs the same linears."""
    from omniserver_amd import synth
    from omniserver_amd.kv_cache import PreallocatedKVCache
    from omniserver_amd.paged_kv import PagedKVCache
    from omniserver_amd.qwen2_llm import Qwen2LLM
    from tests.helpers import compare_logits
    say(f"model over pages quant={quant}")
    shape = synth.DecoderShape()
    gen, build = ((synth.gptq_decoder, Qwen2LLM.from_gptq) if quant
                  else (synth.fp16_decoder, Qwen2LLM.from_fp16))
    shape.num_layers = 2
    llm = build(gen(shape, seed=5, num_layers=2), shape, gpu)
    lens = [40, 17, 65, 100]
    T, n = sum(lens), len(lens)
    ids = [synth.random_ids(L, shape.vocab_size, 5, f"p{L}") for L in lens]
    pool = PreallocatedKVCache(2, n, 2, 160, 128, gpu, n_heads=12)
    pages = PagedKVCache(2, 40, 2, 16, 128, gpu, max_seqs=n, max_len=160, n_heads=12)
    pos = torch.cat([torch.arange(L) for L in lens]).expand(3, 1, T).contiguous().to(gpu)
    last = [sum(lens[:i + 1]) - 1 for i in range(n)]
    with torch.inference_mode():
        emb = llm.embed_tokens(torch.cat(ids).to(gpu)).unsqueeze(0)
        a = llm(emb, pos, None, pool.packed_prefill_cache(range(n), lens), logits_indices=last)[0]
        b = llm(emb, pos, None, pages.prefill_cache(range(n), lens), logits_indices=last)[0]
        assert torch.equal(a, b)
        assert pages.lengths.tolist() == lens == pool.lengths.tolist()
        for turn in range(20):                        # over pages' borders
            new = a.argmax(-1)
            emb = llm.embed_tokens(new)
            a = llm(emb.unsqueeze(1), pool.lengths[:n].expand(3, n).unsqueeze(-1), None,
                    pool.view(n))[:, -1]
            step = pages.decode_cache(n)
            b = llm(emb.unsqueeze(0), step.positions.view(3, 1, n), None, step)[0]
            compare_logits(b, a)
        assert pages.lengths.tolist() == [L + 20 for L in lens] == pool.lengths.tolist()


def oracle_beams(orc, prompt, W, steps, stops):
    """Beam search on the oracle's logits: (sum of log-probabilities, tokens), the best first."""
    from tests.helpers import oracle_stream_logits
    beams = [(0.0, [], False)]
    for _ in range(steps):
        every = []
        for score, line, over in beams:
            if over:
                every.append((score, line, True))
                continue
            rows = oracle_stream_logits(orc, prompt, line + [0], 256)
            lp = torch.log_softmax(rows[len(line)].double(), -1)
            best = lp.topk(W)
            every += [(score + v, line + [t], t in stops)
                      for v, t in zip(best.values.tolist(), best.indices.tolist())]
        every.sort(key=lambda e: -e[0])
        beams = every[:W]
    return beams


@pytest.mark.parametrize("quant,use_graph", [(None, False), (None, True), ("gptq", True)])
def test_runner_beam_search(gpu, quant, use_graph):
    """Beams of two prompts: their sums of log-probabilities are the oracle's for their tokens, the
    best is as good as the oracle's beam search finds, one beam alone is the greedy stream, and running
    sequences are left alone."""
    from omniserver_amd import synth
    from omniserver_amd.request import Request, SamplingParams, Sequence
    from omniserver_amd.runner import NativeQwenVLRunner
    from tests.helpers import oracle_from_fp16, oracle_from_gptq, oracle_stream_logits
    say(f"runner beam search quant={quant} use_graph={use_graph}")
    shape = synth.DecoderShape()
    w = (synth.gptq_decoder if quant else synth.fp16_decoder)(shape, seed=5, num_layers=2)
    prompts = [synth.random_ids(L, shape.vocab_size, 5, f"p{L}").tolist() for L in (40, 17)]
    orc = oracle_from_gptq(w, shape) if quant else oracle_from_fp16(w, shape)
    r = NativeQwenVLRunner(max_running=2, max_len=128, use_graph=use_graph, weights=w, quant=quant)
    mk = lambda p, steps: Sequence(Request(prompt=p, sampling=SamplingParams(max_new_tokens=steps)))  # noqa: E731
    running = [mk(p, 30) for p in prompts]
    for s in running:
        r.tokenize(s)
    r.prefill(running)
    r.decode(running)
    before = [list(s.output_token_ids) for s in running]
    W, steps = 3, 6
    seqs = [mk(prompts[0], steps), mk(prompts[1], steps - 1)]
    found = r.beam_search(seqs, beams=W, page_size=16)
    for s, beams in zip(seqs, found):
        p, limit = s.request.prompt, s.request.sampling.max_new_tokens
        assert len(beams) == W and not s.output_token_ids
        assert [b.score for b in beams] == sorted((b.score for b in beams), reverse=True)
        assert len({tuple(b.tokens) for b in beams}) == W
        want = oracle_beams(orc, p, W, limit, s.request.sampling.stop_token_ids)
        # logits within 2e-2 of the oracle's: a log-probability within twice that
        slack = 2 * 2e-2 * limit
        for b in beams:
            rows = oracle_stream_logits(orc, p, b.tokens, 256)
            lp = torch.log_softmax(torch.as_tensor(rows).double(), -1)
            exact = sum(float(lp[i, t]) for i, t in enumerate(b.tokens))
            assert abs(b.logprob - exact) <= slack
            assert abs(b.score - b.logprob / len(b.tokens)) < 1e-6 and len(b.tokens) == limit
        assert max(b.logprob for b in beams) >= want[0][0] - slack
    stop = found[0][0].tokens[2]
    seq = mk(prompts[0], steps)
    seq.request.sampling.stop_token_ids = [stop]
    for b in r.beam_search([seq], beams=W)[0]:
        assert stop not in b.tokens[:-1] and (b.tokens[-1] == stop or len(b.tokens) == steps)
    greedy = r.beam_search([mk(prompts[0], steps)], beams=1)[0]
    assert len(greedy) == 1 and len(greedy[0].tokens) == steps
    r.decode(running)
    assert [s.output_token_ids[:len(b)] for s, b in zip(running, before)] == before
    for bad in ({"beams": 0}, {"beams": 33}, {"page_size": 24}):
        with pytest.raises(ValueError):
            r.beam_search([mk(prompts[0], 4)], **bad)
    with pytest.raises(ValueError):
        r.beam_search([Sequence(Request(prompt=prompts[0], sampling=SamplingParams(temperature=0.5)))])
    assert r.beam_search([]) == []
