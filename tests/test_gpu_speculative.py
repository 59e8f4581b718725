"""Speculative decoding's operators on the GPU against the 64-bit oracle: attention of drafted
trees over the pool, verification of drafted tokens, the cache after acceptance, the three as a
step runs them."""

import math
import random

import pytest
import torch

from oracle import speculative_ref as ref

pytestmark = pytest.mark.gpu

HD = 128


def say(msg):
    print(f"[gpu-test] {msg}", flush=True)


def make_pool(gpu, layers, rows, nh, nkv, max_len, seed):
    from omniserver_amd.kv_cache import PreallocatedKVCache
    pool = PreallocatedKVCache(layers, rows, nkv, max_len, HD, gpu, n_heads=nh)
    g = torch.Generator().manual_seed(seed)
    pool.storage.copy_(torch.randn(pool.storage.shape, generator=g).half())
    return pool, g


def trees(rng, n, T, kind):
    if kind == "chain":
        return [[i - 1 for i in range(T)] for _ in range(n)]
    if kind == "star":
        return [[-1] + [0] * (T - 1) for _ in range(n)]
    if kind == "roots":                # nodes that see no other
        return [[-1] * T for _ in range(n)]
    return [[-1] + [rng.randint(max(0, i - 5), i - 1) for i in range(1, T)] for _ in range(n)]


def i32(x, gpu):
    return torch.tensor(x, dtype=torch.int32, device=gpu)


def check_attention(out, q, pool, layer, starts, parents, counts, slots, fill):
    """out [n, T, nh, hd] against the oracle; rows not in use still hold fill."""
    k, v = pool.k[layer].cpu(), pool.v[layer].cpu()
    want, mag, seen = ref.tree_attention(q, k, v, starts, parents, counts, slots, HD ** -0.5)
    vf = v.float()
    bound = ref.attention_bound(want, mag, seen, vf[vf.isfinite()].abs().max().item())
    out = out.cpu().double()
    used = ~want.isnan()
    worst = ((out - want).abs() / bound)[used].max().item() if used.any() else 0.0
    say(f"  worst error {worst:.2f} of the bound")
    assert worst <= 1.0
    assert (out[~used] == fill).all()


ATTENTION = [
    # n, T, nh, nkv, starts, kind, ragged
    (1, 1, 12, 2, (0, 0), "chain", False),
    (2, 1, 12, 2, (1, 70), "chain", False),
    (3, 2, 12, 2, (0, 40), "tree", False),
    (2, 8, 12, 2, (250, 300), "tree", False),
    (4, 7, 12, 2, (0, 130), "tree", True),
    (3, 16, 12, 2, (60, 66), "tree", True),
    (2, 33, 12, 2, (31, 33), "star", False),
    (2, 63, 12, 2, (90, 200), "tree", True),
    (2, 64, 12, 2, (0, 65), "chain", False),
    (1, 64, 12, 2, (700, 700), "tree", False),
    (2, 20, 28, 4, (10, 500), "tree", False),
    (2, 9, 16, 16, (33, 180), "tree", True),
    (3, 11, 8, 1, (64, 64), "roots", False),
    (1, 64, 32, 1, (100, 100), "tree", False),
    (1, 5, 64, 1, (129, 129), "tree", False),
    (1, 12, 12, 2, (2000, 2000), "tree", False),
    (6, 3, 12, 2, (0, 1000), "chain", True),
]


@pytest.mark.parametrize("n,T,nh,nkv,span,kind,ragged", ATTENTION)
def test_tree_attention(gpu, n, T, nh, nkv, span, kind, ragged):
    say(f"tree attention n={n} T={T} heads {nh}/{nkv} starts {span} {kind} ragged={ragged}")
    rng = random.Random(n * 1000 + T)
    starts = [rng.randint(*span) for _ in range(n)]
    counts = [rng.randint(0, T) for _ in range(n)] if ragged else [T] * n
    parents = trees(rng, n, T, kind)
    pool, g = make_pool(gpu, 2, n + 2, nh, nkv, max(starts) + T + 3, n + T)
    slots = rng.sample(range(n + 2), n)
    for s, L in zip(slots, starts):
        pool.lengths[s] = L
    rows = torch.randn(n * T, (nh + 2 * nkv) * HD, generator=g).half()
    q = rows[:, :nh * HD].reshape(n, T, nh, HD)
    cache = pool.tree_cache(parents, counts=counts if ragged else None, slots=slots)
    fill = 7.0
    out = torch.full((n * T, nh, HD), fill, device=gpu, dtype=torch.float16)
    cache.attend_qkv(rows.to(gpu), 1, HD ** -0.5, out)
    torch.cuda.synchronize()
    check_attention(out.view(n, T, nh, HD), q, pool, 1, starts, parents, counts, slots, fill)
    again = torch.full_like(out, fill)
    cache.attend_qkv(rows.to(gpu), 1, HD ** -0.5, again)
    assert torch.equal(out, again)


CUT = [
    # n, T, nh, nkv, starts, capacity, the plan's (rows, groups), cut or not
    (1, 8, 12, 2, (3000, 3000), 4096, (64, 4, True)),
    (5, 10, 12, 2, (0, 1700), 2048, (64, 4, True)),
    (70, 3, 8, 1, (0, 150), 1600, (32, 8, True)),        # more sequences than lanes
    (33, 2, 12, 2, (0, 300), 4096, (32, 8, True)),
    (9, 40, 12, 2, (0, 900), 8192, (128, 2, True)),
    (2, 64, 28, 4, (1200, 1800), 16384, (128, 2, True)),
    (3, 64, 64, 1, (0, 200), 2000, (128, 2, True)),      # 32 row blocks
    (150, 2, 12, 2, (0, 700), 4096, (32, 8, True)),      # more items than columns
    (1, 64, 64, 1, (500, 500), 1024, (32, 8, False)),     # 128 row blocks, enough to leave uncut
]


@pytest.mark.parametrize("n,T,nh,nkv,span,capacity,form", CUT)
def test_tree_attention_cut(gpu, n, T, nh, nkv, span, capacity, form):
    """Long pools, where the keys of all sequences are cut evenly over the workgroups: very
    different contexts, sequences without nodes, rows outside the pool, every cut merged."""
    say(f"tree attention cut: n={n} T={T} heads {nh}/{nkv} starts {span} capacity {capacity}")
    rng = random.Random(n * 100 + T)
    starts = [rng.randint(*span) for _ in range(n)]
    counts = [rng.randint(0, T) if n > 2 else T for _ in range(n)]
    parents = trees(rng, n, T, "tree")
    pool, g = make_pool(gpu, 1, n, nh, nkv, 16, T)
    from omniserver_amd.kv_cache import PreallocatedKVCache
    pool = PreallocatedKVCache(1, n, nkv, capacity, HD, gpu, n_heads=nh)
    most = max(starts) + T
    pool.storage[:, :, :, :most].copy_(torch.randn(1, 2, n, most, nkv, HD, generator=g).half())
    slots = rng.sample(range(n), n)
    pool.lengths[torch.tensor(slots, device=gpu)] = torch.tensor(starts, device=gpu)
    given = torch.tensor(slots, device=gpu)
    if n > 8:
        given[4], given[n - 1] = -1, n + 7
        counts[4] = counts[n - 1] = 0
    q = torch.randn(n * T, nh * HD, generator=g).half()
    used = i32([max(c, 1) if s in (4, n - 1) else c for s, c in enumerate(counts)], gpu)
    cache = pool.tree_cache(parents, counts=used, slots=given)
    assert (*cache.form[:2], cache.form[3] > 0) == form
    for _ in range(2):
        out = torch.full((n * T, nh, HD), 7.0, device=gpu, dtype=torch.float16)
        cache.attend_qkv(q.to(gpu), 0, HD ** -0.5, out)
        if n > 8:
            check = [0 if s in (4, n - 1) else c for s, c in enumerate(counts)]
        else:
            check = counts
        check_attention(out.view(n, T, nh, HD), q.view(n, T, nh, HD), pool, 0, starts, parents,
                        check, slots, 7.0)


@pytest.mark.parametrize("n,T,nkv,long", [(100, 3, 2, 3900), (60, 9, 2, 4000), (40, 6, 6, 3000)])
def test_tree_attention_cut_one_long(gpu, n, T, nkv, long):
    """One long context among short ones: its keys go over many columns, which others end in."""
    say(f"tree attention, one of {n} sequences {long} tokens long, T={T} nkv={nkv}")
    rng = random.Random(n)
    starts = [rng.randint(0, 60) for _ in range(n)]
    starts[n // 3], starts[n - 1] = long, long // 3
    parents = trees(rng, n, T, "tree")
    from omniserver_amd.kv_cache import PreallocatedKVCache
    pool = PreallocatedKVCache(1, n, nkv, 4096, HD, gpu, n_heads=12)
    g = torch.Generator(device=gpu).manual_seed(n)
    pool.storage.normal_(generator=g)
    pool.lengths.copy_(torch.tensor(starts))
    q = torch.randn(n * T, 12 * HD, device=gpu, generator=g).half()
    cache = pool.tree_cache(parents)
    assert cache.form[3] > 0
    out = torch.full((n * T, 12, HD), 7.0, device=gpu, dtype=torch.float16)
    cache.attend_qkv(q, 0, HD ** -0.5, out)
    check_attention(out.view(n, T, 12, HD), q.cpu().view(n, T, 12, HD), pool, 0, starts, parents,
                    [T] * n, list(range(n)), 7.0)


def test_tree_attention_cut_keeps_infinities_apart(gpu):
    """As test_tree_attention_nodes_keep_to_themselves, where the rows' states are merged."""
    T, start = 30, 1500
    rng = random.Random(3)
    parents = trees(rng, 2, T, "tree")
    pool, g = make_pool(gpu, 1, 2, 12, 2, 2048, 5)
    pool.lengths.copy_(torch.tensor([start, 40]))
    clean = set(ref.lineage(parents[0], T - 1))
    for j in range(T):
        if j not in clean:
            pool.v[0][0, start + j] = math.inf if j % 2 else math.nan
            pool.k[0][0, start + j] = math.nan
    q = torch.randn(2 * T, 12 * HD, generator=g).half()
    cache = pool.tree_cache(parents)
    assert cache.form[3] > 0
    out = torch.zeros(2 * T, 12, HD, device=gpu, dtype=torch.float16)
    cache.attend_qkv(q.to(gpu), 0, HD ** -0.5, out)
    rows = [i for i in range(T) if set(ref.lineage(parents[0], i)) <= clean]
    want, mag, seen = ref.tree_attention(q.view(2, T, 12, HD), pool.k[0].cpu(), pool.v[0].cpu(),
                                         [start, 40], parents, [T, T], [0, 1], HD ** -0.5)
    v = pool.v[0].cpu().float()
    bound = ref.attention_bound(want, mag, seen, v[v.isfinite()].abs().max().item())
    err = (out.view(2, T, 12, HD).cpu().double() - want).abs() / bound
    assert len(rows) > 3 and err[0, rows].max().item() <= 1.0 and err[1].max().item() <= 1.0


def test_tree_plan(gpu):
    """Ancestors, positions and where the K/V goes; bad parents are roots, rows outside the pool
    and nodes past it go nowhere."""
    pool, _ = make_pool(gpu, 1, 3, 12, 2, 40, 1)
    pool.lengths.copy_(torch.tensor([5, 36, 0]))
    delta = torch.tensor([100, -3, 0], device=gpu)
    parents = [[-1, 0, 0, 1, 3, 2], [-1, 0, 1, 2, 3, 4], [-1, 0, 7, -9, 3, 5]]
    cache = pool.tree_cache(i32(parents, gpu), counts=[6, 5, 6], rope_delta=delta)
    m = cache.ancestors.view(3, 6).cpu().tolist()
    for s in range(3):
        for i in range([6, 5, 6][s]):
            assert m[s][i] == sum(1 << j for j in ref.lineage(parents[s], i)), (s, i)
    assert m[1][5] == 0
    pos = cache.positions.view(3, 3, 6).cpu()
    assert torch.equal(pos[0], pos[1]) and torch.equal(pos[0], pos[2])
    assert pos[0, 0].tolist() == [105, 106, 106, 107, 108, 107]
    assert pos[0, 1].tolist() == [33, 34, 35, 36, 37, 0]
    assert cache.token_slot.view(3, 6).cpu().tolist() == [[0] * 6, [1] * 4 + [-1] * 2, [2] * 6]
    assert cache.token_pos.view(3, 6).cpu()[0].tolist() == list(range(5, 11))
    pool.lengths.zero_()
    assert cache.starts.cpu().tolist() == [5, 36, 0]                # a copy
    far = pool.tree_cache(i32([[-1, 0]], gpu), slots=torch.tensor([9], device=gpu))
    assert far.token_slot.cpu().tolist() == [-1, -1]
    q = torch.randn(2, 16 * HD, device=gpu).half()
    out = torch.full((2, 12, HD), 3.0, device=gpu, dtype=torch.float16)
    far.attend_qkv(q, 0, 0.1, out)
    assert (out == 3.0).all()


@pytest.mark.parametrize("T,start", [(8, 20), (40, 100), (64, 0), (6, 2050)])
def test_tree_attention_nodes_keep_to_themselves(gpu, T, start):
    """NaN and infinities in other branches, in the padding and behind the last node reach no
    row that does not attend to them."""
    say(f"tree attention with NaN off the path, T={T} start={start}")
    rng = random.Random(T)
    parents = trees(rng, 1, T, "tree")
    counts = [T - 2]
    pool, g = make_pool(gpu, 1, 1, 12, 2, start + T + 70, T)
    pool.lengths[0] = start
    clean = set(ref.lineage(parents[0], T - 3))
    bad = [j for j in range(T) if j not in clean]
    for n, j in enumerate(bad):
        pool.k[0][0, start + j] = [math.nan, math.inf, -math.inf][n % 3]
        pool.v[0][0, start + j] = [math.inf, math.nan, -math.inf][n % 3]
    pool.k[0][0, start + T:] = math.nan
    pool.v[0][0, start + T:] = math.inf
    q = torch.randn(T, 12 * HD, generator=g).half()
    out = torch.zeros(T, 12, HD, device=gpu, dtype=torch.float16)
    pool.tree_cache(parents, counts=counts).attend_qkv(q.to(gpu), 0, HD ** -0.5, out)
    rows = [i for i in range(T - 2) if set(ref.lineage(parents[0], i)) <= clean]
    want, mag, seen = ref.tree_attention(q.view(1, T, 12, HD), pool.k[0].cpu(), pool.v[0].cpu(),
                                         [start], parents, counts, [0], HD ** -0.5)
    v = pool.v[0].cpu().float()
    bound = ref.attention_bound(want, mag, seen, v[v.isfinite()].abs().max().item())
    err = ((out.cpu().double() - want[0]).abs() / bound[0])[rows]
    assert len(rows) > 2 and err.max().item() <= 1.0
    tainted = [i for i in range(T - 2) if i not in rows]
    assert not out[tainted].isfinite().all()


def test_tree_attention_past_max_len(gpu):
    """Nodes behind the pool's end are not stored and not seen; the others are as ever."""
    pool, g = make_pool(gpu, 1, 2, 12, 2, 50, 3)
    starts, T = [47, 50], 8
    pool.lengths.copy_(torch.tensor(starts))
    parents = trees(random.Random(2), 2, T, "tree")
    before = pool.storage.clone()
    q, k, v = (torch.randn(2 * T, h, HD, generator=g).half().to(gpu) for h in (12, 2, 2))
    cache = pool.tree_cache(parents)
    out = cache.flash_prefill(q, k, v, 0, HD ** -0.5)
    for i in range(3):
        assert torch.equal(pool.k[0][0, 47 + i], k[i]) and torch.equal(pool.v[0][0, 47 + i], v[i])
    assert torch.equal(pool.storage[:, :, 0, :47], before[:, :, 0, :47])
    assert torch.equal(pool.storage[:, :, 1], before[:, :, 1])
    check_attention(out.view(2, T, 12, HD), q.cpu().view(2, T, 12, HD), pool, 0, starts, parents,
                    [T, T], [0, 1], 0.0)


def test_tree_attention_large_pool(gpu):
    """Rows whose offsets pass 32 bits, byte and element counts alike."""
    from omniserver_amd.kv_cache import PreallocatedKVCache
    T, L, rows, max_len = 16, 600, 36, 1 << 17
    say(f"tree attention in a pool of {rows * max_len * 512} elements a tensor")
    big = PreallocatedKVCache(1, rows, 4, max_len, HD, gpu, n_heads=28)
    small, g = make_pool(gpu, 1, 1, 28, 4, 640, 5)
    slot = rows - 1
    assert slot * max_len * 4 * HD > 1 << 31
    big.storage[0, :, slot, :640] = small.storage[0, :, 0]
    big.lengths[slot], small.lengths[0] = L, L
    parents = trees(random.Random(1), 1, T, "tree")
    q, k, v = (torch.randn(T, h, HD, generator=g).half().to(gpu) for h in (28, 4, 4))
    a = big.tree_cache(parents, slots=[slot])
    b = small.tree_cache(parents)
    oa, ob = a.flash_prefill(q, k, v, 0, 0.09), b.flash_prefill(q, k, v, 0, 0.09)
    # the same sums in another order: two probabilities' and two outputs' half steps
    assert (oa.float() - ob.float()).abs().max().item() <= 2.0 ** -9 * 4.5
    path = i32([[0, 2, 5, 9] + [-1] * (T - 4)], gpu)
    for c in (a, b):
        c.accept(path, i32([4], gpu))
    assert torch.equal(big.storage[0, :, slot, :640], small.storage[0, :, 0])
    assert big.lengths[slot].item() == L + 4


def test_tree_attention_strides_and_streams(gpu):
    """Query rows of a wider buffer, work on a side stream, a prefix of the longest scores."""
    pool, g = make_pool(gpu, 1, 2, 12, 2, 300, 9)
    pool.lengths.copy_(torch.tensor([100, 217]))
    parents = trees(random.Random(5), 2, 10, "tree")
    wide = torch.randn(20, 12 * HD + 40, generator=g).half().to(gpu)
    pool.k[0][:, 50] *= 12.0                       # one key takes nearly all of the mass
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cache = pool.tree_cache(parents)
        out = torch.zeros(20, 12, HD, device=gpu, dtype=torch.float16)
        cache.attend_qkv(wide, 0, HD ** -0.5, out)
    torch.cuda.current_stream().wait_stream(side)
    q = wide[:, :12 * HD].cpu().reshape(2, 10, 12, HD)
    check_attention(out.view(2, 10, 12, HD), q, pool, 0, [100, 217], parents, [10, 10], [0, 1], 0.0)
    with pytest.raises(ValueError):
        cache.attend_qkv(wide[:10], 0, 0.1, out)
    with pytest.raises(ValueError):
        cache.attend_qkv(wide, 0, 0.1, out[:10])
    with pytest.raises(TypeError):
        cache.attend_qkv(wide.float(), 0, 0.1, out)
    with pytest.raises(RuntimeError):
        cache.attend_qkv(wide, 0, -0.1, out)
    with pytest.raises(RuntimeError):                    # off a 16-byte boundary
        cache.attend_qkv(wide.view(-1)[4:4 + 20 * 1536].view(20, 1536), 0, 0.1, out)


def test_tree_attention_far_rows(gpu):
    """Query rows further apart than 32-bit offsets reach."""
    pool, g = make_pool(gpu, 1, 1, 2, 1, 64, 12)
    pool.lengths[0] = 33
    q = torch.randn(2, 2 * HD, generator=g).half()
    far = (1 << 31) + 8
    room = torch.empty(far + 2 * HD, device=gpu, dtype=torch.float16)
    rows = room.as_strided((2, 2 * HD), (far, 1))
    rows.copy_(q.to(gpu))
    cache = pool.tree_cache([[-1, 0]])
    out = torch.zeros(2, 2, HD, device=gpu, dtype=torch.float16)
    cache.attend_qkv(rows, 0, HD ** -0.5, out)
    check_attention(out.view(1, 2, 2, HD), q.view(1, 2, 2, HD), pool, 0, [33], [[-1, 0]], [2], [0],
                    0.0)


def test_pool_off_the_current_device(gpu):
    """Whatever the tensors are, a pool elsewhere is refused before a launch."""
    pool, _ = make_pool(gpu, 1, 2, 12, 2, 64, 13)
    parents = i32([[-1, 0], [-1, 0]], gpu)
    cache = pool.tree_cache(parents)
    rows = torch.zeros(4, 16 * HD, device=gpu, dtype=torch.float16)
    q = rows[:, :12 * HD].view(4, 12, HD)
    kv = rows[:, 12 * HD:14 * HD].view(4, 2, HD)
    pool.storage, pool.lengths = pool.storage.cpu(), pool.lengths.cpu()
    with pytest.raises(RuntimeError):
        pool.tree_cache(parents)
    with pytest.raises(RuntimeError):
        cache.attend_qkv(rows, 0, 0.1, torch.zeros(4, 12, HD, device=gpu, dtype=torch.float16))
    with pytest.raises(RuntimeError):
        cache.flash_prefill(q, kv, kv, 0, 0.1)
    with pytest.raises(RuntimeError):
        cache.accept(i32([[0, -1]] * 2, gpu), i32([1, 1], gpu))


# ----------------------------------------------------------------------------- verification
def rows_like_a_model(g, n, T, V, dtype, std=2.0):
    x = torch.randn(n, T, V, generator=g) * std
    top = torch.randint(0, V, (n, T, min(V, 6)), generator=g)
    x.scatter_(2, top, 8 + 4 * torch.rand(top.shape, generator=g))
    return x.to(dtype)


def check_verify(gpu, logits, tokens, u, temps, parents=None, draft=None, counts=None, scalar=None):
    from omniserver_amd.speculative import verify
    d = lambda x, t: None if x is None else torch.as_tensor(x, dtype=t).to(gpu)  # noqa: E731
    got = verify(logits.to(gpu), d(tokens, torch.int64), None if u is None else d(u, torch.float32),
                 scalar if scalar is not None else d(temps, torch.float32),
                 parents=d(parents, torch.int32),
                 draft_logits=None if draft is None else draft.to(gpu), counts=d(counts, torch.int32))
    n, T = logits.shape[:2]
    temps = torch.tensor(temps, dtype=torch.float32).tolist()
    uu = [[0.0] * T] * n if u is None else torch.as_tensor(u, dtype=torch.float32).tolist()
    want = ref.verify(logits, torch.as_tensor(tokens).tolist(), uu, temps,
                      None if parents is None else parents, draft, counts)
    assert got.emitted.cpu().tolist() == want[2].tolist()
    assert got.path.cpu().tolist() == want[0].tolist()
    assert got.tokens.cpu().tolist() == want[1].tolist()
    return want[2]


VERIFY = [
    # n, T, V, dtype, mode
    (1, 1, 1, "float32", "tree"), (1, 1, 151936, "float16", "tree"), (3, 2, 2, "float16", "tree"),
    (4, 8, 7, "bfloat16", "tree"), (8, 8, 1000, "float16", "tree"), (5, 16, 4096, "float32", "tree"),
    (6, 13, 4097, "bfloat16", "tree"), (3, 64, 333, "float16", "tree"),
    (4, 9, 32003, "float32", "tree"), (4, 8, 151936, "float16", "tree"),
    (2, 5, 151936, "bfloat16", "star"), (9, 6, 1000, "float16", "plain chain"),
    (2, 2, 1, "float16", "chain"), (6, 8, 9, "float32", "chain"), (8, 8, 1000, "float16", "chain"),
    (5, 5, 8193, "bfloat16", "chain"), (4, 8, 32003, "float32", "chain"),
    (4, 8, 151936, "float16", "chain"), (2, 64, 2000, "float16", "chain"),
]


@pytest.mark.parametrize("n,T,V,dtype,mode", VERIFY)
def test_verify(gpu, n, T, V, dtype, mode):
    say(f"verify n={n} T={T} V={V} {dtype} {mode}")
    rng = random.Random(T * V)
    g = torch.Generator().manual_seed(n + T + V)
    dtype = getattr(torch, dtype)
    for ragged in (False, True):
        logits = rows_like_a_model(g, n, T, V, dtype)
        temps = [rng.choice([0.0, rng.uniform(0.3, 1.5), 1.0]) for _ in range(n)]
        counts = [rng.randint(0, T) for _ in range(n)] if ragged else None
        u = torch.rand(n, T, generator=g)
        tokens = torch.randint(0, V, (n, T), generator=g)
        if mode == "chain":
            draft = (logits[:, :T - 1].float()
                     + 0.7 * torch.randn(n, T - 1, V, generator=g)).to(dtype)
            q = torch.softmax(draft.double(), -1).reshape(-1, V)
            if T > 1:
                tokens[:, 1:] = torch.multinomial(q, 1, generator=g).view(n, T - 1)
            total = check_verify(gpu, logits, tokens, u, temps, draft=draft, counts=counts)
        else:
            parents = trees(rng, n, T, "tree" if mode == "tree" else
                            "star" if mode == "star" else "chain")
            for s in range(n):                       # mostly the target's own best tokens
                for i in range(1, T):
                    rank = sum(parents[s][j] == parents[s][i] for j in range(i))
                    best = logits[s, parents[s][i]].float().topk(min(V, rank + 1)).indices
                    if rng.random() < 0.8:
                        tokens[s, i] = best[-1]
            total = check_verify(gpu, logits, tokens, u, temps,
                                 parents=None if mode == "plain chain" else parents, counts=counts)
    say(f"  emitted {total.tolist()}")


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_verify_borders(gpu, dtype):
    """Random numbers 0 and just below 1, tokens proposed twice or outside the vocabulary, masked
    rows, NaN and infinities, nothing left to draw from."""
    g = torch.Generator().manual_seed(3)
    V, T = 40, 6
    below = 1.0 - 2.0 ** -24
    rows, toks, us, temps, pars = [], [], [], [], []

    def case(row, tok, u, temp=0.8, par=(-1, 0, 0, 0, 1, 2)):
        rows.append(row)
        toks.append(tok)
        us.append(u)
        temps.append(temp)
        pars.append(list(par))

    base = torch.randn(T, V, generator=g)
    only = torch.full((T, V), -math.inf)
    only[:, 17] = 0.5
    two = only.clone()
    two[:, 30] = 0.25
    nan = base.clone()
    nan[:, ::3] = math.nan
    inf = base.clone()
    inf[:, 5] = math.inf
    inf2 = inf.clone()
    inf2[:, 33] = math.inf
    none = torch.full((T, V), -math.inf)
    tie = torch.zeros(T, V)
    low = base.clone()
    low[:, 20:] = torch.finfo(torch.float32).min
    for temp in (0.0, 0.8, 0.01, 50.0):
        for row in (base, only, two, nan, inf, inf2, none, tie, low):
            for u0 in (0.0, 0.37, below):
                for u1 in (0.0, 0.5, below):
                    case(row, [0, 17, 17, 30, 5, -1], [u0] + [u1] * 5, temp)
                    case(row, [0, V, 5, 0, 3, 17], [u0] + [u1] * 5, temp)
    logits = torch.stack(rows).to(dtype)
    check_verify(gpu, logits, toks, us, temps, parents=pars)
    # chains against their own distribution, another one, a masked one and an empty one
    draft = torch.stack([(base, two, only, none, nan, inf)[k % 6][:T - 1] for k in range(len(rows))]).to(dtype)
    check_verify(gpu, logits, toks, us, temps, draft=draft)
    check_verify(gpu, logits, toks, us, temps, draft=logits[:, :T - 1].contiguous())


def test_verify_open_tests(gpu):
    """Random numbers on the border of a test, where the rows' 32-bit sums leave it open: the 64-bit
    sum decides, as the oracle does, for trees and chains, at the first node and further down."""
    g = torch.Generator().manual_seed(12)
    n, T, V = 48, 4, 9001
    logits = rows_like_a_model(g, n, T, V, torch.float16)
    draft = (logits[:, :T - 1].float() + 0.3 * torch.randn(n, T - 1, V, generator=g)).half()
    tokens = logits.float().argmax(-1).roll(1, 1)
    p = torch.softmax(logits.double(), -1)
    q = torch.softmax(draft.double(), -1)
    at = tokens[:, 1:, None]
    px, qx = p[:, :-1].gather(2, at)[..., 0], q.gather(2, at)[..., 0]
    for d, parents in ((None, [[-1, 0, 1, 2]] * n), (draft, None)):
        border = px / (1.0 if d is None else qx)
        u = torch.rand(n, T, generator=g)
        for k in range(1, T):
            # on one node a sequence the nearest fp32 number to the border, or its neighbours
            u[:, 1:] = torch.where(torch.arange(1, T) < k, torch.zeros(()), u[:, 1:])
            near = border[:, k - 1].float().clamp(max=1 - 2.0 ** -24)
            step = torch.tensor([-1, 0, 1])[torch.arange(n) % 3]
            u[:, k] = torch.where(step == 0, near, torch.nextafter(near, near + step.float()))
            u[:, k].clamp_(0, 1 - 2.0 ** -24)
            check_verify(gpu, logits, tokens, u, [1.0] * n, parents=parents, draft=d)


def test_verify_scalars_strides_and_repeats(gpu):
    from omniserver_amd.speculative import chain_parents, verify
    g = torch.Generator().manual_seed(8)
    n, T, V = 5, 7, 2003
    logits = rows_like_a_model(g, n, T, V, torch.float16)
    tokens = logits.float().argmax(-1).roll(1, 1)           # the greedy chain: all stand
    parents = chain_parents(n, T, "cpu").tolist()
    total = check_verify(gpu, logits, tokens, None, [0.0] * n, scalar=0.0)
    assert total.tolist() == [T] * n
    u = torch.rand(n, T, generator=g)
    for scalar in (0.0, 0.7):
        check_verify(gpu, logits, tokens, u, [scalar] * n, parents=parents, scalar=scalar)
    wide = torch.zeros(n, T + 2, V + 5, dtype=torch.float16)   # rows off every alignment
    wide[:, 1:T + 1, 3:V + 3] = logits
    view = wide.to(gpu)[:, 1:T + 1, 3:V + 3]
    args = (tokens.to(gpu), u.to(gpu), 0.7)
    a, b = verify(view, *args), verify(logits.to(gpu), *args)
    flip = verify(logits.to(gpu).flip(0).contiguous(), tokens.flip(0).contiguous().to(gpu),
                  u.flip(0).contiguous().to(gpu), 0.7)
    for x, y, z in zip(a, b, flip):
        assert torch.equal(x, y) and torch.equal(x, z.flip(0))


def test_verify_emits_the_target_distribution(gpu):
    """First tokens over a grid of random numbers, shares against the target's probabilities: a
    border moves at most a share of 1 / m for each number on the grid."""
    from omniserver_amd.speculative import verify
    logits = torch.tensor([0.3, -1.0, 1.2, 0.0, -0.4, 0.9])
    V = logits.numel()
    p = ref.weights(logits, 1.0)
    m = 64
    us = ((torch.arange(m).float() + 0.5) / m)
    grid = torch.cartesian_prod(us, us, us).to(gpu)                     # u_0, u_1, u_2
    n = grid.shape[0]
    rows = logits.to(gpu).expand(n, 3, V)
    tokens = torch.tensor([0, 2, 5], device=gpu).repeat(n, 1)
    got = verify(rows, tokens, grid, 1.0, parents=i32([-1, 0, 0], gpu).repeat(n, 1))
    share = torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double() / n
    assert (share - p).abs().max() <= 3 / m
    draft = torch.tensor([1.0, 0.2, -0.5, 0.1, -2.0, 0.0])
    q = ref.weights(draft, 1.0)
    grid = torch.cartesian_prod(us, us).to(gpu)
    n = grid.shape[0]
    share = torch.zeros(V, dtype=torch.float64)
    for x in range(V):
        tokens = torch.tensor([0, x], device=gpu).repeat(n, 1)
        got = verify(rows[:n, :2], tokens, grid, 1.0, draft_logits=draft.to(gpu).expand(n, 1, V))
        share += q[x] * torch.bincount(got.tokens[:, 0].cpu(), minlength=V).double() / n
    assert (share - p).abs().max() <= 2 / m


# ----------------------------------------------------------------------------- acceptance
@pytest.mark.parametrize("n,T,nkv,layers", [(1, 1, 2, 1), (3, 8, 2, 3), (5, 26, 2, 28), (2, 64, 16, 2),
                                            (32, 9, 4, 2)])
def test_accept(gpu, n, T, nkv, layers):
    say(f"accept n={n} T={T} nkv={nkv} layers={layers}")
    rng = random.Random(n + T)
    starts = [rng.randint(0, 90) for _ in range(n)]
    pool, _ = make_pool(gpu, layers, n + 1, 2 * nkv, nkv, 90 + T, T)
    slots = rng.sample(range(n + 1), n)
    for s, L in zip(slots, starts):
        pool.lengths[s] = L
    before, old = pool.storage.cpu(), pool.lengths.cpu().tolist()
    cache = pool.tree_cache(trees(rng, n, T, "chain"), slots=slots)
    path, emitted = [], []
    for _ in range(n):
        k = rng.randint(0, T)
        nodes = sorted(rng.sample(range(T), k)) if rng.random() < 0.7 else list(range(k))
        path.append(nodes + [-1] * (T - k))
        emitted.append(k)
    cache.accept(i32(path, gpu), i32(emitted, gpu))
    want, lengths = ref.accept(before, starts, path, emitted, slots)
    assert torch.equal(pool.storage.cpu(), want)
    for row, L in enumerate(old):
        assert pool.lengths[row].item() == lengths.get(row, L)


def test_accept_borders(gpu):
    """The pool's end, rows outside it, paths that do not ascend, more tokens than nodes."""
    pool, _ = make_pool(gpu, 2, 6, 12, 2, 60, 4)
    starts = [56, 60, 10, 20, 30, 40]
    pool.lengths.copy_(torch.tensor(starts))
    before = pool.storage.cpu()
    slots = torch.tensor([0, 1, 2, 3, 4, 77], device=gpu)
    cache = pool.tree_cache(i32([[i - 1 for i in range(6)]] * 6, gpu), slots=slots)
    path = [[0, 2, 3, 5, -1, -1], [0, 1, 2, 3, 4, 5], [0, 3, 2, 5, -1, -1], [1, 2, 9, 10, 11, 12],
            [0, 1, 2, 3, 4, 5], [1, 2, 3, 4, 5, -1]]
    emitted = [4, 6, 4, 4, 50, 4]
    cache.accept(i32(path, gpu), i32(emitted, gpu))
    want, lengths = ref.accept(before, starts[:5], path[:5], [4, 6, 4, 4, 6], [0, 1, 2, 3, 4])
    assert torch.equal(pool.storage.cpu(), want)
    assert pool.lengths.cpu().tolist() == [lengths[s] for s in range(5)] + [40]
    assert lengths == {0: 59, 1: 60, 2: 12, 3: 22, 4: 36}
    with pytest.raises(ValueError):
        cache.accept(i32(path[:5], gpu), i32(emitted, gpu))
    with pytest.raises(TypeError):
        cache.accept(i32(path, gpu).long(), i32(emitted, gpu))


# ----------------------------------------------------------------------------- together
def spec_step(pool, layers, parents, tokens, u, temps, q, k, v, logits):
    """What a step makes of a drafted tree beside the model's own products."""
    from omniserver_amd.speculative import verify
    cache = pool.tree_cache(parents)
    outs = [cache.flash_prefill(q, k, v, l, HD ** -0.5) for l in range(layers)]
    got = verify(logits, tokens, u, temps, parents=parents)
    cache.accept(got.path, got.emitted)
    return outs, got


@pytest.mark.parametrize("capacity", [200, 2048])      # keys whole, and cut with a merge
def test_step_in_graphs(gpu, capacity):
    """Two captured steps of one pool, replayed in turn with eager work between the replays, give
    what the eager step gives."""
    n, T, layers, V = 3, 12, 2, 5003
    pool, g = make_pool(gpu, layers, n, 12, 2, capacity, 6)
    assert (pool.tree_cache([[-1] * T] * n).form[3] > 0) == (capacity > 512)
    rng = random.Random(6)
    starts = torch.tensor([30, 0, 111], device=gpu)
    sets = []
    for _ in range(2):
        parents = i32(trees(rng, n, T, "tree"), gpu)
        logits = rows_like_a_model(g, n, T, V, torch.float16).to(gpu)
        tokens = logits.float().argmax(-1).gather(1, parents.long().clamp(min=0))
        u = torch.rand(n, T, generator=g).to(gpu)
        temps = torch.tensor([0.0, 0.9, 1.3], device=gpu)
        q, k, v = (torch.randn(n * T, h, HD, generator=g).half().to(gpu) for h in (12, 2, 2))
        sets.append((parents, tokens, u, temps, q, k, v, logits))
    clean = pool.storage.clone()

    def reset():
        pool.storage.copy_(clean)
        pool.lengths[:n] = starts

    eager = []
    for args in sets:
        reset()
        outs, got = spec_step(pool, layers, *args)
        eager.append([x.clone() for x in (*outs, *got, pool.storage, pool.lengths)])
    graphs = []
    for args in sets:
        reset()
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs, got = spec_step(pool, layers, *args)
        graphs.append((gr, [*outs, *got, pool.storage, pool.lengths]))
    for turn in range(3):
        for (gr, res), want in zip(graphs, eager):
            reset()
            gr.replay()
            torch.cuda.synchronize()
            for x, y in zip(res, want):
                assert torch.equal(x, y), turn
            spec_step(pool, layers, *sets[turn % 2])


# ----------------------------------------------------------------------------- the runner
def corrupt(rng, tokens, vocab, rate):
    return [rng.randrange(vocab) if rng.random() < rate else t for t in tokens]


@pytest.mark.parametrize("quant,use_graph", [(None, False), (None, True), ("gptq", True)])
def test_runner_speculates_greedily(gpu, quant, use_graph):
    """Drafts taken from the decoded stream, some tokens replaced, as chains and as trees with
    the right token on one branch: every emitted token the oracle's wherever it is decisive, more
    than one a step, and decode() goes on from there."""
    from omniserver_amd import synth
    from omniserver_amd.request import Request, SamplingParams, Sequence
    from omniserver_amd.runner import NativeQwenVLRunner
    from tests.helpers import (check_stream, compare_logits, oracle_from_fp16, oracle_from_gptq,
                               oracle_stream_logits, record_sampled_logits)
    say(f"runner speculates quant={quant} use_graph={use_graph}")
    shape = synth.DecoderShape()
    gen = synth.gptq_decoder if quant else synth.fp16_decoder
    w = gen(shape, seed=5, num_layers=2)
    prompts = [synth.random_ids(L, shape.vocab_size, 5, f"p{L}").tolist() for L in (40, 17, 65)]
    steps = 14

    def start():
        r = NativeQwenVLRunner(max_running=4, max_len=256, use_graph=use_graph, weights=w,
                               quant=quant)
        seen = record_sampled_logits(r)
        seqs = [Sequence(Request(prompt=p, sampling=SamplingParams(max_new_tokens=steps)))
                for p in prompts]
        for s in seqs:
            r.tokenize(s)
        r.prefill(seqs)
        return r, seqs, seen

    plain, ref_seqs, seen = start()
    while any(s.num_output_tokens < steps for s in ref_seqs):
        plain.decode(ref_seqs)
    streams = [list(s.output_token_ids) for s in ref_seqs]
    runner, seqs, _ = start()
    rng = random.Random(1)
    gained = calls = 0
    while min(s.num_output_tokens for s in seqs) < steps - 5:
        drafts = []
        for b, s in enumerate(seqs):
            at = s.num_output_tokens
            right = streams[b][at:at + 3] if s.output_token_ids == streams[b][:at] else [1, 2, 3]
            if calls % 3 == 2:                       # two branches, the right one second
                wrong = corrupt(rng, right, shape.vocab_size, 1.0)
                drafts.append((wrong + right, [-1] + list(range(len(right) - 1))
                               + [-1] + list(range(len(right), 2 * len(right) - 1))))
            else:
                drafts.append(corrupt(rng, right[:rng.randint(0, 3)], shape.vocab_size, 0.2))
        before = [s.num_output_tokens for s in seqs]
        got = runner.speculate(seqs, drafts)
        assert got == [s.num_output_tokens - x for s, x in zip(seqs, before)]
        assert runner.pool.lengths[:3].tolist() == runner._kv_len
        gained += sum(got)
        calls += 1
    runner.decode(seqs)
    orc = oracle_from_gptq(w, shape) if quant else oracle_from_fp16(w, shape)
    rows = [oracle_stream_logits(orc, p, s.output_token_ids, 256) for p, s in zip(prompts, seqs)]
    err, _ = compare_logits(seen[0], torch.stack([r[0] for r in rows]))
    total = sum(check_stream(s.output_token_ids, r, 2 * err + 1e-3, 0, f"seq {b}")
                for b, (s, r) in enumerate(zip(seqs, rows)))
    assert total >= sum(s.num_output_tokens for s in seqs) // 2
    say(f"  {gained} tokens in {calls} calls for 3 sequences")
    assert gained > 1.5 * 3 * calls


def test_runner_speculates_sampled(gpu):
    """Sampled and greedy sequences, chains with draft logits and proposals without: graph and
    eager steps give the same tokens for the same random numbers; a sequence given in another order
    than its slot gets its own draft."""
    from omniserver_amd import synth
    from omniserver_amd.request import Request, SamplingParams, Sequence
    from omniserver_amd.runner import NativeQwenVLRunner
    say("runner speculates, sampled")
    shape = synth.DecoderShape()
    w = synth.fp16_decoder(shape, seed=6, num_layers=2)
    V = shape.vocab_size
    results = []
    for use_graph in (False, True):
        r = NativeQwenVLRunner(max_running=4, max_len=128, use_graph=use_graph, weights=w)
        seqs = [Sequence(Request(prompt=synth.random_ids(20 + b, V, 6, f"s{b}").tolist(),
                                 sampling=SamplingParams(max_new_tokens=60, temperature=t)))
                for b, t in enumerate((0.8, 0.0, 1.2))]
        for s in seqs:
            r.tokenize(s)
        torch.manual_seed(9)
        r.prefill(seqs)
        g = torch.Generator().manual_seed(4)
        shuffled = [seqs[2], seqs[0], seqs[1]]
        for step in range(5):
            draft = (torch.randn(3, 3, V, generator=g) * 2).half()
            tokens = torch.multinomial(torch.softmax(draft.float(), -1).view(9, V), 1,
                                       generator=g).view(3, 3).tolist()
            r.speculate(shuffled, tokens, draft_logits=draft.to(gpu))
            r.speculate(shuffled, [(t, [-1, -1, 0]) for t in tokens])
        r.decode(seqs)
        results.append([list(s.output_token_ids) for s in seqs])
        assert r.pool.lengths[:3].tolist() == r._kv_len
    assert results[0] == results[1]


def test_runner_speculate_limits(gpu):
    """The pool's end, the token limit and a stop token inside a draft; refusals."""
    from omniserver_amd import synth
    from omniserver_amd.request import Request, SamplingParams, Sequence, Status
    from omniserver_amd.runner import NativeQwenVLRunner
    shape = synth.DecoderShape()
    w = synth.fp16_decoder(shape, seed=7, num_layers=1)
    r = NativeQwenVLRunner(max_running=2, max_len=48, use_graph=False, weights=w)
    mk = lambda L, **kw: Sequence(Request(  # noqa: E731
        prompt=synth.random_ids(L, shape.vocab_size, 7, f"l{L}").tolist(),
        sampling=SamplingParams(**kw)))
    a, b = mk(45, max_new_tokens=99), mk(9, max_new_tokens=3)
    for s in (a, b):
        r.tokenize(s)
    r.prefill([a, b])
    for bad in ([[1]], [[1], [2], [3]], [[1], [shape.vocab_size]], [[1], [-1]],
                [[1] * 64, [1]], [([1, 2], [-1, 1]), [1]], [([1, 2], [-1]), [1]]):
        with pytest.raises(ValueError):
            r.speculate([a, b], bad)
    with pytest.raises(ValueError):
        r.speculate([a, b], [[1], [2]], draft_logits=torch.zeros(2, 2, shape.vocab_size))
    with pytest.raises(AssertionError):
        r.speculate([b], [[1]])
    assert r.speculate([], []) == []
    # greedy continuation of both, by decoding copies of them
    twin = NativeQwenVLRunner(max_running=2, max_len=64, use_graph=False, weights=w)
    ta, tb = mk(45, max_new_tokens=99), mk(9, max_new_tokens=99)
    for s in (ta, tb):
        twin.tokenize(s)
    twin.prefill([ta, tb])
    for _ in range(5):
        twin.decode([ta, tb])
    got = r.speculate([a, b], [ta.output_token_ids[1:6], tb.output_token_ids[1:6]])
    assert got[0] <= 3 and r._kv_len[0] <= 48          # positions 45, 46, 47
    assert b.num_output_tokens <= 3
    if got == [3, 2]:                                   # no near tie on the way
        assert b.status == Status.FINISHED
        with pytest.raises(RuntimeError):
            r.speculate([a, b], [[], []])


def test_runner_speculate_without_a_token(gpu, monkeypatch):
    """A sequence that nothing can be drawn for is an error, and the others' lengths still hold."""
    from omniserver_amd import runner as runner_mod
    from omniserver_amd import synth
    from omniserver_amd.request import Request, SamplingParams, Sequence
    shape = synth.DecoderShape()
    r = runner_mod.NativeQwenVLRunner(max_running=2, max_len=48, use_graph=False,
                                      weights=synth.fp16_decoder(shape, seed=8, num_layers=1))
    seqs = [Sequence(Request(prompt=synth.random_ids(L, shape.vocab_size, 8, f"n{L}").tolist(),
                             sampling=SamplingParams(max_new_tokens=9))) for L in (5, 11)]
    for s in seqs:
        r.tokenize(s)
    r.prefill(seqs)
    verify = runner_mod.verify

    def without(*a, **kw):
        v = verify(*a, **kw)
        v.tokens[0].fill_(-1)
        return v

    monkeypatch.setattr(runner_mod, "verify", without)
    with pytest.raises(RuntimeError):
        r.speculate(seqs, [[1, 2], [3, 4]])
    assert r.pool.lengths[:2].tolist() == r._kv_len[:2]
