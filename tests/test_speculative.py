"""Speculative decoding's operators without a GPU: refusals before any launch, and the 64-bit
oracle's own properties (what is emitted is distributed as the target)."""

import ctypes

import pytest
import torch

from oracle import speculative_ref as ref

P = ctypes.c_void_p(16)          # never read: the checks fail first


def pool(max_batch=4, max_len=128, **kw):
    from omniserver_amd.kv_cache import PreallocatedKVCache
    return PreallocatedKVCache(2, max_batch, 2, max_len, 128, "cpu", n_heads=12, **kw)


def test_tree_attention_refusals():
    from omniserver_amd._lib import lib

    def rc(q=P, q_stride=1536, rows=4, max_len=256, plan=P, n=2, nodes=8, out=P, out_stride=1536,
           nh=12, nkv=2, hd=128, scale=0.1, form=(64, 4), columns=4, least=0, ws=None, floats=0):
        return lib().omni_tree_attention(q, q_stride, P, P, rows, max_len, P, n, nodes, out,
                                         out_stride, nh, nkv, hd, scale, *form, columns, least,
                                         plan, ws, floats, None)

    assert rc(n=-1) == rc(nodes=0) == rc(nh=0) == rc(nkv=0) == rc(rows=0) == rc(max_len=0) == -1
    assert rc(nodes=65) == rc(hd=64) == rc(nh=13) == -2
    assert rc(scale=0.0) == rc(scale=-1.0) == rc(scale=float("nan")) == rc(scale=1e-39) == -2
    assert rc(scale=float("inf")) == rc(scale=2.5e38) == -2       # x log2(e) is infinite
    big = {"nodes": 1, "q_stride": 1 << 31, "out_stride": (1 << 31) - 8}
    assert rc(nh=1 << 17, nkv=1, **big) == -2
    assert rc(n=1 << 24, columns=1 << 25) == rc(columns=1 << 15, least=1) == -2
    assert rc(n=1 << 12, columns=1 << 13, max_len=(1 << 31) - 1) == -2
    assert rc(q_stride=1535) == rc(q_stride=1532) == rc(out_stride=8) == rc(out_stride=1540) == -1
    assert rc(form=(64, 2)) == rc(form=(128, 1)) == rc(form=(0, 0)) == rc(form=(16, 16)) == -1
    assert rc(columns=0) == rc(columns=5) == rc(least=-1) == -1
    assert rc(q=None) == rc(out=None) == rc(plan=None) == -1
    assert rc(q=ctypes.c_void_p(24)) == rc(out=ctypes.c_void_p(8)) == rc(plan=ctypes.c_void_p(4)) == -1
    cut = {"least": 1, "columns": 3, "nodes": 16, "form": (64, 4)}
    assert rc(**cut) == rc(**cut, ws=P, floats=3 * 2 * 2 * 64 * 132 - 1) == -1
    assert rc(n=0) == 0


def test_tree_plan_and_row_write_refusals():
    from omniserver_amd._lib import lib

    def plan(parents=P, lengths=P, n=2, nodes=8, rows=4, max_len=64, slots=None, starts=P, nkv=2,
             form=(64, 4), columns=4, least=0, ints=1 << 20):
        return lib().omni_tree_plan(parents, None, slots, lengths, None, n, nodes, rows, max_len,
                                    starts, P, P, P, P, nkv, *form, columns, least, P, ints, None)

    assert plan(n=-1) == plan(nodes=0) == plan(rows=0) == plan(max_len=0) == plan(nkv=0) == -1
    assert plan(n=5, columns=10) == plan(columns=3) == plan(columns=0) == plan(least=-1) == -1
    assert plan(form=(128, 4)) == plan(ints=4 * 2 + 8 * 4 + 2 * 2 * 2 - 1) == -1
    assert plan(columns=1 << 24, least=1) == plan(nodes=65) == -2
    assert plan(columns=32767, least=1, max_len=(1 << 31) - 1) == -2
    assert plan(n=1 << 24, rows=1 << 24, columns=1 << 25) == -2
    assert plan(parents=None) == plan(lengths=None) == plan(starts=None) == -1
    assert plan(n=0) == 0

    def write(k=P, ks=256, vs=256, kc=P, slots=P, rows=4, max_len=64, halfs=256, tokens=3):
        return lib().omni_kv_write_rows(k, ks, P, vs, kc, P, slots, P, rows, max_len, halfs,
                                        tokens, None)

    assert write(tokens=-1) == write(rows=0) == write(max_len=0) == write(halfs=0) == -1
    assert write(halfs=250) == write(ks=260) == write(vs=257) == -2
    assert write(ks=248) == write(vs=0) == write(k=None) == write(slots=None) == -1
    assert write(kc=ctypes.c_void_p(8)) == -1
    assert write(tokens=0) == 0


def test_kv_accept_refusals():
    from omniserver_amd._lib import lib

    def rc(kv=P, layers=2, rows=4, max_len=64, halfs=256, starts=P, path=P, n=2, nodes=8,
           lengths=P, slots=None):
        return lib().omni_kv_accept(kv, layers, rows, max_len, halfs, slots, starts, path, P, n,
                                    nodes, lengths, None)

    assert rc(layers=0) == rc(rows=0) == rc(max_len=0) == rc(halfs=0) == rc(n=-1) == -1
    assert rc(nodes=0) == rc(n=5) == -1
    assert rc(halfs=252) == rc(n=70000, slots=P) == rc(nodes=65) == -2
    assert rc(kv=None) == rc(starts=None) == rc(path=None) == rc(lengths=None) == -1
    assert rc(kv=ctypes.c_void_p(8)) == -1
    assert rc(n=0) == 0


def test_spec_verify_refusals():
    from omniserver_amd._lib import lib
    work = lib().omni_spec_verify_work(2, 8, 1000, 1)
    assert work >= 0
    assert lib().omni_spec_verify_work(-1, 8, 1000, 0) == -1
    assert lib().omni_spec_verify_work(2, 0, 1000, 0) == lib().omni_spec_verify_work(2, 8, 0, 0) == -1
    assert lib().omni_spec_verify_work(2, 65, 1000, 0) == -2

    def rc(logits=P, dtype=0, ss=8000, rs=1000, draft=None, tokens=P, parents=None, u=P, temps=None,
           temp=0.5, n=2, nodes=8, vocab=1000, path=P, emitted=P, ws=P, doubles=work):
        return lib().omni_spec_verify(logits, dtype, ss, rs, draft, 7000, 1000, tokens, parents,
                                      None, u, temps, temp, n, nodes, vocab, path, P, emitted, ws,
                                      doubles, None)

    assert rc(n=-1) == rc(nodes=0) == rc(vocab=0) == rc(dtype=3) == rc(dtype=-1) == rc(rs=-1) == -1
    assert rc(nodes=65) == rc(draft=P, parents=P) == -2
    assert rc(temp=-0.1) == rc(temp=float("nan")) == rc(u=None) == rc(u=None, temps=P) == -1
    assert rc(logits=None) == rc(tokens=None) == rc(path=None) == rc(emitted=None) == -1
    assert rc(n=0) == 0


def test_tree_cache_refusals():
    p = pool()
    for bad in ([[0, 0]], [[-1, 1]], [[-1, -2]], [[-1, 0], [-1]], [], [[]],
                torch.zeros(3, dtype=torch.int32), torch.zeros(5, 2, dtype=torch.int32),
                [[-1] + [0] * 64]):
        with pytest.raises(ValueError):
            p.tree_cache(bad)
    with pytest.raises(ValueError):
        pool(max_len=4).tree_cache([[-1, 0, 1, 2, 3]])
    ok = [[-1, 0], [-1, 0]]
    for kw in ({"counts": [1]}, {"counts": [1, 3]}, {"counts": [-1, 1]}, {"slots": [0, 0]},
               {"slots": [0, 4]}, {"slots": [1]},
               {"rope_delta": torch.zeros(2, dtype=torch.int64)}):
        with pytest.raises(ValueError):
            p.tree_cache(ok, **kw)
    with pytest.raises(TypeError):
        p.tree_cache(torch.zeros(2, 2, dtype=torch.int64))
    with pytest.raises(TypeError):
        p.tree_cache(ok, counts=torch.ones(2, dtype=torch.int64))
    with pytest.raises(RuntimeError):                 # no CPU path
        p.tree_cache(ok)


def test_tree_plan_rule():
    """What the attention's plan asks for is what the C entry points take, at any size."""
    from omniserver_amd.kv_cache import tree_plan
    for n in (1, 2, 3, 7, 32, 100, 1000):
        for T in (1, 2, 8, 17, 64):
            for nh, nkv in ((12, 2), (28, 4), (16, 16), (64, 1), (8, 8)):
                for capacity in (64, 512, 513, 1536, 1537, 4096, 131072):
                    rows, groups, columns, least = tree_plan(n, T, nh, nkv, capacity, 256)
                    assert (rows, groups) in ((32, 8), (64, 4), (128, 2))
                    if least == 0:
                        assert columns == n * nkv
                        continue
                    blocks = -(-T * (nh // nkv) // rows)
                    assert 1 <= columns <= 256 and (blocks > 32 or columns * blocks <= 256)
                    assert columns <= n * nkv or columns % (n * nkv) == 0 \
                        or columns == n * nkv * -(-capacity // (256 if groups == 8 else 128))


def test_verify_refusals():
    from omniserver_amd.speculative import verify
    L, tok, u = torch.zeros(2, 4, 9), torch.zeros(2, 4, dtype=torch.int64), torch.rand(2, 4)
    draft = torch.zeros(2, 3, 9)
    par = torch.zeros(2, 4, dtype=torch.int32)

    def refuse(err, *a, **kw):
        with pytest.raises(err):
            verify(*a, **kw)

    refuse(ValueError, L[0], tok, u, 1.0)
    refuse(ValueError, torch.zeros(2, 65, 9), torch.zeros(2, 65, dtype=torch.int64), None, 0.0)
    refuse(TypeError, L.double(), tok, u, 1.0)
    refuse(ValueError, torch.zeros(2, 9, 4).transpose(1, 2), tok, u, 1.0)
    refuse(ValueError, L, tok, u, -1.0)
    refuse(ValueError, L, tok, u, float("nan"))
    refuse(ValueError, L, tok, u, float("inf"))
    refuse(ValueError, L, tok, None, 1.0)
    refuse(ValueError, L, tok, None, torch.zeros(2))
    refuse(ValueError, L, tok[:, :3], u, 1.0)
    refuse(ValueError, L, tok, u[:1], 1.0)
    refuse(TypeError, L, tok.int(), u, 1.0)
    refuse(TypeError, L, tok, u.double(), 1.0)
    refuse(TypeError, L, tok, u, 1.0, parents=par.long())
    refuse(ValueError, L, tok, u, 1.0, parents=par, draft_logits=draft)
    refuse(ValueError, L, tok, u, 1.0, draft_logits=L)
    refuse(ValueError, L, tok, u, 1.0, draft_logits=draft.half())
    refuse(ValueError, L, tok, u, torch.zeros(3))
    refuse(TypeError, L, tok, u, torch.zeros(2, dtype=torch.float64))
    refuse(ValueError, L, tok, u, 1.0, counts=torch.ones(3, dtype=torch.int32))
    refuse(RuntimeError, L, tok, u, 1.0)              # no CPU path


def spread(m):
    return (torch.arange(m).double() + 0.5) / m


def grid_first_tokens(logits, children, draft=None, m=48):
    """Share of first emitted tokens over a grid of the random numbers, for one node with the given
    children (trees) or, with draft, one child drawn from it."""
    V = logits.shape[0]
    got = torch.zeros(V, dtype=torch.float64)
    firsts = [(x, 1.0) for x in [None]] if draft is None else \
        [(x, float(w)) for x, w in enumerate(ref.weights(draft, 1.0))]
    us = spread(m).tolist()
    for x, w in firsts:
        kids = children if draft is None else [x]
        T = 1 + len(kids)
        grid = torch.cartesian_prod(*[torch.tensor(us)] * T).tolist()
        n = len(grid)
        rows = logits.expand(n, T, V)
        _, out, _ = ref.verify(rows, [[0] + kids] * n, grid, [1.0] * n,
                               parents=None if draft is not None else [[-1] + [0] * len(kids)] * n,
                               draft=None if draft is None else draft.expand(n, T - 1, V))
        got += w * torch.bincount(out[:, 0], minlength=V).double() / n
    return got


def test_oracle_emits_the_target_distribution():
    """Over a grid of m points a border moves a share of at most 1 / m a random number."""
    logits = torch.tensor([0.3, -1.0, 1.2, 0.0, -0.4])
    p = ref.weights(logits, 1.0)
    got = grid_first_tokens(logits, [2, 4], m=16)
    assert (got - p).abs().max() < 3 / 16
    got = grid_first_tokens(logits, [], draft=torch.tensor([1.0, 0.2, -0.5, 0.1, -2.0]), m=48)
    assert (got - p).abs().max() < 2 / 48
