"""The operators of speculative decoding over the KV pool, as cases that can be timed and checked.

A draft proposes, for each running sequence, a small tree of tokens: node 0 is the sequence's last
emitted token, every other node names an earlier node as its parent.  One forward of the target
model scores all nodes, and three operators beside the model's own work turn that into tokens:

``attn``    attention of the nodes over the sequence's cached prefix and, among the nodes, over the
            node itself and its ancestors (``PreallocatedKVCache.tree_cache``).
``verify``  acceptance of drafted tokens against the target's probabilities from given random
            numbers (``speculative.verify``), for trees of proposed tokens and for chains drawn
            from a draft distribution.
``accept``  the cache after acceptance: the K/V rows of the accepted path moved, in every layer, to
            where a sequence that had decoded them one by one would hold them
            (``TreeCache.accept``).

``own`` selects the framework's kernels; without it every operator runs in its plain form.
"""

import math
import random

import torch

own = False

NL, NH, NKV, HD, V = 28, 12, 2, 128, 151936      # the 2B decoder's layers, heads, vocabulary
SCALE = HD ** -0.5


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest call: one sequence, 8 nodes, a short context, from the drafted parents to
        # the written K/V rows and the attention of one layer
        attn("attn_1x8_300_whole", 1, 8, (300, 300), layout=1, whole=True),
        # one user, a bushy tree, the longest context the default pool holds
        attn("attn_1x26_4096", 1, 26, (4000, 4000), layout=2),
        # a small batch with very different contexts and tree sizes
        attn("attn_8x16_ragged", 8, 16, (40, 3000), ragged=True, layout=3),
        # the serving step: 32 sequences, short chains
        attn("attn_32x8_2048", 32, 8, (2040, 2048), shape="chain", layout=4),
        # the most work: 32 sequences with the largest trees at full contexts
        attn("attn_32x64_4096", 32, 64, (3900, 4032), layout=5),
        # one long document, other head counts
        attn("attn_1x48_32k_28h", 1, 48, (32000, 32000), nh=28, nkv=4, layout=6),
        # one sequence, a tree of proposed tokens (prompt lookup, top-k heads)
        verify("verify_1x8_tree", 1, 8, "tree", layout=7),
        # the serving step: 32 chains of up to 7 drafted tokens and the draft's distributions
        verify("verify_32x8_chain", 32, 8, "chain", ragged=True, layout=8),
        # greedy and sampled requests in one batch, fp32 logits, an odd vocabulary
        verify("verify_6x13_mixed_f32", 6, 13, "tree", dtype="float32", vocab=32003, temps="mixed",
               layout=9),
        # the most rows
        verify("verify_32x16_tree", 32, 16, "tree", ragged=True, layout=10),
        # the accepted path of one sequence, all layers
        accept("accept_1x8_5", 1, 8, 5, (500, 500), layout=11),
        # the serving step's accepted paths, all layers
        accept("accept_32x26_6", 32, 26, 6, (100, 400), layout=12),
    ]


def attn(name, n, nodes, ctx, nh=NH, nkv=NKV, shape="tree", ragged=False, whole=False, layout=0):
    """n sequences with contexts drawn from ctx (by layout) and trees of `nodes` nodes (ragged: up
    to that many); whole: the tree's plan and the K/V rows' write as well."""
    return {"name": name, "family": "attn", "n": n, "nodes": nodes, "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "nh": nh, "nkv": nkv, "shape": shape, "ragged": ragged,
            "whole": whole, "layout": layout}


def verify(name, n, nodes, mode, dtype="float16", vocab=V, temps="sampled", ragged=False, layout=0):
    """n trees of `nodes` nodes: "tree" proposed tokens, "chain" tokens drawn from draft logits."""
    return {"name": name, "family": "verify", "n": n, "nodes": nodes, "mode": mode, "dtype": dtype,
            "vocab": vocab, "temps": temps, "ragged": ragged, "layout": layout}


def accept(name, n, nodes, kept, ctx, layout=0):
    """n sequences that each keep the root and `kept` of their other nodes, none in its place."""
    return {"name": name, "family": "accept", "n": n, "nodes": nodes, "kept": kept,
            "ctx_lo": ctx[0], "ctx_hi": ctx[1], "layout": layout}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "verify", "verify", "accept"])
    layout = rng.randrange(1 << 20)
    n = _log(rng, 1, 32)
    if kind == "attn":
        nodes = _log(rng, 1, 64)
        hi = _log(rng, 16, min(32000, 32 * 4032 // n))
        nh, nkv = rng.choice([(12, 2), (12, 2), (28, 4), (16, 16), (8, 1), (32, 8)])
        if n * nodes * hi * nh > 32 * 64 * 4032 * 12:
            nodes = max(1, 32 * 64 * 4032 * 12 // (n * hi * nh))
        if n * hi * nkv > 32 * 4032 * 2:
            nh, nkv = 12, 2
        c = attn("", n, nodes, (hi // rng.choice([1, 3, 20]), hi), nh, nkv,
                 rng.choice(["tree", "chain"]), rng.random() < 0.5, False, layout)
        if rng.random() < 0.2:
            c["whole"], c["ragged"] = True, False
    elif kind == "verify":
        nodes = _log(rng, 1, min(64, 512 // n))
        mode = rng.choice(["tree", "chain"])
        dtype = rng.choice(["float16", "float16", "float32", "bfloat16"])
        if (mode == "chain") + (dtype == "float32") and n * nodes > 256:
            nodes = 256 // n
        vocab = rng.choice([V, V, V, _log(rng, 500, V)])
        if mode == "chain" and dtype == "float32" and n * nodes > 128:
            nodes = max(1, 128 // n)
        c = verify("", n, nodes, mode, dtype, vocab, rng.choice(["sampled", "mixed"]),
                   rng.random() < 0.5, layout)
    else:
        nodes = _log(rng, 4, 64)
        hi = _log(rng, 16, 400)
        c = accept("", n, nodes, rng.randint(1, min(6, nodes - 2)), (hi // 4, hi), layout)
    c.pop("name")
    return c


# ------------------------------------------------------------------------- seeded inputs
class _Rand:
    """Tensors on the GPU from a seed, in the order asked for, and host numbers beside them."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) * 7919 + 13)
        self.host = random.Random(int(seed) * 104729 + 7)

    def normal(self, *shape, std=1.0, dtype=torch.float16):
        return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=self.g)

    def uniform(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.g)


def _i(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _starts(case):
    rng = random.Random(case["layout"])
    return [rng.randint(case["ctx_lo"], case["ctx_hi"]) for _ in range(case["n"])]


def _counts(case):
    """Nodes in use for each sequence."""
    rng = random.Random(case["layout"] + 1)
    T = case["nodes"]
    return [rng.randint(1, T) if case["ragged"] else T for _ in range(case["n"])]


def _parents(case, rng):
    """One parent list a sequence: a chain, or a tree that grows at its newest nodes most."""
    T = case["nodes"]
    if case.get("shape", case.get("mode")) == "chain":
        return [[i - 1 for i in range(T)] for _ in range(case["n"])]
    return [[-1] + [rng.randint(max(0, i - 6), i - 1) for i in range(1, T)]
            for _ in range(case["n"])]


def _round(x, to):
    return -(-x // to) * to


def _attn_prepare(case, seed):
    r = _Rand(seed)
    n, T, nh, nkv = case["n"], case["nodes"], case["nh"], case["nkv"]
    starts, counts = _starts(case), _counts(case)
    parents = _parents(case, r.host)
    max_len = _round(max(starts) + T, 256)
    return {"case": case, "kind": "attn", "max_len": max_len, "starts": _i(starts),
            "counts": _i(counts, torch.int32), "parents": _i(parents, torch.int32),
            "longest": max(starts) + T,
            "storage": r.normal(1, 2, n, max_len, nkv, HD),
            "qkv": r.normal(n * T, (nh + 2 * nkv) * HD),
            "out": torch.zeros(n * T, nh, HD, device="cuda", dtype=torch.float16)}


def _verify_prepare(case, seed):
    r = _Rand(seed)
    n, T, vocab = case["n"], case["nodes"], case["vocab"]
    dtype = getattr(torch, case["dtype"])
    parents = _i(_parents(case, r.host), torch.int32)
    # a language model's rows: a wide floor and a few tokens far above it
    logits = r.normal(n * T, vocab, std=2.0, dtype=dtype)
    part = vocab // 12
    top = torch.randint(0, part, (n * T, 12), device="cuda", generator=r.g)
    top += part * torch.arange(12, device="cuda")
    logits.scatter_add_(1, top, (9 + 4 * r.uniform(n * T, 12)).to(dtype))
    temp = [0.0 if case["temps"] == "mixed" and r.host.random() < 0.5 else r.host.uniform(0.5, 1.2)
            for _ in range(n)]
    # the draft's rows: the target's with its own errors
    draft = logits + r.normal(n * T, vocab, std=0.5, dtype=dtype)
    t = _i([x or 1.0 for x in temp], torch.float32)
    tokens = torch.randint(0, vocab, (n, T), device="cuda", generator=r.g)
    draft = draft.reshape(n, T, vocab)
    state = {"case": case, "kind": "verify", "logits": logits.reshape(n, T, vocab),
             "parents": parents, "counts": _i(_counts(case), torch.int32),
             "uniforms": r.uniform(n, T), "temperature": _i(temp, torch.float32), "draft": None}
    if T > 1 and case["mode"] == "chain":
        state["draft"] = draft[:, :T - 1].contiguous()
        rows = state["draft"].float() / t[:, None, None]
        noise = r.uniform(*rows.shape).clamp_(1e-20, 1 - 1e-7)
        tokens[:, 1:] = (rows - noise.log_().neg_().log_()).argmax(-1)
    elif T > 1:
        # the r-th child of a node is the draft's r-th best token there
        p = parents.long()
        rank = (torch.tril(p[:, :, None] == p[:, None, :], -1)).sum(-1)
        best = draft.topk(min(8, vocab), -1).indices
        at = best[torch.arange(n, device="cuda")[:, None], p.clamp(min=0)]
        tokens[:, 1:] = at.gather(2, rank.clamp(max=best.shape[-1] - 1)[..., None])[..., 0][:, 1:]
    state["tokens"] = tokens
    return state


def _accept_prepare(case, seed):
    r = _Rand(seed)
    n, T, kept = case["n"], case["nodes"], case["kept"]
    starts = _starts(case)
    max_len = _round(max(starts) + T, 64)
    parents = _parents(case, r.host)
    path = torch.full((n, T), -1, dtype=torch.int32)
    for s in range(n):
        nodes = [0] + sorted(r.host.sample(range(2, T), kept))
        for a, b in zip(nodes, nodes[1:]):
            parents[s][b] = a
        path[s, :kept + 1] = torch.tensor(nodes, dtype=torch.int32)
    return {"case": case, "kind": "accept", "max_len": max_len, "starts": _i(starts),
            "lengths": _i(starts), "parents": _i(parents, torch.int32), "path": path.cuda(),
            "emitted": torch.full((n,), kept + 1, dtype=torch.int32, device="cuda"),
            "storage": r.normal(NL, 2, n, max_len, NKV, HD)}


def prepare(case, seed):
    """The pool, the tree and the tensors that a serving loop holds when it makes the call."""
    make = {"attn": _attn_prepare, "verify": _verify_prepare, "accept": _accept_prepare}
    state = make[case["family"]](case, seed)
    if own:
        _own_handles(state)
    return state


# ------------------------------------------------------------------------- the framework's calls
def _own_handles(s):
    """The pool over the case's K/V and, where it is not part of the pass, the step's tree."""
    if s["kind"] == "verify":
        return
    from omniserver_amd.kv_cache import PreallocatedKVCache
    c = s["case"]
    L, _, n, max_len, nkv, _ = s["storage"].shape
    pool = PreallocatedKVCache(L, n, nkv, max_len, HD, "cuda", n_heads=c.get("nh", NH))
    pool.storage.copy_(s["storage"])
    pool.lengths.copy_(s["starts"])
    s["storage"], s["pool"] = pool.storage, pool
    if not c.get("whole"):
        s["tree"] = pool.tree_cache(s["parents"], counts=s.get("counts"))


def _own_run(s):
    c = s["case"]
    if s["kind"] == "verify":
        from omniserver_amd.speculative import verify as check
        tree = {"parents": s["parents"]} if s["draft"] is None else {"draft_logits": s["draft"]}
        v = check(s["logits"], s["tokens"], s["uniforms"], s["temperature"], counts=s["counts"],
                  **tree)
        return {"path": v.path, "tokens": v.tokens, "emitted": v.emitted}
    pool = s["pool"]
    if s["kind"] == "accept":
        s["tree"].accept(s["path"], s["emitted"])
        return {"kv": pool.storage, "lengths": pool.lengths}
    if c["whole"]:
        q, k, v = _split(s)
        out = pool.tree_cache(s["parents"]).flash_prefill(q, k, v, 0, SCALE)
        return {"out": out, "kv": pool.storage}
    return {"out": s["tree"].attend_qkv(s["qkv"], 0, SCALE, s["out"])}


def _split(s):
    c = s["case"]
    return s["qkv"].view(-1, c["nh"] + 2 * c["nkv"], HD).split((c["nh"], c["nkv"], c["nkv"]), 1)


# ------------------------------------------------------------------------- the plain forms
def _ancestors(parents):
    """[n, T, T] bool: node j is node i or above it.  A step to the parent is a 0/1 matrix; its
    powers' sum, by squaring, holds every number of steps up to 64."""
    n, T = parents.shape
    at = torch.arange(T, device=parents.device)
    a = (at == parents[..., None]).float() + torch.eye(T, device=parents.device)
    for _ in range(6):
        a = (a @ a > 0).float()
    return a > 0


def _plain_attn(s):
    c = s["case"]
    n, T, nh, nkv, K = c["n"], c["nodes"], c["nh"], c["nkv"], s["longest"]
    q, k, v = _split(s)
    starts, used = s["starts"], torch.arange(T, device="cuda") < s["counts"][:, None]
    at = torch.arange(K, device="cuda") - starts[:, None]             # [n, K] node of each key
    if c["whole"]:
        rows = (torch.arange(n, device="cuda")[:, None], starts[:, None] + torch.arange(T, device="cuda"))
        s["storage"][0, 0].index_put_(rows, k.reshape(n, T, nkv, HD))
        s["storage"][0, 1].index_put_(rows, v.reshape(n, T, nkv, HD))
    node = at.clamp(0, T - 1)[:, None].expand(n, T, K)
    seen = (at < 0)[:, None] | (_ancestors(s["parents"]).gather(2, node) & (at < T)[:, None])
    kk, vv = s["storage"][0, :, :, :K].float().permute(0, 1, 3, 2, 4)       # [n, nkv, K, HD]
    qq = q.reshape(n, T, nkv, nh // nkv, HD).permute(0, 2, 3, 1, 4).float()
    w = qq.reshape(n, nkv, -1, HD) @ kk.transpose(2, 3).contiguous() * SCALE
    w = w.reshape(n, nkv, nh // nkv, T, K).masked_fill_(~seen[:, None, None], -math.inf)
    w = (w - w.amax(-1, keepdim=True)).exp_()
    w /= w.sum(-1, keepdim=True)
    o = (w.reshape(n, nkv, -1, K) @ vv.contiguous()).reshape(n, nkv, nh // nkv, T, HD)
    o = o.permute(0, 3, 1, 2, 4).reshape(n, T, nh, HD) * used[..., None, None]
    out = {"out": o.half().reshape(n * T, nh, HD)}
    return dict(out, kv=s["storage"]) if c["whole"] else out


def _weights(logits, temperature):
    """Unnormalised probabilities in 64 bits; a temperature of zero keeps the best token alone."""
    x = logits.double()
    t = temperature.double().reshape(-1, *[1] * (x.dim() - 1))
    w = ((x - x.amax(-1, keepdim=True)) / torch.where(t > 0, t, 1.0)).exp_()
    best = torch.arange(x.shape[-1], device=x.device) == x.argmax(-1, keepdim=True)
    return torch.where(t > 0, w, best.double())


def _plain_verify(s):
    """Every node's own test at once; the path is the run of nodes whose ancestors all passed."""
    logits, tokens, u, temp = s["logits"], s["tokens"], s["uniforms"].double(), s["temperature"]
    n, T, vocab = logits.shape
    seq, at = torch.arange(n, device="cuda"), torch.arange(T, device="cuda")
    used = at < s["counts"][:, None]
    chain = s["draft"] is not None
    parents = (at - 1).expand(n, T) if chain or T == 1 else s["parents"].long()
    up = parents.clamp(min=0)
    p = _weights(logits, temp)
    total = p.sum(-1)
    mine = p[seq[:, None], up, tokens]                  # [n, T] each node's token at its parent
    tried = torch.tril(parents[:, :, None] == parents[:, None, :], -1) & used[:, None]
    if chain:
        p /= total[..., None]
        q = _weights(s["draft"], temp)
        q /= q.sum(-1, keepdim=True)
        passed = u * q[seq[:, None], up.clamp(max=T - 2), tokens] < mine / total.gather(1, up)
    else:
        # earlier siblings take their mass with them; a token proposed twice has none left
        twice = (tried & (tokens[:, :, None] == tokens[:, None, :])).any(-1)
        mine = mine * ~twice
        left = total.gather(1, up) - (tried * mine[:, None]).sum(-1)
        passed = u * left < mine
    passed &= used
    # the chosen child of a node is its first that passes
    first = passed & ~((tried & passed[:, None]).any(-1))
    first[:, 0] = used[:, 0]
    on = (first[:, None] | ~_ancestors(parents)).all(-1) & _ancestors(parents)[..., 0] & used
    emitted = on.sum(-1)
    order = torch.where(on, at, T).sort(-1).values
    path = torch.where(order < T, order, -1)
    last = path.gather(1, (emitted - 1).clamp(min=0)[:, None])[:, 0].clamp(min=0)
    w = p[seq, last]
    if chain:
        more = (last + 1 < s["counts"]) & (last + 1 < T)
        less = (w - q[seq, last.clamp(max=T - 2)]).clamp_(min=0)
        w = torch.where((more & (less.sum(-1) > 0))[:, None], less, w)
    else:
        child = (parents == last[:, None]) & used & (at > 0)
        gone = torch.zeros_like(w).scatter_add_(1, tokens, child.double())
        less = w.masked_fill(gone > 0, 0.0)
        w = torch.where(less.sum(-1, keepdim=True) > 0, less, w)
    run = w.cumsum(-1)
    drawn = (run > u[:, :1] * run[:, -1:]).to(torch.int8).argmax(-1)
    out = tokens.gather(1, path.clamp(min=0).roll(-1, 1))
    out = torch.where(at == emitted[:, None] - 1, drawn[:, None], out)
    out = torch.where(at < emitted[:, None], out, -1)
    return {"path": path.int(), "tokens": out, "emitted": emitted.int()}


def _plain_accept(s):
    """Rows start + path[j] of every layer to start + j; the lengths after them."""
    n, T = s["path"].shape
    keep = torch.arange(T, device="cuda") < s["emitted"][:, None]
    to = s["starts"][:, None] + torch.arange(T, device="cuda")
    at = s["starts"][:, None] + torch.where(keep, s["path"].long(), torch.arange(T, device="cuda"))
    seq = torch.arange(n, device="cuda")[:, None]
    s["storage"][:, :, seq, to] = s["storage"][:, :, seq, at]
    torch.add(s["starts"], s["emitted"], out=s["lengths"])
    return {"kv": s["storage"], "lengths": s["lengths"]}


def run(state):
    if own:
        return _own_run(state)
    return {"attn": _plain_attn, "verify": _plain_verify, "accept": _plain_accept}[state["kind"]](
        state)


# ------------------------------------------------------------------------- bytes and operations
def work(case):
    n, T = case["n"], case["nodes"]
    if case["family"] == "accept":
        moved = n * case["kept"] * NL * 2 * NKV * HD * 2
        return {"bytes": 2.0 * moved + n * (T * 4 + 12), "flops": 0.0}
    counts = _counts(case)
    if case["family"] == "verify":
        size = {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
        rows = sum(counts) + (sum(c - 1 for c in counts) if case["mode"] == "chain" else 0)
        return {"bytes": rows * case["vocab"] * size + n * T * 24.0,
                "flops": 3.0 * rows * case["vocab"]}
    starts, nh, nkv = _starts(case), case["nh"], case["nkv"]
    keys = sum(starts) + sum(counts)
    pairs = sum(c * st for c, st in zip(counts, starts)) + 4 * sum(counts)
    extra = sum(counts) * 2 * nkv * HD * 4 if case["whole"] else 0
    return {"bytes": keys * 2 * nkv * HD * 2 + 2 * sum(counts) * nh * HD * 2 + extra,
            "flops": 4.0 * pairs * nh * HD}


# ------------------------------------------------------------------------- in 64 bits
def _lineage(parents, i):
    """Node i and its ancestors."""
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def _exact_attn(case, s):
    T, nh, nkv = case["nodes"], case["nh"], case["nkv"]
    q, k, v = (x.double() for x in _split(s))
    kc, vc = s["storage"][0, 0].double(), s["storage"][0, 1].double()
    out = torch.zeros(case["n"] * T, nh, HD, dtype=torch.float64, device="cuda")
    parents, starts, counts = s["parents"].tolist(), _starts(case), _counts(case)
    for b, (st, m) in enumerate(zip(starts, counts)):
        if case["whole"]:
            kc[b, st:st + T], vc[b, st:st + T] = k[b * T:b * T + T], v[b * T:b * T + T]
        off = torch.full((m, st + m), -math.inf, dtype=torch.float64, device="cuda")
        off[:, :st] = 0.0
        for i in range(m):
            off[i, [st + j for j in _lineage(parents[b], i)]] = 0.0
        for h in range(nh):
            g = h // (nh // nkv)
            w = torch.softmax(q[b * T:b * T + m, h] @ kc[b, :st + m, g].t() * SCALE + off, -1)
            out[b * T:b * T + m, h] = w @ vc[b, :st + m, g]
    if not case["whole"]:
        return {"out": out}
    return {"out": out, "kv": torch.stack([kc, vc])[None]}


def _exact_verify(case, s):
    """The walk from the root, one node and one child after another."""
    n, T, vocab = case["n"], case["nodes"], case["vocab"]
    tokens, uniforms, parents = s["tokens"].tolist(), s["uniforms"].tolist(), s["parents"].tolist()
    chain, counts, temps = s["draft"] is not None, _counts(case), s["temperature"].tolist()
    path, out, emitted = [], [], []

    def distribution(row, t):
        if t <= 0:
            w = torch.zeros(vocab, dtype=torch.float64, device="cuda")
            w[int(torch.nonzero(row == row.max())[0])] = 1.0
            return w
        return torch.softmax(row.double() / t, -1)

    for b in range(n):
        here, got, m = 0, [0], counts[b]
        while True:
            p = distribution(s["logits"][b, here], temps[b])
            children = [i for i in range(here + 1, m)
                        if (i - 1 if chain else parents[b][i]) == here]
            taken = None
            for i in children:
                x = tokens[b][i]
                if chain:
                    q = distribution(s["draft"][b, here], temps[b])
                else:
                    q = torch.zeros_like(p)
                    q[x] = 1.0
                if uniforms[b][i] * float(q[x]) < float(p[x]):
                    taken = i
                    break
                rest = (p - q).clamp(min=0.0)
                if float(rest.sum()) > 0:
                    p = rest / rest.sum()
            if taken is None:
                break
            got.append(taken)
            here = taken
        run = p.cumsum(0)
        x = int(torch.nonzero(run > uniforms[b][0] * float(run[-1]))[0])
        emitted.append(len(got))
        path.append(got + [-1] * (T - len(got)))
        out.append([tokens[b][i] for i in got[1:]] + [x] + [-1] * (T - len(got)))
    return {"path": torch.tensor(path, dtype=torch.int32), "tokens": torch.tensor(out),
            "emitted": torch.tensor(emitted, dtype=torch.int32)}


def _exact_accept(case, s):
    kv = s["storage"].double()
    starts, path = _starts(case), s["path"].tolist()
    new = kv.clone()
    for b, st in enumerate(starts):
        for j in range(case["kept"] + 1):
            new[:, :, b, st + j] = kv[:, :, b, st + path[b][j]]
    return {"kv": new, "lengths": torch.tensor([st + case["kept"] + 1 for st in starts])}


def exact(case, seed):
    make = {"attn": _attn_prepare, "verify": _verify_prepare, "accept": _accept_prepare}
    s = make[case["family"]](case, seed)
    return {"attn": _exact_attn, "verify": _exact_verify, "accept": _exact_accept}[case["family"]](
        case, s)
