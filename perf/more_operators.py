"""The operators of a paged KV cache and of beam search over it, as cases that can be timed and checked.

Sequences keep their keys and values in pages of a few dozen tokens, named by a block table per
sequence, so that beams of one prompt share its pages.  A step takes four operators beside the
model's own work:

``attn``     attention of one new token per sequence over the pages its table names
             (``PagedKVCache.decode_cache``).
``slots``    pages for the tokens that sequences are about to bring: block tables extended, and for
             every token the page and the place in it (``PagedKVCache.reserve``).
``select``   the best continuations over all beams of a request and the vocabulary
             (``beam.select``).
``reorder``  the cache after that choice: rows take their parents' tables, and every child but a
             parent's first its own copy of the page that is still being filled
             (``PagedKVCache.reorder``).

``own`` selects the framework's kernels; without it every operator runs in its plain form.
"""

import math
import random

import torch

own = False

NL, NH, NKV, HD, V = 28, 12, 2, 128, 151936      # the 2B decoder's layers, heads, vocabulary


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # the smallest call: one sequence, from its length to the attention of one layer
        attn("attn_1x300_whole", 1, (300, 300), 16, whole=True, layout=1),
        # one long document, other head counts
        attn("attn_1x32k_28h", 1, (32000, 32000), 64, nh=28, nkv=4, layout=2),
        # the serving step
        attn("attn_32x2048", 32, (2040, 2048), 16, layout=3),
        # very different contexts, a head of its own for every query, half the width, bf16
        attn("attn_64_ragged_16h_bf16", 64, (20, 4000), 128, nh=16, nkv=16, hd=64, dtype="bfloat16",
             layout=4),
        # the most work: many beams of long prompts
        attn("attn_128x4096_beams", 128, (3800, 4096), 32, beams=4, layout=5),
        # a decode step's slots
        slots("slots_32x1_2048", 32, 33, (2000, 2048), (1, 1), 16, layout=6),
        # the most sequences, with prompts, decode tokens and idle rows, and too few pages for all
        slots("slots_384_prompts", 384, 512, (0, 4096), (0, 256), 16, short=True, layout=7),
        # one request, four beams
        select("select_1x4", 1, 4, 4, layout=8),
        # a batch of requests
        select("select_32x4", 32, 4, 4, layout=9),
        # twice the candidates, some beams at their end, fp32 logits, an odd vocabulary
        select("select_6x5_f32", 6, 5, 10, dtype="float32", vocab=32003, ended=True, layout=10),
        # one request's beams, all layers
        reorder("reorder_1x4", 1, 4, (500, 500), 16, layout=11),
        # a batch of requests, all layers
        reorder("reorder_32x4", 32, 4, (200, 600), 16, layout=12),
    ]


def attn(name, n, ctx, page, nh=NH, nkv=NKV, hd=HD, dtype="float16", beams=1, whole=False, layout=0):
    """n sequences with ctx tokens (by layout) and one new one; beams: that many of them share their
    prompt's pages; whole: the step's slots and the K/V rows' write as well."""
    return {"name": name, "family": "attn", "n": n, "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "page": page, "nh": nh, "nkv": nkv, "hd": hd, "dtype": dtype, "beams": beams,
            "whole": whole, "layout": layout}


def slots(name, n, seqs, ctx, new, page, short=False, layout=0):
    """new tokens for each of the first n of seqs sequences that hold ctx tokens; short: the pool
    has fewer pages than they need."""
    return {"name": name, "family": "slots", "n": n, "seqs": seqs, "ctx_lo": ctx[0],
            "ctx_hi": ctx[1], "new_lo": new[0], "new_hi": new[1], "page": page, "short": short,
            "beams": 1, "layout": layout}


def select(name, n, beams, k, dtype="float16", vocab=V, ended=False, layout=0):
    """k continuations for each of n requests with that many beams; ended: some beams are finished
    and some not in use."""
    return {"name": name, "family": "select", "n": n, "beams": beams, "k": k, "dtype": dtype,
            "vocab": vocab, "ended": ended, "layout": layout}


def reorder(name, n, beams, ctx, page, layout=0):
    """n requests of that many beams, ctx tokens each, of which the last few are a beam's own."""
    return {"name": name, "family": "reorder", "n": n * beams, "ctx_lo": ctx[0], "ctx_hi": ctx[1],
            "page": page, "nkv": NKV, "hd": HD, "beams": beams, "layout": layout}


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["attn", "attn", "attn", "slots", "select", "select", "reorder"])
    layout = rng.randrange(1 << 20)
    page = rng.choice([16, 16, 32, 64, 128, 256])
    if kind == "attn":
        nh, nkv = rng.choice([(12, 2), (12, 2), (28, 4), (16, 16), (8, 1), (32, 8), (40, 2)])
        hd = rng.choice([128, 128, 64])
        beams = rng.choice([1, 1, 1, 4, 5])
        tokens = 128 * 4096 * NKV * HD // (nkv * hd)      # the largest case's bytes
        n = _log(rng, 1, 256)
        n += -n % beams
        hi = _log(rng, 1, max(2, min(32000, tokens // n)))
        c = attn("", n, (hi // rng.choice([1, 3, 20]), hi), page, nh, nkv, hd,
                 rng.choice(["float16", "float16", "bfloat16"]), beams, rng.random() < 0.2, layout)
    elif kind == "slots":
        n = _log(rng, 1, 384)
        hi = _log(rng, 1, 4096)
        new = rng.choice([1, 1, _log(rng, 1, 256)])
        c = slots("", n, n + rng.randrange(1 + n // 3), (hi // rng.choice([1, 4, 50]), hi),
                  (rng.choice([0, 1, new]), new), page, rng.random() < 0.3, layout)
    elif kind == "select":
        beams = _log(rng, 1, 16)
        n = _log(rng, 1, max(1, 128 // beams))
        dtype = rng.choice(["float16", "float16", "bfloat16", "float32"])
        vocab = rng.choice([V, V, _log(rng, 500, V)])
        if dtype == "float32" and n * beams * vocab > 64 * V:
            n = max(1, 64 * V // (beams * vocab))
        c = select("", n, beams, rng.choice([beams, beams, 2 * beams, _log(rng, 1, 32)]), dtype,
                   vocab, rng.random() < 0.5, layout)
    else:
        beams = _log(rng, 1, 16)
        n = _log(rng, 1, max(1, min(128, 128 * 32 // page) // beams))
        hi = _log(rng, 8, 600)
        c = reorder("", n, beams, (hi // rng.choice([1, 3]), hi), page, layout)
    c.pop("name")
    return c


# ------------------------------------------------------------------------- seeded inputs
class _Rand:
    """Tensors on the GPU from a seed, in the order asked for, and host numbers beside them."""

    def __init__(self, seed):
        self.g = torch.Generator(device="cuda")
        self.g.manual_seed(int(seed) * 7919 + 29)
        self.host = random.Random(int(seed) * 104729 + 11)

    def normal(self, *shape, std=1.0, dtype=torch.float16):
        return torch.empty(*shape, device="cuda", dtype=dtype).normal_(0.0, std, generator=self.g)

    def uniform(self, *shape):
        return torch.rand(*shape, device="cuda", generator=self.g)


def _i(values, dtype=torch.int64):
    return torch.tensor(values, dtype=dtype, device="cuda")


def _contexts(case):
    """Tokens of every sequence and, of those, the ones that its request's beams share."""
    rng = random.Random(case["layout"])
    rows, shared = [], []
    while len(rows) < case.get("seqs", case["n"]):
        ctx = rng.randint(case["ctx_lo"], case["ctx_hi"])
        # beams have grown by up to 40 tokens of their own behind the prompt
        prompt = max(0, ctx - rng.randint(1, 40)) if case["beams"] > 1 else 0
        for _ in range(case["beams"]):
            rows.append(ctx)
            shared.append(prompt)
    return rows, shared


def _new(case):
    """Tokens that each of the first n sequences brings."""
    if case["family"] != "slots":
        return [1] * case["n"]
    rng = random.Random(case["layout"] + 1)
    return [rng.randint(case["new_lo"], case["new_hi"]) for _ in range(case["n"])]


def _geometry(case):
    """(pages of the pool, columns of the block tables)."""
    rows, shared = _contexts(case)
    new, page = _new(case), case["page"]
    new += [0] * (len(rows) - len(new))
    width = max(-(-(a + b) // page) for a, b in zip(rows, new))
    held = sum(-(-a // page) - (b // page if i % case["beams"] else 0)
               for i, (a, b) in enumerate(zip(rows, shared)))
    if case["family"] == "reorder":
        need = len(rows)
    else:
        need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(rows, new))
    return held + (need // 2 if case.get("short") else need + 3), max(1, width)


def _tables(case, r):
    """Block tables in which every sequence's pages are anywhere in the pool."""
    rows, shared = _contexts(case)
    pages, width = _geometry(case)
    free = list(range(pages))
    r.host.shuffle(free)
    table = [[0] * width for _ in rows]
    for i, (ctx, common) in enumerate(zip(rows, shared)):
        held, keep = -(-ctx // case["page"]), 0
        if i % case["beams"]:
            keep = common // case["page"]
            table[i][:keep] = table[i - 1][:keep]
        for j in range(keep, held):
            table[i][j] = free.pop()
    return _i(table, torch.int32), _i(rows)


def _cache_prepare(case, seed):
    r = _Rand(seed)
    pages, width = _geometry(case)
    tables, lengths = _tables(case, r)
    new = _new(case)
    s = {"case": case, "kind": case["family"], "tables": tables, "lengths": lengths,
         "counts": _i(new, torch.int32), "tokens": max(1, sum(new)), "pages": pages,
         "max_len": width * case["page"]}
    if case["family"] == "slots":
        return s
    n, page, nkv, hd = case["n"], case["page"], case["nkv"], case["hd"]
    dtype = getattr(torch, case.get("dtype", "float16"))
    layers = NL if case["family"] == "reorder" else 1
    s["storage"] = r.normal(layers, 2, pages, page, nkv, hd, dtype=dtype)
    if case["family"] == "attn":
        s["qkv"] = r.normal(n, (case["nh"] + 2 * nkv) * hd, dtype=dtype)
        s["out"] = torch.zeros(n, case["nh"], hd, device="cuda", dtype=dtype)
    else:
        W = case["beams"]
        # the better beams have more children
        s["parents"] = _i([sorted(min(r.host.randrange(W), r.host.randrange(W)) for _ in range(W))
                           for _ in range(n // W)], torch.int32)
    return s


def _select_prepare(case, seed):
    r = _Rand(seed)
    n, W, vocab = case["n"], case["beams"], case["vocab"]
    dtype = getattr(torch, case["dtype"])
    # a language model's rows: a wide floor and a few tokens far above it
    logits = r.normal(n * W, vocab, std=2.0, dtype=dtype)
    part = vocab // 12
    top = torch.randint(0, part, (n * W, 12), device="cuda", generator=r.g)
    top += part * torch.arange(12, device="cuda")
    logits.scatter_add_(1, top, (9 + 4 * r.uniform(n * W, 12)).to(dtype))
    scores = -4.0 - 3.0 * r.uniform(n, W)
    done = torch.zeros(n, W, dtype=torch.bool, device="cuda")
    if case["ended"]:
        done = r.uniform(n, W) < 0.3
        scores[r.uniform(n, W) < 0.2] = -math.inf
    # the tokens that end a sequence: one of them is likely
    stop = torch.stack([top[::W, 3], torch.randint(0, vocab, (n,), device="cuda", generator=r.g)], 1)
    return {"case": case, "kind": "select", "logits": logits.reshape(n, W, vocab), "scores": scores,
            "done": done, "stop": stop.contiguous()}


def prepare(case, seed):
    """The cache, tables and tensors that a serving loop holds when it makes the call."""
    if case["family"] == "select":
        return _select_prepare(case, seed)
    state = _cache_prepare(case, seed)
    if own:
        _own_handles(state)
    elif state["kind"] == "attn" and not case["whole"]:
        _plain_reserve(state)        # the new token's page is in the table
    return state


# ------------------------------------------------------------------------- the framework's calls
def _own_handles(s):
    """The cache over the case's pages and, where it is not part of the pass, the step's slots."""
    from omniserver_amd.paged_kv import PagedKVCache
    c = s["case"]
    shape = s["storage"].shape if "storage" in s else (1, 2, s["pages"], c["page"], 1, HD)
    pool = PagedKVCache(shape[0], s["pages"], shape[4], c["page"], shape[5], "cuda",
                        max_seqs=len(s["tables"]), max_len=s["max_len"],
                        dtype=s["storage"].dtype if "storage" in s else torch.float16,
                        n_heads=c.get("nh", 6 * shape[4]))
    pool.tables.copy_(s["tables"])
    pool.lengths.copy_(s["lengths"])
    if "storage" in s:
        pool.storage.copy_(s["storage"])
        s["storage"] = pool.storage
    s["pool"] = pool
    if s["kind"] == "attn" and not c["whole"]:
        s["step"] = pool.decode_cache(c["n"])


def _own_run(s):
    c = s["case"]
    if s["kind"] == "select":
        from omniserver_amd.beam import select as choose
        b = choose(s["logits"], s["scores"], c["k"], done=s["done"], stop=s["stop"])
        return {"scores": b.scores, "parents": b.parents, "tokens": b.tokens, "done": b.done}
    pool = s["pool"]
    if s["kind"] == "slots":
        t = pool.reserve(s["counts"], tokens=s["tokens"])
        return {"tables": pool.tables, "pages": t.token_page, "places": t.token_pos,
                "positions": t.positions, "granted": t.granted}
    if s["kind"] == "reorder":
        pool.reorder(s["parents"])
        return {"kv": pool.storage, "tables": pool.tables, "lengths": pool.lengths}
    if c["whole"]:
        _, k, v = _split(s)
        step = pool.decode_cache(c["n"])
        step.write(k, v, 0)
        return {"out": step.attend_qkv(s["qkv"], 0, c["hd"] ** -0.5, s["out"]), "kv": pool.storage}
    return {"out": s["step"].attend_qkv(s["qkv"], 0, c["hd"] ** -0.5, s["out"])}


def _split(s):
    c = s["case"]
    return s["qkv"].view(-1, c["nh"] + 2 * c["nkv"], c["hd"]).split((c["nh"], c["nkv"], c["nkv"]), 1)


# ------------------------------------------------------------------------- the plain forms
def _free_pages(s, tables, lengths, keep=None):
    """The pages that no sequence holds, ascending, then the held ones; how many are free."""
    page, pages = s["case"]["page"], s["pages"]
    at = torch.arange(tables.shape[1], device="cuda")
    held = at < ((lengths + page - 1) // page)[:, None]
    if keep is not None:
        held &= keep
    used = torch.zeros(pages + 1, dtype=torch.int64, device="cuda")
    used[torch.where(held, tables.long(), pages)] = 1
    used = used[:pages]
    return used.sort(stable=True).indices, pages - used.sum()


def _plain_reserve(s):
    """Pages for counts[i] tokens behind each sequence's length, in order; where they go."""
    page, T, n, dev = s["case"]["page"], s["tokens"], len(s["counts"]), "cuda"
    tables, counts = s["tables"], s["counts"].long()
    at = s["lengths"][:n]
    after = at + counts
    first, last = (at + page - 1) // page, (after + page - 1) // page
    need = last - first
    order, left = _free_pages(s, tables, s["lengths"])
    ends = need.cumsum(0)
    ok = (counts > 0) & ((need == 0) | (ends <= left))
    column = torch.arange(tables.shape[1], device=dev)
    fresh = (column >= first[:, None]) & (column < last[:, None]) & ok[:, None]
    rank = (ends - need - first)[:, None] + column
    tables[:n] = torch.where(fresh, order[rank.clamp(0, len(order) - 1)].int(), tables[:n])
    cu = counts.cumsum(0)
    t = torch.arange(T, device=dev)
    seq = torch.searchsorted(cu, t, right=True).clamp(max=n - 1)
    good = ok[seq] & (t < cu[-1])
    pos = at[seq] + t - (cu - counts)[seq]
    slot = tables[seq, (pos // page).clamp(0, tables.shape[1] - 1)].long()
    none = torch.full_like(t, -1)
    return {"tables": tables, "pages": torch.where(good, slot, none),
            "places": torch.where(good, pos % page, none), "positions": torch.where(good, pos, none),
            "granted": torch.where(ok, counts, 0).int()}


def _plain_attn(s):
    c = s["case"]
    n, nh, nkv, hd, page = c["n"], c["nh"], c["nkv"], c["hd"], c["page"]
    q, k, v = _split(s)
    if c["whole"]:
        t = _plain_reserve(s)
        s["storage"][0, 0].index_put_((t["pages"], t["places"]), k)
        s["storage"][0, 1].index_put_((t["pages"], t["places"]), v)
    K = max(_contexts(c)[0]) + 1
    pages = s["tables"][:, :-(-K // page)].long()
    # [n, nkv, K, hd]
    kk, vv = (s["storage"][0, i][pages].reshape(n, -1, nkv, hd)[:, :K].transpose(1, 2).float()
              .contiguous() for i in (0, 1))
    w = q.reshape(n, nkv, nh // nkv, hd).float() @ kk.transpose(2, 3) * hd ** -0.5
    w.masked_fill_((torch.arange(K, device="cuda") > s["lengths"][:, None])[:, None, None], -math.inf)
    w = (w - w.amax(-1, keepdim=True)).exp_()
    w /= w.sum(-1, keepdim=True)
    out = (w @ vv).reshape(n, nh, hd).to(q.dtype)
    return {"out": out, "kv": s["storage"]} if c["whole"] else {"out": out}


def _plain_select(s):
    """The best of each beam by (logit, lowest token), then the best of those in 64 bits."""
    c, logits, scores, done = s["case"], s["logits"], s["scores"].double(), s["done"]
    n, W, vocab = logits.shape
    k = c["k"]
    # logits as whole numbers of the same order, and below them the token, the lowest first
    bits = logits.float().view(torch.int32).long()
    key = torch.where(bits < 0, -2147483648 - bits, bits) * vocab
    key += vocab - 1 - torch.arange(vocab, device="cuda")
    at = key.topk(min(k, vocab), -1).indices
    x = logits.double()
    top = x.amax(-1, keepdim=True)
    norm = (x - top).exp_().sum(-1, keepdim=True).log_()
    value = scores[..., None] + (x.gather(2, at) - top - norm)
    # a finished beam stays as it is
    first = torch.arange(at.shape[-1], device="cuda") == 0
    value = torch.where(done[..., None], torch.where(first, scores[..., None], -math.inf), value)
    at = torch.where(done[..., None], 0, at)
    value = torch.nan_to_num(value, nan=-math.inf, neginf=-math.inf).reshape(n, -1)
    value, order = value.sort(dim=-1, descending=True, stable=True)
    short = max(0, k - value.shape[1])
    value = torch.nn.functional.pad(value[:, :k], (0, short), value=-math.inf)
    order = torch.nn.functional.pad(order[:, :k], (0, short))
    found = value > -math.inf
    parents = torch.where(found, order // at.shape[-1], -1)
    tokens = torch.where(found, at.reshape(n, -1).gather(1, order), -1)
    ended = done.gather(1, parents.clamp(min=0)) | (tokens[..., None] == s["stop"][:, None]).any(-1)
    return {"scores": value.float(), "parents": parents.int(), "tokens": tokens,
            "done": ended | ~found}


def _plain_reorder(s):
    page, W = s["case"]["page"], s["case"]["beams"]
    tables, lengths, parents = s["tables"], s["lengths"], s["parents"].long()
    n = parents.numel()
    at = torch.arange(W, device="cuda")
    up = (parents + W * torch.arange(n // W, device="cuda")[:, None]).reshape(-1)
    tables[:n], lengths[:n] = tables[up], lengths[up]
    # every child of a beam but the first one needs a page for the tokens of an unfinished page
    later = (torch.tril(parents[:, :, None] == parents[:, None], -1)).any(-1).reshape(-1)
    copies = later & (lengths[:n] % page > 0)
    tail = lengths[:n] // page
    column = torch.arange(tables.shape[1], device="cuda")
    keep = torch.ones_like(tables, dtype=torch.bool)
    keep[:n] = ~(copies[:, None] & (column == tail[:, None]))
    order, _ = _free_pages(s, tables, lengths, keep)
    tail.clamp_(max=tables.shape[1] - 1)
    row = torch.arange(n, device="cuda")
    source = tables[row, tail].long()
    fresh = order[(copies.long().cumsum(0) - 1).clamp(0, len(order) - 1)]
    tables[row, tail] = torch.where(copies, fresh, source).int()
    # the places that hold tokens; what is behind them stays
    row = copies.nonzero()[:, 0]
    fresh, source = fresh[row], source[row]
    filled = torch.arange(page, device="cuda") < (lengths[row] % page)[:, None]
    s["storage"][:, :, fresh] = torch.where(filled[..., None, None], s["storage"][:, :, source],
                                            s["storage"][:, :, fresh])
    return {"kv": s["storage"], "tables": tables, "lengths": lengths}


def run(state):
    if own:
        return _own_run(state)
    return {"attn": _plain_attn, "slots": _plain_reserve, "select": _plain_select,
            "reorder": _plain_reorder}[state["kind"]](state)


# ------------------------------------------------------------------------- bytes and operations
def work(case):
    n = case["n"]
    if case["family"] == "select":
        size = {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
        rows = n * case["beams"]
        return {"bytes": rows * (case["vocab"] * size + 5.0) + n * case["k"] * 17.0,
                "flops": 3.0 * rows * case["vocab"]}
    rows, shared = _contexts(case)
    page = case["page"]
    entries = sum(-(-a // page) for a in rows)
    if case["family"] == "slots":
        new = _new(case)
        return {"bytes": 4.0 * entries + 8 * len(rows) + 24 * sum(new) + 8 * n, "flops": 0.0}
    token = 2 * case["nkv"] * case["hd"] * 2
    if case["family"] == "reorder":
        W = case["beams"]
        moved = sum(a % page for a in rows[::W]) * (W - 1) / 2     # a beam in two has a sibling
        return {"bytes": 2.0 * moved * token * NL + 8.0 * entries + 20 * n, "flops": 0.0}
    keys = sum(a + 1 - (b if i % case["beams"] else 0) for i, (a, b) in enumerate(zip(rows, shared)))
    return {"bytes": float(keys) * token + 4 * entries + 4 * n * case["nh"] * case["hd"],
            "flops": 4.0 * (sum(rows) + n) * case["nh"] * case["hd"]}


# ------------------------------------------------------------------------- in 64 bits
def _unheld(case, tables, lengths, pages):
    """Pages that no sequence's tokens are in, ascending."""
    held = set()
    for row, m in zip(tables, lengths):
        held.update(row[:-(-m // case["page"])])
    return [p for p in range(pages) if p not in held]


def _exact_reserve(case, s):
    tables, lengths, page = s["tables"].tolist(), s["lengths"].tolist(), case["page"]
    free = _unheld(case, tables, lengths, s["pages"])
    out = {"pages": [], "places": [], "positions": [], "granted": []}
    asked = 0
    for i, m in enumerate(_new(case)):
        have = -(-lengths[i] // page)
        more = -(-(lengths[i] + m) // page) - have
        start, asked = asked, asked + more
        ok = m > 0 and (more == 0 or asked <= len(free))
        out["granted"].append(m if ok else 0)
        if ok:
            tables[i][have:have + more] = free[start:asked]
        for p in range(lengths[i], lengths[i] + m):
            out["pages"].append(tables[i][p // page] if ok else -1)
            out["places"].append(p % page if ok else -1)
            out["positions"].append(p if ok else -1)
    for name in ("pages", "places", "positions"):
        out[name] += [-1] * (s["tokens"] - len(out[name]))
    out = {name: torch.tensor(v) for name, v in out.items()}
    out["granted"] = out["granted"].int()
    return dict(out, tables=torch.tensor(tables, dtype=torch.int32))


def _exact_attn(case, s):
    n, nh, nkv, hd, page = case["n"], case["nh"], case["nkv"], case["hd"], case["page"]
    q, k, v = (x.double() for x in _split(s))
    t = _exact_reserve(case, s)
    tables, lengths = t["tables"].cuda().long(), s["lengths"].tolist()
    kv = s["storage"].clone() if case["whole"] else s["storage"]
    if case["whole"]:
        for i in range(n):
            kv[0, :, int(t["pages"][i]), int(t["places"][i])] = torch.stack([k[i], v[i]]).to(kv.dtype)
    out = torch.zeros(n, nh, hd, dtype=torch.float64, device="cuda")
    for i in range(n):
        held = tables[i, :lengths[i] // page + 1]
        keys = kv[0, 0, held].double().reshape(-1, nkv, hd)[:lengths[i] + 1]
        values = kv[0, 1, held].double().reshape(-1, nkv, hd)[:lengths[i] + 1]
        for g in range(nkv):
            mine = slice(g * (nh // nkv), (g + 1) * (nh // nkv))
            w = torch.softmax(q[i, mine] @ keys[:, g].t() / math.sqrt(hd), -1)
            out[i, mine] = w @ values[:, g]
    return {"out": out, "kv": kv.double()} if case["whole"] else {"out": out}


def _exact_select(case, s):
    """All continuations of a request in one line, the best taken out one after another."""
    n, W, vocab, k = case["n"], case["beams"], case["vocab"], case["k"]
    scores, done, stop = s["scores"].tolist(), s["done"].tolist(), s["stop"].tolist()
    out = {"scores": [], "parents": [], "tokens": [], "done": []}
    for i in range(n):
        line = torch.full((W, vocab), -math.inf, dtype=torch.float64, device="cuda")
        for b in range(W):
            if scores[i][b] == -math.inf:
                continue
            if done[i][b]:
                line[b, 0] = scores[i][b]
            else:
                line[b] = torch.log_softmax(s["logits"][i, b].double(), -1) + scores[i][b]
        line = line.reshape(-1)
        rows = {name: [] for name in out}
        for _ in range(k):
            best = float(line.max())
            if best == -math.inf:
                b = token = -1
            else:
                where = int(torch.nonzero(line == best)[0])
                line[where] = -math.inf
                b, token = divmod(where, vocab)
            rows["scores"].append(best)
            rows["parents"].append(b)
            rows["tokens"].append(token)
            rows["done"].append(b < 0 or done[i][b] or token in stop[i])
        for name, v in rows.items():
            out[name].append(v)
    kinds = {"scores": torch.float64, "parents": torch.int32, "tokens": torch.int64, "done": torch.bool}
    return {name: torch.tensor(v, dtype=kinds[name]) for name, v in out.items()}


def _exact_reorder(case, s):
    W, page = case["beams"], case["page"]
    old, lengths = s["tables"].tolist(), s["lengths"].tolist()
    parents = s["parents"].tolist()
    tables, after, wants = [], [], []
    for i in range(len(old)):
        b = parents[i // W][i % W]
        up = i - i % W + b
        tables.append(list(old[up]))
        after.append(lengths[up])
        if lengths[up] % page and b in parents[i // W][:i % W]:
            wants.append((i, up))
    held = [row[:-(-m // page)] for row, m in zip(tables, after)]
    for i, _ in wants:
        held[i] = held[i][:-1]
    used = {p for row in held for p in row}
    free = (p for p in range(s["pages"]) if p not in used)
    kv, new = s["storage"], s["storage"].clone()
    for i, up in wants:
        j, m = after[i] // page, after[i] % page
        tables[i][j] = next(free)
        new[:, :, tables[i][j], :m] = kv[:, :, old[up][j], :m]
    return {"kv": new, "tables": torch.tensor(tables, dtype=torch.int32),
            "lengths": torch.tensor(after)}


def exact(case, seed):
    s = _select_prepare(case, seed) if case["family"] == "select" else _cache_prepare(case, seed)
    return {"attn": _exact_attn, "slots": _exact_reserve, "select": _exact_select,
            "reorder": _exact_reorder}[case["family"]](case, s)
