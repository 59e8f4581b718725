"""Speculative decoding's operators in 64 bits on the CPU, one sequence and one node at a time:
attention of drafted trees over a cached prefix, verification of drafted tokens from given random
numbers, the cache after acceptance."""

from __future__ import annotations

import math

import torch


def lineage(parents, i: int) -> list:
    """Node i and its ancestors; an entry that is not an earlier node ends the walk."""
    out = [i]
    while 0 <= parents[out[-1]] < out[-1]:
        out.append(parents[out[-1]])
    return out


def tree_attention(q, k_pool, v_pool, starts, parents, counts, slots, scale: float):
    """q [n, T, nh, hd], pools [rows, max_len, nkv, hd] -> (out [n, T, nh, hd], the same sums with
    |v| in the place of v, keys seen [n, T]), float64; rows not in use are NaN in out."""
    n, T, nh, hd = q.shape
    max_len, nkv = k_pool.shape[1], k_pool.shape[2]
    out = torch.full((n, T, nh, hd), math.nan, dtype=torch.float64)
    mag, seen = out.clone(), torch.zeros(n, T, dtype=torch.int64)
    for s in range(n):
        for i in range(counts[s]):
            keys = list(range(starts[s])) + [starts[s] + j for j in sorted(lineage(parents[s], i))]
            keys = torch.tensor([x for x in keys if x < max_len], dtype=torch.int64)
            kk = k_pool[slots[s], keys].double()                       # [K, nkv, hd]
            vv = v_pool[slots[s], keys].double()
            seen[s, i] = len(keys)
            for h in range(nh):
                g = h // (nh // nkv)
                p = torch.softmax(kk[:, g] @ q[s, i, h].double() * scale, 0)
                out[s, i, h] = p @ vv[:, g]
                mag[s, i, h] = p @ vv[:, g].abs()
            if not len(keys):
                out[s, i] = mag[s, i] = 0.0
    return out, mag, seen


def attention_bound(out, mag, seen, v_max: float):
    """How far an fp16 output may be off: its own rounding (half a step: 2^-11 relative, 2^-25
    below the normal range); fp16 probabilities relative to a largest of 1, each off by 2^-11 of
    itself and, below the normal range, by 2^-25, over a sum of at least 1; and fp32 scores, sums
    and exponentials, a quarter of the probabilities' step."""
    return out.abs() * 2.0 ** -11 + 2.0 ** -25 + mag * (2.0 ** -11 + 2.0 ** -13) \
        + (seen * 2.0 ** -25 * v_max)[:, :, None, None]


def weights(row, temperature: float):
    """Probabilities of a logits row, float64: NaN counts as -inf, all zero without a token."""
    x = torch.where(torch.isnan(row), torch.full_like(row, -math.inf), row).double()
    m = x.max()
    if m == -math.inf:
        return torch.zeros_like(x)
    if temperature <= 0 or math.isnan(temperature):
        w = torch.zeros_like(x)
        w[int(torch.nonzero(x == m)[0])] = 1.0
        return w
    w = torch.where(x == m, torch.ones_like(x), torch.exp((x - m) / temperature))
    w[x == -math.inf] = 0.0
    return w / w.sum()


def draw(p, u: float) -> int:
    """First token whose running sum exceeds u times the total; -1 where all weights are zero."""
    run = p.cumsum(0)
    if float(run[-1]) <= 0:
        return -1
    hit = torch.nonzero((run > u * float(run[-1])) & (p > 0))
    return int(hit[0]) if len(hit) else int(torch.nonzero(p > 0)[-1])


def verify(logits, tokens, uniforms, temps, parents=None, draft=None, counts=None):
    """logits [n, T, V], tokens / uniforms / parents nested lists -> (path, tokens, emitted)."""
    n, T, V = logits.shape
    paths, outs, emitted = [], [], []
    for s in range(n):
        m = T if counts is None else counts[s]
        if m == 0:
            paths.append([-1] * T)
            outs.append([-1] * T)
            emitted.append(0)
            continue
        here, path = 0, [0]
        while True:
            own = p = weights(logits[s, here], temps[s])
            taken = None
            for i in range(here + 1, m):
                if (i - 1 if parents is None else parents[s][i]) != here:
                    continue
                x, u = tokens[s][i], uniforms[s][i]
                q = torch.zeros_like(p)
                if draft is not None and temps[s] > 0:
                    q = weights(draft[s, here], temps[s])
                elif 0 <= x < V:
                    q[x] = 1.0
                if 0 <= x < V and u * float(q[x]) < float(p[x]):
                    taken = i
                    break
                rest = (p - q).clamp(min=0.0)
                p = rest / rest.sum() if float(rest.sum()) > 0 else torch.zeros_like(p)
            if taken is None:
                break
            path.append(taken)
            here = taken
        if float(p.sum()) <= 0:
            p = own
        out = [tokens[s][i] for i in path[1:]] + [draw(p, uniforms[s][0])]
        emitted.append(len(path))
        paths.append(path + [-1] * (T - len(path)))
        outs.append(out + [-1] * (T - len(out)))
    return torch.tensor(paths), torch.tensor(outs), torch.tensor(emitted)


def accept(storage, starts, path, emitted, slots):
    """storage [layers, 2, rows, max_len, nkv, hd] -> (the storage after, lengths by row)."""
    out, lengths = storage.clone(), {}
    max_len = storage.shape[3]
    for s, slot in enumerate(slots):
        keep = []
        for j in range(emitted[s]):
            a = path[s][j]
            if a < (keep[-1] + 1 if keep else 0) or a >= len(path[s]) or starts[s] + a >= max_len:
                break
            keep.append(a)
        for j, a in enumerate(keep):
            out[:, :, slot, starts[s] + j] = storage[:, :, slot, starts[s] + a]
        lengths[slot] = starts[s] + len(keep)
    return out, lengths
