"""Plain restatements of the paged cache's operators and of beam search's choice, for the tests:
whole numbers on Python lists, attention and log-probabilities in 64 bits."""

from __future__ import annotations

import math

import torch


def pages_of(tokens: int, page: int) -> int:
    return -(-tokens // page)


def free_pages(tables, lengths, pages: int, page: int) -> list:
    held = {p for row, m in zip(tables, lengths) for p in row[:pages_of(m, page)]}
    return [p for p in range(pages) if p not in held]


def reserve(tables, lengths, counts, rows, pages: int, page: int, max_len: int, tokens: int,
            dense: bool = False):
    """(tables, granted, starts, after, per packed row (page, place, position))."""
    tables = [list(row) for row in tables]
    free = free_pages(tables, lengths, pages, page)
    slots = [(-1, -1, -1)] * tokens
    granted, starts, after, used, at = [], [], [], 0, 0
    for i, (row, c) in enumerate(zip(rows, counts)):
        c = min(max(c, 0), 1) if dense else max(c, 0)
        L = lengths[row]
        at, end = (i, i + 1) if dense else (at, at + c)
        fits = c > 0 and L + c <= max_len and end <= tokens
        need = pages_of(L + c, page) - pages_of(L, page) if fits else 0
        used += need
        if fits and need and used > len(free):
            fits = False
        elif fits:
            tables[row][pages_of(L, page):pages_of(L + c, page)] = free[used - need:used]
            for j in range(c):
                p = L + j
                slots[at + j] = (tables[row][p // page], p % page, p)
        granted.append(c if fits else 0)
        starts.append(L)
        after.append(L + granted[-1])
        at = end
    return tables, granted, starts, after, slots


def reorder(tables, lengths, parents, pages: int, page: int):
    """(tables, lengths, copies) with copies a list of (from page, to page, tokens)."""
    W = len(parents[0])
    old, had = [list(row) for row in tables], list(lengths)
    tables, lengths = [list(row) for row in tables], list(lengths)
    wants = []
    for s, request in enumerate(parents):
        for w, p in enumerate(request):
            r = s * W + w
            if not 0 <= p < W:
                lengths[r] = 0
                continue
            tables[r], lengths[r] = list(old[s * W + p]), had[s * W + p]
            if lengths[r] % page and p in request[:w]:
                wants.append(r)
    # a page that is not full belongs to the first child alone
    free = free_pages(tables, [m - m % page if r in wants else m for r, m in enumerate(lengths)], pages,
                      page)
    copies = []
    for r in wants:
        if not free:
            lengths[r] = 0
            continue
        j = lengths[r] // page
        copies.append((tables[r][j], free[0], lengths[r] % page))
        tables[r][j] = free.pop(0)
    return tables, lengths, copies


def attention(q, k, v, scale: float):
    """One query a head over keys: q [nh, hd], k / v [L, nkv, hd] -> ([nh, hd], sum of weights times
    |v| alike), in 64 bits."""
    nh, hd = q.shape
    nkv = k.shape[1]
    q, k, v = q.double(), k.double(), v.double()
    out, mag = torch.zeros(nh, hd, dtype=torch.float64), torch.zeros(nh, hd, dtype=torch.float64)
    for h in range(nh):
        g = h // (nh // nkv)
        w = torch.softmax(k[:, g] @ q[h] * scale, 0)
        out[h], mag[h] = w @ v[:, g], w @ v[:, g].abs()
    return out, mag


def attention_bound(out, mag, keys: int, v_max: float, dtype):
    """How far an output may be off: its own rounding; probabilities rounded to the same type,
    relative to a largest of 1 over a sum of at least 1; and fp32 scores, sums and exponentials, 2^-13
    of the probabilities.  fp16 steps stay at 2^-24 below the normal range."""
    half = torch.finfo(dtype).eps / 2
    low = 2.0 ** -25 if dtype == torch.float16 else 0.0
    return out.abs() * half + low + mag * (half + 2.0 ** -13) + keys * low * v_max


def select(logits, scores, k: int, done=None, stop=None, pad: int = 0):
    """Lists of k (score, beam, token, finished) per request."""
    out = []
    for s in range(logits.shape[0]):
        every = []
        for b in range(logits.shape[1]):
            score = float(scores[s, b])
            if not math.isfinite(score):
                continue
            if done is not None and bool(done[s, b]):
                every.append((-score, b, 0, pad, True))
                continue
            x = logits[s, b].double()
            x = torch.where(torch.isnan(x), torch.full_like(x, -math.inf), x)
            m = float(x.max())
            if m == -math.inf:
                continue
            if m == math.inf:
                lp = torch.where(x == m, -math.log(int((x == m).sum())), -math.inf)
            else:
                lp = (x - m) - torch.log(torch.exp(x - m).sum())
            # the first k by logit and token are enough
            order = torch.argsort(x, descending=True, stable=True)[:k].tolist()
            every += [(-(score + float(lp[v])), b, rank, v, False) for rank, v in enumerate(order)
                      if float(lp[v]) > -math.inf]
        every.sort()
        rows = []
        for value, b, _, v, over in every[:k]:
            ends = stop is not None and v in (stop[s] if isinstance(stop[0], list) else stop)
            rows.append((-value, b, v, over or ends))
        out.append(rows + [(-math.inf, -1, -1, True)] * (k - len(rows)))
    return out
