"""The paged cache's operators and beam search's choice without a GPU: refusals before any launch, the
plain forms' own properties, and what the runner makes of the choices."""

import ctypes
import math
import random

import pytest
import torch

from oracle import paged_ref as ref

P = ctypes.c_void_p(16)          # never read: the checks fail first


def cache(num_pages=8, page_size=16, max_seqs=4, max_len=64, hd=128, **kw):
    from omniserver_amd.paged_kv import PagedKVCache
    return PagedKVCache(2, num_pages, 2, page_size, hd, "cpu", max_seqs=max_seqs, max_len=max_len, **kw)


def test_reserve_refusals():
    from omniserver_amd._lib import lib

    def rc(tables=P, lengths=P, seqs=4, width=4, pages=8, page=16, max_len=64, counts=P, rows=None,
           n=2, tokens=8, dense=0, axes=1, starts=P, token_page=P, positions=P, granted=P,
           schedule=None, columns=0, most=0):
        return lib().omni_page_reserve(tables, lengths, seqs, width, pages, page, max_len, counts, rows,
                                       None, n, tokens, dense, axes, starts, P, token_page, P,
                                       positions, granted, P, schedule, columns, most, None)

    assert rc(n=-1) == rc(tokens=-1) == rc(axes=0) == rc(n=5) == -1
    assert rc(seqs=0) == rc(width=0) == rc(pages=0) == rc(max_len=0) == rc(page=0) == -1
    assert rc(page=8) == rc(page=24) == rc(page=2048) == rc(pages=(1 << 19) + 1) == rc(seqs=2049) == -2
    assert rc(max_len=(1 << 30) + 1, width=1 << 27) == rc(seqs=2048, width=(1 << 19) + 1) == -2
    assert rc(tokens=(1 << 28) + 1) == rc(axes=4) == -2
    assert rc(max_len=65) == rc(tables=None) == rc(lengths=None) == -1
    assert rc(starts=None) == rc(granted=None) == rc(token_page=None) == rc(positions=None) == -1
    plan = {"schedule": P, "columns": 4, "most": 5}
    dense = {"dense": 1, "tokens": 2, **plan}
    assert rc(dense=1) == rc(**plan) == rc(**{**dense, "columns": 0}) == rc(**{**dense, "most": 0}) == -1
    assert rc(**dense, rows=P) == rc(**{**dense, "schedule": ctypes.c_void_p(8)}) == -1
    assert rc(**{**dense, "columns": 65536}) == -2
    assert rc(**{**dense, "n": 2048, "tokens": 2048}, seqs=2048, max_len=1 << 27, width=1 << 19,
              page=256) == -2
    assert rc(n=0) == 0


def test_reorder_refusals():
    from omniserver_amd._lib import lib

    def rc(pool=P, layers=2, halfs=256, tables=P, lengths=P, seqs=8, width=4, pages=8, page=16,
           max_len=64, parents=P, n=2, beams=4, work=P, ints=32):
        return lib().omni_page_reorder(pool, layers, halfs, tables, lengths, seqs, width, pages, page,
                                       max_len, parents, n, beams, work, ints, None)

    assert rc(layers=0) == rc(halfs=0) == rc(n=-1) == rc(beams=0) == rc(n=3) == -1
    assert rc(halfs=260) == rc(page=20) == rc(halfs=1 << 25) == -2
    assert rc(pool=None) == rc(parents=None) == rc(work=None) == rc(ints=31) == rc(tables=None) == -1
    assert rc(pool=ctypes.c_void_p(24)) == rc(work=ctypes.c_void_p(8)) == -1
    assert rc(n=0) == 0


def test_attention_refusals():
    from omniserver_amd._lib import lib

    def rc(q=P, q_stride=1536, k=P, dtype=0, pages=8, page=16, tables=P, width=4, n=2, schedule=P,
           columns=4, most=5, out=P, out_stride=1536, nh=12, nkv=2, hd=128, scale=0.1, ws=P,
           floats=1 << 30):
        return lib().omni_paged_attention(q, q_stride, k, P, dtype, pages, page, tables, width, n,
                                          schedule, columns, most, out, out_stride, nh, nkv, hd, scale,
                                          ws, floats, None)

    assert rc(n=-1) == rc(pages=0) == rc(page=0) == rc(width=0) == rc(columns=0) == rc(most=0) == -1
    assert rc(nh=0) == rc(nkv=0) == -1
    assert rc(dtype=2) == rc(hd=96) == rc(nh=13) == rc(page=20) == rc(columns=65536) == rc(n=65536) == -2
    assert rc(scale=0.0) == rc(scale=-1.0) == rc(scale=float("nan")) == rc(scale=float("inf")) == -2
    assert rc(most=6) == -2                                       # 36 queries
    assert rc(q_stride=1528) == rc(q_stride=1540) == rc(out_stride=8) == rc(out_stride=1540) == -1
    assert rc(q=None) == rc(k=None) == rc(tables=None) == rc(schedule=None) == rc(out=None) == -1
    assert rc(ws=None) == rc(q=ctypes.c_void_p(24)) == rc(out=ctypes.c_void_p(8)) == -1
    need = 12 * ((4 * 5 + 2) + (4 + 2)) * 132
    assert rc(floats=need - 1) == rc(most=1, floats=12 * 6 * 132 - 1) == -1
    assert rc(columns=65535, n=60000, nh=1024, nkv=1024, q_stride=1 << 17, out_stride=1 << 17) == -2
    assert rc(n=0) == 0


def test_select_refusals():
    from omniserver_amd._lib import lib

    assert lib().omni_beam_select_work(1, 4, 151936, 4) > 0
    assert lib().omni_beam_select_work(-1, 4, 100, 4) == lib().omni_beam_select_work(1, 0, 100, 4) == -1
    assert lib().omni_beam_select_work(1, 4, 0, 4) == lib().omni_beam_select_work(1, 4, 100, 0) == -1
    for bad in ((1, 33, 100, 4), (1, 4, 100, 65), (1, 4, 524289, 4), (65536, 1, 100, 1),
                (60000, 32, 524288, 64)):
        assert lib().omni_beam_select_work(*bad) == -2

    def rc(logits=P, dtype=0, strides=(400, 100), scores=P, stop=None, stops=0, n=1, W=4, V=100, k=4,
           out=P, ws=P, words=1 << 20):
        return lib().omni_beam_select(logits, dtype, *strides, scores, None, stop, stops, 0, 0, n, W, V,
                                      k, out, P, P, P, ws, words, None)

    assert rc(dtype=3) == rc(k=65) == -2
    assert rc(strides=(-1, 100)) == rc(strides=(400, -1)) == rc(stops=-1) == rc(stops=1) == -1
    assert rc(logits=None) == rc(scores=None) == rc(out=None) == rc(ws=None) == -1
    assert rc(words=lib().omni_beam_select_work(1, 4, 100, 4) - 1) == rc(ws=ctypes.c_void_p(8)) == -1
    assert rc(n=0) == 0


def test_cache_checks_its_arguments():
    for bad in ({"page_size": 8}, {"page_size": 48}, {"hd": 96}, {"num_pages": 0},
                {"num_pages": (1 << 19) + 1}, {"max_seqs": 0}, {"max_seqs": 2049}, {"max_len": 0},
                {"n_heads": 13}, {"n_heads": 0}, {"dtype": torch.float32}):
        with pytest.raises(ValueError):
            cache(**bad)
    c = cache(max_len=65)
    assert c.tables.shape == (4, 5) and c.storage.shape == (2, 2, 8, 16, 2, 128) and c.n_heads == 12
    with pytest.raises(ValueError):
        c.reserve(torch.ones(2, dtype=torch.int32))                    # how many rows?
    for bad in ([], [1] * 5, [-1], [66]):
        with pytest.raises(ValueError):
            c.reserve(bad)
    for rows in ([0], [0, 0], [0, 4], [-1, 0]):
        with pytest.raises(ValueError):
            c.reserve([1, 1], rows=rows)
    with pytest.raises(ValueError):
        c.reserve([1, 1], tokens=-1)
    with pytest.raises(TypeError):
        c.reserve(torch.ones(2, dtype=torch.int64), tokens=2)
    with pytest.raises(RuntimeError, match="GPU only"):
        c.reserve([1, 1])
    for bad in ([[0, 2]], [[0, 0], [0]], [], [[0] * 5]):
        with pytest.raises(ValueError):
            c.reorder(bad)
    with pytest.raises(TypeError):
        c.reorder(torch.zeros(1, 2, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="GPU only"):
        c.reorder([[0, 0]])
    for rows in ([4], [-1], [1, 1]):
        with pytest.raises(ValueError):
            c.free(rows)
    c.lengths.fill_(5)
    c.free([2, 0])
    assert c.lengths.tolist() == [0, 5, 0, 5]
    for bad in (([0], []), ([0], [66]), ([0, 1], [3]), ([0], [0]), ([], [])):
        with pytest.raises(ValueError):
            c.prefill_cache(*bad)
    with pytest.raises(ValueError):
        cache(dtype=torch.bfloat16).prefill_cache([0], [4])


def test_refused_prompts_leave_their_rows():
    """Sequences are forgotten for prompts that are taken, not for those that are refused."""
    c = cache(page_size=1024, max_len=1 << 28)
    c.lengths.fill_(5)
    step = c._step
    for error, rows, lens in ((ValueError, [0, 1], [1 << 28, 1]), (ValueError, [0, 4], [1, 1]),
                              (ValueError, [2, 2], [1, 1]), (RuntimeError, [0, 3], [4, 7])):
        with pytest.raises(error):
            c.prefill_cache(rows, lens)
        assert c.lengths.tolist() == [5] * 4 and c._step == step, rows


def test_adapters_check_their_rows():
    """Rows, outputs and positions of other sizes or types never reach a kernel."""
    from omniserver_amd.paged_kv import PagedDecode, PagedPrefill
    c = cache()
    qkv, out = torch.zeros(3, 16 * 128).half(), torch.empty(3, 12, 128).half()
    pos = torch.zeros(3, 3, dtype=torch.int64)
    q, k = torch.zeros(3, 12, 128).half(), torch.zeros(3, 2, 128).half()
    for kind in (PagedDecode, PagedPrefill):
        step = object.__new__(kind)
        step.pool, step.n, step.T, step._step = c, 3, 3, c._step
        attend = lambda x, y: step.attend_qkv(x, 0, 0.1, y)
        rotate = lambda x, p: step.rope_and_write(x, 0, p, None, None, (16, 24, 24))
        flash = step.flash_decode if kind is PagedDecode else step.flash_prefill
        for x, y in ((qkv[:2], out), (qkv[:, :1535], out), (qkv.view(-1), out), (qkv, out[:2]),
                     (qkv.t().contiguous().t(), out), (qkv, out.transpose(0, 1))):
            with pytest.raises(ValueError):
                attend(x, y)
        for x, y in ((qkv.float(), out), (qkv, out.float()), (qkv.bfloat16(), out.bfloat16())):
            with pytest.raises(TypeError):
                attend(x, y)
        for x, p in ((qkv[:, :2047], pos), (qkv[:2], pos), (qkv, pos[:2]), (qkv, pos.int()), (qkv, pos.t()[:2])):
            with pytest.raises(ValueError):
                rotate(x, p)
        with pytest.raises(TypeError):
            rotate(qkv.float(), pos)
        for bad in (q[:2], q[:, :11], q[..., :64], q.float()):
            with pytest.raises(ValueError):
                flash(bad, k, k, 0, 0.1)
        for call in (lambda: attend(qkv, out), lambda: rotate(qkv, pos), lambda: flash(q, k, k, 0, 0.1)):
            with pytest.raises(RuntimeError, match="GPU only"):
                call()


def test_select_checks_its_arguments():
    from omniserver_amd.beam import select
    logits, scores = torch.zeros(2, 3, 50), torch.zeros(2, 3)
    for bad in ({"k": 0}, {"k": 65}, {"done": torch.zeros(2, 2, dtype=torch.bool)},
                {"stop": torch.zeros(3, 1, dtype=torch.int64)}, {"stop": torch.tensor(1)}):
        with pytest.raises(ValueError):
            select(logits, scores, **bad)
    for bad in ({"done": torch.zeros(2, 3)}, {"stop": torch.zeros(1)}):
        with pytest.raises(TypeError):
            select(logits, scores, **bad)
    for x, y in ((logits[0], scores), (torch.zeros(2, 33, 50), torch.zeros(2, 33)),
                 (logits, torch.zeros(2, 2)), (logits.transpose(1, 2), torch.zeros(2, 50)),
                 (torch.zeros(2, 3, 0), scores)):
        with pytest.raises(ValueError):
            select(x, y)
    with pytest.raises(TypeError):
        select(logits.double(), scores)
    with pytest.raises(TypeError):
        select(logits, scores.half())
    with pytest.raises(RuntimeError, match="GPU only"):
        select(logits, scores, stop=[1])


def test_attention_columns():
    from omniserver_amd.paged_kv import attention_columns, attention_group
    assert attention_columns(1, 12, 2, 300, 256) == 3            # a column a unit
    assert attention_columns(32, 12, 2, 4096, 256) == 256
    assert attention_columns(64, 16, 16, 4096, 256) == 32
    assert attention_columns(1, 64, 1, 1 << 20, 256) == 256       # two groups of 32 heads
    assert attention_columns(4, 8192, 1024, 4096, 256) == 1
    assert [attention_group(nh, 1) for nh in (1, 6, 16, 17, 64)] == [32, 5, 2, 1, 1]


def test_reserve_plain_form():
    tables = [[3, 9, 9], [9, 9, 9], [0, 1, 9]]
    t, granted, starts, after, slots = ref.reserve(tables, [16, 0, 20], [2, 40, 3], [0, 1, 2], 6, 16, 48, 45)
    # pages 2, 4, 5 are free: one for the first, the second's three are not all there, the third
    # needs none
    assert granted == [2, 0, 3] and starts == [16, 0, 20] and after == [18, 0, 23]
    assert t == [[3, 2, 9], [9, 9, 9], [0, 1, 9]]
    assert slots[:3] == [(2, 0, 16), (2, 1, 17), (-1, -1, -1)] and slots[42:] == [(1, 4, 20), (1, 5, 21), (1, 6, 22)]


def test_reorder_plain_form_keeps_every_beams_tokens():
    """Random reorderings, tokens added between them: what a beam's table names is the beam's tokens."""
    rng = random.Random(1)
    n, W, page, pages, width = 2, 4, 4, 60, 12
    tables, lengths = [[0] * width for _ in range(n * W)], [0] * (n * W)
    store, lines = [[None] * page for _ in range(pages)], [[] for _ in range(n * W)]
    for step in range(30):
        counts = [1 if step else rng.randint(1, 9) for _ in range(n * W)]
        tables, granted, _, after, slots = ref.reserve(tables, lengths, counts, range(n * W), pages, page,
                                                       width * page, sum(counts))
        assert granted == counts
        at = 0
        for r, c in enumerate(counts):
            for j in range(c):
                p, place, _ = slots[at]
                store[p][place] = (r, step, j)
                lines[r] = lines[r] + [(r, step, j)]
                at += 1
        parents = [[rng.randrange(W) for _ in range(W)] for _ in range(n)]
        tables, lengths, copies = ref.reorder(tables, after, parents, pages, page)
        for a, b, m in copies:
            store[b][:m] = store[a][:m]
        lines = [lines[s * W + p] for s, q in enumerate(parents) for p in q]
        for r, line in enumerate(lines):
            assert lengths[r] == len(line)
            assert [store[tables[r][t // page]][t % page] for t in range(len(line))] == line


def test_select_plain_form():
    logits = torch.log(torch.tensor([[[0.5, 0.25, 0.25], [0.1, 0.8, 0.1]]]))
    got = ref.select(logits, torch.tensor([[math.log(0.5), math.log(0.4)]]), 4, stop=[1])[0]
    assert [(b, t, d) for _, b, t, d in got] == [(1, 1, True), (0, 0, False), (0, 1, True), (0, 2, False)]
    assert [round(math.exp(v), 4) for v, *_ in got] == [0.32, 0.25, 0.125, 0.125]
    done = torch.tensor([[False, True]])
    got = ref.select(logits, torch.tensor([[-math.inf, -1.0]]), 2, done, pad=7)[0]
    assert got == [(-1.0, 1, 7, True), (-math.inf, -1, -1, True)]


def test_beams_of_choices():
    """Lines of tokens from the steps' choices: a finished beam goes on with -1, and counts as long as
    it is; a beam that was never there is left out."""
    from omniserver_amd.runner import _beams_of
    tokens = [[[5, 6, 7]], [[8, -1, 9]], [[1, -1, 2]]]
    parents = [[[0, 0, 0]], [[1, 0, 1]], [[0, 1, 0]]]
    found = _beams_of(tokens, parents, [[-3.0, -1.5, -math.inf]], 1.0)[0]
    assert [(b.tokens, b.score) for b in found] == [([6, 8, 1], -1.0), ([5], -1.5)]
    assert [b.tokens for b in _beams_of(tokens, parents, [[-3.0, -1.5, -math.inf]], 0.0)[0]] == [[5], [6, 8, 1]]
