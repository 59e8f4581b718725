"""Speculative decoding without a GPU where it ends badly: what the runner leaves behind, sizes that
the kernels do not take."""

import ctypes
from types import SimpleNamespace

import numpy as np
import pytest
import torch

VOCAB = 50
P = ctypes.c_void_p(16)          # never read: the checks fail first


def bare_runner(lengths, emitted_tokens):
    """A runner over a CPU pool, its step replaced: emitted_tokens [n][..] is what verification
    gives, the pool's lengths move as acceptance moves them."""
    from omniserver_amd.kv_cache import PreallocatedKVCache
    from omniserver_amd.request import Request, SamplingParams, Sequence
    from omniserver_amd.runner import MultimodalRunner
    from omniserver_amd.speculative import Verified
    n = len(lengths)
    r = MultimodalRunner.__new__(MultimodalRunner)
    r.adapter = SimpleNamespace(model=SimpleNamespace(cfg=SimpleNamespace(vocab_size=VOCAB)))
    r.device = torch.device("cpu")
    r._pool = PreallocatedKVCache(1, n + 1, 2, 64, 128, "cpu", n_heads=12)
    r._pool.lengths[:n] = torch.tensor(lengths)
    r._kv_len = list(lengths)
    r._use_graph, r._ahead, r._dev_ids_for = False, None, None
    seqs = [Sequence(Request(prompt=list(range(L)), sampling=SamplingParams(max_new_tokens=9)),
                     prompt_token_ids=list(range(L)), kv_handle={"slot": s, "rope_delta": 0})
            for s, L in enumerate(lengths)]
    for s in seqs:
        s.append_token(7)

    def step(step):
        T = step["ids"].shape[1]
        tokens = torch.tensor([row + [-1] * (T - len(row)) for row in emitted_tokens])
        emitted = torch.tensor([len(row) for row in emitted_tokens], dtype=torch.int32)
        r._pool.lengths[:n] += emitted
        return Verified(torch.zeros(n, T, dtype=torch.int32), tokens, emitted)

    r._spec_step = step
    return r, seqs


def test_speculate_keeps_the_others_tokens():
    """Sequences that nothing can be drawn for, one of them after a drafted token that stands: the
    others have their tokens, everyone's cached rows are its tokens but the last."""
    lengths = [10, 11, 12, 13]
    emitted = [[5, 6], [-1], [8, -1], [9, 3, 4]]
    r, seqs = bare_runner(lengths, emitted)
    with pytest.raises(RuntimeError, match=r"\[1, 2\]"):
        r.speculate(seqs, [[3, 0]] * 4)
    assert [s.output_token_ids for s in seqs] == [[7, 5, 6], [7], [7, 8], [7, 9, 3, 4]]
    assert r._kv_len == [s.total_len - 1 for s in seqs]
    assert r._pool.lengths[:4].tolist() == r._kv_len


def test_speculate_that_fails_behind_acceptance():
    """An error once the lengths have moved (a capture out of memory): the lengths as before, so
    that the same call can be made again."""
    r, seqs = bare_runner([10, 11], [[5, 6], [4]])
    step = r._spec_step

    def fails(s):
        step(s)
        raise MemoryError

    r._spec_step = fails
    with pytest.raises(MemoryError):
        r.speculate(seqs, [[3], [3]])
    assert r._pool.lengths[:2].tolist() == r._kv_len == [10, 11]
    assert [s.output_token_ids for s in seqs] == [[7], [7]]
    r._spec_step = step
    assert r.speculate(seqs, [[3], [3]]) == [2, 1]
    assert r._pool.lengths[:2].tolist() == r._kv_len == [12, 12]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64])
def test_speculate_refuses_draft_logits_of_another_type(dtype):
    r, seqs = bare_runner([10, 11], [[5], [4]])
    for temperature in (0.0, 0.7):
        seqs[0].request.sampling.temperature = temperature
        with pytest.raises(TypeError):
            r.speculate(seqs, [[3], [3]], draft_logits=torch.zeros(2, 1, VOCAB, dtype=dtype))
    assert r._pool.lengths[:2].tolist() == r._kv_len == [10, 11]


# ----------------------------------------------------------------------------- sizes
def attention_rc(n=2, nodes=8, nh=12, nkv=2, form=(64, 4), columns=4, least=0, q=None):
    from omniserver_amd._lib import lib
    return lib().omni_tree_attention(q, nh * 128, P, P, max(n, 1), 256, P, n, nodes, P, nh * 128, nh,
                                     nkv, 128, 0.1, *form, columns, least, P, None, 0, None)


@pytest.mark.parametrize("nodes,widest", [(64, 8192), (63, 8256), (17, 15894), (1, 65536)])
def test_tree_attention_head_ratio(nodes, widest):
    """Up to the widest ratio that is taken every row's node comes out right by the 32-bit
    reciprocal; wider ones are refused (q is null: what passes the sizes ends there, -1)."""
    for ratio in (widest, widest - 1, 6):
        rows, magic = np.arange(nodes * ratio, dtype=np.uint64), np.uint64(0xffffffff // ratio + 1)
        assert (rows * magic >> np.uint64(32) == rows // np.uint64(ratio)).all()
        assert attention_rc(nodes=nodes, nh=ratio, nkv=1, columns=2) == -1
    assert attention_rc(nodes=nodes, nh=widest + 1, nkv=1, columns=2) == -2


def test_tree_attention_head_ratio_goes_wrong():
    """Why: 64 nodes and a ratio of 16383 put row 278510 one node too far."""
    row, ratio = 278510, 16383
    assert row < 64 * ratio
    assert row * (0xffffffff // ratio + 1) >> 32 == row // ratio + 1
    assert attention_rc(nodes=64, nh=ratio, nkv=1, columns=2) == -2


def test_launches_that_do_not_count_in_32_bits():
    """A launch counts its threads in 32 bits: more rows are refused before any of a call's launches
    goes out."""
    from omniserver_amd._lib import lib
    work = lib().omni_spec_verify_work
    assert work((1 << 18) - 1, 64, 100, 0) > 0 and work(1 << 18, 64, 100, 0) == -2
    assert work((1 << 18) - 1, 33, 100, 1) == -2 and work(1 << 12, 64, 8192 * 64, 0) == -2
    assert work(1 << 17, 64, 8192, 0) > 0 and work(1 << 17, 64, 8193, 0) == -2
    for n, rc in (((1 << 18) - 1, -1), (1 << 18, -2)):          # without a workspace
        assert lib().omni_spec_verify(P, 0, 6400, 100, None, 0, 0, P, None, None, None, None, 0.0, n,
                                      64, 100, P, P, P, None, 0, None) == rc
    write = lambda n: lib().omni_kv_write_rows(None, 256, P, 256, P, P, P, P, 4, 64, 256, n, None)  # noqa: E731
    assert write((1 << 24) - 1) == -1 and write(1 << 24) == -2
    # 8 workgroups a column at 64 nodes of 16 heads, columns in eights
    wide = {"nodes": 64, "nkv": 16, "nh": 256, "form": (128, 2)}
    assert attention_rc(n=(1 << 16) - 2, columns=16 * ((1 << 16) - 2), **wide) == -1
    assert attention_rc(n=1 << 16, columns=1 << 20, **wide) == -2
    # a merge of a wave's half a row, eight rows a workgroup
    cut = {"nodes": 64, "nkv": 8, "nh": 64, "form": (128, 2), "columns": 32760, "least": 1}
    assert attention_rc(n=(1 << 15) - 1, **cut) == -1 and attention_rc(n=1 << 15, **cut) == -2


def test_verify_outputs_over_inputs():
    """Outputs that lie over an input other workgroups still read: refused, before a launch."""
    from omniserver_amd._lib import lib
    n, T = 3, 8
    at = {"tokens": (1 << 20, 8 * n * T), "parents": (2 << 20, 4 * n * T), "counts": (3 << 20, 4 * n),
          "u": (4 << 20, 4 * n * T), "temps": (5 << 20, 4 * n)}
    outs = {"path": 4 * n * T, "out": 8 * n * T, "emitted": 4 * n}

    def rc(**kw):
        a = {k: v[0] for k, v in at.items()} | {"path": 6 << 20, "out": 7 << 20, "emitted": 9 << 20} | kw
        p = {k: ctypes.c_void_p(v) for k, v in a.items()}
        return lib().omni_spec_verify(P, 0, 800, 100, None, 0, 0, p["tokens"], p["parents"],
                                      p["counts"], p["u"], p["temps"], 0.0, n, T, 100, p["path"],
                                      p["out"], p["emitted"], P, 1 << 20, None)

    for name, (start, size) in at.items():
        for o, osize in outs.items():
            assert rc(**{o: start}) == rc(**{o: start + size - 4}) == rc(**{o: start - osize + 4}) == -1
