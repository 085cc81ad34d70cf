"""CPU pins of oracle/spans.py, and the host side of windows, trees and page moves."""
import ctypes
import random

import numpy as np
import pytest
import torch

import nano_qwen_amd.utils.context as C
from nano_qwen_amd import _lib, kernels
from nano_qwen_amd.engine import ModelRunner, Sequence
from nano_qwen_amd.layers import Attention
from oracle import paged, spans
from tests.spans import Case, random_tree, tree_reference


def test_wide_window_is_causal_attention():
    c = Case([5, 9], [20, 0], 4, 2, 128, torch.bfloat16, block=32)
    ref, _ = c.window_reference(10 ** 6, 0)
    f = lambda t: t.double().numpy()    # noqa: E731
    want = paged.varlen_prefill(f(c.q), np.nan_to_num(f(c.k)), np.nan_to_num(f(c.v)), c.cu_q.numpy(), c.cu_k.numpy(),
                                c.scale, c.table.numpy())
    np.testing.assert_allclose(ref.numpy(), np.asarray(want).reshape(ref.shape), rtol=1e-12, atol=1e-12)


def test_chain_is_causal_and_star_sees_itself():
    chain, star = [-1, 0, 1, 2, 3], [-1, 0, 0, 0, 0]
    c = Case([5, 5], [7, 0], 4, 2, 128, torch.bfloat16, block=32)
    mask = torch.tensor(spans.ancestors(chain, 1) + spans.ancestors(star, 1))
    ref, _ = tree_reference(c, mask)
    causal, _ = c.window_reference(10 ** 6, 0)
    torch.testing.assert_close(ref[:5], causal[:5])
    k, _ = spans.keys_of(c.k, c.table[1], 5)
    v, _ = spans.keys_of(c.v, c.table[1], 5)
    for i in range(5):
        idx = [0] if i == 0 else [0, i]
        for h in range(4):
            w = torch.softmax(k[idx, h // 2] @ c.q[5 + i, h].double() * c.scale, 0)
            torch.testing.assert_close(ref[5 + i, h], w @ v[idx, h // 2])


def test_window_brute_force():
    c = Case([3], [6], 2, 1, 128, torch.float16, block=32)
    ref, _ = c.window_reference(4, 2)
    k, _ = spans.keys_of(c.k, c.table[0], 9)
    v, _ = spans.keys_of(c.v, c.table[0], 9)
    for i in range(3):
        p = 6 + i
        idx = [j for j in range(p + 1) if p - j < 4 or j < 2]
        for h in range(2):
            e = [float(torch.exp(k[j, 0] @ c.q[i, h].double() * c.scale)) for j in idx]
            want = sum(x * v[j, 0] for x, j in zip(e, idx)) / sum(e)
            torch.testing.assert_close(ref[i, h], want)


def test_accepted_path():
    #       0 -> 1, 2, 3;  2 -> 4, 5
    parents, tokens = [-1, 0, 0, 0, 2, 2], [9, 5, 6, 6, 7, 8]
    assert spans.accepted_path(parents, tokens, [6, 1, 8, 1, 1, 3]) == ([0, 2, 5], 3)    # the first of two 6s
    assert spans.accepted_path(parents, tokens, [4, 1, 8, 1, 1, 3]) == ([0], 4)


def test_tree_masks():
    r = random.Random(2)
    trees = [random_tree(r, n) for n in (1, 5, 64, 100)]
    got = kernels.tree_masks(trees)
    assert got.dtype == torch.int64 and got.tolist() == [row for t in trees for row in spans.ancestors(t, 2)]
    assert kernels.tree_masks([[-1, 0]], words=3).tolist() == [[1, 0, 0], [3, 0, 0]]
    assert kernels.tree_masks([]).shape == (0, 1)
    with pytest.raises(ValueError, match="parent"):
        kernels.tree_masks([[-1, 1]])
    with pytest.raises(ValueError, match="words"):
        kernels.tree_masks([[-1] + [0] * 64], words=1)


def _runner(block=32, blocks=40, layers=2, device="cpu"):
    runner = ModelRunner(block_size=block, max_num_seqs=8, device=device)
    attns = torch.nn.ModuleList(Attention(4, 128, 128 ** -0.5, 2) for _ in range(layers))
    runner.allocate_kv_cache(attns, layers, blocks, 2, 128, torch.bfloat16)
    return runner, attns


def test_prepare_tree():
    runner, _ = _runner()
    a, b = Sequence(list(range(100, 140)), [3, 5]), Sequence([7], [9])
    ids, pos = runner.prepare_tree([a, b], [[1, 2, 3], []], [[0, 0, 2], []])
    ctx = C.get_context()
    assert ctx.is_prefill and isinstance(ctx, C.TreeContext)
    assert ids.tolist() == [139, 1, 2, 3, 7] and pos.tolist() == [39, 40, 40, 41, 0]
    assert ctx.cu_seqlens_q.tolist() == [0, 4, 5] and ctx.cu_seqlens_k.tolist() == [0, 43, 44]
    assert (ctx.max_seqlen_q, ctx.max_seqlen_k) == (4, 43)
    assert ctx.slot_mapping.tolist() == [5 * 32 + 7, 5 * 32 + 8, 5 * 32 + 9, 5 * 32 + 10, 9 * 32]
    assert ctx.tree_mask.tolist() == [[1], [3], [5], [13], [1]]
    assert ctx.block_tables.tolist() == [[3, 5], [9, -1]]
    C.reset_context()
    assert not hasattr(C.get_context(), "tree_mask")
    with pytest.raises(ValueError, match="blocks"):
        runner.prepare_tree([a], [[0] * 30], [[0] * 30])
    with pytest.raises(ValueError, match="parent"):
        runner.prepare_tree([a], [[1]], [[1]])
    with pytest.raises(ValueError, match="parents"):
        runner.prepare_tree([a], [[1]], [[]])
    # the accepted path of a: nodes 0, 2, 3
    runner.accept_tree([a, b], [[1, 2, 3], []], torch.tensor([[0, 2, 3, -1], [0, -1, -1, -1]]), torch.tensor([3, 1]),
                       torch.tensor([55, 66]))
    assert a.token_ids[-4:] == [139, 2, 3, 55] and len(a) == 43 and b.token_ids == [7, 66]


def test_release_window_blocks():
    runner, _ = _runner()
    s = Sequence(list(range(200)), list(range(10, 17)))    # 200 tokens, 7 pages of 32
    assert runner.release_window_blocks(s, 200) == []
    assert runner.release_window_blocks(s, 100, 4) == [11, 12]    # keys 0 .. 3 and 100 .. 199 are seen
    assert s.block_table == [10, -1, -1, 13, 14, 15, 16]
    assert runner.release_window_blocks(s, 100, 4) == []
    assert runner.release_window_blocks(s, 9, 33) == [13, 14]
    assert runner.release_window_blocks(s, 1) == [10, 15]
    assert s.block_table == [-1, -1, -1, -1, -1, -1, 16]


def test_copy_blocks_refusals():
    runner, _ = _runner()
    for src, dst, what in (([1, 2], [3], "pages"), ([1, 2], [3, 3], "another pair"), ([1, 2], [2, 3], "another pair"),
                           ([1], [40], "outside"), ([-1], [2], "outside")):
        with pytest.raises(ValueError, match=what):
            runner.copy_blocks(src, dst)
    with pytest.raises(ValueError, match="pages"):
        runner.copy_blocks([1], [2], [3, 4])


def test_attention_window_arguments():
    with pytest.raises(ValueError):
        Attention(4, 128, 1.0, 2, window=0)
    with pytest.raises(ValueError):
        Attention(4, 128, 1.0, 2, window=3, num_sinks=-1)
    with pytest.raises(ValueError):
        Attention(4, 128, 1.0, 2, num_sinks=4)
    a = Attention(4, 128, 1.0, 2, window=8)
    C.set_tree_context(None, None, 1, 1, None, None, torch.zeros(1, 1, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="window"):
        a(None, None, None)
    C.reset_context()


def test_no_cpu_fallback():
    q = torch.zeros(2, 4, 128, dtype=torch.bfloat16)
    cache = torch.zeros(4, 32, 2, 128, dtype=torch.bfloat16)
    i32 = lambda *x: torch.tensor(x, dtype=torch.int32)    # noqa: E731
    calls = [lambda: kernels.tree_attention(q, cache, cache, i32(0, 2), i32(0, 5), 2, 5, 0.1, i32([0]), torch.zeros(2, 1, dtype=torch.int64)),
             lambda: kernels.window_prefill(q, q[:, :2], q[:, :2], i32(0, 2), i32(0, 2), 2, 2, 0.1, 4),
             lambda: kernels.window_decode(q, cache, cache, i32(1, 1), i32([0], [1]), 0.1, 4),
             lambda: kernels.copy_kv_blocks(cache, i32(0), i32(1)),
             lambda: kernels.commit_tree(cache, i32([0]), i32(0, 2), i32(0, 5), 2, path=i32([0, -1]), num_accepted=i32(1))]
    for call in calls:
        with pytest.raises(RuntimeError, match="HIP device"):
            call()


P = ctypes.c_void_p(1 << 20)


def _tree(**kw):
    a = dict(q=P, q_rs=512, q_hs=128, k=P, v=P, cu_q=P, cu_k=P, mq=8, mk=100, bt=P, bts=4, mb=4, nb=64, mask=P, mrs=1,
             words=1, out=P, o_rs=512, o_hs=128, n=1, total=8, hq=4, hkv=2, d=128, bs=32, scale=0.1, qt=2, kt=2, ks=None,
             vs=None, gate=None, g_rs=0, g_hs=0, ws=None, wsb=0, need=None, stream=None)
    a.update(kw)
    return _lib.lib().nq_tree_attention(*a.values())


def _prefill(**kw):
    a = dict(q=P, q_rs=512, q_hs=128, k=P, v=P, kv_rs=256, tk=8, cu_q=P, cu_k=P, mq=8, mk=8, bt=None, bts=0, mb=0, nb=0,
             window=4, sinks=0, out=P, o_rs=512, o_hs=128, n=1, total=8, hq=4, hkv=2, d=128, bs=0, scale=0.1, qt=2, kt=2,
             ks=None, vs=None, gate=None, g_rs=0, g_hs=0, ws=None, wsb=0, need=None, stream=None)
    a.update(kw)
    return _lib.lib().nq_window_prefill(*a.values())


def _decode(**kw):
    a = dict(q=P, q_rs=512, q_hs=128, k=P, v=P, bt=P, bts=4, mb=4, lens=P, window=4, sinks=0, kn=None, kn_rs=256, vn=P,
             vn_rs=256, slots=P, nt=2, out=P, o_rs=512, o_hs=128,
             n=2, hq=4, hkv=2, d=128, bs=32, nb=64, scale=0.1, qt=2, kt=2, ks=None, vs=None, gate=None, g_rs=0, g_hs=0,
             ws=None, wsb=0, need=None, stream=None)
    a.update(kw)
    return _lib.lib().nq_window_decode(*a.values())


@pytest.mark.parametrize("call", [_tree, _prefill, _decode])
@pytest.mark.parametrize("kw,rc,text", [
    (dict(hq=5), -1, "multiple"), (dict(hq=34), -2, "group"), (dict(d=64), -2, "head_dim"), (dict(qt=0), -2, "q dtype"),
    (dict(kt=1), -2, "kv dtype"), (dict(kt=3), -1, "scales"), (dict(scale=0.0), -1, "softmax_scale"),
    (dict(scale=float("nan")), -1, "softmax_scale"), (dict(q=None), -1, "null"), (dict(out=None), -1, "null"),
    (dict(q_rs=511), -1, "alignment"), (dict(q=ctypes.c_void_p((1 << 20) + 8)), -1, "alignment"),
    (dict(o_hs=126), -1, "alignment"), (dict(gate=P, g_rs=3), -1, "gate"), (dict(n=-1), -1, "counts"),
    (dict(hkv=0), -1, "counts")])
def test_span_refusals(call, kw, rc, text):
    assert call(**kw) == rc and text in _lib.lib().nq_last_error().decode()


def test_more_span_refusals():
    err = lambda: _lib.lib().nq_last_error().decode()    # noqa: E731
    for call in (_prefill, _decode):
        assert call(window=0) == -1 and "window" in err()
        assert call(sinks=-1) == -1 and "sinks" in err()
    for call in (_tree, _decode):
        assert call(bs=48) == -2 and "block_size" in err()
        assert call(bts=3) == -1 and "width" in err()
        assert call(bt=None) == -1 and "null" in err()
        assert call(nb=1 << 31, bs=1 << 20) == -1 and "pool" in err()
    assert _tree(mq=257, words=4, mrs=4) == -2 and "nodes" in err()
    assert _tree(mq=65) == -1 and "words" in err()
    assert _tree(mask=None) == -1 and _tree(mrs=0) == -1
    assert _decode(kn=P, slots=None) == -1 and _decode(kn=P, vn=None) == -1 and _decode(kn=P, kn_rs=255) == -1
    assert _decode(kn=P, nt=1) == -2 and _decode(kn=P, nt=3) == -2 and "new rows" in err()
    assert _prefill(kv_rs=255) == -1 and _prefill(cu_q=None) == -1
    # nothing to do: no launch
    assert _tree(n=0) == 0 and _tree(total=0) == 0 and _tree(mq=0) == 0
    assert _prefill(n=0) == 0 and _prefill(total=0) == 0 and _decode(n=0) == 0


def test_page_refusals():
    lib = _lib.lib()
    err = lambda: lib.nq_last_error().decode()    # noqa: E731
    copy = lambda pool=P, slabs=2, nb=4, bs=32, row=512, src=P, n=1: lib.nq_copy_kv_blocks(    # noqa: E731
        pool, slabs, nb, bs, row, src, P, None, n, None)
    assert copy(row=24) == -1 and "16-byte" in err()
    assert copy(pool=None) == -1 and copy(src=None) == -1 and copy(n=-1) == -1 and copy(bs=0) == -1
    assert copy(slabs=65536) == -2 and copy(bs=1 << 30, row=1 << 20, n=100) == -1
    assert copy(n=0) == 0 and copy(slabs=0) == 0
    commit = lambda mq=8, n=1, bt=P, target=P, parents=P, nxt=P, row=512, bts=4, path=P: lib.nq_commit_tree(    # noqa: E731
        P, 2, 4, 32, row, bt, bts, 4, P, P, n, 8, mq, parents, P, target, path, P, nxt, None)
    assert commit(mq=257) == -2 and "nodes" in err()
    assert commit(bt=None) == -1 and commit(path=None) == -1 and commit(row=8) == -1 and commit(bts=3) == -1
    assert commit(parents=None) == -1 and commit(nxt=None) == -1 and commit(n=65536) == -1 and commit(n=-1) == -1
    assert commit(n=0) == 0
