"""Windowed and tree attention where a workgroup has many items, one after the other: the entries of its stream of
tiles full, partly filled, empty and missing by turns, lists of more than 64 tiles, items dealt out over several rounds."""
import pytest
import torch

from oracle import spans
from tests.spans import Case, check, tree_masks, tree_reference

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _lose_pages(case, every=3):
    """Some visible pages are missing: one in the middle, the last, or all of a sequence's."""
    pages = [(case.table[i] >= 0).nonzero()[:, 0].tolist() for i in range(len(case.have))]
    for i in range(0, len(pages), every):
        if pages[i]:
            lost = (pages[i][len(pages[i]) // 2:][:1], pages[i][-1:], pages[i])[(i // every) % 3]
            for j in lost:
                case.table[i, j] = (-1, 10 ** 6)[i % 2]
    return case


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("dtype,fp8", [(BF, False), (HF, False), (BF, True), (HF, True)])
def test_one_wave_entries(cuda, d, dtype, fp8):
    """Rows of one wave (decode, the smallest trees and prefills): long items behind items of one tile or none, last
    tiles of one key, missing pages; whole items and equal ranges (a window of 65, of all)."""
    pre = [0, 330, 31, 32, 33, 400, -1, 64, 5, 250, 95, 1, 160] * 10
    c = _lose_pages(Case([1] * len(pre), pre, 8, 8, d, dtype, block=32, fp8=fp8, seed=d)).to(cuda)
    for window, sinks in ((65, 3), (1, 0), (5000, 0)):
        check(c.window_decode(window, sinks), *c.window_reference(window, sinks), dtype, f"decode {window}")
    new, pre = [2, 1, 3, 0, 1, 2, 3] * 8, [max(p, 0) for p in pre[:56]]
    t = _lose_pages(Case(new, pre, 8, 2, d, dtype, block=32, fp8=fp8, seed=d + 1)).to(cuda)
    trees, mask = tree_masks([n for n in new if n], seed=d)
    check(t.tree_attention(mask), *tree_reference(t, mask), dtype, "trees")
    check(t.window_prefill(40, 5), *t.window_reference(40, 5), dtype, "paged prefill")
    if not fp8:    # packed, the last sequence's last tile at the tensor's end
        for seed, last in enumerate((1, 31, 32, 33, 70)):
            p = Case(new + [2], [k % 90 for k in pre] + [last - 2 if last > 2 else 0], 8, 2, d, dtype, paged=False,
                     seed=seed).to(cuda)
            check(p.window_prefill(50, 1), *p.window_reference(50, 1), dtype, f"packed prefill {last}")


def test_lengths_beyond_32_bits(cuda):
    """Largest lengths that no int holds mean no bound; windows and sinks far below zero are refused."""
    c = Case([3, 2], [100, 40], 8, 2, 128, BF, block=32).to(cuda)
    p = Case([40, 3], [0, 0], 8, 2, 128, BF, paged=False).to(cuda)
    trees, mask = tree_masks([3, 2])
    want = c.tree_attention(mask), c.window_prefill(50, 2)
    for far in (2 ** 31, 2 ** 32, 2 ** 40 + 7):
        c.max_k = far
        assert torch.equal(c.tree_attention(mask), want[0]) and torch.equal(c.window_prefill(50, 2), want[1])
        for case, window, sinks in ((c, -far + 5, 0), (c, 5, -far + 1), (p, -far + 5, 0)):
            with pytest.raises(RuntimeError):
                case.window_prefill(window, sinks)
        with pytest.raises(RuntimeError):
            Case([1], [9], 8, 2, 128, BF, block=32).to(cuda).window_decode(-far + 5, 0)
        p.max_k = far    # packed keys of a length that no tensor has
        with pytest.raises(RuntimeError):
            p.window_prefill(50, 2)
        p.max_k = 40
    c.max_q = -2 ** 32 + 3
    with pytest.raises(RuntimeError):
        c.tree_attention(mask)


@pytest.mark.parametrize("d", [128, 256])
def test_scales_of_zero(cuda, d):
    """Keys of a head whose scale is 0 are all 0: the mean of the visible values."""
    for new, pre in (([1, 1, 1], [70, 0, 300]), ([2, 9, 40], [33, 0, 90])):
        c = Case(new, pre, 8, 2, d, BF, block=32, fp8=True, seed=d)
        c.k_scale[1] = 0.0
        c.to(cuda)
        trees, mask = tree_masks(new, seed=1)
        check(c.tree_attention(mask), *tree_reference(c, mask), BF, "tree")
        check(c.window_prefill(40, 3), *c.window_reference(40, 3), BF, "prefill")
        if max(new) == 1:
            check(c.window_decode(40, 3), *c.window_reference(40, 3), BF, "decode")
