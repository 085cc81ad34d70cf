"""Windowed and tree attention on the GPU against float64, value by value."""
import pytest
import torch

from tests.spans import Case, check, tree_masks, tree_reference

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16

# new tokens, cached tokens before them, window, sinks
WINDOWS = [
    ([1], [0], 4, 0),
    ([1, 7], [0, 3], 1, 0),
    ([33], [0], 32, 1),
    ([5, 64, 1, 130], [300, 0, 31, 513], 40, 4),
    ([300, 17], [0, 700], 128, 33),
    ([200, 90], [40, 0], 100000, 0),
    ([257], [255], 256, 65),
    ([40, 0, 3], [0, 9, 500], 16, 1000),
]


@pytest.mark.parametrize("paged", [True, False])
@pytest.mark.parametrize("new,pre,window,sinks", WINDOWS)
def test_window_prefill(cuda, new, pre, window, sinks, paged):
    c = Case(new, pre, 8, 2, 128, BF, block=32 if paged else 0, paged=paged, seed=len(new) + window)
    if paged:
        c.free_before(window, sinks)
    out = c.to(cuda).window_prefill(window, sinks)
    check(out, *c.window_reference(window, sinks), BF)


@pytest.mark.parametrize("hq,hkv,d,dtype,fp8,block", [
    (4, 4, 128, HF, False, 64), (6, 2, 128, BF, True, 32), (16, 1, 128, BF, False, 256), (32, 2, 128, HF, True, 256),
    (10, 2, 256, BF, False, 96), (4, 2, 256, HF, True, 64), (8, 1, 256, BF, True, 32), (3, 3, 256, HF, False, 256),
    (24, 8, 128, BF, False, 64), (7, 7, 128, BF, False, 32)])
def test_window_prefill_heads_and_types(cuda, hq, hkv, d, dtype, fp8, block):
    for new, pre in (([70, 3, 150], [100, 600, 0]), ([2, 5], [77, 10])):
        c = Case(new, pre, hq, hkv, d, dtype, block=block, fp8=fp8, seed=hq).free_before(90, 5)
        check(c.to(cuda).window_prefill(90, 5), *c.window_reference(90, 5), dtype, f"{new}")


@pytest.mark.parametrize("hq,hkv,d,dtype,fp8,block", [
    (8, 2, 128, BF, False, 32), (4, 4, 128, HF, True, 64), (32, 2, 128, BF, True, 256), (10, 2, 256, HF, False, 96),
    (8, 8, 256, BF, True, 256), (3, 1, 256, BF, False, 32)])
@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 4), (200, 64), (100000, 0)])
def test_window_decode(cuda, hq, hkv, d, dtype, fp8, block, window, sinks):
    pre = [0, 1, 31, 32, 255, 256, 700, 40]
    c = Case([1] * len(pre), pre, hq, hkv, d, dtype, block=block, fp8=fp8, seed=window).free_before(window, sinks)
    check(c.to(cuda).window_decode(window, sinks), *c.window_reference(window, sinks), dtype)


def test_window_decode_empty_rows(cuda):
    c = Case([1, 1, 1], [-1, 4, -1], 8, 2, 128, BF, block=32)
    out = torch.full((3, 1, 8, 128), 7.0, dtype=BF, device=cuda)
    c.to(cuda).window_decode(8, 1, out=out)
    ref, mag = c.window_reference(8, 1)
    check(out[:, 0], ref, mag, BF)
    assert (out[[0, 2]] == 0).all()


def test_window_rows_before_the_cache(cuda):
    """More query tokens than cached ones: the first rows see nothing."""
    c = Case([9, 40], [-4, 2], 4, 2, 128, BF, block=32)
    out = c.to(cuda).window_prefill(3, 2)
    check(out, *c.window_reference(3, 2), BF)
    assert (out[:4] == 0).all()


TREES = [
    ([1], [0]),
    ([1, 1], [5, 700]),
    ([2, 3], [31, 0]),
    ([8], [777]),
    ([16, 1, 33, 7], [100, 0, 64, 500]),
    ([64, 63], [300, 33]),
    ([65, 130], [90, 7]),
    ([256], [40]),
    ([26] * 5, [60, 61, 62, 63, 64]),
]


@pytest.mark.parametrize("new,pre", TREES)
@pytest.mark.parametrize("hq,hkv,d,dtype,fp8,block", [(8, 2, 128, BF, False, 32), (8, 1, 128, HF, True, 64),
                                                     (2, 2, 256, BF, True, 256), (6, 2, 256, HF, False, 32)])
def test_tree(cuda, new, pre, hq, hkv, d, dtype, fp8, block):
    if max(new) > 130 and hq == 6:
        new = [100]
    trees, mask = tree_masks(new, seed=sum(pre))
    c = Case(new, pre, hq, hkv, d, dtype, block=block, fp8=fp8, seed=sum(new))
    check(c.to(cuda).tree_attention(mask), *tree_reference(c, mask), dtype)


def test_tree_arbitrary_masks(cuda):
    """Bits in any pattern: empty rows, rows without themselves, bits of nodes that the tree does not have."""
    g = torch.Generator().manual_seed(5)
    new, pre = [40, 70, 3], [0, 100, 0]
    mask = torch.randint(-2 ** 62, 2 ** 62, (sum(new), 2), generator=g) * 2 + 1
    mask[3] = 0           # sees nothing: no context
    mask[50] = 0          # the context alone
    mask[-1] = -8         # only bits past its tree of 3
    c = Case(new, pre, 8, 2, 128, BF, block=32)
    out = c.to(cuda).tree_attention(mask)
    check(out, *tree_reference(c, mask), BF)
    assert (out[3] == 0).all() and (out[-1] == 0).all()


def _odd(case, g, share=0.02):
    """NaN and infinities in some of the cached values and keys; fp8 has NaN only."""
    nb, bs = case.k.shape[:2]
    for cache, vals, share in ((case.k, [float("nan")], share / 6), (case.v, [float("nan"), float("inf"), float("-inf")], share)):
        raw = cache.view(torch.uint8) if case.fp8 else cache
        for i, h in enumerate(case.have):
            for j in range(h):
                if torch.rand((), generator=g) < share:
                    at = raw[case.table[i, j // bs].long(), j % bs, int(torch.randint(0, case.hkv, (), generator=g))]
                    dims = torch.randint(0, case.d, (3,), generator=g)
                    x = vals[int(torch.randint(0, len(vals), (), generator=g))]
                    at[dims] = 0x7F if case.fp8 else x
    return case


def _check_odd(out, visible_rows, case, dtype):
    """Rows that see nothing odd are as close as ever, and every output is finite or not as the oracle's."""
    ref, mag = visible_rows
    o = out.double().cpu()
    fine = torch.isfinite(ref)
    assert fine.any() and not fine.all()
    assert torch.equal(fine, torch.isfinite(o))
    assert torch.equal(torch.isnan(ref), torch.isnan(o))
    assert torch.equal(ref[~fine & ~torch.isnan(ref)], o[~fine & ~torch.isnan(ref)])
    ok = fine & torch.isfinite(mag)
    check(torch.where(ok, o, 0.0), torch.where(ok, ref, 0.0), torch.where(ok, mag, 0.0), dtype)


@pytest.mark.parametrize("hq,hkv,d,dtype,fp8", [(8, 2, 128, BF, False), (2, 2, 128, HF, False), (4, 2, 256, HF, False),
                                                (8, 1, 256, BF, False), (8, 2, 128, BF, True), (4, 1, 256, HF, True)])
def test_masked_nan_and_infinity(cuda, hq, hkv, d, dtype, fp8):
    """Odd values reach the rows that see them, and no others: in windows (prefill and decode) and trees."""
    for seed, new, pre, window, sinks in ((1, [50, 30], [60, 200], 24, 3), (2, [1, 1, 1, 1, 1, 1], [30, 80, 130, 200, 9, 64], 20, 2),
                                          (3, [150], [0], 12, 1)):
        c = Case(new, pre, hq, hkv, d, dtype, block=32, fp8=fp8, seed=seed)
        _odd(c, torch.Generator().manual_seed(seed), 0.01).to(cuda)
        ref = c.window_reference(window, sinks)
        _check_odd(c.window_prefill(window, sinks), ref, c, dtype)
        if max(new) == 1:
            _check_odd(c.window_decode(window, sinks), ref, c, dtype)
    for seed, new in ((4, [2, 3, 1, 2] * 4), (5, [60, 40]), (6, [8, 7, 6])):
        trees, mask = tree_masks(new, seed)
        c = Case(new, [0] * len(new), hq, hkv, d, dtype, block=32, fp8=fp8, seed=seed)
        _odd(c, torch.Generator().manual_seed(seed), 0.06).to(cuda)
        _check_odd(c.tree_attention(mask), tree_reference(c, mask), c, dtype)


@pytest.mark.parametrize("hq,hkv,d,dtype,fp8,block", [
    (8, 2, 128, BF, False, 64), (8, 8, 128, HF, True, 32), (12, 3, 128, BF, True, 256), (16, 1, 128, BF, False, 32),
    (8, 2, 256, BF, False, 32), (4, 4, 256, HF, True, 64), (8, 1, 256, HF, False, 64), (8, 2, 256, BF, True, 32)])
@pytest.mark.parametrize("new,pre", [([3], [4100]), ([14], [2600]), ([40, 1, 33], [2000, 900, 70])])
def test_items_cut_into_pieces(cuda, new, pre, hq, hkv, d, dtype, fp8, block):
    """Few long items: each cut into many pieces, for every launch shape; trees, windows and decode."""
    c = Case(new, pre, hq, hkv, d, dtype, block=block, fp8=fp8, seed=sum(new)).to(cuda)
    trees, mask = tree_masks(new, seed=sum(pre))
    check(c.tree_attention(mask), *tree_reference(c, mask), dtype)
    check(c.window_prefill(1500, 40), *c.window_reference(1500, 40), dtype)
    one = Case([1] * len(pre), pre, hq, hkv, d, dtype, block=block, fp8=fp8, seed=1).to(cuda)
    check(one.window_decode(1900, 3), *one.window_reference(1900, 3), dtype)
