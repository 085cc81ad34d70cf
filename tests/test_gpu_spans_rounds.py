"""Windowed and tree attention where a workgroup has many items, one after the other: the entries of its stream of
tiles full, partly filled, empty and missing by turns, lists of more than 64 tiles, items dealt out over several rounds."""
import pytest
import torch

from nano_qwen_amd import kernels
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


class Shared:
    """Sequences whose tables point into one small pool, in any order, some entries missing: long contexts without
    the memory.  References are formed for a few query rows of every sequence."""

    def __init__(self, new, have, hq, hkv, d, dtype, fp8, block, seed, missing=0.0):
        g = torch.Generator().manual_seed(seed)
        n, pool = len(have), 24
        self.new, self.have, self.d, self.dtype, self.block = new, have, d, dtype, block
        x = torch.randn(2, pool, block, hkv, d, generator=g).to(dtype)
        self.scales = [None, None]
        if fp8:
            s = x.float().abs().amax(dim=(1, 2, 4)) / 448
            x = (x.float() / s[:, None, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
            self.scales = [s[0].contiguous(), s[1].contiguous()]
        self.k, self.v = x[0].contiguous(), x[1].contiguous()
        self.table = torch.randint(0, pool, (n, -(-max(have) // block)), generator=g, dtype=torch.int32)
        self.table[torch.rand(self.table.shape, generator=g) < missing] = -1
        self.q = torch.randn(sum(new), hq, d, generator=g).to(dtype)
        self.dev = {k: v.to("cuda:0") for k, v in dict(q=self.q, k=self.k, v=self.v, table=self.table).items()}
        self.dev_scales = [None if t is None else t.to("cuda:0") for t in self.scales]
        cu = lambda v: torch.tensor([0, *torch.tensor(v).cumsum(0).tolist()], dtype=torch.int32, device="cuda:0")    # noqa: E731
        self.cu_q, self.cu_k = cu(new), cu(have)

    def decode(self, window, sinks):
        lens = torch.tensor(self.have, dtype=torch.int32, device="cuda:0")
        x = self.dev
        return kernels.window_decode(x["q"], x["k"], x["v"], lens, x["table"], self.d ** -0.5, window, sinks,
                                     *self.dev_scales)

    def prefill(self, window, sinks):
        x = self.dev
        return kernels.window_prefill(x["q"], x["k"], x["v"], self.cu_q, self.cu_k, max(self.new), max(self.have),
                                      self.d ** -0.5, window, sinks, x["table"], *self.dev_scales)

    def tree(self, mask):
        x = self.dev
        return kernels.tree_attention(x["q"], x["k"], x["v"], self.cu_q, self.cu_k, max(self.new), max(self.have),
                                      self.d ** -0.5, x["table"], mask.to("cuda:0"), *self.dev_scales)

    def check(self, out, visible, rows_of, what, every=1):
        """``visible(sequence, rows)`` over a sequence's keys, for the rows ``rows_of(sequence)``."""
        out, at = out.cpu(), 0
        for i, (n, have) in enumerate(zip(self.new, self.have)):
            if i % every == 0:
                k, has = spans.keys_of(self.k, self.table[i], have, self.scales[0])
                v, _ = spans.keys_of(self.v, self.table[i], have, self.scales[1])
                rows = sorted({r % n for r in rows_of(i)})
                ref = spans.attend(self.q[at:at + n][rows], k, v, visible(i, rows) & has, self.d ** -0.5)
                check(out[at:at + n][rows], *ref, self.dtype, f"{what}, sequence {i}")
            at += n

    def check_window(self, out, window, sinks, what, rows_of=lambda i: (0, -1), every=1):
        self.check(out, lambda i, rows: spans.window_visible(torch.tensor(rows) + self.have[i] - self.new[i], self.have[i],
                                                            window, sinks), rows_of, what, every)

    def check_tree(self, out, mask, what, rows_of=lambda i: (0, -1), every=1):
        at = [sum(self.new[:i]) for i in range(len(self.new))]
        self.check(out, lambda i, rows: spans.tree_visible(mask[at[i]:at[i] + self.new[i]].tolist(), self.new[i],
                                                          self.have[i] - self.new[i])[rows], rows_of, what, every)


LONG = [(128, BF, False), (128, HF, True), (256, HF, False), (256, BF, True)]


@pytest.mark.parametrize("d,dtype,fp8", LONG)
@pytest.mark.parametrize("batch,hkv", [(128, 8), (512, 2)])
def test_long_whole_items_of_one_wave(cuda, batch, hkv, d, dtype, fp8):
    """More than 64 tiles to an item that one wave has whole, in sequences that the kernel keeps the bounds of, and
    more of them than that; visible pages missing."""
    have = [2049 + (37 * i) % 190 if i % 5 else 1 + i % 70 for i in range(batch)]
    c = Shared([1] * batch, have, hkv, hkv, d, dtype, fp8, 32, batch + d, missing=0.02)
    c.check_window(c.decode(5000, 0), 5000, 0, "all", every=3)
    c.check_window(c.decode(2060, 9), 2060, 9, "window", every=7)


@pytest.mark.parametrize("d,dtype,fp8", [LONG[0], LONG[3]])
def test_long_ranges(cuda, d, dtype, fp8):
    """More than 64 tiles of an item in each of its ranges: decode, one node, rows of several waves."""
    have = [35001 + 977 * i for i in range(7)] + [5, 45000]
    n = len(have)
    c = Shared([1] * n, have, 8, 8, d, dtype, fp8, 64, d, missing=0.01)
    one = torch.ones(n, 1, dtype=torch.int64)
    c.check_window(c.decode(10 ** 6, 0), 10 ** 6, 0, "decode", every=4)
    c.check_tree(c.tree(one), one, "nodes", every=7)
    new = [5, 3, 1, 5, 2, 4, 3, 5, 4]
    c = Shared(new, have, 32, 8, d, dtype, fp8, 64, d + 1, missing=0.01)
    trees, mask = tree_masks(new, seed=d)
    c.check_tree(c.tree(mask), mask, "trees", rows_of=lambda i: (-1,), every=4)
    c.check_window(c.prefill(35000, 4), 35000, 4, "prefill", rows_of=lambda i: (0,), every=7)


@pytest.mark.parametrize("d,dtype,fp8", LONG)
@pytest.mark.parametrize("nodes", [12, 32])
def test_long_whole_items_of_several_waves(cuda, nodes, d, dtype, fp8):
    """More than 64 tiles to an item that a workgroup of four or eight waves has whole."""
    new = [nodes - i % 3 for i in range(64)]
    have = [2080 + (41 * i) % 150 if i % 6 else nodes + i for i in range(64)]
    trees, mask = tree_masks(new, seed=d)
    for missing in (0.0, 0.02):
        c = Shared(new, have, 32, 8, d, dtype, fp8, 32, nodes, missing)
        c.check_tree(c.tree(mask), mask, "trees", every=5)
    c.check_window(c.prefill(3000, 0), 3000, 0, "prefill", every=5)


@pytest.mark.parametrize("batch", [200, 300])
@pytest.mark.parametrize("d,dtype,fp8", LONG)
def test_decode_in_rounds(cuda, batch, d, dtype, fp8):
    """Two to five rounds of whole items, in sequences that the kernel keeps the bounds of and more than those."""
    have = [(37 * i) % 400 + 1 for i in range(batch)]
    c = Shared([1] * batch, have, 16, 8, d, dtype, fp8, 32, batch)
    c.check_window(c.decode(65, 3), 65, 3, "decode")


def _edges(i):
    """Rows of a prompt at its ends and on both sides of the edges of row tiles, in odd sequences others."""
    return (0, 1, 31, 32, 63, 64, 127, 128, 255, 256, 400, -1) if i % 2 == 0 else (0, 15, 16, 47, 95, 96, 191, 192, 300, -2, -1)


@pytest.mark.parametrize("hq,d,dtype,fp8", [(32, 128, BF, False), (32, 128, BF, True), (16, 256, HF, False),
                                            (8, 256, BF, False), (16, 256, BF, True), (8, 128, HF, True)])
def test_prefill_in_rounds(cuda, hq, d, dtype, fp8):
    """Prompts behind cached ones, their row tiles dealt out over several rounds, every sequence looked at."""
    new = [700, 33, 1200, 5, 900, 350, 64, 1100, 1, 128, 640, 257] * 2
    have = [n + (0, 90, 300)[i % 3] for i, n in enumerate(new)]
    c = Shared(new, have, hq, 8, d, dtype, fp8, 64, hq + d)
    c.check_window(c.prefill(300, 4), 300, 4, "prefill", _edges)


def test_packed_prefill_in_rounds(cuda):
    """The same over packed keys, where the first and the last sequences' items lie far apart."""
    new = [700, 33, 1200, 5, 900, 350, 64, 1100] * 3
    c = Case(new, [0] * len(new), 32, 8, 128, BF, paged=False, seed=4).to(cuda)
    out, at = c.window_prefill(300, 4).cpu(), 0
    for i, n in enumerate(new):
        rows = sorted({r % n for r in _edges(i)})
        ref = spans.attend(c.q[at:at + n][rows], c.k[at:at + n].double(), c.v[at:at + n].double(),
                           spans.window_visible(torch.tensor(rows), n, 300, 4), c.scale)
        check(out[at:at + n][rows], *ref, BF, f"sequence {i}")
        at += n


@pytest.mark.parametrize("nodes", [3, 12, 40])
@pytest.mark.parametrize("d,dtype,fp8", LONG)
def test_trees_in_rounds(cuda, nodes, d, dtype, fp8):
    """Many short trees: rounds of whole items of one, four and eight waves."""
    new = [1 + (7 * i) % nodes for i in range(150)]
    have = [n + (13 * i) % 70 for i, n in enumerate(new)]
    trees, mask = tree_masks(new, seed=nodes)
    c = Shared(new, have, 32, 8, d, dtype, fp8, 32, nodes)
    c.check_tree(c.tree(mask), mask, "trees", rows_of=lambda i: (0, 5, 15, 16, -1))
