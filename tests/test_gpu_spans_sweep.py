"""Windowed and tree attention over drawn heads, types, lengths, tables and strides, every output row against float64."""
import random

import pytest
import torch

from nano_qwen_amd import kernels
from tests.spans import check, tree_masks

pytestmark = pytest.mark.gpu


def _log(r, lo, hi):
    return min(hi, int(lo * (hi / lo) ** r.random() + 0.5))


def _reference(q, k, v, visible, scale):
    """(output, weighted mean of |v|) of ``q [R, Hq, D]`` over ``k, v [N, Hkv, D]`` in float64 on the device."""
    r, hq, d = q.shape
    n, hkv, _ = k.shape
    if n == 0:
        return torch.zeros(r, hq, d, dtype=torch.float64), torch.zeros(r, hq, d, dtype=torch.float64)
    x = q.double().reshape(r, hkv, -1, d).transpose(0, 1).reshape(hkv, -1, d).contiguous()
    s = torch.matmul(x, k.permute(1, 2, 0).contiguous()) * scale
    s = s.masked_fill(~visible.repeat_interleave(hq // hkv, 0)[None], float("-inf"))
    top = s.amax(-1, keepdim=True)
    w = torch.exp(s - torch.where(top.isinf(), 0.0, top))
    w = w / w.sum(-1, keepdim=True).clamp_min(1e-300)
    y = v.transpose(0, 1).contiguous()
    back = lambda t: t.reshape(hkv, r, -1, d).transpose(0, 1).reshape(r, hq, d).cpu()    # noqa: E731
    return back(torch.matmul(w, y)), back(torch.matmul(w, y.abs()))


def _drawn(seed, cuda):
    r, g = random.Random(seed), torch.Generator(device=cuda).manual_seed(seed)
    kind = ("tree", "prefill", "packed", "decode")[seed % 4]
    d, dtype = r.choice((128, 256)), r.choice((torch.bfloat16, torch.float16))
    hkv = r.choice((1, 2, 3, 4, 5, 8, 12))
    grp = r.choice((1, 2, 3, 4, 7, 8, 16))
    fp8 = kind != "packed" and r.random() < 0.4
    block, batch = r.choice((32, 64, 96, 256)), r.choice((1, 2, 5, 20, 70, 260))
    budget = 60000 // (batch * hkv) + 40    # of cached tokens
    top = {"tree": 256, "decode": 1}.get(kind, 1500)
    most = max(1, min(top, 40000 // (batch * hkv * grp)))
    most = _log(r, 1, most)
    new = [1 if kind == "decode" else r.choice((0, 1, r.randint(1, most), most)) for _ in range(batch)]
    pre = [0 if kind == "packed" and r.random() < 0.5 else r.choice((0, 1, 31, 32, r.randint(0, budget))) for _ in range(batch)]
    have = [a + b for a, b in zip(new, pre)]
    if sum(new) == 0:
        new[0], have[0] = 1, have[0] + 1
    for i in range(batch):
        if r.random() < 0.05 and new[i] > 1:    # rows before the cache
            have[i] = r.randint(0, new[i] - 1)
    window, sinks = _log(r, 1, 3000), r.choice((0, 0, 1, 4, 33, 500))
    rows, pad = sum(new), r.choice((0, 3))
    wide = torch.randn(rows + pad, grp * hkv, r.choice((d, 2 * d, d + 8)), generator=g, device=cuda).to(dtype)
    q = wide[:, :, :d]
    out = torch.full((rows + pad, grp * hkv + 1, d + 4), 5.0, dtype=dtype, device=cuda)
    scales, nan = [None, None], float("nan")
    if kind == "packed":
        both = torch.randn(max(sum(have), 1), 2 * hkv, d, generator=g, device=cuda).to(dtype)
        k, v = both[:, :hkv], both[:, hkv:]
        table = None
    else:
        counts = [-(-h // block) for h in have]
        blocks = sum(counts) + 2
        x = torch.randn(2, blocks, block, hkv, d, generator=g, device=cuda).to(dtype)
        if fp8:
            s = x.float().abs().amax(dim=(1, 2, 4)) / 448
            x = (x.float() / s[:, None, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
            scales = [s[0].contiguous(), s[1].contiguous()]
        perm = r.sample(range(blocks), blocks)
        table = torch.full((batch + 1, max(max(counts), 1) + 2), -1, dtype=torch.int32)
        own = torch.zeros(blocks, block, dtype=torch.bool)
        lost, at = r.choice((0.0, 0.0, 0.1)), 0
        for i, c in enumerate(counts):
            for j in range(c):
                page = perm[at + j]
                if r.random() >= lost:
                    table[i, j] = page
                    own[page, :max(0, min(block, have[i] - j * block))] = True
            at += c
        raw = x.view(torch.uint8).view(2, blocks, block, -1)
        raw[:, ~own.to(cuda)] = 0xFF if fp8 else torch.full((1,), nan, dtype=dtype).view(torch.uint8).repeat(raw.shape[-1] // 2).to(cuda)
        k, v = x[0].contiguous(), x[1].contiguous()
    cu = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32, device=cuda)    # noqa: E731
    mask = None
    if kind == "tree":
        trees, mask = tree_masks([n for n in new if n], seed, words=r.choice((None, 4)))
        mask = torch.cat([mask, torch.full((pad, mask.shape[1]), -1)])
    print(f"seed {seed}: {kind} batch {batch} new {max(new)} have {max(have)} hkv {hkv} group {grp} d {d} {dtype} fp8 {fp8} "
          f"block {block} window {window} sinks {sinks}", flush=True)
    torch.cuda.synchronize()
    args = (q, k, v, cu(new), cu(have), max(new), max(max(have), 1), d ** -0.5)
    dev_table = None if table is None else table.to(cuda)[:, :-1]
    o = out[:, :-1, :d]
    if kind == "tree":
        kernels.tree_attention(*args, dev_table, mask.to(cuda), *scales, out=o)
    elif kind == "decode":
        kernels.window_decode(q[:rows], k, v, torch.tensor(have, dtype=torch.int32, device=cuda), dev_table, d ** -0.5,
                              window, sinks, *scales, out=o[:rows])
    else:
        kernels.window_prefill(*args, window, sinks, dev_table, *scales, out=o)
    at = key = 0
    for i, (n, h) in enumerate(zip(new, have)):
        if n == 0:
            key += h
            continue
        j, p = torch.arange(h, device=cuda), torch.arange(h - n, h, device=cuda)[:, None]
        if kind == "tree":
            c = h - n
            words = mask[at:at + n].to(cuda)
            bit = (j - c).clamp_min(0)
            visible = (j < c) | (((words[:, bit // 64] >> (bit % 64)) & 1) != 0)
        else:
            visible = (j <= p) & ((j > p - window) | (j < sinks))
        if table is None:
            kk, vv = k[key:key + h].double(), v[key:key + h].double()
        else:
            page = table[i, torch.arange(h) // block].to(cuda)
            visible = visible & (page >= 0)
            row = page.clamp_min(0).long() * block + j % block
            kk, vv = (t.view(torch.uint8).view(-1, hkv, d * t.element_size())[row].view(t.dtype).double() for t in (k, v))
            if fp8:
                kk, vv = (t * s.double()[:, None] for t, s in zip((kk, vv), scales))
            kk, vv = (torch.where((page >= 0)[:, None, None], t, 0.0) for t in (kk, vv))
        ref = _reference(q[at:at + n], kk, vv, visible, d ** -0.5)
        check(o[at:at + n], *ref, dtype, f"sequence {i} of seed {seed}")
        at, key = at + n, key + h
    o[:rows] = 5.0
    assert (out == 5.0).all(), "rows or columns beside the output"


@pytest.mark.parametrize("first", range(0, 160, 16))
def test_drawn_spans(cuda, first):
    for seed in range(first, first + 16):
        _drawn(seed, cuda)
