"""Attention over caches with a scale for each block of tokens and head, on the GPU, against float64 value by value."""
import pytest
import torch

from nano_qwen_amd import kernels
from tests.blocks import CODE, Case, check

pytestmark = pytest.mark.gpu

BF, HF = torch.bfloat16, torch.float16

HEADS = [    # query heads, kv heads, dim, type, page, tokens of a block
    (8, 2, 128, BF, 256, 64), (4, 4, 128, HF, 64, 32), (32, 8, 128, BF, 256, 256), (16, 1, 128, HF, 128, 128),
    (10, 2, 256, BF, 96, 32), (16, 2, 256, HF, 64, 64), (8, 1, 256, BF, 256, 128), (6, 3, 128, BF, 32, 32),
    (24, 8, 128, HF, 256, 32), (7, 7, 128, BF, 32, 32), (16, 16, 256, BF, 64, 32), (64, 8, 128, BF, 256, 64)]


@pytest.mark.parametrize("hq,hkv,d,dtype,block,unit", HEADS)
@pytest.mark.parametrize("fine", [False, True])
def test_decode(cuda, hq, hkv, d, dtype, block, unit, fine):
    pre = [0, 1, 31, 32, 33, 63, 64, 255, 256, 700, 40, 1500]
    c = Case([1] * len(pre), pre, hq, hkv, d, dtype, block, unit, seed=hq + unit, fine=fine).to(cuda)
    check(c.decode(), c.reference(), dtype)


@pytest.mark.parametrize("hq,hkv,d,dtype,block,unit", HEADS[:7])
def test_decode_of_one(cuda, hq, hkv, d, dtype, block, unit):
    for n in (1, 2, 32, 65, 3000):
        c = Case([1], [n - 1], hq, hkv, d, dtype, block, unit, seed=n).to(cuda)
        check(c.decode(), c.reference(), dtype, f"{n}")


@pytest.mark.parametrize("hq,hkv,d,dtype,block,unit,batch,longest", [
    (32, 8, 128, BF, 256, 64, 40, 4000), (16, 2, 256, HF, 64, 32, 24, 3000), (8, 4, 128, HF, 32, 32, 70, 1500),
    (32, 8, 128, BF, 256, 128, 3, 20000), (16, 4, 256, BF, 256, 256, 2, 30000), (4, 1, 128, BF, 256, 64, 300, 900)])
def test_decode_batches(cuda, hq, hkv, d, dtype, block, unit, batch, longest):
    """Batches on either side of the one-launch and stream-K plans."""
    r = torch.Generator().manual_seed(batch)
    pre = (torch.rand(batch, generator=r) ** 2 * longest).int().tolist()
    pre[0], pre[-1] = longest - 1, 0
    c = Case([1] * batch, pre, hq, hkv, d, dtype, block, unit, seed=batch).to(cuda)
    check(c.decode(), c.reference(), dtype)


def test_decode_plans_are_all_taken(monkeypatch):
    plan = lambda b, hq, hkv, d, w, bs: kernels._decode_config(b, hq, hkv, d, w, bs, CODE)    # noqa: E731
    assert plan(12, 8, 2, 128, 7, 256)[0] > 0 and plan(1, 32, 8, 128, 13, 256)[0] > 0
    big = plan(40, 32, 8, 128, 17, 256)
    assert big[0] == 0 and big[1] > 1
    assert kernels.decode_schedule(40, 32, 8, 128, 17, 256, CODE, big[1], big[3]) == "stream-K"


def test_decode_split_k(cuda, monkeypatch):
    monkeypatch.setenv("NQ_DECODE_STREAMK", "0")
    for split in ("128", "512"):
        monkeypatch.setenv("NQ_DECODE_SPLIT_TOKENS", split)
        for hq, hkv, d in ((32, 8, 128), (8, 2, 256)):
            c = Case([1] * 5, [1300, 0, 127, 128, 600], hq, hkv, d, BF, 256, 64, seed=hq).to(cuda)
            check(c.decode(), c.reference(), BF, split)


def test_decode_empty_rows_and_gate(cuda):
    """Padding rows of a captured batch give zeros; an output gate; an output of another layout."""
    c = Case([1, 1, 1], [-1, 90, -1], 8, 2, 128, BF, 64, 32).to(cuda)
    wide = torch.full((3, 8, 256), 7.0, dtype=BF, device=cuda)
    out = c.decode(out=wide[:, :, :128])
    assert (out[[0, 2]] == 0).all() and (wide[:, :, 128:] == 7).all()
    check(out, c.reference(), BF)
    gate = torch.randn(3, 8, 128, device=cuda).to(BF)
    gated = c.decode(gate=gate)
    assert torch.equal(gated, kernels.output_gate(c.decode(), gate))
    assert torch.equal(c.decode(), c.decode(out=torch.empty(3, 8, 128, dtype=BF, device=cuda)))
    four = kernels.paged_decode(c.q_dev[:, None], c.k_dev, c.v_dev, c.lens_dev, c.table_dev, c.scale, c.k_scale_dev, c.v_scale_dev)
    assert four.shape == (3, 1, 8, 128) and torch.equal(four[:, 0], c.decode())


@pytest.mark.parametrize("d", [128, 256])
def test_missing_pages(cuda, kernel, d):
    """Keys without a page, or with one outside the pool, are not seen."""
    lost = [(0, 1), (0, 2), (1, 0), (2, 5)]
    c = Case([1, 1, 1], [300, 63, 400], 8, 2, d, BF, 64, 32, lost=lost).to(cuda)
    check(c.decode(), c.reference(), BF)
    check(c.decode(100000, 0), c.reference(), BF)
    c = Case([40, 3, 70], [300, 61, 400], 8, 2, d, BF, 64, 32, lost=lost).to(cuda)
    check(c.prefill(), c.reference(), BF)


STEPS = [([1], [0]), ([1, 7], [0, 3]), ([33], [0]), ([5, 64, 1, 130], [300, 0, 31, 513]), ([300, 17], [0, 700]),
         ([200, 90], [40, 0]), ([257], [255]), ([40, 0, 3], [0, 9, 500])]


@pytest.fixture(params=["causal", "window"])
def kernel(request, monkeypatch):
    """Either kernel of the causal prefill, where both can."""
    monkeypatch.setenv("NQ_PREFILL_BLOCKS", request.param)
    return request.param


@pytest.mark.parametrize("new,pre", STEPS)
@pytest.mark.parametrize("fine", [False, True])
def test_prefill(cuda, kernel, new, pre, fine):
    c = Case(new, pre, 8, 2, 128, BF, 64, 32, seed=len(new) + new[0], fine=fine).to(cuda)
    check(c.prefill(), c.reference(), BF)


@pytest.mark.parametrize("hq,hkv,d,dtype,block,unit", HEADS)
def test_prefill_heads_and_types(cuda, kernel, hq, hkv, d, dtype, block, unit):
    for new, pre in (([70, 3, 150], [100, 600, 0]), ([2, 5], [77, 10]), ([1, 1], [40, 3])):
        c = Case(new, pre, hq, hkv, d, dtype, block, unit, seed=hq).to(cuda)
        check(c.prefill(), c.reference(), dtype, f"{new}")


@pytest.mark.parametrize("new,pre,d,dtype", [([1500, 900], [600, 0], 128, BF), ([20], [9000], 128, BF), ([700], [3000], 256, HF),
                                             ([260] * 12, [500] * 12, 128, HF)])
def test_prefill_long(cuda, kernel, new, pre, d, dtype):
    """More than 64 tiles to an item, items that are cut and those that are dealt out whole."""
    c = Case(new, pre, 4, 2, d, dtype, 256, 64, seed=new[0]).to(cuda)
    check(c.prefill(), c.reference(), dtype)


@pytest.mark.parametrize("new,pre,hq,hkv,d,dtype", [([900, 1000, 17], [8000, 3000, 9000], 32, 8, 128, BF),
                                                    ([1500] * 6, [0, 100, 700, 33, 256, 2000], 16, 4, 256, HF),
                                                    ([300] * 40, [64] * 40, 32, 8, 128, BF), ([3000], [5000], 64, 8, 128, HF)])
def test_prefill_large(cuda, new, pre, hq, hkv, d, dtype):
    """What the rules give to the causal kernel: queues and ranges.  (The oracle's products on the device, in float64.)"""
    c = Case(new, pre, hq, hkv, d, dtype, 256, 64, seed=new[0]).to(cuda)
    check(c.prefill(), c.reference(device=cuda), dtype)


def test_gated_prefill(cuda, kernel):
    c = Case([70, 3], [100, 600], 8, 2, 128, BF, 64, 32).to(cuda)
    gate = torch.randn(73, 8, 256, device=cuda).to(BF)[:, :, 128:]
    wide = torch.full((73, 8, 256), 7.0, dtype=BF, device=cuda)
    out = c.prefill(gate=gate, out=wide[:, :, :128])
    assert torch.equal(out, kernels.output_gate(c.prefill(), gate)) and (wide[:, :, 128:] == 7).all()


@pytest.mark.parametrize("window,sinks", [(1, 0), (33, 4), (200, 64), (100000, 0)])
@pytest.mark.parametrize("hq,hkv,d,dtype,block,unit", [HEADS[0], HEADS[1], HEADS[4]])
def test_windows(cuda, window, sinks, hq, hkv, d, dtype, block, unit):
    pre = [0, 1, 31, 32, 255, 256, 700, 40]
    c = Case([1] * len(pre), pre, hq, hkv, d, dtype, block, unit, seed=window).to(cuda)
    check(c.decode(window, sinks), c.reference(window, sinks), dtype)
    c = Case([5, 64, 1, 130], [300, 0, 31, 513], hq, hkv, d, dtype, block, unit, seed=window).to(cuda)
    check(c.prefill(window, sinks), c.reference(window, sinks), dtype)


@pytest.mark.parametrize("d", [128, 256])
def test_values_that_are_not_finite(cuda, kernel, d):
    """NaN among the values reaches the rows that see it, and no others."""
    c = Case([40, 33], [70, 0], 8, 2, d, BF, 64, 32, seed=d)
    c.v.view(torch.uint8)[c.table[0, 1].long(), 30, 1, 5] = 0x7F    # token 94 of sequence 0: its query row 24 sees it
    c.v.view(torch.uint8)[c.table[1, 0].long(), 32, 0, 9] = 0xFF    # the last token of sequence 1
    ok = Case([40, 33], [70, 0], 8, 2, d, BF, 64, 32, seed=d)
    for x in (c, ok):
        x.to(cuda)
    bad, good = c.prefill(), ok.prefill()
    nan = torch.zeros_like(bad, dtype=torch.bool)
    nan[24:40, 4:, 5] = True
    nan[72, :4, 9] = True
    assert torch.equal(torch.isnan(bad), nan)
    check(torch.where(nan, good, bad), ok.reference(), BF)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_scales_far_apart(cuda, kernel, dtype):
    """Values of neighbouring blocks 2^40 apart, and one block of scale 0: what a 16-bit weight must not lose."""
    c = Case([1, 1, 30], [200, 700, 170], 8, 2, 128, dtype, 64, 32, seed=4)
    far = torch.tensor([2.0 ** -40, 1.0, 2.0 ** -20]).repeat(c.v_scale.numel())[:c.v_scale.numel()].view(c.v_scale.shape)
    c.v_scale *= far
    c.to(cuda)
    ref = c.reference()
    check(c.prefill(), ref, dtype)
    one = Case([1, 1], [200, 700], 8, 2, 128, dtype, 64, 32, seed=4)
    one.v_scale *= torch.tensor([2.0 ** -40, 1.0, 2.0 ** -20]).repeat(one.v_scale.numel())[:one.v_scale.numel()].view(one.v_scale.shape)
    one.v_scale[one.table[1, 2].long(), 1] = 0.0
    one.k_scale[one.table[1, 3].long(), 0] = 0.0
    one.to(cuda)
    ref = one.reference()
    check(one.decode(), ref, dtype)
    check(one.prefill(), ref, dtype)


def test_captured_and_on_other_streams(cuda, kernel):
    """Replays follow their inputs, the scales among them; streams and threads that decode at once."""
    c = Case([1] * 4, [800, 20, 300, 1999], 8, 2, 128, BF, 64, 32, seed=1).to(cuda)
    p = Case([30, 70], [900, 10], 8, 2, 128, BF, 64, 32, seed=2).to(cuda)
    c.decode(), p.prefill(), c.decode(100, 4)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = c.decode(), p.prefill(), c.decode(100, 4)
    for t in range(4):
        c.v_scale_dev *= 2
        p.k_scale_dev *= 0.75
        c.lens_dev.copy_(torch.tensor([801 - t, 21 - 5 * t, 301 - 100 * t, 2000 - 7 * t]))
        for o in outs:
            o.fill_(7)
        graph.replay()
        want = c.decode(), p.prefill(), c.decode(100, 4)
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want)), t
    want = [x.clone() for x in want]
    streams = [torch.cuda.Stream() for _ in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for _ in range(10):
        got = []
        for s in streams:
            with torch.cuda.stream(s):
                got.append((c.decode(), p.prefill(), c.decode(100, 4)))
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def refusals(dev):
    """(name of the call, arguments that are refused)."""
    c = Case([2, 3], [40, 5], 8, 2, 128, BF, 64, 32).to(dev)
    s = torch.ones_like(c.k_scale_dev)
    q = c.q_dev
    one = Case([1, 1], [40, 5], 8, 2, 128, BF, 64, 32).to(dev)
    bad = [dict(k_scale=s[:, :1]), dict(k_scale=s[..., :1]), dict(k_scale=s.double()), dict(v_scale=s[:1]), dict(v_scale=None),
           dict(v_scale=s[0, 0]), dict(k_scale=s[:-1], v_scale=s[:-1]), dict(gate=q[:1]), dict(out=q[:1])]
    eights = torch.ones(s.shape[0], 4, 2, device=dev)
    bad += [dict(k_scale=eights, v_scale=eights)]    # blocks of 16 tokens
    for kw in bad:
        yield "prefill", c, (), kw
        yield "prefill", c, (40, 1), kw
        yield "decode", one, (), kw
        yield "decode", one, (40, 1), kw
    yield "prefill", c, (), dict(causal=False)
    yield "prefill", c, (), dict(block_table=None)
    yield "prefill", c, (0, 0), {}
    yield "prefill", c, (4, -1), {}
    yield "decode", one, (0, 0), {}
    rows = torch.zeros(2, 2, 128, dtype=BF, device=dev)
    new = dict(k=rows, v=rows, slot_mapping=torch.zeros(2, dtype=torch.int32, device=dev))
    yield "decode", one, (), new
    yield "decode", one, (40, 1), new
    half = Case([1, 1], [40, 5], 8, 2, 128, BF, 64, 32).to(dev)
    half.k_dev, half.v_dev = half.k_dev.to(BF), half.v_dev.to(BF)
    yield "decode", half, (), {}
    yield "prefill", half, (), {}
    wide = Case([1, 1], [40, 5], 34, 2, 128, BF, 64, 32).to(dev)    # 17 query heads to a kv head
    yield "decode", wide, (), {}
    yield "prefill", wide, (), {}


def test_refusals(cuda):
    for call, c, args, kw in refusals(cuda):
        with pytest.raises(RuntimeError):
            getattr(c, call)(*args, **kw)
    c = Case([2, 3], [40, 5], 8, 2, 128, BF, 64, 32).to(cuda)
    mask = torch.ones(5, 1, dtype=torch.int64, device=cuda)
    with pytest.raises(RuntimeError):
        kernels.tree_attention(c.q_dev, c.k_dev, c.v_dev, c.cu_q_dev, c.cu_k_dev, 3, 45, c.scale, c.table_dev, mask,
                               c.k_scale_dev, c.v_scale_dev)
    with pytest.raises(RuntimeError):
        c.prefill(out=torch.empty(5, 8, 128, dtype=HF, device=cuda))
