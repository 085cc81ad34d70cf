"""Drawn calls of the operators over caches with a scale for each block of tokens and head; pools past 32 bits of bytes;
host threads on one stream."""
import random
import threading

import pytest
import torch

from nano_qwen_amd import kernels
from tests import test_gpu_append as append
from tests.blocks import Case, check

pytestmark = pytest.mark.gpu

BF, HF, CODE = torch.bfloat16, torch.float16, torch.float8_e4m3fn


def drawn_shape(r):
    hkv = r.choice([1, 2, 3, 4, 5, 8, 16])
    hq = hkv * r.choice([1, 2, 3, 4, 6, 8])
    block, unit = r.choice([(32, 32), (64, 32), (64, 64), (96, 32), (128, 64), (128, 128), (192, 64), (256, 32), (256, 64),
                            (256, 256), (512, 128)])
    return dict(hq=hq, hkv=hkv, d=r.choice([128, 256]), dtype=r.choice([BF, HF]), block=block, unit=unit)


def drawn_length(r, longest):
    return min(longest, int(2 ** r.uniform(0, 12)) - 1 + r.choice([0, 0, 1, 31, 32, 63]))


@pytest.mark.parametrize("seed", range(24))
def test_drawn_decode(cuda, seed):
    r = random.Random(seed)
    kw = drawn_shape(r)
    batch = r.choice([1, 2, 3, 7, 16, 33])
    pre = [drawn_length(r, 3000) for _ in range(batch)]
    if batch > 2:
        pre[r.randrange(batch)] = -1    # (a row with no keys)
    c = Case([1] * batch, pre, seed=seed, fine=r.random() < 0.5, **kw).to(cuda)
    check(c.decode(), c.reference(), c.dtype, f"{kw} {pre}")
    window, sinks = r.choice([1, 17, 64, 300, 5000]), r.choice([0, 0, 4, 100])
    check(c.decode(window, sinks), c.reference(window, sinks), c.dtype, f"{kw} {pre} {window} {sinks}")


@pytest.mark.parametrize("choice", ["causal", "window", ""])
@pytest.mark.parametrize("seed", range(16))
def test_drawn_prefill(cuda, monkeypatch, seed, choice):
    monkeypatch.setenv("NQ_PREFILL_BLOCKS", choice) if choice else monkeypatch.delenv("NQ_PREFILL_BLOCKS", raising=False)
    r = random.Random(1000 + seed)
    kw = drawn_shape(r)
    n = r.choice([1, 2, 3, 6])
    new, pre = [max(1, drawn_length(r, 500)) for _ in range(n)], [drawn_length(r, 1200) for _ in range(n)]
    c = Case(new, pre, seed=seed, fine=r.random() < 0.5, **kw).to(cuda)
    check(c.prefill(), c.reference(), c.dtype, f"{kw} {new} {pre}")
    if not choice:
        window, sinks = r.choice([1, 17, 64, 300, 5000]), r.choice([0, 0, 4, 100])
        check(c.prefill(window, sinks), c.reference(window, sinks), c.dtype, f"{kw} {new} {pre} {window} {sinks}")


@pytest.mark.parametrize("seed", range(24))
def test_drawn_append(cuda, seed):
    r = random.Random(2000 + seed)
    kw = drawn_shape(r)
    n = r.choice([1, 2, 5, 30])
    new = [1] * n if r.random() < 0.4 else [max(1, drawn_length(r, 900)) for _ in range(n)]
    pre = [drawn_length(r, 700) for _ in range(n)]
    skip = (r.randrange(n),) if n > 2 else ()
    rot = r.choice([0, 16, kw["d"] // 4, kw["d"] // 2, kw["d"]])
    append.run(cuda, new, pre, rot=rot, norm=r.random() < 0.5, seed=seed, skip=skip, scale=2.0 ** r.randint(-6, 6),
               strided=r.random() < 0.5, query=r.random() < 0.8, **kw)


@pytest.mark.parametrize("choice", ["causal", "window"])
def test_pool_past_32_bits(cuda, monkeypatch, choice):
    """Pages behind 4 GiB of codes give, and take, what the same pages give at the front."""
    monkeypatch.setenv("NQ_PREFILL_BLOCKS", choice)
    c = Case([70, 1, 130], [900, 333, 0], 32, 8, 128, BF, 256, 64).to(cuda)
    one = Case([1, 1, 1], [900, 333, 0], 32, 8, 128, BF, 256, 64).to(cuda)
    pages = 4 * 1024 ** 3 // (256 * 8 * 128) + 40
    k, v = (torch.zeros(pages, 256, 8, 128, dtype=torch.uint8, device=cuda) for _ in range(2))
    ks, vs = (torch.ones(pages, 4, 8, device=cuda) for _ in range(2))

    def far(x):
        m = x.k_dev.shape[0]
        for to, of in ((k, x.k_dev), (v, x.v_dev)):
            to[pages - m:] = of.view(torch.uint8)
        for to, of in ((ks, x.k_scale_dev), (vs, x.v_scale_dev)):
            to[pages - m:] = of
        y = Case.__new__(Case)
        y.__dict__.update(x.__dict__, k_dev=k.view(CODE), v_dev=v.view(CODE), k_scale_dev=ks, v_scale_dev=vs,
                          table_dev=torch.where(x.table_dev >= 0, x.table_dev + (pages - m), x.table_dev))
        return y
    y = far(c)
    assert torch.equal(c.prefill(), y.prefill())
    assert torch.equal(c.prefill(200, 4), y.prefill(200, 4))
    y = far(one)
    assert torch.equal(one.decode(), y.decode())
    assert torch.equal(one.decode(200, 4), y.decode(200, 4))
    # appends behind the first 100 tokens of the last page
    g = torch.Generator().manual_seed(1)
    key, value = (torch.randn(90, 8, 128, generator=g).to(BF).to(cuda) for _ in range(2))
    m = one.k_dev.shape[0]
    near = [t.clone() for t in (one.k_dev.view(torch.uint8), one.v_dev.view(torch.uint8), one.k_scale_dev, one.v_scale_dev)]
    for t in (*near[2:], ks, vs):
        t[-1] = 2.0 ** -9
    for t in (*near[:2], k, v):
        t[-1] = 0x31
    slots = torch.arange(100, 190, dtype=torch.int32, device=cuda)
    kernels.append_kvcache(key, value, near[0].view(CODE), near[1].view(CODE), slots + (m - 1) * 256, *near[2:])
    kernels.append_kvcache(key, value, k.view(CODE), v.view(CODE), slots + (pages - 1) * 256, ks, vs)
    for a, b in zip(near, (k, v, ks, vs)):
        assert torch.equal(a[-1], b[-1])
    assert (near[2][-1, 1:3] > 2.0 ** -9).all() and (near[0][-1, 100:190] != 0x31).any()


@pytest.mark.parametrize("d", [128, 256])
def test_graphs_replayed_at_once(cuda, d):
    """Decodes of several pieces in two graphs captured on one stream: each has a workspace of its own."""
    cases = [Case([1] * 40, [1500 + 7 * j + i for j in range(40)], 16, 2, d, BF, 256, 64, seed=i).to(cuda) for i in range(2)]
    want = [c.decode() for c in cases]
    torch.cuda.synchronize()
    graphs, outs = [torch.cuda.CUDAGraph() for _ in cases], []
    for g, c in zip(graphs, cases):
        with torch.cuda.graph(g):
            outs.append(c.decode())
    streams = [torch.cuda.Stream() for _ in cases]
    for _ in range(5):
        for o in outs:
            o.fill_(7)
        torch.cuda.synchronize()
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                for _ in range(10):
                    g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("what", ["decode", "prefill"])
def test_threads_on_one_stream(cuda, what):
    cases = [Case([1] * 3 if what == "decode" else [300, 90], [3000, 1500 + 64 * i, 77][:3 if what == "decode" else 2], 16, 2,
                  256 if i % 2 else 128, BF, 256, 64, seed=i).to(cuda) for i in range(4)]
    calls = [c.decode if what == "decode" else c.prefill for c in cases]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    start, fails = threading.Barrier(4), []

    def body(i):
        start.wait()
        for _ in range(10):
            if not torch.equal(calls[i](), want[i]):
                fails.append(i)
    threads = [threading.Thread(target=body, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not fails
