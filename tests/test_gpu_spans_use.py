"""Windowed and tree attention, page copies and commits as an engine uses them: through the layer and the runner,
captured, on several streams, with strides, padding and long caches."""
import threading

import pytest
import torch

import nano_qwen_amd.utils.context as C
from nano_qwen_amd import kernels
from nano_qwen_amd.engine import ModelRunner, Sequence
from nano_qwen_amd.layers import Attention
from oracle import spans
from tests.spans import Case, check, half_step, tree_masks, tree_reference

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


def _gated(ref, mag, gate, dtype):
    """Reference and tolerance of a gated output: o and sigmoid(g) rounded, their product rounded."""
    s = torch.sigmoid(gate.double().cpu())
    u = half_step(dtype)
    want = ref * s
    tol = 1.02 * (s * (u * mag + u * ref.abs() + 5e-4 * mag) + 2 * u * want.abs()) + 1e-6
    return want, tol


@pytest.mark.parametrize("hq,hkv,d,dtype,fp8", [(8, 2, 128, BF, False), (4, 2, 256, HF, True), (16, 1, 128, HF, False)])
def test_strides_gate_and_rows_behind(cuda, hq, hkv, d, dtype, fp8):
    """q and gate as halves of one projection, out with strides, rows behind the last sequence left alone."""
    for new, pre in (([1, 1, 1], [40, 0, 90]), ([9, 33], [70, 5]), ([130], [64])):
        c = Case(new, pre, hq, hkv, d, dtype, block=32, fp8=fp8, seed=3, extra_rows=3, qstride=2 * d).to(cuda)
        T, gate = sum(new), c.q_full_dev[:, :, d:]
        trees, mask = tree_masks(new, 1)
        full_mask = torch.cat([mask, torch.full((3, 1), -1)]) if mask.shape[1] == 1 else torch.cat([mask, -torch.ones(3, mask.shape[1], dtype=torch.int64)])
        wide = torch.full((T + 3, hq + 1, d + 8), 9.0, dtype=dtype, device=cuda)
        for call, ref in ((lambda **kw: c.window_prefill(20, 2, **kw), c.window_reference(20, 2)),
                          (lambda **kw: c.tree_attention(full_mask, **kw), tree_reference(c, mask))):
            out = wide.clone()
            call(out=out[:, :hq, :d], gate=gate)
            want, tol = _gated(*ref, gate[:T], dtype)
            off = (out[:T, :hq, :d].double().cpu() - want).abs()
            assert (off <= tol).all(), (off - tol).max()
            out[:T, :hq, :d] = 9.0
            assert (out == 9.0).all()
        if max(new) == 1:
            cd = Case(new, pre, hq, hkv, d, dtype, block=32, fp8=fp8, seed=3, qstride=2 * d).to(cuda)
            g = cd.q_full_dev[:, :, d:]
            out = cd.window_decode(20, 2, gate=g)
            want, tol = _gated(*cd.window_reference(20, 2), g, dtype)
            assert ((out.double().cpu() - want).abs() <= tol).all()


def test_table_wider_than_rows_and_more_rows(cuda):
    """Tables with a row stride, and with more rows than sequences (a captured step's)."""
    c = Case([1, 1], [70, 500], 8, 2, 128, BF, block=32).to(cuda)
    big = torch.full((6, 64), -7, dtype=torch.int32, device=cuda)
    big[:2, :c.table.shape[1]] = c.table_dev
    plain = c.window_decode(100, 4)
    c.table_dev = big[:, :40]
    assert torch.equal(c.window_decode(100, 4), plain)


@pytest.mark.parametrize("batch", [1, 7, 300])
def test_decode_batches(cuda, batch):
    """Few sequences and more than the kernel keeps the bounds of; some of them empty."""
    pre = [(-1 if i % 9 == 4 else (37 * i) % 400) for i in range(batch)]
    c = Case([1] * batch, pre, 8, 2, 128, BF, block=32, seed=batch).to(cuda)
    check(c.window_decode(65, 3), *c.window_reference(65, 3), BF)


def test_prefill_of_many_sequences(cuda):
    new = [1 + (29 * i) % 40 for i in range(270)]
    pre = [(17 * i) % 50 for i in range(270)]
    c = Case(new, pre, 4, 1, 128, BF, block=32, seed=2).to(cuda)
    check(c.window_prefill(24, 2), *c.window_reference(24, 2), BF)
    trees, mask = tree_masks(new, 2)
    check(c.tree_attention(mask), *tree_reference(c, mask), BF)


def test_whole_items_equal_ranges(cuda):
    """Enough prompts that items are dealt out whole: each sequence as close as alone, where it is cut."""
    new = [700, 33, 1200, 5, 900, 350, 64, 1100] * 3
    c = Case(new, [0] * len(new), 32, 8, 128, BF, paged=False, seed=4).to(cuda)
    out = c.window_prefill(300, 4)
    at = 0
    for i, n in enumerate(new[:8]):
        cu = torch.tensor([0, n], dtype=torch.int32, device=cuda)
        one = kernels.window_prefill(c.q_dev[at:at + n], c.k_dev[at:at + n], c.v_dev[at:at + n], cu, cu, n, n, c.scale, 300, 4)
        # both round P and the output once: twice the tolerance of one, whose mean of |v| is at most max |v|
        d = (out[at:at + n].float() - one.float()).abs()
        assert d.max() <= 2 * 1.02 * (2 * half_step(BF) + 5e-4) * float(c.v.abs().max())
        assert d.mean() < 2e-3 * float(one.float().abs().mean()) + 1e-4
        at += n
    short = Case([33, 5, 64], [0, 0, 0], 32, 8, 128, BF, paged=False, seed=4)
    check(short.to(cuda).window_prefill(300, 4), *short.window_reference(300, 4), BF)


def test_missing_pages_are_invisible(cuda):
    c = Case([3, 40, 1], [200, 100, 150], 8, 2, 128, BF, block=32)
    c.table[0, 5] = -1
    c.table[1, 0] = 10 ** 6
    c.table[2, 4] = -5
    c.to(cuda)
    check(c.window_prefill(90, 40), *c.window_reference(90, 40), BF)
    trees, mask = tree_masks([3, 40, 1])
    check(c.tree_attention(mask), *tree_reference(c, mask), BF)


def test_long_cache_offsets(cuda):
    """Cache rows whose byte offsets pass 32 bits."""
    blocks, bs, hkv, d = 5000, 256, 8, 256    # 5000 * 256 * 8 * 256 * 2 bytes = 4.9 GiB per cache
    k = torch.zeros(blocks, bs, hkv, d, dtype=BF, device=cuda)
    v = torch.zeros_like(k)
    table = torch.tensor([[4999, 3, 4500]], dtype=torch.int32, device=cuda)
    g = torch.Generator(device=cuda).manual_seed(0)
    for b in (4999, 3, 4500):
        k[b].normal_(generator=g)
        v[b].normal_(generator=g)
    q = torch.randn(4, 16, d, generator=g, device=cuda).to(BF)
    cu_q, cu_k = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 4], [0, 700]))
    mask = kernels.tree_masks([[-1, 0, 0, 1]]).to(cuda)
    out = kernels.tree_attention(q, k, v, cu_q, cu_k, 4, 700, d ** -0.5, table, mask)
    kk = torch.cat([k[b] for b in (4999, 3, 4500)])[:700].double().cpu()
    vv = torch.cat([v[b] for b in (4999, 3, 4500)])[:700].double().cpu()
    check(out, *spans.attend(q.cpu(), kk, vv, spans.tree_visible(mask.tolist(), 4, 696), d ** -0.5), BF)
    win = kernels.window_prefill(q, k, v, cu_q, cu_k, 4, 700, d ** -0.5, 300, 4, block_table=table)
    check(win, *spans.attend(q.cpu(), kk, vv, spans.window_visible(torch.arange(696, 700), 700, 300, 4), d ** -0.5), BF)
    before = k[4999].clone()
    kernels.copy_kv_blocks(k, *(torch.tensor([x], dtype=torch.int32, device=cuda) for x in (4999, 4998)))
    assert torch.equal(k[4998], before)


def test_graphs_replayed_with_eager_work_between(cuda):
    """Every entry point captured, two graphs of it, new lengths and values at each replay."""
    c = Case([1, 1, 1, 1], [300, 0, 77, 900], 8, 2, 128, BF, block=32).to(cuda)
    t = Case([9, 20, 1], [100, 0, 300], 8, 2, 128, BF, block=32, seed=5).to(cuda)
    trees, mask = tree_masks([9, 20, 1])
    mask = mask.to(cuda)
    lens = torch.tensor(c.have, dtype=torch.int32, device=cuda)
    pool = torch.randn(2, 2, 6, 32, 2, 128, device=cuda).to(BF)
    src, dst = (torch.tensor(x, dtype=torch.int32, device=cuda) for x in ([0, 1], [4, 5]))

    def step():
        kernels.copy_kv_blocks(pool, src, dst)
        return (kernels.window_decode(c.q_dev, c.k_dev, c.v_dev, lens, c.table_dev, c.scale, 70, 4),
                t.window_prefill(33, 2), t.tree_attention(mask))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step())
        graphs.append(g)
    for turn in range(5):
        c.q_dev.copy_(torch.randn_like(c.q_dev, dtype=torch.float32))
        t.q_full_dev.copy_(torch.randn_like(t.q_full_dev, dtype=torch.float32))
        lens.copy_(torch.tensor([[301, 1, 78, 901], [5, 0, 40, 130], [64, 1, 2, 3], [200, 1, 0, 880], [301, 1, 78, 901]][turn]))
        pool.normal_()
        for o in outs:
            for x in o:
                x.fill_(7.0)
        for g in graphs:
            g.replay()
        want = step()
        for o in outs:
            for a, b in zip(o, want):
                assert torch.equal(a, b), turn
        assert torch.equal(pool[:, :, 4:6], pool[:, :, 0:2])
        torch.cuda.synchronize()


def test_streams_and_threads(cuda):
    """Host threads with a stream each, and two that share one."""
    c = Case([1] * 3, [300, 20, 900], 8, 2, 128, BF, block=32).to(cuda)
    t = Case([26, 9], [600, 40], 8, 2, 128, BF, block=32, seed=5).to(cuda)
    trees, mask = tree_masks([26, 9])
    mask = mask.to(cuda)
    want = c.window_decode(200, 4), t.tree_attention(mask), t.window_prefill(50, 1)
    torch.cuda.synchronize()
    shared = torch.cuda.Stream()
    streams = [torch.cuda.Stream(), torch.cuda.Stream(), shared, shared]
    failed = []

    def work(stream):
        try:
            with torch.cuda.stream(stream):
                for _ in range(30):
                    got = c.window_decode(200, 4), t.tree_attention(mask), t.window_prefill(50, 1)
                    stream.synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want)):
                        failed.append("another result")
        except Exception as e:    # noqa: BLE001
            failed.append(e)

    threads = [threading.Thread(target=work, args=(s,)) for s in streams]
    for x in threads:
        x.start()
    for x in threads:
        x.join()
    assert not failed, failed[0]


def test_refusals(cuda):
    c = Case([2, 3], [40, 5], 8, 2, 128, BF, block=32).to(cuda)
    trees, mask = tree_masks([2, 3])
    mask = mask.to(cuda)
    q, k, v, cq, ck, bt = c.q_dev, c.k_dev, c.v_dev, c.cu_q_dev, c.cu_k_dev, c.table_dev
    tree = lambda q=q, k=k, v=v, cq=cq, ck=ck, bt=bt, m=mask, **kw: kernels.tree_attention(    # noqa: E731
        q, k, v, cq, ck, 3, 45, c.scale, bt, m, **kw)
    for kw in (dict(q=q[:, :, ::2]), dict(q=q[0]), dict(cq=cq.long()), dict(ck=ck[:2]), dict(bt=bt.long()), dict(bt=bt[:1]),
               dict(bt=bt.t()), dict(m=mask.int()), dict(m=mask[:3]), dict(k=k.half(), v=v.half()), dict(v=v[:3]),
               dict(out=torch.empty_like(q, dtype=HF)), dict(gate=q[:2]), dict(q=q.float()),
               dict(k=k.to(torch.float8_e4m3fn), v=v.to(torch.float8_e4m3fn)), dict(m=mask.cpu())):
        with pytest.raises(RuntimeError):
            tree(**kw)
    with pytest.raises(RuntimeError):
        kernels.window_prefill(q, k, v, cq, ck, 3, 45, c.scale, 0, block_table=bt)
    with pytest.raises(RuntimeError):
        kernels.window_prefill(q, k, v, cq, ck, 3, 45, -1.0, 4, block_table=bt)
    with pytest.raises(RuntimeError):
        kernels.window_prefill(q, q[:, :2], q[:, 2:4].contiguous(), cq, cq, 3, 3, c.scale, 4)
    lens = torch.tensor([3, 4], dtype=torch.int32, device=cuda)
    for args in ((q[:2], k, v, lens.long(), bt), (q[:2], k, v, lens[:1], bt), (q[:2][None], k, v, lens, bt)):
        with pytest.raises(RuntimeError):
            kernels.window_decode(*args, c.scale, 4)
    with pytest.raises(RuntimeError):    # a stored row of another shape
        kernels.window_decode(q[:2], k, v, lens, bt, c.scale, 4, k=q[:2], v=q[:2], slot_mapping=lens)
    ids = torch.tensor([0, 1], dtype=torch.int32, device=cuda)
    for args in ((k[:, :, :1], ids, ids), (k, ids.long(), ids), (k, ids, ids[:1]), (k, ids, ids, ids[:1]), (k[0], ids, ids)):
        with pytest.raises(RuntimeError):
            kernels.copy_kv_blocks(*args)
    tok = torch.zeros(5, dtype=torch.int64, device=cuda)
    par = torch.zeros(5, dtype=torch.int32, device=cuda)
    path, num = torch.zeros(2, 3, dtype=torch.int32, device=cuda), torch.zeros(2, dtype=torch.int32, device=cuda)
    for kw in (dict(parents=par, tokens=tok), dict(parents=par.long(), tokens=tok, target_tokens=tok), dict(path=path),
               dict(path=path[:, :2], num_accepted=num), dict(parents=par[:4], tokens=tok, target_tokens=tok),
               dict(path=path, num_accepted=num, tokens=tok)):
        with pytest.raises(RuntimeError):
            kernels.commit_tree(k, bt, cq, ck, 3, **kw)


# ------------------------------------------------------- through the engine

def _engine(cuda, layers, block=32, blocks=60, dtype=BF, kv=None, **attn):
    runner = ModelRunner(block_size=block, max_num_seqs=8, device=cuda)
    attns = torch.nn.ModuleList(Attention(8, 128, 128 ** -0.5, 2, **attn) for _ in range(layers))
    runner.allocate_kv_cache(attns, layers, blocks, 2, 128, dtype, kv_cache_dtype=kv)
    if kv is None:
        runner.kv_cache.fill_(float("nan"))
    else:
        runner.kv_cache.view(torch.uint8).fill_(0xFF)
        runner.kv_scales.fill_(0.02)
    return runner, attns


def _token_rows(tokens, positions, layer, cuda):
    """A toy model's q, k, v rows: of a token at a position, the same in whatever step they are computed."""
    out = [], [], []
    for t, p in zip(tokens, positions):
        g = torch.Generator().manual_seed(1000003 * layer + 977 * int(t) + int(p))
        x = torch.randn(12, 128, generator=g)
        for o, part in zip(out, (x[:8], x[8:10], x[10:])):
            o.append(part)
    return [torch.stack(o).to(BF).to(cuda) for o in out]


def _run(attns, ids, pos, cuda):
    rows = [_token_rows(ids.tolist(), pos.tolist(), i, cuda) for i in range(len(attns))]
    return [a(*r) for a, r in zip(attns, rows)]


@pytest.mark.parametrize("kv", [None, torch.float8_e4m3fn])
def test_speculation_equals_decoding(cuda, kv):
    """Prefill, fork, verify a tree, commit, decode on: the same cache and outputs as token by token."""
    runner, attns = _engine(cuda, 3, kv=kv)
    a = Sequence(list(range(50, 95)), [7, 2, 11], 0, 45)
    b = Sequence([5, 6, 7], [4], 0, 3)
    for s in (a, b):
        s.num_scheduled_tokens = len(s)
    ids, pos = runner.prepare_prefill([a, b])
    _run(attns, ids, pos, cuda)
    a.append_token(500)
    b.append_token(600)
    # continuations that decode token by token from a copy of the last pages
    c, d = runner.fork([a, b], [20, 21])
    assert c.block_table == [7, 20] and d.block_table == [21]
    # trees: the model "chooses" 501 after 500, 502 after 501, then 503; and 601 after 600
    drafts = [[499, 501, 9, 502, 8], [1, 2]]
    parents = [[0, 0, 2, 2, 4], [0, 0]]
    follows = {500: 501, 501: 502, 502: 503, 600: 601}
    ids, pos = runner.prepare_tree([a, b], drafts, parents)
    outs = _run(attns, ids, pos, cuda)
    targets = torch.tensor([follows.get(t, 77) for t in ids.tolist()], device=cuda)
    path, count, following = runner.commit_tree(targets)
    assert path.tolist() == [[0, 2, 4, -1, -1, -1], [0, -1, -1, -1, -1, -1]] and count.tolist() == [3, 1]
    runner.accept_tree([a, b], drafts, path, count, following)
    assert a.token_ids[-4:] == [500, 501, 502, 503] and b.token_ids[-2:] == [600, 601]
    C.reset_context()
    # the same tokens decoded one by one in the continuations
    for step in range(3):
        seqs = [c, d] if step == 0 else [c]
        runner.sampled_token_ids_gpu[:2] = torch.tensor([c.last_token, d.last_token])
        ids, pos = runner.prepare_decode(seqs)
        got = _run(attns, ids, pos, cuda)
        for tree, one in zip(outs, got):
            # rounding of P and of the output in both; values of |v| <= 5 (fp8: the same codes in both)
            assert (tree[[0, 2, 4][step]].float() - one[0, 0].float()).abs().max() <= 2 * 1.02 * (2 * half_step(BF) + 5e-4) * 5
        c.append_token([501, 502, 503][step])
    raw = runner.kv_cache.view(torch.uint8)
    for s, o in ((a, c), (b, d)):
        for p in range(len(s) - 1 if s is a else 4):
            x, y = (raw[:, :, t.block_table[p // 32], p % 32] for t in (s, o))
            assert torch.equal(x, y), p
    # and on: one more decode step of both, over caches that went different ways
    outs = []
    for s in (a, c):
        s.block_table = s.block_table[:2]    # 48 tokens and the new one: two pages
        runner.sampled_token_ids_gpu[:1] = torch.tensor([s.last_token])
        ids, pos = runner.prepare_decode([s])
        outs.append(_run(attns, ids, pos, cuda))
    assert all(torch.equal(x, y) for x, y in zip(*outs))
    # the pool compacted: the same attention from other pages
    n = runner.compact([a, b, c, d])
    assert n == 5 and max(x for s in (a, b, c, d) for x in s.block_table) == 4
    runner.sampled_token_ids_gpu[:1] = torch.tensor([a.last_token])
    ids, pos = runner.prepare_decode([a])
    assert all(torch.equal(x, y) for x, y in zip(_run(attns, ids, pos, cuda), outs[0]))
    C.reset_context()


@pytest.mark.parametrize("kv", [None, torch.float8_e4m3fn])
def test_windowed_layers_release_pages(cuda, kv):
    """Prefill in two chunks, then decode through a captured graph, while pages behind the window are given back."""
    window, sinks = 40, 3
    runner, attns = _engine(cuda, 2, kv=kv, window=window, num_sinks=sinks)
    tokens = list(range(300, 300 + 150))
    s = Sequence(tokens, [9, 3, 14, 1, 22], 0, 100)
    chunks = []
    for start, n in ((0, 100), (100, 50)):
        s.num_cached_tokens, s.num_scheduled_tokens = start, n
        ids, pos = runner.prepare_prefill([s])
        chunks.append(_run(attns, ids, pos, cuda))
    rows = [_token_rows(tokens, range(150), i, "cpu") for i in range(2)]

    def as_cached(x, which, layer):
        if kv is None:
            return x.double()
        t = runner.kv_scales[which, layer].cpu()
        return (x.float() * (1.0 / t)[:, None]).clamp(-448, 448).to(kv).double() * t.double()[:, None]

    for layer in range(2):
        q, k, v = rows[layer]
        vis = spans.window_visible(torch.arange(150), 150, window, sinks)
        exact = spans.attend(q[:100], k[:100].double(), v[:100].double(), vis[:100, :100], 128 ** -0.5)    # packed
        check(chunks[0][layer], *exact, BF)
        exact = spans.attend(q[100:], as_cached(k, 0, layer), as_cached(v, 1, layer), vis[100:], 128 ** -0.5)
        check(chunks[1][layer], *exact, BF)

    class Model:
        def __call__(self, ids, pos):
            x = self.rows
            return torch.cat([a(*r)[:, 0].flatten(1) for a, r in zip(attns, x)], 1)

    model = Model()
    model.rows = [[torch.zeros(8, h, 128, dtype=BF, device=cuda)[:1] for h in (8, 2, 2)] for _ in range(2)]
    runner.max_num_seqs = 1
    runner.capture_cudagraph(model, 2 * 8 * 128, 6 * 32, dtype=BF)
    for step in range(30):
        s.append_token(1000 + step)
        if len(s) == 161:    # the last page of a table holds the last token
            s.block_table.append(6)
        freed = runner.release_window_blocks(s, window, sinks)
        for b in freed:    # whoever takes the page writes anything
            runner.kv_cache.view(torch.uint8)[:, :, b] = 0xFF
        runner.sampled_token_ids_gpu[:1] = torch.tensor([s.last_token])
        ids, pos = runner.prepare_decode([s])
        p = len(s) - 1
        for layer in range(2):
            new = _token_rows([s.last_token], [p], layer, cuda)
            for to, x in zip(model.rows[layer], new):
                to.copy_(x)
            rows[layer] = [torch.cat([x, y.cpu()]) for x, y in zip(rows[layer], new)]
        out = runner.run_model(ids, pos, False).view(2, 8, 128)
        for layer in range(2):
            q, k, v = rows[layer]
            exact = spans.attend(q[p:], as_cached(k, 0, layer), as_cached(v, 1, layer),
                                 spans.window_visible(torch.tensor([p]), p + 1, window, sinks), 128 ** -0.5)
            check(out[layer][None], *exact, BF, f"step {step}")
    assert s.block_table == [9, -1, -1, -1, 22, 6]    # 180 tokens: 140 .. 179 are seen
    C.reset_context()


@pytest.mark.parametrize("d,dtype,fp8,new_dtype", [(128, BF, False, BF), (256, HF, False, HF), (128, BF, True, BF),
                                                   (256, HF, True, torch.float32), (128, HF, True, HF)])
def test_decode_stores_the_new_token(cuda, d, dtype, fp8, new_dtype):
    """The fused store leaves the bytes and outputs of the store followed by the decode; skipped and odd slots too."""
    pre = [0, 31, 32, 255, 700, 63, -1, 90]
    for sinks, window in ((4, 40), (0, 1), (64, 10 ** 6)):
        g = torch.Generator(device=cuda).manual_seed(window)
        cases = [Case([1] * 8, pre, 8, 2, d, dtype, block=32, fp8=fp8, seed=9).to(cuda) for _ in range(2)]
        base = torch.randn(8, 5, 2, d, device=cuda, generator=g).to(new_dtype)
        k, v = base[:, 1], base[:, 3]    # rows of one projection
        slots = [int(cases[0].table[i, p // 32]) * 32 + p % 32 if p >= 0 else -1 for i, p in enumerate(pre)]
        spare = next(b for b in range(cases[0].k.shape[0]) if b not in cases[0].table)
        slots[5], slots[6], slots[7] = -1, spare * 32 + 7, 10 ** 7    # skipped, a row nobody reads, outside the pool
        slots = torch.tensor(slots, dtype=torch.int32, device=cuda)
        a, b = cases
        got = a.window_decode(window, sinks, k=k, v=v, slot_mapping=slots)
        kernels.store_kvcache(k, v, b.k_dev, b.v_dev, slots, b.k_scale_dev, b.v_scale_dev)
        want = b.window_decode(window, sinks)
        assert torch.equal(got, want)
        for x, y in ((a.k_dev, b.k_dev), (a.v_dev, b.v_dev)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8))


def test_captured_decode_stores_the_new_token(cuda):
    """The fused store in a graph: new rows, slots and lengths at every replay, against the separate store."""
    a, b = (Case([1] * 3, [255, 31, 90], 8, 2, 128, BF, block=32, seed=9).to(cuda) for _ in range(2))
    k, v = (torch.zeros(3, 2, 128, dtype=BF, device=cuda) for _ in range(2))
    slots, lens = (torch.zeros(3, dtype=torch.int32, device=cuda) for _ in range(2))

    def step(c, **new):
        return kernels.window_decode(c.q_dev, c.k_dev, c.v_dev, lens, c.table_dev, c.scale, 50, 2, **new)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    slots.fill_(-1)
    with torch.cuda.stream(side):
        step(a, k=k, v=v, slot_mapping=slots)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(a, k=k, v=v, slot_mapping=slots)
    for turn, pos in enumerate([[255, 31, 90], [0, 32, 64], [254, 0, 63], [31, 31, 31]]):
        k.normal_()
        v.normal_()
        lens.copy_(torch.tensor([p + 1 for p in pos]))
        slots.copy_(torch.tensor([int(a.table[i, p // 32]) * 32 + p % 32 for i, p in enumerate(pos)]))
        graph.replay()
        kernels.store_kvcache(k, v, b.k_dev, b.v_dev, slots)
        want = step(b)
        assert torch.equal(out, want), turn
        for x, y in ((a.k_dev, b.k_dev), (a.v_dev, b.v_dev)):
            assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)), turn


def test_windows_beyond_32_bits(cuda):
    """A window (or sinks) that no int holds is one that every token sees through."""
    c = Case([1, 1], [300, 40], 8, 2, 128, BF, block=32).to(cuda)
    p = Case([40, 3], [0, 90], 8, 2, 128, BF, block=32).to(cuda)
    for case, call in ((c, c.window_decode), (p, p.window_prefill)):
        want = call(4096, 0)
        assert torch.equal(call(2 ** 32 + 3, 0), want) and torch.equal(call(1, 2 ** 32 + 3), want)
