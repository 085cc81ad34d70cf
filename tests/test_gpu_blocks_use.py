"""A cache with a scale for each block of tokens and head, through the layer and the runner: prompts in chunks, decoding,
forks, compaction, windows and captured steps, against a cache and an attention in float64."""
import types

import numpy as np
import pytest
import torch

from nano_qwen_amd import kernels
from nano_qwen_amd.engine import ModelRunner, Sequence
from nano_qwen_amd.layers import Attention, qk_norm_rope_store
from nano_qwen_amd.utils.context import get_context, set_context
from oracle import block_scales as o
from oracle import spans
from tests.blocks import CODE
from tests.spans import tolerance

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HQ, HKV, D, LAYERS = 8, 2, 128, 2


class Engine:
    """A toy model's layers over a runner's pool, and the same pool in float64."""

    def __init__(self, cuda, block=64, unit=32, blocks=24, **attn):
        self.cuda, self.block, self.unit = cuda, block, unit
        self.runner = ModelRunner(block_size=block, max_num_seqs=8, device=cuda)
        self.attns = torch.nn.ModuleList(Attention(HQ, D, D ** -0.5, HKV, **attn) for _ in range(LAYERS))
        self.runner.allocate_kv_cache(self.attns, LAYERS, blocks, HKV, D, BF, kv_cache_dtype=CODE, kv_scale_block=unit)
        self.runner.kv_cache.view(torch.uint8).fill_(0x7F)    # NaN
        self.codes = np.full((2, LAYERS, blocks * block, HKV, D), 0x7F, np.uint8)
        self.scales = np.ones((2, LAYERS, blocks * block // unit, HKV), np.float32)

    def rows(self, ids, pos, layer):
        """q, k, v of tokens at positions, the same in whatever step they are computed; magnitudes rise and fall."""
        out = [], [], []
        for t, p in zip(ids, pos):
            g = torch.Generator().manual_seed(1000003 * layer + 977 * int(t) + int(p))
            x = torch.randn(HQ + 2 * HKV, D, generator=g)
            x[HQ:] *= 2.0 ** float(torch.randint(-2, 1, (1,), generator=g))
            x[HQ + HKV:] *= 2.0 ** float(torch.randint(-4, 5, (1,), generator=g))
            for to, part in zip(out, (x[:HQ], x[HQ:HQ + HKV], x[HQ + HKV:])):
                to.append(part)
        return [torch.stack(x).to(BF) for x in out]

    def step(self, ids, pos, seqs, have, new, packed, window=1 << 40, sinks=0):
        """One step of all layers; ``packed``: attention over the new keys and values themselves."""
        ids, pos = ids.tolist(), pos.tolist()
        slots = get_context().slot_mapping.cpu().numpy()
        for i, attn in enumerate(self.attns):
            q, k, v = self.rows(ids, pos, i)
            out = attn(*(x.to(self.cuda) for x in (q, k, v)))
            for kv, z in enumerate((k, v)):
                self.codes[kv, i], self.scales[kv, i] = o.append(z.double().numpy(), self.codes[kv, i], self.scales[kv, i], slots,
                                                                 self.unit)
            out, at = out.reshape(len(ids), HQ, D).double().cpu(), 0
            for s, h, n in zip(seqs, have, new):
                if packed:
                    kk, vv = (x[at:at + n].double() for x in (k, v))
                else:
                    rows = [s.block_table[p // self.block] * self.block + p % self.block for p in range(h)]
                    seen = [r if r >= 0 else 0 for r in rows]    # pages given back: not in any window
                    kk, vv = (torch.from_numpy(np.nan_to_num(o.values(self.codes[x, i], self.scales[x, i], self.unit)[seen]))
                              for x in (0, 1))
                vis = spans.window_visible(torch.arange(h - n, h), h, window, sinks)
                ref, mag = spans.attend(q[at:at + n], kk, vv, vis, D ** -0.5)
                off = (out[at:at + n] - ref).abs()
                assert (off <= tolerance(ref, mag, BF)).all(), (i, off.max())
                at += n
        self.check_pool()

    def check_pool(self):
        got = self.runner.kv_cache.view(torch.uint8).cpu().numpy().reshape(self.codes.shape)
        assert np.array_equal(got, self.codes)
        assert np.array_equal(self.runner.kv_scales.cpu().numpy().reshape(self.scales.shape), self.scales)

    def prefill(self, seqs, scheduled, **kw):
        for s, n in zip(seqs, scheduled):
            s.num_scheduled_tokens = n
        ids, pos = self.runner.prepare_prefill(seqs)
        self.step(ids, pos, seqs, [s.num_cached_tokens + n for s, n in zip(seqs, scheduled)], scheduled,
                  get_context().block_tables is None, **kw)
        for s, n in zip(seqs, scheduled):
            s.num_cached_tokens += n

    def decode(self, seqs, tokens, **kw):
        for i, (s, t) in enumerate(zip(seqs, tokens)):
            s.append_token(t)
            self.runner.sampled_token_ids_gpu[i] = t
        ids, pos = self.runner.prepare_decode(seqs)
        self.step(ids, pos, seqs, [len(s) for s in seqs], [1] * len(seqs), False, **kw)

    def move(self, src, dst):
        """Pages in the float64 pool, whole."""
        b, u = self.block, self.block // self.unit
        codes, scales = self.codes.copy(), self.scales.copy()
        for x, y in zip(src, dst):
            self.codes[:, :, y * b:(y + 1) * b] = codes[:, :, x * b:(x + 1) * b]
            self.scales[:, :, y * u:(y + 1) * u] = scales[:, :, x * u:(x + 1) * u]


@pytest.mark.parametrize("block,unit", [(64, 32), (64, 64), (256, 64)])
def test_serving(cuda, block, unit):
    e = Engine(cuda, block, unit)
    a = Sequence(list(range(50, 50 + 150)), [7, 2, 11, 5][:4], 0, 0)
    b = Sequence([5, 6, 7], [4], 0, 0)
    e.prefill([a, b], [90, 3])            # packed: no prefix yet
    e.prefill([a], [60])                  # the rest, behind a partly filled block
    for t in range(3):
        e.decode([a, b], [500 + t, 600 + t])
    c, d = e.runner.fork([a, b], [20, 21])
    full_a, full_b = (len(a) - 1) // block, (len(b) - 1) // block
    src, dst = [a.block_table[full_a], b.block_table[full_b]], [20, 21]
    for s, y, rows in zip(src, dst, ((len(a) - 1) % block, (len(b) - 1) % block)):
        u = block // unit
        e.codes[:, :, y * block:y * block + rows] = e.codes[:, :, s * block:s * block + rows]
        e.scales[:, :, y * u:(y + 1) * u] = e.scales[:, :, s * u:(s + 1) * u]
    e.check_pool()
    for s in (c, d):    # the fork's last token is computed again, as after any fork
        s.token_ids = s.token_ids[:-1]
        s.num_tokens = len(s.token_ids)
    for t in range(4):
        e.decode([a, c, b, d], [700 + t, 710 + t, 720 + t, 730 + t])
    seqs = [a, b, c, d]
    before = sorted({x for s in seqs for x in s.block_table})
    old = [list(s.block_table) for s in seqs]
    used = e.runner.compact(seqs)
    moved = {x: y for s, t in zip(old, seqs) for x, y in zip(s, t.block_table) if x != y}
    e.move(list(moved), list(moved.values()))
    assert used == len(before) and max(x for s in seqs for x in s.block_table) < used
    e.check_pool()
    e.decode(seqs, [800, 810, 820, 830])


def test_windowed_layers(cuda):
    kw = dict(window=40, sinks=2)
    e = Engine(cuda, 32, 32, window=40, num_sinks=2)
    a = Sequence(list(range(300)), [3, 9, 1, 0, 7, 12, 15, 2, 21, 22, 23], 0, 0)
    e.prefill([a], [200], **kw)
    e.runner.release_window_blocks(a, 40, 2)
    e.prefill([a], [100], **kw)
    for t in range(20):
        e.decode([a], [400 + t], **kw)
        freed = e.runner.release_window_blocks(a, 40, 2)
        for x in freed:    # another sequence's pages now
            e.runner.kv_cache[:, :, x].view(torch.uint8).fill_(0x7F)
            e.codes[:, :, x * 32:(x + 1) * 32] = 0x7F


class Rotary:
    rotary_dim = 128

    def __init__(self, cuda):
        self.cos_sin_cache = torch.randn(512, 1, 128, generator=torch.Generator().manual_seed(0)).to(cuda)


class Model(torch.nn.Module):
    """Rotation (and norms) and attention of one layer, from hidden states that embed the tokens."""

    def __init__(self, cuda, norm):
        super().__init__()
        g = torch.Generator().manual_seed(1)
        self.table = torch.randn(64, HQ + 2 * HKV, D, generator=g).to(BF).to(cuda)
        self.attn = Attention(HQ, D, D ** -0.5, HKV)
        self.rotary = Rotary(cuda)
        self.norms = [types.SimpleNamespace(weight=torch.randn(D, generator=g).to(BF).to(cuda) * 0.1, eps=1e-6) for _ in range(2)] \
            if norm else [None, None]

    def forward(self, ids, positions):
        x = self.table[ids]
        q, k, v = x[:, :HQ], x[:, HQ:HQ + HKV].contiguous(), x[:, HQ + HKV:].contiguous()
        q, k = qk_norm_rope_store(positions, q, k, v, *self.norms, self.rotary, self.attn)
        return self.attn(q, k, v, kv_stored=True).reshape(len(ids), -1)


@pytest.mark.parametrize("norm", [False, True])
def test_captured_decode_equals_eager(cuda, norm):
    """The runner's captured steps, padded batches among them, bit for bit: outputs, codes and scales."""
    pools = []
    for graphs in (False, True):
        model = Model(cuda, norm)
        runner = ModelRunner(block_size=64, max_num_seqs=4, device=cuda)
        set_context(True)    # before there is a pool: nothing is stored
        q = model.table[:2]
        qk_norm_rope_store(torch.tensor([0, 1], device=cuda), q[:, :HQ], q[:, HQ:HQ + HKV].contiguous(),
                           q[:, HQ + HKV:].contiguous(), *model.norms, model.rotary, model.attn)
        runner.allocate_kv_cache([model.attn], 1, 8, HKV, D, BF, kv_cache_dtype=CODE, kv_scale_block=32)
        runner.kv_cache.view(torch.uint8).zero_()
        runner.model = model
        if graphs:
            runner.capture_cudagraph(model, HQ * D, 256, dtype=BF)
            assert (runner.kv_cache.view(torch.uint8) == 0).all() and (runner.kv_scales == 1).all()
        seqs = [Sequence(list(range(40)), [1, 3], 0, 40), Sequence([9, 8, 7], [5, 6], 0, 3), Sequence([3], [2, 0], 0, 1)]
        outs = [runner.run_model(*runner.prepare_prefill(seqs), True).clone()]
        for t in range(36):
            batch = seqs[:1 + t % 3] if t < 30 else seqs
            for i, s in enumerate(batch):
                s.append_token((7 * t + i) % 64)
                runner.sampled_token_ids_gpu[i] = s.last_token
            ids, pos = runner.prepare_decode(batch)
            outs.append(runner.run_model(ids, pos, False).clone())
        pools.append((outs, runner.kv_cache.view(torch.uint8).clone(), runner.kv_scales.clone()))
    (a, ka, sa), (b, kb, sb) = pools
    assert all(torch.equal(x, y) for x, y in zip(a, b)) and torch.equal(ka, kb) and torch.equal(sa, sb)
    assert torch.isfinite(torch.cat(a)).all()


def test_layer_path_equals_the_calls(cuda):
    """qk_norm_rope_store and Attention make the calls of kernels, in prefill and decode."""
    model = Model(cuda, True)
    runner = ModelRunner(block_size=64, max_num_seqs=4, device=cuda)
    runner.allocate_kv_cache([model.attn], 1, 8, HKV, D, BF, kv_cache_dtype=CODE, kv_scale_block=64)
    seq = Sequence(list(range(40)), [1, 3], 0, 40)
    ids, pos = runner.prepare_prefill([seq])
    out = model(ids, pos)
    cache, scale = runner.kv_cache.clone(), runner.kv_scales.clone()
    c = get_context()
    x = model.table[ids]
    q, k, v = x[:, :HQ], x[:, HQ:HQ + HKV].contiguous(), x[:, HQ + HKV:].contiguous()
    q, k = kernels.append_kvcache(k, v, runner.kv_cache[0, 0], runner.kv_cache[1, 0], c.slot_mapping, runner.kv_scales[0, 0],
                                  runner.kv_scales[1, 0], query=q, positions=pos, cos_sin_cache=model.rotary.cos_sin_cache,
                                  rotary_dim=128, q_weight=model.norms[0].weight, k_weight=model.norms[1].weight, eps=1e-6)
    want = kernels.varlen_prefill(q, k, v, c.cu_seqlens_q, c.cu_seqlens_k, 40, 40, D ** -0.5)
    assert torch.equal(out, want.reshape(40, -1))
    assert torch.equal(cache.view(torch.uint8), runner.kv_cache.view(torch.uint8)) and torch.equal(scale, runner.kv_scales)


def test_refusals(cuda):
    e = Engine(cuda)
    s = Sequence(list(range(10)), [1], 0, 10)
    with pytest.raises(RuntimeError):
        e.runner.prepare_tree([s], [[1]], [[0]])
    with pytest.raises(RuntimeError):
        e.runner.calibrate_kv_scales([(None, None)] * LAYERS)
    for kw in (dict(kv_cache_dtype=BF, kv_scale_block=32), dict(kv_cache_dtype=CODE, kv_scale_block=16),
               dict(kv_cache_dtype=CODE, kv_scale_block=128), dict(kv_scale_block=32)):
        with pytest.raises(ValueError):
            ModelRunner(block_size=64, max_num_seqs=2, device=cuda).allocate_kv_cache(e.attns, LAYERS, 4, HKV, D, BF, **kw)
    with pytest.raises(RuntimeError):
        kernels.copy_kv_scales(e.runner.kv_scales[:, :, :, :, :1], *(torch.zeros(1, dtype=torch.int32, device=cuda),) * 2)
    plain = Attention(HQ, D, D ** -0.5, HKV)
    plain.k_cache = plain.v_cache = torch.zeros(2, 64, HKV, D, dtype=BF, device=cuda)
    x = torch.zeros(1, HQ, D, dtype=BF, device=cuda)
    with pytest.raises(RuntimeError):
        qk_norm_rope_store(torch.zeros(1, dtype=torch.int64, device=cuda), x, x[:, :HKV], x[:, :HKV], None, None, Rotary(cuda), plain)


def test_copy_scales(cuda):
    scales = torch.randn(2, 3, 9, 4, 3, device=cuda)
    want = scales.clone()
    src, dst = torch.tensor([0, 5, 8, -1, 3, 20], dtype=torch.int32), torch.tensor([1, 2, 4, 6, 9, 7], dtype=torch.int32)
    want[:, :, [1, 2, 4]] = scales[:, :, [0, 5, 8]]
    kernels.copy_kv_scales(scales, src.to(cuda), dst.to(cuda))
    assert torch.equal(scales, want)
    kernels.copy_kv_scales(scales, src[:0].to(cuda), dst[:0].to(cuda))
    assert torch.equal(scales, want)


def test_budget_counts_the_scales():
    r = ModelRunner(block_size=256, max_num_seqs=1, device="cpu")
    plain = r.kv_block_bytes(3, 8, 128, CODE)
    assert r.kv_block_bytes(3, 8, 128, CODE, 64) == plain + 2 * 3 * 8 * 4 * 4
