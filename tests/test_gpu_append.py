"""Appends to a cache with a scale for each block of tokens and head, on the GPU, against float64 value by value."""
import numpy as np
import pytest
import torch

from nano_qwen_amd import kernels
from oracle import block_scales as o
from oracle.fp8 import decode_e4m3fn

pytestmark = pytest.mark.gpu

BF, HF, CODE = torch.bfloat16, torch.float16, torch.float8_e4m3fn
EPS = 1e-6


def slots_of(new, pre, block, seed=0, skip=()):
    """(slots, positions, pages of the pool) of sequences in pages of their own; sequences in ``skip`` are not stored."""
    perm = np.random.default_rng(seed).permutation(sum(-(-(n + c) // block) for n, c in zip(new, pre)) + 2)
    at, slots, pos = 0, [], []
    for i, (n, c) in enumerate(zip(new, pre)):
        for p in range(c, c + n):
            slots.append(-1 if i in skip else int(perm[at + p // block]) * block + p % block)
            pos.append(p)
        at += -(-(n + c) // block)
    return np.array(slots, dtype=np.int64), np.array(pos, dtype=np.int64), len(perm)


def one_nan(codes):
    """Codes with one for NaN, whose sign means nothing."""
    return np.where((codes & 0x7F) == 0x7F, np.uint8(0x7F), codes)


class Pool:
    """Random codes (NaN among them) and scales of K and V."""

    def __init__(self, pages, block, unit, hkv, d, seed, cuda):
        r = np.random.default_rng(seed)
        self.unit = unit
        self.codes = [one_nan(r.integers(0, 256, size=(pages * block, hkv, d)).astype(np.uint8)) for _ in range(2)]
        self.scales = [(2.0 ** r.integers(-9, 2, size=(pages * block // unit, hkv))).astype(np.float32) for _ in range(2)]
        self.cache = [torch.from_numpy(c).to(cuda).view(CODE).view(pages, block, hkv, d) for c in self.codes]
        self.scale = [torch.from_numpy(s).to(cuda).view(pages, block // unit, hkv) for s in self.scales]

    def now(self):
        return ([one_nan(c.view(torch.uint8).cpu().numpy().reshape(self.codes[0].shape)) for c in self.cache],
                [s.cpu().numpy().reshape(self.scales[0].shape) for s in self.scale])


def fp32_off(x, weight, rot, z):
    """What fp32 may be off in a transformed row.  Norm: the sum of at most 256 squares in 8 + 5 or fewer steps, the
    root, the division and two products, 2^-24 each: under 20 * 2^-24 of a value.  Rotation: two products and a sum of
    normed values, each at most as large as the two magnitudes.  In all under 2^-19 of their sum."""
    y = np.abs(o.transform(x, weight[0], weight[1], EPS)) if weight is not None else np.abs(np.asarray(x, np.float64))
    m = y.copy()
    if rot:
        h = rot // 2
        m[..., :h] += y[..., h:rot]
        m[..., h:rot] += y[..., :h]
    return np.where(np.isnan(z), 0.0, m * 2.0 ** -19 if (rot or weight is not None) else 0.0)


def check_rows(out, z, off, dtype):
    got = out.double().cpu().numpy()
    nan = np.isnan(z)
    assert np.array_equal(nan, np.isnan(got))
    u = torch.finfo(dtype).eps / 2
    tol = np.maximum(u * (np.abs(z) + off), 2.0 ** -25 if dtype == HF else 0.0) + off    # fp16: subnormals
    with np.errstate(invalid="ignore"):
        same = got == z    # infinities
        assert (same | nan | (np.abs(got - z) <= tol)).all()


def check_cache(got, pool, which, z, off, slots):
    """Codes and scales between those of z - off and of z + off; what is not appended to, bit for bit."""
    codes, scales = got[0][which], got[1][which]
    unit = pool.unit
    mag = np.abs(z)
    sign = np.where(np.signbit(z), -1.0, 1.0)
    lo, hi = sign * np.maximum(mag - off, 0.0), sign * (mag + off)
    (c_lo, s_lo), (c_hi, s_hi) = (o.append(x, pool.codes[which], pool.scales[which], slots, unit) for x in (lo, hi))
    c_lo, c_hi = one_nan(c_lo), one_nan(c_hi)
    assert ((scales >= s_lo) & (scales <= s_hi)).all()
    assert (np.log2(scales) == np.round(np.log2(scales))).all()
    sure = np.repeat((s_lo == s_hi), unit, 0)[:, :, None]    # blocks whose scale is certain: nearly all
    assert sure.mean() > 0.99
    a, b = (np.where(x & 0x80, -(x & 0x7F).astype(int), (x & 0x7F).astype(int)) for x in (c_lo, c_hi))
    g = np.where(codes & 0x80, -(codes & 0x7F).astype(int), (codes & 0x7F).astype(int))
    ok = (g >= np.minimum(a, b)) & (g <= np.maximum(a, b))
    assert (ok | ~np.broadcast_to(sure, ok.shape)).all(), f"{(~ok & sure).sum()} codes"
    same = c_lo == c_hi
    assert (codes == c_lo)[same & np.broadcast_to(sure, ok.shape)].mean() > 0.999 or off.max() > 0


def run(cuda, new, pre, hq, hkv, d, dtype, block, unit, rot=0, norm=False, seed=0, skip=(), scale=1.0, values=None, query=True,
        strided=False, max_pos=None):
    r = np.random.default_rng(seed)
    slots, pos, pages = slots_of(new, pre, block, seed, skip)
    n = len(slots)
    pool = Pool(pages, block, unit, hkv, d, seed + 1, cuda)
    mk = lambda heads: torch.from_numpy((r.normal(size=(n, heads, d)) * scale * 2.0 ** r.integers(-2, 3, size=(n, 1, 1)))    # noqa: E731
                                        .astype(np.float32)).to(dtype)
    q, k, v = mk(hq), mk(hkv), mk(hkv)
    if values is not None:
        values(k, v)
    table = r.normal(size=(max_pos or int(pos.max(initial=0)) + 1, rot or 16)).astype(np.float32)
    w = [torch.from_numpy(0.3 * r.normal(size=d)).to(dtype) for _ in range(2)] if norm else [None, None]
    dev = lambda t: None if t is None else t.to(cuda)    # noqa: E731
    qd, kd, vd = dev(q), dev(k), dev(v)
    if strided:    # the query half of a wider projection, keys and values of one
        wide = torch.full((n, hq, 2 * d), float("nan"), dtype=dtype, device=cuda)
        wide[:, :, :d] = qd
        qd = wide[:, :, :d]
        kv = torch.cat([kd.reshape(n, -1), vd.reshape(n, -1)], 1)
        kd, vd = kv[:, :hkv * d].view(n, hkv, d), kv[:, hkv * d:].view(n, hkv, d)
    q_out, k_out = kernels.append_kvcache(
        kd, vd, *pool.cache, torch.from_numpy(slots).int().to(cuda), *pool.scale, query=qd if query else None,
        positions=torch.from_numpy(pos).to(cuda) if rot else None,
        cos_sin_cache=torch.from_numpy(table).to(cuda) if rot else None, rotary_dim=rot, q_weight=dev(w[0]),
        k_weight=dev(w[1]), eps=EPS)
    got = pool.now()
    args = lambda i: dict(weight=None if w[i] is None else w[i].double().numpy(), eps=EPS, cos_sin=table, positions=pos, rot=rot)    # noqa: E731
    zq, zk, zv = (o.transform(q.double().numpy(), **args(0)), o.transform(k.double().numpy(), **args(1)), v.double().numpy())
    pair = lambda i: None if w[i] is None else (w[i].double().numpy(), 1.0)    # noqa: E731
    off = fp32_off(k.double().numpy(), pair(1), rot, zk)
    if query:
        check_rows(q_out, zq, fp32_off(q.double().numpy(), pair(0), rot, zq), dtype)
    else:
        assert q_out is None
    check_rows(k_out, zk, off, dtype)
    check_cache(got, pool, 0, zk, off, slots)
    check_cache(got, pool, 1, zv, np.zeros_like(zv), slots)
    return pool, got


STEPS = [([1], [0]), ([1], [777]), ([1] * 9, [0, 1, 31, 32, 63, 64, 255, 256, 300]), ([5], [3]), ([70, 1, 33, 300], [0, 31, 32, 250])]


@pytest.mark.parametrize("new,pre", STEPS)
@pytest.mark.parametrize("block,unit", [(256, 64), (64, 32), (256, 256), (32, 32), (96, 32), (128, 128)])
def test_append(cuda, new, pre, block, unit):
    run(cuda, new, pre, 8, 2, 128, BF, block, unit, rot=128, seed=block + unit)


@pytest.mark.parametrize("hq,hkv,d,dtype,rot,norm", [
    (4, 4, 128, HF, 0, False), (16, 1, 128, BF, 64, True), (10, 2, 256, BF, 64, True), (3, 3, 256, HF, 256, False),
    (7, 1, 128, HF, 16, True), (32, 8, 128, BF, 128, True), (24, 2, 256, HF, 0, True), (1, 1, 256, BF, 128, False)])
@pytest.mark.parametrize("unit", [32, 256])
def test_heads_types_and_rotations(cuda, hq, hkv, d, dtype, rot, norm, unit):
    run(cuda, [40, 1, 257], [13, 99, 700], hq, hkv, d, dtype, 256, unit, rot=rot, norm=norm, seed=hq, strided=True)


@pytest.mark.parametrize("unit", [32, 64, 128, 256])
def test_many_rows(cuda, unit):
    """Several rows to a workgroup of runs, single ones and long ones among them."""
    r = np.random.default_rng(unit)
    new = [int(x) for x in r.choice([1, 1, 2, 17, 64, 300], size=60)]
    pre = [int(x) for x in r.integers(0, 400, size=60)]
    run(cuda, new, pre, 2, 1, 128, BF, 256, unit, rot=32, seed=unit)


def test_many_single_rows(cuda):
    run(cuda, [1] * 1500, [int(x) for x in np.random.default_rng(5).integers(0, 64, size=1500)], 1, 1, 128, HF, 64, 32)


def test_rows_that_are_not_stored(cuda):
    """Padding rows of a batch, and sequences outside the pool, are transformed and not stored."""
    run(cuda, [1, 1, 1], [5, 9, 40], 4, 2, 128, BF, 64, 32, rot=128, skip=(1,))
    run(cuda, [50, 40], [0, 10], 4, 2, 128, BF, 64, 32, rot=128, skip=(0, 1))


def test_positions_outside_the_table_are_nan(cuda):
    run(cuda, [3, 1], [38, 20], 4, 2, 128, BF, 64, 32, rot=128, max_pos=39)


def test_without_a_query(cuda):
    run(cuda, [33, 1], [0, 50], 1, 2, 128, BF, 64, 32, query=False)


@pytest.mark.parametrize("dtype", [BF, HF])
def test_zeros_and_values_that_are_not_finite(cuda, dtype):
    def values(k, v):
        k[0], v[1] = 0.0, 0.0
        for t in (k, v):
            t[2, 0, 3], t[2, 1, 5], t[3, 0, 0], t[5] = float("inf"), float("-inf"), float("nan"), float("nan")
    run(cuda, [6, 2], [30, 0], 2, 2, 128, dtype, 64, 32, values=values)


@pytest.mark.parametrize("scale", [1e-30, 1e30, 2.0 ** -60, 1e-12])
def test_scales_at_their_ends(cuda, scale):
    run(cuda, [5, 40], [30, 0], 2, 2, 128, BF, 64, 32, scale=scale)


def test_growth_step_by_step(cuda):
    """A decode of 70 tokens whose magnitudes rise and fall: every step against the oracle."""
    r = np.random.default_rng(1)
    pool = Pool(3, 64, 32, 2, 128, 2, cuda)
    for t in range(70):
        k, v = (torch.from_numpy(r.normal(size=(1, 2, 128)) * 2.0 ** r.integers(-8, 9)).to(BF) for _ in range(2))
        slot = np.array([64 + t])
        want = [o.append(x.double().numpy(), c, s, slot, 32) for x, c, s in zip((k, v), pool.codes, pool.scales)]
        kernels.append_kvcache(k.to(cuda), v.to(cuda), *pool.cache, torch.tensor(slot, dtype=torch.int32, device=cuda), *pool.scale)
        codes, scales = pool.now()
        for i in range(2):
            assert np.array_equal(scales[i], want[i][1]) and np.array_equal(codes[i], one_nan(want[i][0])), (t, i)
        pool.codes, pool.scales = codes, scales


def test_given_outputs_and_no_rows(cuda):
    pool = Pool(2, 64, 32, 2, 128, 2, cuda)
    q, k, v = (torch.randn(3, h, 128, device=cuda).to(BF) for h in (4, 2, 2))
    slots = torch.tensor([0, 1, 2], dtype=torch.int32, device=cuda)
    pos, table = torch.tensor([0, 1, 2], device=cuda), torch.randn(3, 128, device=cuda)
    kw = dict(query=q, positions=pos, cos_sin_cache=table, rotary_dim=128)
    a = kernels.append_kvcache(k, v, *pool.cache, slots, *pool.scale, **kw)
    qo = torch.full((3, 4, 256), 7.0, dtype=BF, device=cuda)
    ko = torch.empty_like(k)
    b = kernels.append_kvcache(k, v, *pool.cache, slots, *pool.scale, **kw, q_out=qo[:, :, :128], k_out=ko)
    assert b[1] is ko and torch.equal(a[0], qo[:, :, :128]) and torch.equal(a[1], ko) and (qo[:, :, 128:] == 7).all()
    c = kernels.append_kvcache(k, v, *pool.cache, slots, *pool.scale, **kw | dict(query=q.clone()), q_out=q)    # in place
    assert c[0] is q and torch.equal(a[0], q)
    before = pool.now()
    kernels.append_kvcache(k[:0], v[:0], *pool.cache, slots[:0], *pool.scale, **kw | dict(query=q[:0], positions=pos[:0]))
    after = pool.now()
    assert all(np.array_equal(x, y) for s, t in zip(before, after) for x, y in zip(s, t))


def test_graph_and_streams(cuda):
    """A captured append replays on what its inputs hold then; appends of two streams to their own blocks."""
    pool = Pool(4, 64, 32, 2, 128, 3, cuda)
    k, v = (torch.randn(2, 2, 128, device=cuda).to(BF) for _ in range(2))
    slots = torch.tensor([0, 64], dtype=torch.int32, device=cuda)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        kernels.append_kvcache(k, v, *pool.cache, slots, *pool.scale)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kernels.append_kvcache(k, v, *pool.cache, slots, *pool.scale)
    for t in range(1, 40):
        x = [torch.randn(2, 2, 128, device=cuda).to(BF) * 2.0 ** (t % 7) for _ in range(2)]
        k.copy_(x[0])
        v.copy_(x[1])
        slots.copy_(torch.tensor([t, 64 + t], device=cuda))
        was, scale = pool.now()
        graph.replay()
        torch.cuda.synchronize()
        codes, scales = pool.now()
        for i in range(2):
            want = o.append(x[i].double().cpu().numpy(), was[i], scale[i], slots.cpu().numpy(), 32)
            assert np.array_equal(codes[i], one_nan(want[0])) and np.array_equal(scales[i], want[1]), (t, i)


def refusals(dev):
    """Calls that are refused, each with its arguments."""
    g = torch.Generator().manual_seed(0)
    cache = lambda **kw: torch.zeros(3, 64, 2, 128, dtype=kw.get("dtype", torch.uint8)).to(dev)    # noqa: E731
    good = dict(key=torch.randn(4, 2, 128, generator=g).to(BF), value=torch.randn(4, 2, 128, generator=g).to(BF),
                k_cache=cache().view(CODE), v_cache=cache().view(CODE), slot_mapping=torch.arange(4, dtype=torch.int32),
                k_scale=torch.ones(3, 2, 2), v_scale=torch.ones(3, 2, 2), query=torch.randn(4, 6, 128, generator=g).to(BF),
                positions=torch.arange(4), cos_sin_cache=torch.randn(4, 128, generator=g), rotary_dim=128)
    good = {n: t.to(dev) if isinstance(t, torch.Tensor) else t for n, t in good.items()}
    q, k = good["query"], good["key"]
    w = torch.ones(128, dtype=BF, device=dev)
    bad = [dict(key=k.float()), dict(key=k[:, :, ::2]), dict(value=good["value"][:3]), dict(value=good["value"].half()),
           dict(key=k[0]), dict(k_cache=cache(dtype=BF), v_cache=cache(dtype=BF)), dict(v_cache=cache(dtype=BF)),
           dict(k_cache=good["k_cache"][:2]), dict(slot_mapping=good["slot_mapping"].long()),
           dict(slot_mapping=good["slot_mapping"][:3]), dict(k_scale=torch.ones(2, device=dev)),
           dict(k_scale=torch.ones(3, 2, 2, device=dev).double()), dict(k_scale=torch.ones(3, 2, 3, device=dev)),
           dict(k_scale=torch.ones(3, 4, 2, device=dev), v_scale=torch.ones(3, 4, 2, device=dev)),    # blocks of 16
           dict(k_scale=torch.ones(3, 3, 2, device=dev), v_scale=torch.ones(3, 3, 2, device=dev)),
           dict(k_scale=torch.ones(3, 2, 4, device=dev)[:, :, ::2]), dict(v_scale=None), dict(positions=None),
           dict(positions=good["positions"].int()), dict(cos_sin_cache=None), dict(cos_sin_cache=good["cos_sin_cache"][:, :64]),
           dict(rotary_dim=136, cos_sin_cache=torch.ones(4, 136, device=dev)),
           dict(rotary_dim=8, cos_sin_cache=torch.ones(4, 8, device=dev)), dict(q_weight=w), dict(q_weight=w, k_weight=w[:64]),
           dict(q_weight=w, k_weight=w.half()), dict(query=q.half()), dict(query=q[:3]), dict(q_out=torch.empty_like(q)[:3]),
           dict(query=None, q_out=q), dict(rotary_dim=0, k_out=torch.empty_like(k)), dict(k_out=k), dict(k_out=k[:, :1]),
           dict(rotary_dim=-16)]
    return good, bad


def test_refusals(cuda):
    good, bad = refusals(cuda)
    kernels.append_kvcache(**good)
    for kw in bad:
        with pytest.raises(RuntimeError):
            kernels.append_kvcache(**(good | kw))
    with pytest.raises(RuntimeError):
        kernels.append_kvcache(**(good | dict(slot_mapping=good["slot_mapping"].cpu())))
