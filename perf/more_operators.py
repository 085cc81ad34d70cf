"""Serving over a KV cache of e4m3 codes with a scale for each block of tokens and head: what is measured of it.

Kinds:

* ``append``   one layer's new keys and values into the paged cache: rotation (and, with ``norm``, the q/k RMS norm
               before it) of queries and keys, the blocks' scales, the codes
* ``decode``   one layer's attention of single tokens over that cache
* ``prefill``  one layer's causal attention of packed prompts behind cached tokens, keys and values in that cache

A block of ``unit`` tokens of a page and a head has one scale for its keys and one for its values, a power of two
where the append writes it: the smallest that the block's largest magnitude fits.  Lengths follow from the case alone
(``lens`` seeds them); the seed given to ``prepare`` makes the values and the pages.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
CODE = torch.float8_e4m3fn
HEADS_128 = ((32, 8), (64, 8), (16, 8), (16, 4), (8, 2))
HEADS_256 = ((16, 4), (16, 2), (8, 2))
ROPE_BASE = 1e6
EPS = 1e-6


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one user's next token: latency is all
        dict(name="append_one_user", kind="append", batch=1, lo=1, hi=1, pre_lo=777, pre_hi=777, hq=32, hkv=8, d=128,
             block=256, unit=64, dtype="bf16", norm=False, rot=128, lens=1),
        # a busy server's decode step, normed queries and keys of 256, a quarter of them rotated
        dict(name="append_batch_d256", kind="append", batch=128, lo=1, hi=1, pre_lo=0, pre_hi=8000, hq=16, hkv=4, d=256,
             block=256, unit=64, dtype="bf16", norm=True, rot=64, lens=2),
        # the next turns of a few chats, behind partly filled blocks
        dict(name="append_turns", kind="append", batch=6, lo=40, hi=400, pre_lo=1, pre_hi=5000, hq=16, hkv=8, d=128,
             block=64, unit=32, dtype="f16", norm=False, rot=128, lens=3),
        # as many prompt tokens as one step takes
        dict(name="append_prompts", kind="append", batch=8, lo=1700, hi=2048, pre_lo=0, pre_hi=0, hq=32, hkv=8, d=128,
             block=256, unit=64, dtype="bf16", norm=True, rot=128, lens=4),
        # one user's next token in a chat
        dict(name="decode_one_user", kind="decode", batch=1, lo=1, hi=1, pre_lo=3000, pre_hi=3000, hq=32, hkv=8, d=128,
             block=256, unit=64, dtype="bf16", lens=5),
        # a server's step
        dict(name="decode_batch", kind="decode", batch=64, lo=1, hi=1, pre_lo=1023, pre_hi=4095, hq=32, hkv=8, d=128,
             block=256, unit=64, dtype="bf16", lens=6),
        # few long contexts, 64 query heads
        dict(name="decode_long", kind="decode", batch=8, lo=1, hi=1, pre_lo=20000, pre_hi=32767, hq=64, hkv=8, d=128,
             block=256, unit=128, dtype="bf16", lens=7),
        # many users, some at their first token, small pages, heads of 256 in half precision
        dict(name="decode_ragged_d256", kind="decode", batch=96, lo=1, hi=1, pre_lo=0, pre_hi=5000, hq=16, hkv=2, d=256,
             block=64, unit=32, dtype="f16", lens=8),
        # one user's next turn
        dict(name="prefill_one_user", kind="prefill", batch=1, lo=48, hi=48, pre_lo=1500, pre_hi=1500, hq=32, hkv=8,
             d=128, block=256, unit=64, dtype="bf16", lens=9),
        # a few chats' next turns behind their histories
        dict(name="prefill_chats", kind="prefill", batch=6, lo=40, hi=400, pre_lo=2000, pre_hi=8192, hq=32, hkv=8, d=128,
             block=256, unit=64, dtype="bf16", lens=10),
        # prompts that share a cached beginning, heads of 256 in half precision
        dict(name="prefill_batch_d256", kind="prefill", batch=5, lo=300, hi=1500, pre_lo=256, pre_hi=1024, hq=16, hkv=4,
             d=256, block=64, unit=32, dtype="f16", lens=11),
        # the last chunk of a long document
        dict(name="prefill_long_chunk", kind="prefill", batch=1, lo=2048, hi=2048, pre_lo=14336, pre_hi=14336, hq=32,
             hkv=8, d=128, block=256, unit=256, dtype="bf16", lens=12),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most = [work(c) for c in listed()]
    most = {k: max(w[k] for w in most) for k in ("bytes", "flops")}
    while True:
        case = _draw(rng)
        w = work(case)
        if w["bytes"] <= most["bytes"] and w["flops"] <= most["flops"] and _plain_values(case) <= 1 << 30:
            return case


def _draw(rng):
    kind = rng.choice(("append", "decode", "prefill"))
    d = rng.choice((128, 128, 256))
    hq, hkv = rng.choice(HEADS_128 if d == 128 else HEADS_256)
    block = rng.choice((256, 256, 64, 32))
    case = dict(kind=kind, hq=hq, hkv=hkv, d=d, dtype=rng.choice(("bf16", "bf16", "f16")), block=block,
                unit=rng.choice([u for u in (32, 64, 128, 256) if block % u == 0]), lens=rng.randrange(1 << 30))
    spread = rng.uniform(0.1, 1.0)
    if kind == "append":
        hi, pre = rng.choice((1, _log(rng, 1, 2048))), rng.choice((0, _log(rng, 1, 8192)))
        return dict(case, batch=_log(rng, 1, 128 if hi == 1 else 8), lo=max(1, int(hi * spread)), hi=hi,
                    pre_lo=pre // 8, pre_hi=pre, norm=rng.random() < 0.5, rot=rng.choice((d, d // 2, 64)))
    if kind == "decode":
        pre = _log(rng, 16, 32768) - 1
        return dict(case, batch=_log(rng, 1, 128), lo=1, hi=1, pre_lo=int(pre * spread), pre_hi=pre)
    hi, pre = _log(rng, 2, 2048), _log(rng, 1, 14336)
    return dict(case, batch=_log(rng, 1, 8), lo=max(1, int(hi * spread)), hi=hi, pre_lo=(pre + 1) // 2, pre_hi=pre)


def _lengths(case):
    """(new tokens, cached tokens before them) of each sequence."""
    r = random.Random(case["lens"])
    batch = range(case["batch"])
    return [r.randint(case["lo"], case["hi"]) for _ in batch], [r.randint(case["pre_lo"], case["pre_hi"]) for _ in batch]


def work(case):
    new, pre = _lengths(case)
    rows, item = sum(new), 2
    q, kv = case["hq"] * case["d"] * item, case["hkv"] * case["d"]
    scales = 2 * 4 * case["hkv"]    # of a block
    if case["kind"] == "append":    # q, k read and written, v read, two codes written; a table row, position and slot
        blocks = sum((c + n - 1) // case["unit"] - c // case["unit"] + 1 for n, c in zip(new, pre))
        row = 2 * q + 3 * kv * item + 2 * kv + 4 * case["rot"] + 12
        return {"bytes": float(rows * row + blocks * scales), "flops": 0.0}
    have = [n + c for n, c in zip(new, pre)]
    pairs = sum(n * c + n * (n + 1) / 2 for n, c in zip(new, pre))
    read = sum(have) * 2 * kv + sum(-(-h // case["unit"]) for h in have) * scales
    return {"bytes": float(read + 2 * rows * q), "flops": 4.0 * case["hq"] * case["d"] * pairs}


CHUNK = 256    # rows of a prefill that the plain form takes together


def _plain_values(case):
    """Values of the plain form's largest tensor."""
    new, pre = _lengths(case)
    if case["kind"] == "append":
        return sum(new) * case["hq"] * case["d"]
    rows = min(CHUNK, max(new))
    keys = max(n + c for n, c in zip(new, pre))
    return sum(-(-n // rows) for n in new) * keys * max(case["hkv"] * case["d"], case["hq"] * rows)


# ------------------------------------------------------------------ inputs

def _power(amax):
    """The smallest power of two with ``amax <= 448 * it``, from 2^-60 to 2^60."""
    m, e = torch.frexp(amax)
    e = torch.where(amax > 0, e - 9 + (m > 0.875).to(e.dtype), -60).clamp(-60, 60)
    return torch.ldexp(torch.ones_like(amax), e)


def _codes(x):
    return x.clamp(-448, 448).to(CODE)


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEVICE)


def _values(gen, *shape):
    """Keys or values of tokens: some channels are larger than others, and some tokens."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    x *= torch.exp(0.5 * torch.randn(shape[-1], generator=gen, device=DEVICE))
    x *= torch.exp(0.5 * torch.randn(*shape[:-2], 1, 1, generator=gen, device=DEVICE))
    return x


def _cache(gen, pages, case):
    """Codes and scales of a pool whose every token is stored."""
    units = case["block"] // case["unit"]
    x = _values(gen, pages, units, case["unit"], case["hkv"], case["d"])
    scale = _power(x.abs().amax(dim=(2, 4)))
    codes = _codes(x / scale[:, :, None, :, None])
    return codes.view(pages, case["block"], case["hkv"], case["d"]), scale


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, block = DTYPES[case["dtype"]], case["block"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    new, pre = _lengths(case)
    total = sum(new)
    s = dict(case)
    s["q"] = torch.randn(total, hq, d, generator=gen, device=DEVICE).to(dtype)
    # an append's pool is the pages that it writes to, an attention's the pages that it reads
    first = [c // block if case["kind"] == "append" else 0 for c in pre]
    counts = [-(-(n + c) // block) - f for n, c, f in zip(new, pre, first)]
    pages = math.ceil(1.1 * sum(counts)) + 1
    perm = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    at = [sum(counts[:i]) for i in range(len(counts))]
    s["k_cache"], s["k_scale"] = _cache(gen, pages, case)
    s["v_cache"], s["v_scale"] = _cache(gen, pages, case)
    if case["kind"] == "append":
        s["k"], s["v"] = (_values(gen, total, hkv, d).to(dtype) for _ in range(2))
        s["positions"] = _ints([c + i for n, c in zip(new, pre) for i in range(n)], torch.int64)
        s["slots"] = _ints([perm[a + p // block - f] * block + p % block
                            for n, c, f, a in zip(new, pre, first, at) for p in range(c, c + n)])
        half = torch.arange(0, case["rot"], 2, dtype=torch.float64, device=DEVICE) / case["rot"]
        angle = torch.arange(max(n + c for n, c in zip(new, pre)), dtype=torch.float64, device=DEVICE)[:, None] / ROPE_BASE ** half
        s["cos_sin"] = torch.cat([angle.cos(), angle.sin()], 1).float()
        s["q_weight"] = s["k_weight"] = None
        if case["norm"]:
            s["q_weight"], s["k_weight"] = ((0.2 * torch.randn(d, generator=gen, device=DEVICE)).to(dtype) for _ in range(2))
        return s
    table = torch.full((len(counts), max(counts)), -1, dtype=torch.int32)
    for i, (a, c) in enumerate(zip(at, counts)):
        table[i, :c] = torch.tensor(perm[a:a + c])
    cu = lambda v: _ints([sum(v[:i]) for i in range(len(v) + 1)])    # noqa: E731
    have = [n + c for n, c in zip(new, pre)]
    s.update(block_table=table.to(DEVICE), cu_q=cu(new), cu_k=cu(have), have=_ints(have), max_q=max(new), max_k=max(have),
             total=total, scale=d ** -0.5)
    return s


# -------------------------------------------------------------- plain forms

def _plain_rows(x, weight, s):
    """Rows of queries or keys, normed and rotated, in float32."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt(x.square().mean(-1, keepdim=True) + EPS) * (1.0 + weight.float())
    half = s["rot"] // 2
    table = s["cos_sin"][s["positions"]][:, None]
    c, n = table[..., :half], table[..., half:]
    a, b = x[..., :half], x[..., half:2 * half]
    return torch.cat([a * c - b * n, b * c + a * n, x[..., 2 * half:]], -1)


def _plain_append_one(x, cache, scale, s):
    """Rows ``x [N, Hkv, D]`` into the cache, which is written: codes and scales."""
    unit, (hkv, d) = s["unit"], cache.shape[2:]
    slots = s["slots"].long()
    unit_of = torch.div(slots, unit, rounding_mode="floor")
    old = scale.view(-1, hkv)
    amax = torch.zeros_like(old).scatter_reduce_(0, unit_of[:, None].expand(-1, hkv), x.abs().amax(-1), "amax")
    first = slots.new_full((old.shape[0],), unit)    # place of the call's first token in a block
    first = first.scatter_reduce_(0, unit_of, slots % unit, "amin")[:, None]
    grown = torch.where(first == 0, _power(amax), torch.maximum(old, _power(amax)))
    grown = torch.where(first < unit, grown, old)
    codes = cache.view(-1, unit, hkv, d)
    before = (torch.arange(unit, device=DEVICE)[:, None] < first[:, None]) & (grown > old)[:, None]
    moved = _codes(codes.float() * (old / grown)[:, None, :, None])
    kept = torch.where(before[..., None], moved.view(torch.uint8), codes.view(torch.uint8)).view(-1, hkv, d)
    kept[slots] = _codes(x / grown[unit_of][..., None]).view(torch.uint8)
    cache.view(torch.uint8).copy_(kept.view(cache.shape))
    scale.copy_(grown.view(scale.shape))


def _plain_append(s):
    q, k = _plain_rows(s["q"], s["q_weight"], s), _plain_rows(s["k"], s["k_weight"], s)
    _plain_append_one(k, s["k_cache"], s["k_scale"], s)
    _plain_append_one(s["v"].float(), s["v_cache"], s["v_scale"], s)
    return q.to(s["q"].dtype), k.to(s["k"].dtype), s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]


def _gathered(cache, scale, pages):
    """The cached values of pages ``[nb, P]`` in float32: ``[nb, P * block, Hkv, D]``."""
    nb, (block, hkv, d) = pages.shape[0], cache.shape[1:]
    x = cache.view(torch.uint8)[pages].view(CODE).float().view(nb, -1, block // scale.shape[1], hkv, d)
    return (x * scale[pages].view(nb, -1, 1, hkv, 1)).view(nb, -1, hkv, d)


def _plain_attention(s):
    """The rows of every sequence in chunks of CHUNK, all at once."""
    cu_q, new = s["cu_q"].long(), s["cu_q"].long().diff()
    have = s["have"].long()
    chunk = min(CHUNK, s["max_q"])
    parts = torch.div(new + chunk - 1, chunk, rounding_mode="floor")
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEVICE), parts)      # sequence of each chunk
    first = torch.arange(len(seq), device=DEVICE) - (torch.cumsum(parts, 0) - parts)[seq]
    row = first[:, None] * chunk + torch.arange(chunk, device=DEVICE)                # rows within the sequence
    live = row < new[seq][:, None]
    pos = (have - new)[seq][:, None] + row
    pages = s["block_table"].long().clamp_min(0)[seq]
    k, v = _gathered(s["k_cache"], s["k_scale"], pages), _gathered(s["v_cache"], s["v_scale"], pages)
    nb, keys, hkv, d = k.shape
    hq = s["q"].shape[1]
    seen = torch.arange(keys, device=DEVICE) <= torch.where(live, pos, -1)[:, :, None]    # nb, R, S
    x = s["q"][(cu_q[seq][:, None] + row).clamp_max(s["total"] - 1)].float()
    x = x.view(nb, chunk, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(nb, hkv, -1, d)
    p = torch.matmul(x, k.permute(0, 2, 3, 1).contiguous()).view(nb, hkv, hq // hkv, chunk, keys) * s["scale"]
    p = p.masked_fill(~seen[:, None, None], -math.inf)
    top = p.amax(-1, keepdim=True)
    p = torch.exp(p - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.view(nb, hkv, -1, keys), v.permute(0, 2, 1, 3).contiguous()).view(nb, hkv, hq // hkv, chunk, d)
    o = o / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(nb, chunk, hq, d)[live].to(s["q"].dtype)


# ------------------------------------------------------------ one pass

def _own(s):
    from nano_qwen_amd import kernels
    if s["kind"] == "append":
        q, k = kernels.append_kvcache(s["k"], s["v"], s["k_cache"], s["v_cache"], s["slots"], s["k_scale"], s["v_scale"],
                                      query=s["q"], positions=s["positions"], cos_sin_cache=s["cos_sin"],
                                      rotary_dim=s["rot"], q_weight=s["q_weight"], k_weight=s["k_weight"], eps=EPS)
        return q, k, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    if s["kind"] == "decode":
        return kernels.paged_decode(s["q"], s["k_cache"], s["v_cache"], s["have"], s["block_table"], s["scale"],
                                    s["k_scale"], s["v_scale"])
    return kernels.varlen_prefill(s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["cu_k"], s["max_q"], s["max_k"],
                                  s["scale"], block_table=s["block_table"], k_scale=s["k_scale"], v_scale=s["v_scale"])


def run(state):
    if own:
        return _own(state)
    return _plain_append(state) if state["kind"] == "append" else _plain_attention(state)


# ------------------------------------------------------------------ in 64 bits

def _exact_rows(x, weight, s):
    x = x.double()
    if weight is not None:
        x = x / torch.sqrt((x * x).mean(-1, keepdim=True) + EPS) * (1.0 + weight.double())
    half = s["rot"] // 2
    cos, sin = s["cos_sin"][s["positions"]].double()[:, None].split(half, -1)
    z = x.clone()
    z[..., :half] = x[..., :half] * cos - x[..., half:2 * half] * sin
    z[..., half:2 * half] = x[..., half:2 * half] * cos + x[..., :half] * sin
    return z


def _exact_append(x, cache, scale, s):
    """Block by block, in the order of the slots."""
    unit, block = s["unit"], s["block"]
    slots = s["slots"].tolist()
    at = 0
    while at < len(slots):
        end = at + 1
        while end < len(slots) and slots[end] == slots[end - 1] + 1 and slots[end] % unit:
            end += 1
        page, off = divmod(slots[at], block)
        u, o = divmod(off, unit)
        lo = u * unit
        rows = x[at:end]
        amax = rows.abs().amax(dim=(0, 2)).cpu().tolist()
        need = torch.tensor([2.0 ** min(60, max(-60, math.ceil(math.log2(a / 448)) if a else -60)) for a in amax],
                            dtype=torch.float64, device=DEVICE)
        was = scale[page, u].double()
        now = need if o == 0 else torch.maximum(was, need)
        if o:
            old = cache[page, lo:lo + o].double()
            again = (old * (was / now)[:, None]).clamp(-448, 448).to(CODE)
            cache.view(torch.uint8)[page, lo:lo + o] = again.view(torch.uint8)
        cache.view(torch.uint8)[page, off:off + end - at] = (rows / now[:, None]).clamp(-448, 448).to(CODE).view(torch.uint8)
        scale[page, u] = now.float()
        at = end


def exact(case, seed):
    s = prepare(case, seed)
    if case["kind"] == "append":
        q, k = _exact_rows(s["q"], s["q_weight"], s), _exact_rows(s["k"], s["k_weight"], s)
        _exact_append(k, s["k_cache"], s["k_scale"], s)
        _exact_append(s["v"].double(), s["v_cache"], s["v_scale"], s)
        return q, k, s["k_cache"], s["v_cache"], s["k_scale"], s["v_scale"]
    new, pre = _lengths(case)
    hq, hkv, unit, block = case["hq"], case["hkv"], case["unit"], case["block"]
    out, q0 = [], 0
    for b, (n, c) in enumerate(zip(new, pre)):
        have = n + c
        pages = s["block_table"][b, :-(-have // block)].long()
        k, v = (cache.view(torch.uint8)[pages].view(CODE).double() * scale[pages].double().repeat_interleave(unit, 1)[..., None]
                for cache, scale in ((s["k_cache"], s["k_scale"]), (s["v_cache"], s["v_scale"])))
        k, v = k.flatten(0, 1)[:have], v.flatten(0, 1)[:have]
        for lo in range(0, n, 512):
            hi = min(n, lo + 512)
            hidden = torch.arange(have, device=DEVICE) > c + torch.arange(lo, hi, device=DEVICE)[:, None]
            heads = []
            for h in range(hq):
                t = s["q"][q0 + lo:q0 + hi, h].double() @ k[:, h * hkv // hq].T * s["scale"]
                t = t.masked_fill(hidden, -math.inf)
                e = torch.exp(t - t.amax(1, keepdim=True))
                heads.append(e @ v[:, h * hkv // hq] / e.sum(1, keepdim=True))
            out.append(torch.stack(heads, 1))
        q0 += n
    return torch.cat(out)
