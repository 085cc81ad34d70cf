"""Speculative and windowed serving over the paged KV cache: what is measured of it.

Kinds:

* ``tree``     one layer's attention for trees of drafted tokens over the paged cache
* ``wdecode``  one layer's decode step with a sliding window and sinks; with ``store``
               the new token's store too, else the q/k norm's launch has stored it
* ``wprefill`` one layer's prefill with a sliding window and sinks, over packed K/V, or
               over the paged cache when a prefix is cached
* ``copy``     copies of cache pages in all layers (forks, compaction of the pool)
* ``commit``   the end of a verification step: the accepted path of every tree and its
               K/V rows moved into place in all layers

Lengths follow from the case alone (``lens`` seeds them); the seed given to ``prepare``
makes the values, the block permutation and the trees.
"""
import math
import random

import torch

own = False

DEVICE = "cuda"
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
VOCAB = 32000
HEADS_128 = ((32, 8), (64, 8), (16, 8), (16, 4), (8, 2))
HEADS_256 = ((16, 4), (16, 2), (8, 2))


# ------------------------------------------------------------------- cases

def listed():
    return [
        # one user's chat with a small static tree: latency is all
        dict(name="tree_one_user", kind="tree", batch=1, lo=777, hi=777, n_lo=8, n_hi=8, hq=32, hkv=8, d=128,
             block=256, dtype="bf16", kv="same", lens=1),
        # a server's verification step, ragged trees of about 26 nodes
        dict(name="tree_batch", kind="tree", batch=16, lo=1024, hi=4096, n_lo=16, n_hi=32, hq=32, hkv=8, d=128,
             block=256, dtype="bf16", kv="same", lens=2),
        # long contexts held as fp8, full trees, 64 query heads
        dict(name="tree_long_fp8", kind="tree", batch=4, lo=16000, hi=32768, n_lo=60, n_hi=64, hq=64, hkv=8, d=128,
             block=256, dtype="bf16", kv="fp8", lens=3),
        # one user's windowed layer deep into a long chat
        dict(name="wdecode_one_user", kind="wdecode", batch=1, lo=9001, hi=9001, window=1024, sinks=4, hq=16, hkv=4,
             d=256, block=256, dtype="bf16", kv="same", store=True, lens=4),
        # a busy server's windowed layer, some contexts shorter than the window
        dict(name="wdecode_batch", kind="wdecode", batch=96, lo=500, hi=20000, window=4096, sinks=4, hq=32, hkv=8,
             d=128, block=256, dtype="bf16", kv="same", store=False, lens=5),
        # the next turns of a few long chats, their histories held as fp8
        dict(name="wprefill_chat_fp8", kind="wprefill", batch=4, lo=40, hi=400, pre_lo=4000, pre_hi=8192, window=1024,
             sinks=4, hq=32, hkv=8, d=128, block=256, dtype="bf16", kv="fp8", lens=6),
        # an ordinary batch of prompts at head_dim 256, half precision
        dict(name="wprefill_batch_d256", kind="wprefill", batch=6, lo=200, hi=2567, pre_lo=0, pre_hi=0, window=512,
             sinks=1, hq=16, hkv=4, d=256, block=256, dtype="f16", kv="same", lens=7),
        # two long documents, as many tokens as one prefill step takes
        dict(name="wprefill_long", kind="wprefill", batch=2, lo=7900, hi=8192, pre_lo=0, pre_hi=0, window=2048, sinks=4,
             hq=32, hkv=8, d=128, block=256, dtype="bf16", kv="same", lens=8),
        # two continuations forked from one prompt: their last, partly filled pages
        dict(name="copy_fork", kind="copy", pairs=2, partial=True, layers=16, hkv=8, d=128, block=256, dtype="bf16",
             lens=9),
        # a pool compacted: whole pages moved
        dict(name="copy_pool", kind="copy", pairs=48, partial=False, layers=16, hkv=8, d=128, block=256, dtype="bf16",
             lens=10),
        # one user's step: a few rows in every layer
        dict(name="commit_one_user", kind="commit", batch=1, lo=300, hi=300, n_lo=8, n_hi=8, layers=16, hkv=8, d=128,
             block=256, dtype="bf16", lens=11),
        # a server's step
        dict(name="commit_batch", kind="commit", batch=64, lo=64, hi=500, n_lo=16, n_hi=64, layers=16, hkv=8, d=128,
             block=256, dtype="bf16", lens=12),
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
    kind = rng.choice(("tree", "tree", "wdecode", "wdecode", "wprefill", "wprefill", "copy", "commit"))
    dtype = rng.choice(("bf16", "bf16", "f16"))
    d = rng.choice((128, 128, 256))
    hq, hkv = rng.choice(HEADS_128 if d == 128 else HEADS_256)
    base = dict(kind=kind, hq=hq, hkv=hkv, d=d, dtype=dtype, block=rng.choice((256, 256, 64, 32)),
                lens=rng.randrange(1 << 30))
    spread = rng.uniform(0.1, 1.0)
    if kind == "tree":
        hi, n_hi = _log(rng, 16, 32768), _log(rng, 1, 64)
        return dict(base, batch=_log(rng, 1, 32), lo=max(1, int(hi * spread)), hi=hi, n_lo=(n_hi + 1) // 2, n_hi=n_hi,
                    kv=rng.choice(("same", "fp8")))
    if kind == "wdecode":
        hi, kv = _log(rng, 16, 32768), rng.choice(("same", "same", "fp8"))
        return dict(base, batch=_log(rng, 1, 128), lo=max(1, int(hi * spread)), hi=hi, window=_log(rng, 16, 4096),
                    sinks=rng.choice((0, 1, 4, 33)), kv=kv, store=kv == "same" and rng.random() < 0.5)
    if kind == "wprefill":
        hi, pre = _log(rng, 8, 8192), rng.choice((0, 0, _log(rng, 1, 8192)))
        return dict(base, batch=_log(rng, 1, 16), lo=max(1, int(hi * spread)), hi=hi, pre_lo=(pre + 1) // 2, pre_hi=pre,
                    window=_log(rng, 16, 4096), sinks=rng.choice((0, 1, 4, 33)),
                    kv=rng.choice(("same", "fp8")) if pre else "same")
    base.pop("hq")
    base["layers"] = rng.choice((4, 8, 16))
    if kind == "copy":
        return dict(base, pairs=_log(rng, 1, 48), partial=rng.random() < 0.5)
    hi, n_hi = _log(rng, 16, 500), _log(rng, 1, 64)
    return dict(base, batch=_log(rng, 1, 64), lo=max(1, int(hi * spread)), hi=hi, n_lo=(n_hi + 1) // 2, n_hi=n_hi)


def _lengths(case):
    """(new rows, cached tokens before them) of each sequence."""
    r = random.Random(case["lens"])
    batch = range(case["batch"])
    if case["kind"] == "wprefill":
        new = [r.randint(case["lo"], case["hi"]) for _ in batch]
        return new, [r.randint(case["pre_lo"], case["pre_hi"]) if case["pre_hi"] else 0 for _ in batch]
    if case["kind"] == "wdecode":
        return [1] * case["batch"], [r.randint(case["lo"], case["hi"]) - 1 for _ in batch]
    return [r.randint(case["n_lo"], case["n_hi"]) for _ in batch], [r.randint(case["lo"], case["hi"]) for _ in batch]


def _copied(case):
    r = random.Random(case["lens"])
    return [r.randint(1, case["block"]) if case["partial"] else case["block"] for _ in range(case["pairs"])]


def _seen(case, new, pre):
    """(visible pairs, keys that some row sees) of a windowed sequence."""
    w, s = case["window"], case["sinks"]
    pairs = 0
    for p in (range(pre, pre + new) if new < 64 else (pre, pre + new // 4, pre + new // 2, pre + 3 * new // 4)):
        first = max(0, p - w + 1)
        pairs += p + 1 - first + min(s, first)
    first = max(0, pre - w + 1)
    return pairs if new < 64 else pairs * new // 4, pre + new - first + min(s, first)


def work(case):
    kind, item = case["kind"], 2
    row = case["hkv"] * case["d"] * item
    if kind == "copy":
        return {"bytes": 4.0 * case["layers"] * row * sum(_copied(case)), "flops": 0.0}
    new, pre = _lengths(case)
    if kind == "commit":    # about three nodes of a tree are accepted; the root stays where it is
        moved = sum(min(2, n - 1) for n in new) + 0.25
        return {"bytes": 4.0 * case["layers"] * row * moved + 28.0 * sum(new), "flops": 0.0}
    kv_row = 2 * case["hkv"] * case["d"] * (1 if case["kv"] == "fp8" else item)
    qo = 2 * case["hq"] * case["d"] * item
    if kind == "tree":
        pairs, keys = sum(n * (c + n / 4) for n, c in zip(new, pre)), sum(new) + sum(pre)
    else:
        seen = [_seen(case, n, c) for n, c in zip(new, pre)]
        pairs, keys = sum(p for p, _ in seen), sum(k for _, k in seen)
    store = 4 * row if case.get("store") else 0    # the new token: read, and written to the cache
    return {"bytes": float(keys * kv_row + sum(new) * (qo + store)), "flops": 4.0 * case["hq"] * case["d"] * pairs}


CHUNK = 256    # rows of a prefill that the plain form takes together


def _plain_values(case):
    """Values of the plain form's largest tensor."""
    if case["kind"] in ("copy", "commit"):
        return 0
    new, pre = _lengths(case)
    rows = min(CHUNK, max(new))
    keys = max(n + c for n, c in zip(new, pre))
    if case["kind"] != "tree":
        keys = min(keys, case["window"] + case["sinks"] + rows)
    blocks = sum(-(-n // rows) for n in new)
    return blocks * keys * max(case["hkv"] * case["d"], case["hq"] * rows)


# ------------------------------------------------------------------ inputs

def _randn(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device=DEVICE, dtype=torch.float32).to(dtype)


def _tables(counts, pool, seed):
    perm = torch.randperm(pool, generator=torch.Generator().manual_seed(seed)).to(torch.int32)
    tables = torch.full((len(counts), max(counts)), -1, dtype=torch.int32)
    at = 0
    for i, c in enumerate(counts):
        tables[i, :c] = perm[at:at + c]
        at += c
    return tables


def _tree(r, n):
    """Parents of a tree's nodes (node 0: the root, the last sampled token): breadth first
    with more children near the root, as drafters make them."""
    return [-1] + [min(i - 1, int((i - 1) * r.random() ** 1.5)) for i in range(1, n)]


def _words(parents, words):
    """Ancestors of each node, itself among them, as 64-bit words."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((1 << i) | (rows[p] if p >= 0 else 0))
    signed = [[(m >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for m in rows]
    return [[x - 2 ** 64 if x >= 2 ** 63 else x for x in row] for row in signed]


def _ints(x, dtype=torch.int32):
    return torch.tensor(x, dtype=dtype, device=DEVICE)


def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype, block = DTYPES[case["dtype"]], case["block"]
    s = dict(case)
    if case["kind"] == "copy":
        n = case["pairs"]
        blocks = 2 * n + 2
        s["kv_cache"] = torch.empty(2, case["layers"], blocks, block, case["hkv"], case["d"], dtype=dtype,
                                    device=DEVICE).normal_(generator=gen)
        perm = torch.randperm(blocks, generator=torch.Generator().manual_seed(seed)).to(torch.int32).to(DEVICE)
        s["src"], s["dst"] = perm[:n].contiguous(), perm[n:2 * n].contiguous()
        s["tokens"] = _ints(_copied(case)) if case["partial"] else None
        return s
    new, pre = _lengths(case)
    r = random.Random(seed)
    counts = [-(-(n + c) // block) for n, c in zip(new, pre)]
    blocks = math.ceil(1.1 * sum(counts)) + 1
    tables = _tables(counts, blocks, seed)
    cu = lambda v: _ints([sum(v[:i]) for i in range(len(v) + 1)])    # noqa: E731
    s.update(block_table=tables.to(DEVICE), cu_q=cu(new), cu_k=cu([n + c for n, c in zip(new, pre)]), max_q=max(new),
             max_k=max(n + c for n, c in zip(new, pre)), total=sum(new))
    if case["kind"] in ("tree", "commit"):
        trees = [_tree(r, n) for n in new]
        words = -(-max(new) // 64)
        s["mask"] = _ints([row for t in trees for row in _words(t, words)], torch.int64)
    if case["kind"] == "commit":
        s["kv_cache"] = torch.empty(2, case["layers"], blocks, block, case["hkv"], case["d"], dtype=dtype,
                                    device=DEVICE).normal_(generator=gen)
        tokens, targets = [], []
        for t in trees:    # seven of ten nodes' targets are the token of one of their children, if they have any
            own_tokens = [r.randrange(VOCAB) for _ in t]
            for i in range(len(t)):
                children = [j for j, p in enumerate(t) if p == i]
                targets.append(own_tokens[r.choice(children)] if children and r.random() < 0.7 else r.randrange(VOCAB))
            tokens += own_tokens
        s.update(parents=_ints([p for t in trees for p in t]), tokens=_ints(tokens, torch.int64),
                 targets=_ints(targets, torch.int64))
        return s
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    s["scale"] = d ** -0.5
    s["q"] = _randn(gen, s["total"], hq, d, dtype=dtype)
    s["k_scale"] = s["v_scale"] = None
    if case["kind"] == "wprefill" and not case["pre_hi"]:    # no prefix: the new keys and values, packed
        s["k"], s["v"] = (_randn(gen, s["total"], hkv, d, dtype=dtype) for _ in range(2))
        s["block_table"] = None
        return s
    caches = [_randn(gen, blocks, block, hkv, d, dtype=dtype) for _ in range(2)]
    if case["kv"] == "fp8":
        scales = [c.float().abs().amax(dim=(0, 1, 3)) / 448.0 for c in caches]
        caches = [(c.float() / t[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn) for c, t in zip(caches, scales)]
        s["k_scale"], s["v_scale"] = scales
    s["k_cache"], s["v_cache"] = caches
    if case["kind"] == "wdecode":
        s["lens"] = _ints([c + 1 for c in pre])
        s["k_new"] = s["v_new"] = s["slots"] = None
        if case["store"]:
            s["slots"] = _ints([int(tables[i, c // block]) * block + c % block for i, c in enumerate(pre)])
            s["k_new"], s["v_new"] = (_randn(gen, case["batch"], hkv, d, dtype=dtype) for _ in range(2))
    return s


# -------------------------------------------------------------- plain forms

def _attend(q, kf, vf, rows, keys, visible, scale):
    """Rows ``q[rows] [nb, R]`` over the keys ``keys [nb, S]`` of the flat float32 K/V ``[n, Hkv, D]``, where
    ``visible [nb, R, S]``; rows that see nothing give zeros.  Returns ``[nb, R, Hq, D]`` float32."""
    nb, r = rows.shape
    hq, d = q.shape[1:]
    hkv = kf.shape[1]
    k = kf[keys].permute(0, 2, 3, 1).contiguous()                                    # nb, Hkv, D, S
    v = vf[keys].permute(0, 2, 1, 3).contiguous()                                    # nb, Hkv, S, D
    x = q[rows].float().reshape(nb, r, hkv, hq // hkv, d).permute(0, 2, 3, 1, 4).reshape(nb, hkv, -1, d)
    s = torch.matmul(x, k).reshape(nb, hkv, hq // hkv, r, -1) * scale
    s = s.masked_fill(~visible[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -math.inf, 0.0, top))
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p.reshape(nb, hkv, -1, p.shape[-1]), v).reshape(nb, hkv, hq // hkv, r, d)
    o = o / torch.where(total == 0, 1.0, total)
    return o.permute(0, 3, 1, 2, 4).reshape(nb, r, hq, d)


def _flat(cache, scale):
    x = cache.reshape(-1, *cache.shape[-2:]).float()
    return x if scale is None else x * scale[:, None]


def _slots_of(table, seq, pos, block):
    """Cache rows of positions ``pos`` of sequences ``seq`` (same shapes); 0 where there is none."""
    page = torch.div(pos, block, rounding_mode="floor").clamp(0, table.shape[1] - 1)
    return (table[seq, page].long() * block + pos % block).clamp_min(0)


def _spans(s):
    cu_q, cu_k = s["cu_q"].long(), s["cu_k"].long()
    new, have = cu_q.diff(), cu_k.diff()
    return cu_q, cu_k, new, have


def _plain_tree(s):
    cu_q, cu_k, new, have = _spans(s)
    seq = torch.arange(len(new), device=DEVICE)[:, None]
    node, pos = torch.arange(s["max_q"], device=DEVICE), torch.arange(s["max_k"], device=DEVICE)
    rows = (cu_q[:-1, None] + node).clamp_max(s["total"] - 1)
    at = pos - (have - new)[:, None]                                                 # node that a key belongs to
    bit = at.clamp(0, 64 * s["mask"].shape[1] - 1)
    words = s["mask"][rows[:, :, None], (bit // 64)[:, None, :]]                     # B, R, S
    sees = ((words >> (bit % 64)[:, None, :]) & 1).bool()
    visible = ((at < 0)[:, None] | (sees & (at < new[:, None])[:, None])) & (pos < have[:, None])[:, None]
    keys = _slots_of(s["block_table"], seq.expand(-1, len(pos)), pos.expand(len(new), -1), s["block"])
    o = _attend(s["q"], _flat(s["k_cache"], s["k_scale"]), _flat(s["v_cache"], s["v_scale"]), rows, keys, visible,
                s["scale"])
    return o[node < new[:, None]].to(s["q"].dtype)


def _plain_window(s, cu_q, new, have, kf, vf, key_rows):
    """Windowed attention, the rows of a sequence in chunks: ``key_rows(seq, pos)`` gives a key's row in kf, vf."""
    chunk = min(CHUNK, s["max_q"])
    parts = torch.div(new + chunk - 1, chunk, rounding_mode="floor")
    seq = torch.repeat_interleave(torch.arange(len(new), device=DEVICE), parts)      # sequence of each chunk
    first = torch.arange(len(seq), device=DEVICE) - (torch.cumsum(parts, 0) - parts)[seq]
    row = first[:, None] * chunk + torch.arange(chunk, device=DEVICE)                # rows within the sequence
    live = row < new[seq][:, None]
    q_pos = (have - new)[seq][:, None] + row
    w, sinks = s["window"], s["sinks"]
    low = (q_pos[:, :1] - w + 1).clamp_min(0)                                        # first key of a chunk's windows
    span = min(s["max_k"], w + chunk - 1)
    pos = torch.cat([torch.arange(sinks, device=DEVICE).expand(len(seq), -1), low + torch.arange(span, device=DEVICE)], 1)
    is_sink = torch.arange(sinks + span, device=DEVICE) < sinks
    seen = (pos[:, None] <= q_pos[:, :, None]) & (pos < have[seq][:, None])[:, None]
    near = pos[:, None] > q_pos[:, :, None] - w
    visible = seen & torch.where(is_sink, ~near, near)                               # each key once
    o = _attend(s["q"], kf, vf, (cu_q[seq][:, None] + row).clamp_max(s["q"].shape[0] - 1),
                key_rows(seq[:, None].expand_as(pos), pos), visible, s["scale"])
    return o[live].to(s["q"].dtype)


def _plain_wprefill(s):
    cu_q, cu_k, new, have = _spans(s)
    if s["block_table"] is None:
        rows = lambda seq, pos: (cu_k[seq] + pos).clamp_max(s["k"].shape[0] - 1)     # noqa: E731
        return _plain_window(s, cu_q, new, have, s["k"].float(), s["v"].float(), rows)
    rows = lambda seq, pos: _slots_of(s["block_table"], seq, pos, s["block"])        # noqa: E731
    return _plain_window(s, cu_q, new, have, _flat(s["k_cache"], s["k_scale"]), _flat(s["v_cache"], s["v_scale"]), rows)


def _rows_of(cache, scale, slots):
    """Cache rows in float32 (one-byte values are indexed as bytes)."""
    flat = cache.reshape(-1, *cache.shape[-2:])
    if scale is None:
        return flat[slots].float()
    return flat.view(torch.uint8)[slots].view(cache.dtype).float() * scale[:, None]


def _plain_wdecode(s):
    if s["slots"] is not None:
        s["k_cache"].view(-1, *s["k_new"].shape[1:])[s["slots"].long()] = s["k_new"]
        s["v_cache"].view(-1, *s["v_new"].shape[1:])[s["slots"].long()] = s["v_new"]
    have = s["lens"].long()
    keep = min(s["max_k"], s["window"] + s["sinks"])
    pos = torch.arange(keep, device=DEVICE)
    first = (have - s["window"]).clamp_min(0)                                        # before it only sinks are seen
    pos = torch.where(pos < s["sinks"], pos, pos + (first - s["sinks"]).clamp_min(0)[:, None])
    seen = (pos < have[:, None]) & ((pos >= first[:, None]) | (pos < s["sinks"]))
    seq = torch.arange(len(have), device=DEVICE)[:, None]
    slots = _slots_of(s["block_table"], seq.expand_as(pos), pos, s["block"]).reshape(-1)
    keys = torch.arange(pos.numel(), device=DEVICE).reshape(pos.shape)
    o = _attend(s["q"], _rows_of(s["k_cache"], s["k_scale"], slots), _rows_of(s["v_cache"], s["v_scale"], slots), seq,
                keys, seen[:, None], s["scale"]).to(s["q"].dtype)
    return o if s["slots"] is None else (o, s["k_cache"], s["v_cache"])


def _plain_copy(s):
    pool = s["kv_cache"]
    if s["tokens"] is None:
        pool[:, :, s["dst"].long()] = pool[:, :, s["src"].long()]
        return pool
    rows = torch.arange(s["block"], device=DEVICE)
    take = rows < s["tokens"][:, None]
    src = (s["src"].long()[:, None] * s["block"] + rows)[take]
    dst = (s["dst"].long()[:, None] * s["block"] + rows)[take]
    flat = pool.view(*pool.shape[:2], -1, *pool.shape[-2:])
    flat[:, :, dst] = flat[:, :, src]
    return pool


def _plain_commit(s):
    """A node is accepted where each of its ancestors below the root, and the node itself, is the first child of its
    parent that has the parent's target token."""
    cu_q, cu_k, new, have = _spans(s)
    n, block = s["max_q"], s["block"]
    node = torch.arange(n, device=DEVICE)
    live = node < new[:, None]
    rows = (cu_q[:-1, None] + node).clamp_max(s["total"] - 1)
    parent, token, target = s["parents"].long()[rows], s["tokens"][rows], s["targets"][rows]
    fits = live & (parent >= 0) & (token == target.gather(1, parent.clamp_min(0)))
    earlier = (parent[:, :, None] == parent[:, None, :]) & (node[None, :] < node[:, None])    # [i, j]: j before i
    first = fits & ~(earlier & fits[:, None, :]).any(-1)
    first[:, 0] = live[:, 0]
    above = ((s["mask"][rows][:, :, node // 64] >> (node % 64)) & 1).bool()                  # [i, j]: j is i or above
    taken = live & (first[:, None, :] | ~above).all(-1)
    count = taken.sum(-1)
    rank = torch.cumsum(taken, -1) - 1
    path = torch.full_like(rows, -1).masked_scatter(node < count[:, None], node.expand_as(rows)[taken])
    last = path.gather(1, (count - 1).clamp_min(0)[:, None])
    following = target.gather(1, last.clamp_min(0))[:, 0]
    seq = torch.arange(len(new), device=DEVICE)[:, None].expand_as(rows)
    base = (have - new)[:, None]
    src = _slots_of(s["block_table"], seq, base + node, block)[taken]
    dst = _slots_of(s["block_table"], seq, base + rank, block)[taken]
    flat = s["kv_cache"].view(*s["kv_cache"].shape[:2], -1, *s["kv_cache"].shape[-2:])
    flat[:, :, dst] = flat[:, :, src]
    return path.int(), count.int(), following, s["kv_cache"]


# ------------------------------------------------------------ one pass

def _own(s):
    from nano_qwen_amd import kernels
    kind = s["kind"]
    if kind == "tree":
        return kernels.tree_attention(s["q"], s["k_cache"], s["v_cache"], s["cu_q"], s["cu_k"], s["max_q"], s["max_k"],
                                      s["scale"], s["block_table"], s["mask"], s["k_scale"], s["v_scale"])
    if kind == "wdecode":
        o = kernels.window_decode(s["q"][:, None], s["k_cache"], s["v_cache"], s["lens"], s["block_table"], s["scale"],
                                  s["window"], s["sinks"], s["k_scale"], s["v_scale"], k=s["k_new"], v=s["v_new"],
                                  slot_mapping=s["slots"])
        return o if s["slots"] is None else (o, s["k_cache"], s["v_cache"])
    if kind == "wprefill":
        paged = s["block_table"] is not None
        return kernels.window_prefill(s["q"], s["k_cache"] if paged else s["k"], s["v_cache"] if paged else s["v"],
                                      s["cu_q"], s["cu_k"], s["max_q"], s["max_k"], s["scale"], s["window"], s["sinks"],
                                      block_table=s["block_table"], k_scale=s["k_scale"], v_scale=s["v_scale"])
    if kind == "copy":
        kernels.copy_kv_blocks(s["kv_cache"], s["src"], s["dst"], s["tokens"])
        return s["kv_cache"]
    path, count, following = kernels.commit_tree(s["kv_cache"], s["block_table"], s["cu_q"], s["cu_k"], s["max_q"],
                                                 s["parents"], s["tokens"], s["targets"])
    return path, count, following, s["kv_cache"]


PLAIN = {"tree": _plain_tree, "wdecode": _plain_wdecode, "wprefill": _plain_wprefill, "copy": _plain_copy,
         "commit": _plain_commit}


def run(state):
    if own:
        return _own(state)
    return PLAIN[state["kind"]](state)


# ------------------------------------------------------------------ in 64 bits

def _exact_row_blocks(s, q0, new, have, k, v, see):
    """float64 attention of one sequence, a few hundred rows at a time: ``see(i, j)`` of row and key positions."""
    hq, d = s["q"].shape[1:]
    g = hq // k.shape[1]
    out = []
    at = torch.arange(have, device=DEVICE)
    for lo in range(0, new, CHUNK):
        i = torch.arange(lo, min(lo + CHUNK, new), device=DEVICE)
        ok = see(i[:, None], at[None, :])
        cols = ok.any(0).nonzero()[:, 0]
        ok = ok[:, cols]
        heads = []
        for h in range(hq):
            s64 = s["q"][q0 + i, h].double() @ k[cols, h // g].T * s["scale"]
            e = torch.where(ok, torch.exp(s64 - s64.masked_fill(~ok, -1e300).amax(1, keepdim=True)), 0.0)
            heads.append(e @ v[cols, h // g] / e.sum(1, keepdim=True).clamp_min(1e-300))
        out.append(torch.stack(heads, 1))
    return out


def exact(case, seed):
    s = prepare(case, seed)
    kind = case["kind"]
    if kind == "copy":
        pool = s["kv_cache"]
        was = pool.clone()
        for i, (a, b) in enumerate(zip(s["src"].tolist(), s["dst"].tolist())):
            n = case["block"] if s["tokens"] is None else int(s["tokens"][i])
            pool[:, :, b, :n] = was[:, :, a, :n]
        return pool
    new, pre = _lengths(case)
    block = case["block"]
    table = s["block_table"].cpu() if s["block_table"] is not None else None
    slot = lambda b, p: int(table[b, p // block]) * block + p % block    # noqa: E731
    if kind == "commit":
        parents, tokens, targets = (s[x].tolist() for x in ("parents", "tokens", "targets"))
        paths, nexts, src, dst, at = [], [], [], [], 0
        for b, (n, c) in enumerate(zip(new, pre)):
            path = [0]
            while True:
                cur = path[-1]
                child = [i for i in range(cur + 1, n) if parents[at + i] == cur and tokens[at + i] == targets[at + cur]]
                if not child:
                    break
                path.append(child[0])
            nexts.append(targets[at + path[-1]])
            src += [slot(b, c + i) for i in path]
            dst += [slot(b, c + i) for i in range(len(path))]
            paths.append(path)
            at += n
        flat = s["kv_cache"].view(2, case["layers"], -1, case["hkv"], case["d"])
        flat[:, :, dst] = flat[:, :, src].clone()
        return (_ints([p + [-1] * (max(new) - len(p)) for p in paths]), _ints([len(p) for p in paths]),
                _ints(nexts, torch.int64), s["kv_cache"])
    scales = s["k_scale"], s["v_scale"]
    if kind == "wdecode" and case["store"]:
        for b, n in enumerate(s["slots"].tolist()):
            s["k_cache"][n // block, n % block] = s["k_new"][b]
            s["v_cache"][n // block, n % block] = s["v_new"][b]
    out = []
    words = s["mask"].cpu().tolist() if kind == "tree" else None
    q0 = k0 = 0
    for b, (n, c) in enumerate(zip(new, pre)):
        have = n + c
        if table is None:
            k, v = s["k"][k0:k0 + have].double(), s["v"][k0:k0 + have].double()
        else:
            pages = table[b, :-(-have // block)].long().to(DEVICE)
            k, v = (cache.view(torch.uint8)[pages].view(cache.dtype).double().flatten(0, 1)[:have]
                    for cache in (s["k_cache"], s["v_cache"]))
            if scales[0] is not None:
                k, v = k * scales[0].double()[:, None], v * scales[1].double()[:, None]
        if kind == "tree":
            grid = torch.tensor([[(words[q0 + i][j // 64] >> (j % 64)) & 1 for j in range(n)] for i in range(n)],
                                device=DEVICE).bool()
            see = lambda i, j: (j < c) | ((j >= c) & grid[i, (j - c).clamp_min(0)])    # noqa: E731
        else:
            see = lambda i, j: (j <= c + i) & ((j > c + i - case["window"]) | (j < case["sinks"]))    # noqa: E731
        out += _exact_row_blocks(s, q0, n, have, k, v, see)
        q0, k0 = q0 + n, k0 + have
    o = torch.cat(out)
    if kind != "wdecode":
        return o
    return (o[:, None], s["k_cache"], s["v_cache"]) if case["store"] else o[:, None]
