"""Attention over chosen spans of the paged cache, page copies and tree commits
in float64 torch on the CPU (oracle; test only).

No counterpart in the reference.  The definitions:

* a query token at position p of its sequence sees key j when ``j <= p`` and
  (``j > p - window`` or ``j < sinks``) (windowed); when ``j < C`` or node
  ``j - C`` is in its row of the mask (a tree behind C cached tokens);
* the output is the softmax-weighted mean of the visible values, zeros when
  nothing is visible; masked keys and values take no part, whatever they hold.

Pinned by ``tests/test_oracle_spans.py``: against ``oracle.paged`` (a window
over the whole context is causal attention, a chain is causal, a star sees the
context and itself) and a pure-Python brute force.
"""
from __future__ import annotations

import torch


def keys_of(cache, table_row, n, scale=None):
    """Float64 rows 0 .. n - 1 of one sequence ``[n, Hkv, D]`` and which of them have a page."""
    nb, bs, hkv, d = cache.shape
    out = torch.zeros(n, hkv, d, dtype=torch.float64)
    has = torch.zeros(n, dtype=torch.bool)
    for i in range(-(-n // bs)):
        blk = int(table_row[i])
        take = min(bs, n - i * bs)
        if 0 <= blk < nb:
            out[i * bs:i * bs + take] = cache[blk, :take].to(torch.float64)
            has[i * bs:i * bs + take] = True
    if scale is not None:
        out *= scale.double()[:, None]
    return out, has


def attend(q, k, v, visible, scale):
    """``q [R, Hq, D]`` over ``k, v [N, Hkv, D]`` with ``visible [R, N]``: the output and the weighted mean of
    ``|v|`` (what errors of the weights are relative to), both ``[R, Hq, D]`` float64."""
    r, hq, d = q.shape
    g = hq // k.shape[1]
    o = torch.zeros(r, hq, d, dtype=torch.float64)
    mag = torch.zeros_like(o)
    for i in range(r):
        idx = visible[i].nonzero()[:, 0]
        if len(idx) == 0:
            continue
        for h in range(k.shape[1]):
            s = q[i, h * g:(h + 1) * g].double() @ k[idx, h].T * scale
            w = torch.softmax(s, -1)
            o[i, h * g:(h + 1) * g] = w @ v[idx, h]
            mag[i, h * g:(h + 1) * g] = w @ v[idx, h].abs()
    return o, mag


def window_visible(p, n, window, sinks):
    """``[rows, n]`` for query positions ``p [rows]``."""
    j = torch.arange(n)
    p = p[:, None]
    return (j <= p) & ((j > p - window) | (j < sinks))


def tree_visible(words, n_nodes, context):
    """``[n_nodes, context + n_nodes]`` from the mask words ``[n_nodes, W]`` (Python ints or int64)."""
    out = torch.ones(n_nodes, context + n_nodes, dtype=torch.bool)
    for i in range(n_nodes):
        for j in range(n_nodes):
            out[i, context + j] = bool((int(words[i][j // 64]) >> (j % 64)) & 1)
    return out


def ancestors(parents, words):
    """Mask words of a tree from its parents (node 0: the root, parent -1)."""
    rows = []
    for i, p in enumerate(parents):
        rows.append((1 << i) | (rows[p] if p >= 0 else 0))
    split = [[(m >> (64 * w)) & (2 ** 64 - 1) for w in range(words)] for m in rows]
    return [[x - 2 ** 64 if x >= 2 ** 63 else x for x in row] for row in split]


def accepted_path(parents, tokens, targets):
    """(path, next token) of one tree."""
    path = [0]
    while True:
        cur = path[-1]
        nxt = [i for i in range(cur + 1, len(parents)) if parents[i] == cur and tokens[i] == targets[cur]]
        if not nxt:
            return path, targets[cur]
        path.append(nxt[0])


def move_rows(pool, table_row, context, path):
    """In place: row ``context + path[r]`` to ``context + r`` in ``pool [..., num_blocks, block_size, H, D]``."""
    bs = pool.shape[-3]
    was = pool.clone()
    for r, node in enumerate(path):
        a, b = context + node, context + r
        pool[..., int(table_row[b // bs]), b % bs, :, :] = was[..., int(table_row[a // bs]), a % bs, :, :]
    return pool
