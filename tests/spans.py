"""Cases and checks shared by the tests of windowed and tree attention."""
import random

import torch

from oracle import spans

NAN = float("nan")


def gen(seed):
    return torch.Generator().manual_seed(seed)


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tolerance(ref, mag, dtype, roundings=1):
    """What a kernel's output may be off from the float64 one, value by value.

    Each weight is rounded once to the 16-bit type (half a step, relative): at most u * mag, mag the weighted mean
    of |v|.  The output is rounded once: u * |o|.  The rest is fp32: a score of D = 256 products whose magnitudes
    sum to at most 16 after scaling is off by 256 * 2^-24 * 16 = 2.5e-4 at most, its weight by as much, and the mean
    by twice that (numerator and sum): 5e-4 * mag.  (1 + u)^2 and sums of a few more fp32 roundings: 2%.
    """
    u = half_step(dtype)
    return 1.02 * (u * mag + roundings * u * ref.abs() + 5e-4 * mag) + 1e-30


def check(out, ref, mag, dtype, what=""):
    o = out.double().cpu()
    assert o.shape == ref.shape, (what, o.shape, ref.shape)
    assert torch.isfinite(o).all(), f"{what}: not finite"
    off = (o - ref).abs()
    tol = tolerance(ref, mag, dtype)
    worst = (off - tol).max().item()
    assert (off <= tol).all(), f"{what}: {worst:.3e} past the tolerance; max error {off.max():.3e}"


class Case:
    """Sequences of ``new`` query tokens behind ``pre`` cached ones over a paged pool (or packed K/V).

    Every value that no sequence owns is NaN: pages of no sequence, rows behind a sequence's last token.  ``free``
    takes the pages that no query token sees out of the table (-1)."""

    def __init__(self, new, pre, hq, hkv, d, dtype, block=256, fp8=False, paged=True, seed=0, extra_rows=0, qstride=None):
        g = gen(seed)
        self.new, self.pre, self.hq, self.hkv, self.d, self.dtype, self.block = new, pre, hq, hkv, d, dtype, block
        self.scale = d ** -0.5
        self.fp8, self.paged = fp8, paged
        n = len(new)
        have = [a + b for a, b in zip(new, pre)]
        self.have = have
        cu = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32)    # noqa: E731
        self.cu_q, self.cu_k = cu(new), cu([max(0, h) for h in have])
        self.max_q, self.max_k = max(new), max(max(have), 1)
        total = sum(new)
        width = hq * (qstride or d)
        base = torch.randn(total + extra_rows, width, generator=g).to(dtype)
        self.q_full = base.view(total + extra_rows, hq, qstride or d)
        self.q = self.q_full[:, :, :d]
        if not paged:
            tk = sum(have)
            self.k, self.v = (torch.randn(tk, hkv, d, generator=g).to(dtype) for _ in range(2))
            self.table = None
            self.k_scale = self.v_scale = None
            return
        counts = [-(-max(h, 0) // block) for h in have]
        blocks = sum(counts) + 3
        perm = torch.randperm(blocks, generator=g).to(torch.int32)
        self.table = torch.full((n, max(max(counts), 1) + 1), -1, dtype=torch.int32)
        at = 0
        x = torch.randn(2, blocks, block, hkv, d, generator=g).to(dtype)
        self.k_scale = self.v_scale = None
        if fp8:
            s = x.float().abs().amax(dim=(1, 2, 4)) / 448
            x = (x.float() / s[:, None, None, :, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
            self.k_scale, self.v_scale = s[0].contiguous(), s[1].contiguous()
        own = torch.zeros(blocks, block, dtype=torch.bool)
        for i, c in enumerate(counts):
            self.table[i, :c] = perm[at:at + c]
            at += c
            for j in range(c):
                own[self.table[i, j].long(), :max(0, min(block, have[i] - j * block))] = True
        # what nobody owns is NaN (through bytes: fp8 has no masked fill)
        raw = x.view(torch.uint8).view(2, blocks, block, -1)
        raw[:, ~own] = 0xFF if fp8 else (torch.full((1,), NAN, dtype=dtype).view(torch.uint8).repeat(raw.shape[-1] // 2))
        self.k, self.v = x[0].contiguous(), x[1].contiguous()

    def to(self, dev):
        for name in ("q_full", "k", "v", "table", "cu_q", "cu_k", "k_scale", "v_scale"):
            t = getattr(self, name)
            setattr(self, name + "_dev", None if t is None else t.to(dev))
        self.q_dev = self.q_full_dev[:, :, :self.d]
        return self

    def free_before(self, window, sinks):
        """Takes the pages out of the table that no query token of a window sees."""
        for i, (n, c) in enumerate(zip(self.new, self.pre)):
            vis = spans.window_visible(torch.arange(c, c + n), self.have[i], window, sinks).any(0)
            for j in range(-(-self.have[i] // self.block)):
                if not vis[j * self.block:(j + 1) * self.block].any():
                    self.table[i, j] = -1
        return self

    def reference(self, visible_of):
        """(output, weighted mean of |v|) with ``visible_of(sequence, rows, keys)``."""
        outs, mags = [], []
        q0 = k0 = 0
        for i, n in enumerate(self.new):
            have = max(self.have[i], 0)
            if self.paged:
                k, hask = spans.keys_of(self.k, self.table[i], have, self.k_scale)
                v, _ = spans.keys_of(self.v, self.table[i], have, self.v_scale)
            else:
                k, v = self.k[k0:k0 + have].double(), self.v[k0:k0 + have].double()
                hask = torch.ones(have, dtype=torch.bool)
            vis = visible_of(i, n, have) & hask
            o, mag = spans.attend(self.q[q0:q0 + n], k, v, vis, self.scale)
            outs.append(o)
            mags.append(mag)
            q0, k0 = q0 + n, k0 + have
        return torch.cat(outs), torch.cat(mags)

    def window_reference(self, window, sinks):
        return self.reference(lambda i, n, have: spans.window_visible(torch.arange(have - n, have), have, window, sinks))

    def window_prefill(self, window, sinks, **kw):
        from nano_qwen_amd import kernels
        return kernels.window_prefill(self.q_dev, self.k_dev, self.v_dev, self.cu_q_dev, self.cu_k_dev, self.max_q,
                                      self.max_k, self.scale, window, sinks, block_table=self.table_dev,
                                      k_scale=self.k_scale_dev, v_scale=self.v_scale_dev, **kw)

    def window_decode(self, window, sinks, **kw):
        from nano_qwen_amd import kernels
        lens = torch.tensor(self.have, dtype=torch.int32, device=self.q_dev.device)
        return kernels.window_decode(self.q_dev, self.k_dev, self.v_dev, lens, self.table_dev, self.scale, window,
                                     sinks, self.k_scale_dev, self.v_scale_dev, **kw)

    def tree_attention(self, mask, **kw):
        from nano_qwen_amd import kernels
        return kernels.tree_attention(self.q_dev, self.k_dev, self.v_dev, self.cu_q_dev, self.cu_k_dev, self.max_q,
                                      self.max_k, self.scale, self.table_dev, mask.to(self.q_dev.device),
                                      self.k_scale_dev, self.v_scale_dev, **kw)


def random_tree(r, n):
    return [-1] + [r.randrange(i) if r.random() < 0.5 else min(i - 1, int((i - 1) * r.random() ** 2)) for i in range(1, n)]


def tree_masks(new, seed=0, words=None):
    """(trees, mask ``[T, words]``) of random trees."""
    r = random.Random(seed)
    words = words or -(-max(new) // 64)
    trees = [random_tree(r, n) for n in new]
    rows = [row for t in trees for row in spans.ancestors(t, words)]
    return trees, torch.tensor(rows, dtype=torch.int64)


def tree_reference(case, mask):
    at = [sum(case.new[:i]) for i in range(len(case.new))]
    return case.reference(lambda i, n, have: spans.tree_visible(mask[at[i]:at[i] + n].tolist(), n, have - n))
