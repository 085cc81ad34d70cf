"""Cases and checks of attention over caches with a scale for each block of tokens and head."""
import torch

from oracle import spans
from tests.spans import NAN, gen, tolerance

CODE = torch.float8_e4m3fn


def power(amax):
    m, e = torch.frexp(amax)
    return torch.ldexp(torch.ones_like(amax), (e - 9 + (m > 0.875)).clamp(-60, 60))


class Case:
    """Sequences of ``new`` query tokens behind ``pre`` cached ones.  Codes that no sequence owns and scales of blocks that
    hold no token are NaN.  ``fine``: scales that are no powers of two.  ``lost``: pages (sequence, entry) that the
    table lacks."""

    def __init__(self, new, pre, hq, hkv, d, dtype, block=256, unit=64, seed=0, fine=False, lost=(), spread=6):
        g = gen(seed)
        self.new, self.pre, self.hq, self.hkv, self.d, self.dtype, self.block, self.unit = new, pre, hq, hkv, d, dtype, block, unit
        self.scale = d ** -0.5
        n = len(new)
        self.have = [a + b for a, b in zip(new, pre)]
        cu = lambda v: torch.tensor([sum(v[:i]) for i in range(len(v) + 1)], dtype=torch.int32)    # noqa: E731
        self.cu_q, self.cu_k = cu(new), cu([max(0, h) for h in self.have])
        self.max_q, self.max_k = max(new), max(max(self.have), 1)
        self.q_full = torch.randn(sum(new), hq, d + 64, generator=g).to(dtype)
        self.q = self.q_full[:, :, :d]
        counts = [-(-max(h, 0) // block) for h in self.have]
        blocks = sum(counts) + 3
        perm = torch.randperm(blocks, generator=g).to(torch.int32)
        self.table = torch.full((n, max(max(counts), 1) + 1), -1, dtype=torch.int32)
        units = block // unit
        self.k, self.v, self.k_scale, self.v_scale = [], [], [], []
        own = torch.zeros(blocks, block, dtype=torch.bool)
        at = 0
        for i, c in enumerate(counts):
            self.table[i, :c] = perm[at:at + c]
            at += c
            for j in range(c):
                own[self.table[i, j].long(), :max(0, min(block, self.have[i] - j * block))] = True
        used = own.view(blocks, units, unit).any(-1)
        for is_v in (False, True):
            x = torch.randn(blocks, units, unit, hkv, d, generator=g)
            # V's blocks differ widely; K's as far as the scores of spans.tolerance go
            x *= 2.0 ** torch.randint(-spread, spread + 1, (blocks, units, 1, hkv, 1), generator=g) if is_v else \
                2.0 ** torch.randint(-2, 1, (blocks, units, 1, hkv, 1), generator=g)
            s = power(x.abs().amax(dim=(2, 4)))
            if fine:
                s = s * (1 + torch.rand(s.shape, generator=g))
            codes = (x / s[:, :, None, :, None]).clamp(-448, 448).to(CODE).view(blocks, block, hkv, d)
            codes.view(torch.uint8)[~own] = 0xFF
            s[~used] = NAN
            if is_v:
                self.v, self.v_scale = codes, s
            else:
                self.k, self.k_scale = codes, s
        for i, j in lost:
            self.table[i, j] = -1 if (i + j) % 2 else blocks + 5

    def to(self, dev):
        for name in ("q_full", "k", "v", "table", "cu_q", "cu_k", "k_scale", "v_scale"):
            setattr(self, name + "_dev", getattr(self, name).to(dev))
        self.q_dev = self.q_full_dev[:, :, :self.d]
        self.lens_dev = torch.tensor(self.have, dtype=torch.int32, device=dev)
        return self

    def values_of(self, cache, scale, i, have):
        """Float64 rows of sequence i, their scales, and which have a page."""
        rows, has = spans.keys_of(cache, self.table[i], have)
        each = scale.repeat_interleave(self.unit, 1)[..., None]    # [blocks, block, Hkv, 1]
        s, _ = spans.keys_of(each, self.table[i], have)
        s = torch.where(has[:, None, None], s, 1.0)
        return torch.where(has[:, None, None], rows * s, 0.0), s[..., 0], has

    def reference(self, window=1 << 40, sinks=0, device="cpu"):
        """(output, weighted mean of |v|, what fp16's subnormal weights may be off), in float64 on ``device``."""
        outs, mags, subs, q0 = [], [], [], 0
        g = self.hq // self.hkv
        for i, n in enumerate(self.new):
            have = max(self.have[i], 0)
            k, _, has = self.values_of(self.k, self.k_scale, i, have)
            v, sv, _ = self.values_of(self.v, self.v_scale, i, have)
            vis = (spans.window_visible(torch.arange(have - n, have), have, window, sinks) & has).to(device)
            o, mag, sub = (torch.zeros(n, self.hq, self.d, dtype=torch.float64, device=device) for _ in range(3))
            q, k, v, sv = (x.to(device) for x in (self.q[q0:q0 + n].double(), k, v, sv))
            for h in range(self.hkv if have else 0):
                t = (q[:, h * g:(h + 1) * g].reshape(-1, self.d) @ k[:, h].T.contiguous()).view(n, g, have) * self.scale
                t = t.masked_fill(~vis[:, None], -torch.inf)
                any_ = vis.any(1)[:, None, None]
                p = torch.where(any_, torch.softmax(t, -1), 0.0)
                hs = slice(h * g, (h + 1) * g)
                o[:, hs], mag[:, hs] = p @ v[:, h], p @ v[:, h].abs()
                # weights w = p sv / max(p sv): one below fp16's normal range is off by 2^-25 of the largest, times a code
                top = (p * sv[:, h]).amax(-1, keepdim=True)
                codes = (v[:, h] / torch.where(sv[:, h, None] > 0, sv[:, h, None], 1.0)).abs()
                sub[:, hs] = 2.0 ** -25 * top * (vis[:, None].double() @ codes)
            for to, x in ((outs, o), (mags, mag), (subs, sub)):
                to.append(x.cpu())
            q0 += n
        return torch.cat(outs), torch.cat(mags), torch.cat(subs)

    def prefill(self, window=None, sinks=0, **kw):
        from nano_qwen_amd import kernels
        args = (self.q_dev, self.k_dev, self.v_dev, self.cu_q_dev, self.cu_k_dev, self.max_q, self.max_k, self.scale)
        kw = dict(block_table=self.table_dev, k_scale=self.k_scale_dev, v_scale=self.v_scale_dev) | kw
        return kernels.varlen_prefill(*args, **kw) if window is None else kernels.window_prefill(*args, window, sinks, **kw)

    def decode(self, window=None, sinks=0, **kw):
        from nano_qwen_amd import kernels
        args = (self.q_dev, self.k_dev, self.v_dev, self.lens_dev, self.table_dev, self.scale)
        kw = dict(k_scale=self.k_scale_dev, v_scale=self.v_scale_dev) | kw
        return kernels.paged_decode(*args, **kw) if window is None else kernels.window_decode(*args, window, sinks, **kw)


def check(out, ref, dtype, what=""):
    """Value by value: spans.tolerance (a weight's and an output's rounding to 16 bits, fp32 scores), and fp16's subnormals,
    of the weights and of the output.  The exponents' terms -- a score, V's scale, the maximum -- are at most 64 each:
    another 3 * 64 * 2^-24 < 2e-5 of a weight, inside the 2 % that spans.tolerance leaves of its 5e-4."""
    o, mag, sub = ref
    got = out.double().cpu().reshape(o.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    tol = tolerance(o, mag, dtype)
    if dtype == torch.float16:
        tol = tol + sub + 2.0 ** -25
    off = (got - o).abs()
    assert (off <= tol).all(), f"{what}: {(off - tol).max():.3e} past the tolerance; max error {off.max():.3e}"
