"""Whole batches over a paged 8-bit cache, made and evaluated (in 64 bits) on one device without a loop over blocks."""
import itertools
import math

import torch

import ads_model_kernel_library_b200.gdpa as G
from tests import _paged_oracle as ref

F8 = torch.float8_e4m3fn
# What a P is off by at most, in parts of its row's largest P (both times V's scale): the largest lies at 32 at least, P is rounded to float16 and
# for few queries (up to 64 rows of a K / V head) to the sum of three e4m3 values, the last in steps of 2^-18.
FEW, MANY = 2.0 ** -24, 2.0 ** -29


class Batch:
    """Requests with random caches; rows past a request's length and blocks of no request are NaN."""

    def __init__(self, lens, q_lens, heads, kv_heads, dim, size, seed=0, device="cuda"):
        g = torch.Generator(device=device).manual_seed(seed)
        self.lens, self.size, self.group = list(lens), size, heads // kv_heads
        self.offsets = [0] + list(itertools.accumulate(q_lens))
        self.max_q = max(list(q_lens) + [0])
        held = torch.tensor([-(-n // size) for n in lens], dtype=torch.int64)
        width, total = max(1, int(held.max())), int(held.sum())
        order = torch.randperm(total + 1, generator=torch.Generator().manual_seed(seed))
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        has = torch.arange(width) < held[:, None]
        self.table[has] = order[:total].to(torch.int32)
        self.table = self.table.to(device)
        shape = (total + 1, size, kv_heads, dim)
        unused = torch.ones(total + 1, size, dtype=torch.bool, device=device)
        in_use = torch.arange(width * size).view(width, size) < torch.tensor(lens)[:, None, None]
        unused[self.table[has.to(device)].long()] = ~in_use[has].to(device)

        def cache(scale):
            c = (torch.randn(shape, generator=g, device=device) / scale).to(F8).view(torch.uint8)
            c[unused] = 0x7F
            s = torch.full((total + 1, kv_heads), scale, device=device)
            s[order[total]] = math.nan
            return c, s

        self.k, self.ks = cache(2.0 ** -6)
        self.v, self.vs = cache(2.0 ** -6)
        self.q = torch.randn(self.offsets[-1], heads, dim, generator=g, device=device).bfloat16()

    def int32(self, x):
        return torch.tensor(x, dtype=torch.int32, device=self.q.device)

    def run(self, scale, activation="softmax", causal=False, window=None):
        return G.generalized_dot_product_attention_paged_fp8(
            self.q, self.k.view(F8), self.v.view(F8), self.ks, self.vs, self.table, self.int32(self.offsets), self.int32(self.lens), self.max_q,
            qk_scale=scale, activation=activation, is_causal=causal, window_size=window)

    def want(self, scale, activation="softmax", causal=False, window=None, step=None):
        """(O, how far a kernel may be from it).  In parts of what the sums here carry: O's rounding to bf16 and fp32 steps on the way (2^-8 of it);
        P's rounding, a score's and an activation's (2^-7 of sum |P| |V| together); P below the formats' smallest steps (``step``, above),
        which takes no more than the P that are that small."""
        if step is None:
            step = FEW if self.max_q * self.group <= 64 else MANY
        out = torch.zeros(self.q.shape, dtype=torch.float64, device=self.q.device)
        tol = torch.zeros_like(out)
        for b, n in enumerate(self.lens):
            lo, hi = self.offsets[b], self.offsets[b + 1]
            if hi == lo or n == 0:
                continue
            (k8, sk), (v8, sv) = (ref.gather(c, s, self.table[b], n) for c, s in ((self.k, self.ks), (self.v, self.vs)))
            n = len(k8)  # no more than the table can hold; the queries are the last of all tokens
            k, v = (t.repeat_interleave(self.group, 1).transpose(0, 1) for t in (k8 * sk[..., None], v8 * sv[..., None]))
            sv = sv.repeat_interleave(self.group, 1).T[:, None]
            x = self.q[lo:hi].double().transpose(0, 1) @ k.transpose(1, 2)
            p0, j = torch.arange(self.lens[b] - (hi - lo), self.lens[b], device=x.device)[:, None], torch.arange(n, device=x.device)
            off = torch.zeros(hi - lo, n, dtype=torch.bool, device=x.device)
            if causal:
                off |= j > p0
            if window is not None:
                off |= (j - p0).abs() > window
            if activation == "softmax":
                p = torch.softmax((x * scale).masked_fill(off, -math.inf), -1).masked_fill(off.all(1)[:, None], 0)
            else:
                p = (ref.ACT[activation](x) * scale).masked_fill(off, 0)
            out[lo:hi] = (p @ v).transpose(0, 1)
            most = (p.abs() * sv).amax(2, keepdim=True)
            small = torch.minimum(p.abs(), torch.where(sv > 0, step * most / sv, 0))
            if activation in ("gelu_approx", "silu"):  # tanh.approx: 2^-10.98 of a tanh, times |x| / 2
                small = small + (2.0 ** -11 * x.abs() * abs(scale)).masked_fill(off, 0)
            tol[lo:hi] = ((2.0 ** -7 * p.abs() + small) @ v.abs()).transpose(0, 1) + 2.0 ** -8 * out[lo:hi].abs()
        return out, tol

    def check(self, scale, activation="softmax", causal=False, window=None):
        o = self.run(scale, activation, causal, window).double()
        assert G.kernel_status() == 0
        want, tol = self.want(scale, activation, causal, window)
        assert bool(torch.isfinite(o).all())
        over = (o - want).abs() - tol
        assert float(over.max()) <= 0, f"{int((over > 0).sum())} of {over.numel()} elements too far, worst by {float(over.max()):.3g}"
        return o
