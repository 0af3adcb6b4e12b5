"""The operators on either side of the attention in plain 64-bit form, on the CPU, and how far the kernels may be from them."""
import math

import torch

from tests import _paged_oracle as paged

HALF_STEP = {torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}


def angles(inv_freq, positions, sections=None):
    """[tokens, pairs]"""
    p = positions.double()
    if sections is None:
        return p[:, None] * inv_freq.double()
    axis = torch.tensor([a for a, n in enumerate(sections) for _ in range(n)], dtype=torch.int64)
    return p[axis].T * inv_freq.double()


def pairs_of(pairs, interleaved):
    i = torch.arange(pairs)
    return (2 * i, 2 * i + 1) if interleaved else (i, i + pairs)


def rotate(x, angle, interleaved):
    a, b = pairs_of(angle.shape[1], interleaved)
    c, s = torch.cos(angle)[:, None], torch.sin(angle)[:, None]
    y = x.clone()
    y[..., a], y[..., b] = x[..., a] * c - x[..., b] * s, x[..., b] * c + x[..., a] * s
    return y


def mixed(x, pairs, interleaved):
    """|x_a| + |x_b| for both values of a pair, |x| for the others: what a value's rounding errors scale with."""
    a, b = pairs_of(pairs, interleaved)
    y = x.abs().clone()
    y[..., a] = y[..., b] = x[..., a].abs() + x[..., b].abs()
    return y


def norm_rotary(x, weight, eps, norm, angle, interleaved):
    """(y, tolerance without the output's rounding), fp64.

    fp32 steps, each 2^-24 of what it works on: the sum of 128 squares at most 2^-17 of it (2^-18 of its root's inverse), rsqrt and the products 2^-21, cosine
    and sine 2^-22 for the reduced angle and 2^-22 for themselves, of both values of a pair: 2^-16 covers them.
    """
    x = x.double()
    if norm:
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps) * (1.0 if weight is None else weight.double())
    return rotate(x, angle, interleaved), 2.0 ** -16 * mixed(x, angle.shape[1], interleaved)


def norm_rotary_grad(x, dy, weight, eps, norm, angle, interleaved):
    """((dx, tolerance), (dw, tolerance)) by the formulas; tolerances without the output's rounding.

    As above for the gradient turned back; dx = r (g - x r^2 mean(g x)) adds the error of a mean of 128 products, 2^-17 of their magnitudes; dw
    sums products that are off by 2^-16, in fp32 over at most a few hundred at a time: 2^-15 of the magnitudes covers both.
    """
    x, dy = x.double(), dy.double()
    dn = rotate(dy, -angle, interleaved)
    wide = mixed(dy, angle.shape[1], interleaved)
    if not norm:
        return (dn, 2.0 ** -16 * wide), None
    w = torch.ones(x.shape[-1], dtype=torch.float64) if weight is None else weight.double()
    r = torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + eps)
    u, g, gw = x * r, dn * w, wide * w.abs()
    dx = r * (g - u * (g * u).mean(-1, keepdim=True))
    tol = 2.0 ** -15 * r * (gw + u.abs() * (gw * u.abs()).mean(-1, keepdim=True))
    return (dx, tol), ((dn * u).sum((0, 1)), 2.0 ** -15 * (wide * u.abs()).sum((0, 1)))


def check_close(got, want, tol, what=""):
    """`got` (of its own type) within `tol` and half a step of `want`; NaN and infinities where they are wanted."""
    g = got.detach().cpu().double()
    assert torch.equal(torch.isnan(g), torch.isnan(want)), what
    fine = torch.isfinite(want)
    assert torch.equal(g[~fine & ~torch.isnan(want)], want[~fine & ~torch.isnan(want)]), what
    tol = tol.expand_as(want) + HALF_STEP[got.dtype] * (want.abs() + tol) + torch.finfo(got.dtype).tiny
    off = (g - want).abs()[fine] - tol[fine]
    assert off.numel() == 0 or float(off.max()) <= 0, (what, float(off.max()))


def check_append(x, tol, before, scales_before, got, scales, slots, what=""):
    """A cache after rows `x` (fp64, each off by at most `tol` in the kernel) went into their slots: [blocks, size, heads, dim] bytes, scales.

    A run's scale is the rule's for its largest magnitude or, where that lies within `tol` of a power's limit, its neighbour; with that scale every value is
    within half a step of e4m3 (2^-4 of it, 2^-10 of the scale below the smallest normal value) of x, give or take `tol`.
    """
    size, i, slots = before.shape[1], 0, slots.tolist()
    want, touched = before.clone(), torch.zeros(before.shape[:2], dtype=torch.bool)
    while i < len(slots):
        if not 0 <= slots[i] < before.shape[0] * size:
            i += 1
            continue
        n = 1
        while i + n < len(slots) and slots[i + n] == slots[i] + n and slots[i + n] % size:
            n += 1
        blk, row = slots[i] // size, slots[i] % size
        touched[blk, :row + n] = True
        for h in range(before.shape[2]):
            part, t = x[i:i + n, h], tol[i:i + n, h]
            fine = torch.isfinite(part)
            low, high = (paged.least_scale(torch.where(fine, part.abs() + f * t, 0).clamp_min(0)) for f in (-1, 1))
            old = float(scales_before[blk, h]) if row else 0.0
            scale = float(scales[blk, h])
            assert max(low, old) <= scale <= max(high, old), (what, blk, h, scale, low, high, old)
            if row:
                held = before[blk, :row, h]
                if scale != old:
                    held = paged.e4m3_bytes(held.view(torch.float8_e4m3fn).double() * (old / scale))
                assert torch.equal(got[blk, :row, h], held), what
            v = got[blk, row:row + n, h].view(torch.float8_e4m3fn).double() * scale
            assert torch.equal(torch.isnan(v), torch.isnan(part)), what
            y = part.clamp(-448 * scale, 448 * scale)
            bound = t + 2.0 ** -4 * (y.abs() + t) + 2.0 ** -10 * scale
            assert bool(((v - y).abs() <= bound)[~torch.isnan(part)].all()), (what, blk, h)
        i += n
    assert torch.equal(got[~touched], before[~touched]), what
    heads_touched = touched.any(1)
    assert torch.equal(scales[~heads_touched], scales_before[~heads_touched]), what


def read(cache, scales, table, offsets, first, total):
    """Packed rows, fp64."""
    out = torch.zeros(total, *cache.shape[2:], dtype=torch.float64)
    size = cache.shape[1]
    for b in range(len(offsets) - 1):
        for i in range(offsets[b], min(offsets[b + 1], total)):
            p = first[b] + i - offsets[b]
            blk = int(table[b, p // size]) if p // size < table.shape[1] else -1
            if 0 <= blk < cache.shape[0]:
                out[i] = cache[blk, p % size].view(torch.float8_e4m3fn).double() * scales[blk].double()[:, None]
    return out


def _share(x):
    return x if x > 0 and math.isfinite(x) else 0.0


def verify(target, draft, tokens, offsets, draft_offsets, accept, sample, most):
    """(tokens, accepted, refused) as lists, from Python floats of the inputs' values, request by request."""
    out, took, lost = [], [], []
    target = target.double().tolist()
    draft = None if draft is None else draft.double().tolist()
    tokens, accept, sample = tokens.tolist(), accept.double().tolist(), sample.double().tolist()
    for b in range(len(offsets) - 1):
        rows, d0 = offsets[b + 1] - offsets[b], draft_offsets[b]
        line = [-1] * (most + 1)
        if rows <= 0:
            out.append(line), took.append(0), lost.append(0)
            continue
        n = max(0, min(draft_offsets[b + 1] - d0, rows - 1, most))
        a = 0
        while a < n:
            x = tokens[d0 + a]
            if not (0 <= x < len(target[0]) and accept[d0 + a] * (1.0 if draft is None else _share(draft[d0 + a][x])) < _share(target[offsets[b] + a][x])):
                break
            line[a] = x
            a += 1
        p = [_share(v) for v in target[offsets[b] + a]]
        left = p
        if a < n:
            if draft is None:
                left = [0.0 if i == tokens[d0 + a] else v for i, v in enumerate(p)]
            else:
                left = [_share(_share(t) - _share(q)) for t, q in zip(target[offsets[b] + a], draft[d0 + a])]
            if not sum(left) > 0:
                left = p
        mark, below, token = sample[b] * math.fsum(left), 0.0, -1
        for i, v in enumerate(left):
            below += v
            if v > 0:
                token = i
                if below > mark:
                    break
        line[a] = token
        out.append(line), took.append(a), lost.append(n - a)
    return out, took, lost


def drop(table, lens, dropped, free, num_free, size):
    """(lens, number of free blocks, stack)."""
    free, at, after = list(free), max(0, min(num_free, len(free))), []
    for b, (n, d) in enumerate(zip(lens, dropped)):
        n0 = max(n, 0)
        keep = n0 - max(0, min(d, n0))
        after.append(keep)
        for j in range(-(-keep // size), min(-(-n0 // size), table.shape[1])):
            if int(table[b, j]) >= 0:
                if at < len(free):
                    free[at] = int(table[b, j])
                at += 1
    return after, min(at, len(free)), free
