"""Verification of drafts, their way out of the cache, and whole steps with both, on the GPU."""
import math
import os
import subprocess
import sys

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from tests import _heads_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def sums(n):
    out = [0]
    for x in n:
        out.append(out[-1] + x)
    return out


def check_verify(drafts, vocab, dtype=torch.float32, lookup=False, ints=torch.int64, offsets=torch.int32, agree=0.7, seed=0, rows=None, most=None, padded=0, edit=None,
                 exact_sums=False):
    g = torch.Generator().manual_seed(seed)
    n, rows = sum(drafts), [d + 1 for d in drafts] if rows is None else rows
    if exact_sums:  # multiples of 2^-12 below 2^4: every sum of them is exact, so that marks can lie on the borders
        target, draft = (torch.randint(0, 8, (m, vocab), generator=g).double() / 4096 for m in (sum(rows), n))
    else:
        target = torch.softmax(2.5 * torch.randn(sum(rows), vocab, generator=g), 1).double()
        own = torch.tensor([r0 + j for r0, d, r in zip(sums(rows), drafts, rows) for j in range(d)], dtype=torch.int64).clamp(0, max(sum(rows) - 1, 0))
        draft = agree * (target[own] if sum(rows) else 0) + (1 - agree) * torch.softmax(2.5 * torch.randn(n, vocab, generator=g), 1).double()
    target, draft = target.to(dtype), draft.to(dtype)
    tokens = torch.multinomial(draft.float() + 1e-9, 1, generator=g)[:, 0].to(ints) if n else torch.zeros(0, dtype=ints)
    accept, sample = torch.rand(n, generator=g), torch.rand(len(drafts), generator=g)
    if exact_sums:
        sample = torch.randint(0, 65, (len(drafts),), generator=g).float() / 64
    if edit:
        edit(target, draft, tokens, accept, sample)
    most = max(drafts + [0]) if most is None else most
    want = ref.verify(target, None if lookup else draft, tokens, sums(rows), sums(drafts), accept, sample, most)

    def wide(x):
        if not padded:
            return x.to(DEV)
        return torch.nn.functional.pad(x.to(DEV), (1, padded), value=math.nan)[:, 1:vocab + 1]

    got = G.verify_draft_tokens(wide(target), None if lookup else wide(draft), tokens.to(DEV), torch.tensor(sums(rows), dtype=offsets, device=DEV),
                                torch.tensor(sums(drafts), dtype=offsets, device=DEV), accept.to(DEV), sample.to(DEV), most)
    assert got[0].dtype == ints and got[1].dtype == got[2].dtype == torch.int32
    assert tuple(t.tolist() for t in got) == want


@pytest.mark.parametrize("vocab", [1, 2, 31, 33, 1000, 1024, 1025, 4096, 4097, 20011])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_verify_vocabularies(vocab, dtype):
    check_verify([3, 0, 1, 4, 2], vocab, dtype)
    check_verify([2, 1], vocab, dtype, lookup=True, seed=1)


@pytest.mark.parametrize("options", [
    dict(ints=torch.int32), dict(offsets=torch.int64), dict(agree=0.99), dict(agree=0.05), dict(padded=3), dict(lookup=True, padded=1),
    dict(rows=[4, 3, 0, 2, 1, 5]), dict(most=2), dict(most=0), dict(most=9)])
def test_verify_options(options):
    check_verify([3, 2, 2, 0, 1, 4], 3001, **options)


def test_verify_many():
    check_verify([i % 6 for i in range(400)], 150)
    check_verify([40, 0, 70], 90, agree=0.999)  # more drafts than a warp has lanes
    check_verify([1] * 3, 300000)
    check_verify([1], 300000, torch.bfloat16)


@pytest.mark.parametrize("dtype,vocab", [(torch.float32, 65537), (torch.bfloat16, 131079)])
def test_verify_many_long_rows(dtype, vocab):
    """Rows that are enough for the three kernels."""
    def edit(target, draft, tokens, accept, sample):
        target[3, 700], target[4, 65000], draft[2] = math.nan, math.inf, 9.0
        target[9:14] = 0.0
        sample[1], sample[2] = 0.0, 1.0

    drafts = [i % 3 for i in range(32)]
    check_verify(drafts, vocab, dtype, edit=edit)
    check_verify(drafts, vocab, dtype, lookup=True, edit=lambda t, d, x, a, s: a.mul_(1e-4), seed=1)
    check_verify(drafts, vocab, dtype, padded=3, rows=[0, 2, 1] * 10 + [3, 0], ints=torch.int32, agree=0.95, seed=2)


def test_verify_marks_on_borders():
    for seed in range(6):
        check_verify([1, 2, 0, 1] * 8, (50, 1024, 2050, 5000, 9000, 16384)[seed], exact_sums=True, seed=seed)
    check_verify([1, 2, 0, 1] * 8, 65600, exact_sums=True, seed=6)


def test_verify_numbers_that_are_none():
    def edit(target, draft, tokens, accept, sample):
        target[0, 5], target[1, 3], draft[0, 2], draft[0, 7], draft[0, 8], target[2] = math.nan, math.inf, math.nan, math.inf, -0.5, -1.0
        target[3] = 0.0
        draft[1] = 9.0  # nothing is left of the difference
        target[6, :], target[6, 77] = 0.0, 1e-38
        sample[0], sample[1], sample[2] = 1.0, 0.0, 1.5
        tokens[2], tokens[3] = -5, 10 ** 6

    for lookup in (False, True):
        check_verify([1, 1, 1, 1, 0], 100, edit=edit, lookup=lookup)
        check_verify([1, 1, 1, 1, 0], 9001, torch.bfloat16, edit=edit, lookup=lookup)
        check_verify([1, 1, 1, 1, 0], 5000, edit=edit, lookup=lookup, ints=torch.int32)


def test_verify_numbers_that_are_none_for_a_draft():
    def edit(target, draft, tokens, accept, sample):
        tokens[:] = 7
        accept[:] = 0.25
        target[::2, 7] = 0.5
        draft[0, 7], draft[1, 7], draft[2, 7], draft[3, 7] = math.nan, math.inf, -1.0, 0.0  # count as 0: accepted
        for i, bad in enumerate((math.inf, math.nan, -1.0, 0.0)):  # ... and refused
            draft[4 + i, 7], target[2 * (4 + i), 7] = 0.5, bad

    for lookup in (False, True):
        check_verify([1] * 8, 100, edit=edit, lookup=lookup)
        check_verify([1] * 8, 1001, torch.bfloat16, edit=edit, lookup=lookup)


def test_verify_nothing():
    check_verify([], 10)
    check_verify([0, 0], 10)
    check_verify([0], 10, rows=[0])
    check_verify([3], 10, rows=[0])


def test_verify_draws_what_the_target_would():
    """Over many requests the accepted or drawn first token is distributed as the target's: a chi-squared sum of 11 terms stays below 50 but once in 10^6 times."""
    g = torch.Generator(device=DEV).manual_seed(0)
    n, vocab = 40000, 12
    p, q = (torch.softmax(torch.randn(vocab, generator=g, device=DEV), 0) for _ in range(2))
    tokens = torch.multinomial(q.expand(n, vocab), 1, generator=g)[:, 0]
    off = torch.arange(n + 1, dtype=torch.int32, device=DEV)
    out, accepted, _ = G.verify_draft_tokens(p.expand(2 * n, vocab), q.expand(n, vocab), tokens, 2 * off, off, torch.rand(n, generator=g, device=DEV),
                                             torch.rand(n, generator=g, device=DEV), 1)
    count = torch.bincount(out[:, 0], minlength=vocab).double()
    assert float(((count - n * p.double()) ** 2 / (n * p.double())).sum()) < 50
    assert 0.2 < float(accepted.float().mean()) < 0.999


def test_verify_refusals():
    p, t, o = torch.ones(4, 10, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV), i32([0, 4])
    d, u, s = i32([0, 3]), torch.zeros(3, device=DEV), torch.zeros(1, device=DEV)
    good = [p, p[:3], t, o, d, u, s, 3]
    for at, bad, error in ((0, p.half(), TypeError), (0, p[0], ValueError), (0, p[:, :0], ValueError), (0, p.t(), ValueError), (1, p, ValueError),
                           (1, p[:3, :9], ValueError), (1, p[:3].bfloat16(), TypeError), (2, t.float(), TypeError), (2, t[:2], ValueError), (3, o.long(), TypeError),
                           (3, i32([0, 1, 4]), ValueError), (4, i32([0]), ValueError), (5, u.double(), TypeError), (5, u[:2], ValueError), (6, s.double(), TypeError),
                           (6, s.cpu(), RuntimeError), (7, -1, ValueError)):
        with pytest.raises(error):
            G.verify_draft_tokens(*good[:at], bad, *good[at + 1:])
    with pytest.raises(NotImplementedError):
        G.verify_draft_tokens(torch.ones(1, 1, device=DEV).expand(4, (1 << 20) + 1)[:, :].contiguous(), None, *good[2:])
    old = G.set_offset_validation(True)
    try:
        for at, bad in ((3, i32([0, 5])), (3, i32([2, 1])), (4, i32([0, 4]))):
            with pytest.raises(ValueError):
                G.verify_draft_tokens(*good[:at], bad, *good[at + 1:])
    finally:
        G.set_offset_validation(old)


# ------------------------------------------------------------------------------------------ out of the cache


def check_drop(lens, dropped, size, width, holes=0, have=5, capacity=None, ints=torch.int32, stride=0, seed=0):
    g = torch.Generator().manual_seed(seed)
    batch = len(lens)
    table = torch.randint(0, 10 ** 6, (batch, width), generator=g, dtype=torch.int32)
    if holes:
        table[torch.rand(table.shape, generator=g) < holes] = -1
    need = sum(-(-max(n, 0) // size) for n in lens) + max(have, 0) + 3
    free = torch.randint(0, 10 ** 6, (need if capacity is None else capacity,), generator=g, dtype=torch.int32)
    want = ref.drop(table, lens, dropped, free.tolist(), have, size)
    wide = torch.full((max(batch, 1), width + stride), 77, dtype=torch.int32, device=DEV)
    mine = wide[:batch, :width]
    mine.copy_(table)
    stack = free.to(DEV)
    after, left = G.drop_cached_tokens(mine, torch.tensor(lens, dtype=ints, device=DEV), torch.tensor(dropped, dtype=ints, device=DEV), stack, i32([have]), size)
    assert after.tolist() == want[0] and int(left) == want[1] and stack.tolist() == want[2]
    assert torch.equal(mine.cpu(), table)


@pytest.mark.parametrize("size", [16, 32, 64, 128])
def test_drop_lengths(size):
    lens = [0, 1, size, size + 1, 5 * size, 3 * size + 2, 900, 40]
    check_drop(lens, [0, 1, 1, 1, 2 * size + 1, 2, 900, -3], size, 60)
    check_drop(lens, [5, 0, size, size + 1, 10 ** 6, 3, 1, 40], size, 60, holes=0.3, ints=torch.int64, stride=5)
    check_drop(lens, [n // 2 for n in lens], size, 4)  # lengths beyond the table


def test_drop_nothing_and_full_stacks():
    check_drop([], [], 16, 4)
    check_drop([50], [0], 16, 4)
    check_drop([50, 60], [50, 60], 16, 0)
    check_drop([50, 60], [50, 60], 16, 4, have=-7)
    check_drop([50, 60], [50, 60], 16, 4, have=3, capacity=5)
    check_drop([50, 60], [50, 60], 16, 4, have=9, capacity=0)
    check_drop([-5, 60], [3, 7], 16, 4)


def test_drop_long_requests():
    """More entries of a request than a warp has in registers."""
    check_drop([16 * 1500 - 3, 5, 16 * 640, 16 * 129], [16 * 1500 - 3, 1, 16 * 513, 16 * 128 + 4], 16, 1500)
    check_drop([16 * 700] * 300, [16 * 700 - 5] * 300, 16, 700, holes=0.3)


@pytest.mark.parametrize("batch", [31, 256, 257, 2049, 9000])
def test_drop_many(batch):
    g = torch.Generator().manual_seed(batch)
    lens = torch.randint(0, 500, (batch,), generator=g)
    check_drop(lens.tolist(), (torch.rand(batch, generator=g) * (lens + 1)).int().tolist(), 16, 32, holes=0.1)
    check_drop(lens.tolist(), torch.randint(0, 5, (batch,), generator=g).tolist(), 64, 8)


def test_drop_refusals():
    t, n, f, one = i32([[0, 1]]), i32([20]), i32([0] * 4), i32([0])
    good = [t, n, n, f, one, 16]
    for at, bad, error in ((0, t.long(), TypeError), (0, t.expand(2, 2), ValueError), (1, n.float(), TypeError), (2, i32([1, 2]), ValueError),
                           (3, f.long(), TypeError), (4, i32([1, 2]), ValueError), (5, 20, NotImplementedError), (3, f.cpu(), RuntimeError)):
        with pytest.raises(error):
            G.drop_cached_tokens(*good[:at], bad, *good[at + 1:])


# ------------------------------------------------------------------------------------------ whole steps


def served(steps, capture=False):
    """Requests with drafts over one cache, norm and rotation on the way; every step's queries, keys and values are given tensors, so that the tokens that
    stay can be attended to in plain form at the end."""
    g = torch.Generator().manual_seed(4)
    batch, heads, kv, dim, size, vocab, most = 5, 4, 2, 64, 16, 600, 3
    cache = G.PagedKVCache(80, size, kv, dim, batch, 256)
    f = 10000.0 ** -(torch.arange(32, dtype=torch.float64) / 32)
    w = 1 + 0.2 * torch.randn(2, dim, generator=g)
    rotary = dict(inv_freq=f.to(DEV), query_weight=w[0].to(DEV), key_weight=w[1].to(DEV))
    kept = [([], []) for _ in range(batch)]
    lens = [0] * batch
    for step in range(steps):
        prompt = step == 0
        drafts = [0] * batch if prompt else torch.randint(0, most + 1, (batch,), generator=g).tolist()
        new = torch.randint(1, 60, (batch,), generator=g).tolist() if prompt else [d + 1 for d in drafts]
        total = sum(new)
        q, k, v = (torch.randn(total, h, dim, generator=g).bfloat16() for h in (heads, kv, kv))
        out = cache.step(q.to(DEV), k.to(DEV), v.to(DEV), i32(new), max(new), rotary=rotary, qk_scale=dim ** -0.5)
        for b, (x, y) in enumerate(zip(k.split(new), v.split(new))):
            kept[b][0].append(x), kept[b][1].append(y)
            lens[b] += new[b]
        last = (q, new, list(lens), out, [torch.cat(x[0]) for x in kept], [torch.cat(x[1]) for x in kept])
        if prompt:
            continue
        target, draft = (torch.softmax(2 * torch.randn(n, vocab, generator=g), 1) for n in (total, sum(drafts)))
        draft = 0.3 * draft + 0.7 * target[[i for r, d in zip(sums(new), drafts) for i in range(r, r + d)]]
        tokens = torch.multinomial(draft, 1, generator=g)[:, 0] if sum(drafts) else torch.zeros(0, dtype=torch.int64)
        accept, sample = torch.rand(sum(drafts), generator=g), torch.rand(batch, generator=g)
        out_tokens, accepted, refused = G.verify_draft_tokens(target.to(DEV), draft.to(DEV), tokens.to(DEV), i32(sums(new)), i32(sums(drafts)), accept.to(DEV),
                                                              sample.to(DEV), most)
        want = ref.verify(target, draft, tokens, sums(new), sums(drafts), accept, sample, most)
        assert (out_tokens.tolist(), accepted.tolist(), refused.tolist()) == want
        cache.drop(refused)
        for b, r in enumerate(want[2]):
            lens[b] -= r
            kept[b] = ([torch.cat(kept[b][0])[:lens[b]]], [torch.cat(kept[b][1])[:lens[b]]])
        assert cache.seq_lens.tolist() == lens
        used = [set(row[:-(-n // size)]) for row, n in zip(cache.block_tables.tolist(), lens)]
        free = cache.free_blocks[:int(cache.num_free)].tolist()
        assert sum(map(len, used)) + len(free) == 80 and set(free).union(*used) == set(range(80))
    return cache, last, f, w, size


def test_steps_with_drafts():
    cache, (q, new, lens, out, keys, values), f, w, size = served(6)
    at, group = 0, 2
    for b, (n, m) in enumerate(zip(new, lens)):
        p = torch.arange(m)
        qr, _ = ref.norm_rotary(q[at:at + n], w[0], 1e-6, True, ref.angles(f, p[m - n:]), False)
        kr, _ = ref.norm_rotary(keys[b], w[1], 1e-6, True, ref.angles(f, p), False)
        x = torch.einsum("qhd,khd->hqk", qr, kr.repeat_interleave(group, 1)) * 64 ** -0.5
        pr = torch.softmax(x.masked_fill(p > p[m - n:, None], -math.inf), -1)
        vv = values[b].double().repeat_interleave(group, 1)
        want = torch.einsum("hqk,khd->qhd", pr, vv)
        # keys and values have four significant bits: scores of up to 64 / 8 in size move by 2^-4 sqrt(2 / 64) of them, values by 2^-4
        got = out[at:at + n].double().cpu()
        assert float((got - want).norm() / want.norm()) < 0.12
        at += n
    # read back: keys and values as they are held
    held = cache.seq_lens.tolist()
    off = sums(held)
    key, value = cache.read(i32(off), off[-1])
    for b, m in enumerate(held):
        k, _ = ref.norm_rotary(keys[b][:m], w[1], 1e-6, True, ref.angles(f, torch.arange(m)), False)
        for got, want in ((key, k), (value, values[b][:m].double())):
            assert float((got[off[b]:off[b + 1]].cpu().double() - want).norm() / want.norm()) < 2.0 ** -4
    # what was read serves the packed operator as the cache serves the paged one
    q2 = torch.randn(off[-1], 4, 64, device=DEV).bfloat16()
    dense = G.generalized_dot_product_attention(q2, key, value, torch.tensor(off, device=DEV), torch.tensor(off, device=DEV), max(held), max(held),
                                                qk_scale=0.125, activation="softmax")
    paged = cache.attend(q2, i32(off), max(held), qk_scale=0.125)
    assert float((dense.float() - paged.float()).norm() / dense.float().norm()) < 2.0 ** -6  # both round P and O to 8 bits or more
    cache.release(range(5))
    assert int(cache.num_free) == 80


def test_training_through_norm_rotation_and_attention():
    """Gradients of norm, rotation and attention together, against autograd of the plain form in 64 bits."""
    g = torch.Generator().manual_seed(9)
    lens, heads, kv, dim = [40, 1, 130], 4, 2, 64
    q, k, v, do = (torch.randn(sum(lens), h, dim, generator=g).bfloat16() for h in (heads, kv, kv, heads))
    w = 1 + 0.2 * torch.randn(2, dim, generator=g)
    f, p = 10000.0 ** -(torch.arange(32, dtype=torch.float64) / 32), torch.cat([torch.arange(n) for n in lens])
    off = torch.tensor(sums(lens), device=DEV)
    leaves = [t.to(DEV).requires_grad_() for t in (q, k, v, w[0], w[1])]
    a, b = G.qk_norm_rotary(leaves[0], leaves[1], f.to(DEV), p.to(DEV), query_weight=leaves[3], key_weight=leaves[4])
    o = G.generalized_dot_product_attention(a, b, leaves[2], off, off, max(lens), max(lens), qk_scale=0.125, activation="softmax")
    got = [o, *torch.autograd.grad(o, leaves, do.to(DEV))]
    plain = [t.double().requires_grad_() for t in (q, k, v, w[0], w[1])]
    rot = []
    for x, wt in ((plain[0], plain[3]), (plain[1], plain[4])):
        n = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + 1e-6) * wt
        z = torch.complex(n[..., :32], n[..., 32:]) * torch.polar(torch.ones(1, dtype=torch.float64), ref.angles(f, p))[:, None]
        rot.append(torch.cat([z.real, z.imag], -1))
    outs = []
    for qq, kk, vv in zip(rot[0].split(lens), rot[1].split(lens), plain[2].split(lens)):
        s = torch.softmax(torch.einsum("qhd,khd->hqk", qq, kk.repeat_interleave(2, 1)) * 0.125, -1)
        outs.append(torch.einsum("hqk,khd->qhd", s, vv.repeat_interleave(2, 1)))
    want = [torch.cat(outs)]
    want += torch.autograd.grad(want[0], plain, do.double())
    for name, x, y in zip(("o", "dq", "dk", "dv", "dwq", "dwk"), got, want):
        # the attention's operands and P are bf16: 2^-8 each, a handful of them in a row
        assert float(((x.double().cpu() - y).norm() / y.norm()).detach()) < 8 * 2.0 ** -8, name


def test_a_step_replays_from_a_graph():
    """Tables, rotated append, attention, verification and drop captured together: replayed, they do what the calls do."""
    batch, size = 3, 16
    g = torch.Generator().manual_seed(1)
    f = (100.0 ** -(torch.arange(32, dtype=torch.float64) / 32)).to(DEV)
    q, k, v = (torch.randn(9, h, 64, generator=g).bfloat16().to(DEV) for h in (2, 1, 1))
    target, draft = (torch.softmax(torch.randn(n, 2000, generator=g), 1).to(DEV) for n in (9, 6))
    tokens, accept, sample = torch.randint(0, 2000, (6,), generator=g).to(DEV), torch.rand(6, generator=g).to(DEV) * 0.5, torch.rand(3, generator=g).to(DEV)

    def fresh():
        c = G.PagedKVCache(20, size, 1, 64, batch, 96)
        for x in (c.k_cache, c.v_cache):
            x.view(torch.uint8).fill_(0x30)
        return c

    def step(c):
        out = c.step(q, k, v, i32_new, 3, rotary=dict(inv_freq=f), qk_scale=0.125)
        verdict = G.verify_draft_tokens(target, draft, tokens, rows, drafts, accept, sample, 2)
        c.drop(verdict[2])
        return (out, *verdict)

    i32_new, rows, drafts = i32([3, 3, 3]), i32([0, 3, 6, 9]), i32([0, 2, 4, 6])
    eager = fresh()
    want = [step(eager) for _ in range(2)]
    c = fresh()
    lens, left = c.seq_lens, c.num_free  # what a replay reads
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(fresh())
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(c)
        lens.copy_(c.seq_lens)
        left.copy_(c.num_free)
    for w in want:
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(outs, w))
    assert torch.equal(lens, eager.seq_lens) and torch.equal(left, eager.num_free)
    assert torch.equal(c.k_cache.view(torch.uint8), eager.k_cache.view(torch.uint8)) and torch.equal(c.free_blocks, eager.free_blocks)


def test_large_calls_replay_from_two_graphs_on_other_streams():
    """The forms of several launches each (an append of prompts, verification and dropping of many), captured twice, replayed in turn on two streams."""
    g = torch.Generator().manual_seed(2)
    f = (100.0 ** -(torch.arange(32, dtype=torch.float64) / 32)).to(DEV)
    lens = [300, 70, 129, 1]
    q, k, v = (torch.randn(2, sum(lens), h, 64, generator=g).bfloat16().to(DEV) for h in (2, 1, 1))
    batch, vocab = 64, 66000
    target = torch.softmax(3 * torch.randn(2, 2 * batch, vocab, generator=g), 2).bfloat16().to(DEV)
    draft = torch.softmax(3 * torch.randn(2, batch, vocab, generator=g), 2).bfloat16().to(DEV)
    tokens, accept, sample = torch.randint(0, vocab, (2, batch), generator=g).to(DEV), torch.rand(2, batch, generator=g).to(DEV), torch.rand(2, batch, generator=g).to(DEV)
    rows, drafts, held = i32(list(range(0, 2 * batch + 1, 2))), i32(list(range(batch + 1))), i32([200] * 700)
    table, dropped = torch.randint(0, 10 ** 6, (2, 700, 13), generator=g, dtype=torch.int32).to(DEV), torch.randint(0, 200, (2, 700), generator=g, dtype=torch.int32).to(DEV)
    new = i32(lens)

    def call(i):
        c = G.PagedKVCache(40, 16, 1, 64, 4, 400)
        c.k_cache.view(torch.uint8).zero_(), c.v_cache.view(torch.uint8).zero_()
        out = c.step(q[i], k[i], v[i], new, 300, rotary=dict(inv_freq=f), qk_scale=0.125)
        verdict = G.verify_draft_tokens(target[i], draft[i], tokens[i], rows, drafts, accept[i], sample[i], 1)
        free = torch.zeros(9000, dtype=torch.int32, device=DEV)
        left = G.drop_cached_tokens(table[i], held, dropped[i], free, torch.zeros(1, dtype=torch.int32, device=DEV), 16)
        return (out, c.k_cache.view(torch.uint8), c.v_cache.view(torch.uint8), c.k_scales, *verdict, free, *left)

    want = [[x.clone() for x in call(i)] for i in range(2)]
    streams, graphs, outs = [torch.cuda.Stream() for _ in range(2)], [], []
    torch.cuda.synchronize()
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i], stream=streams[i]):
            outs.append(call(i))
    for _ in range(3):
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                for x in outs[i]:
                    x.view(torch.uint8).fill_(77)
                graphs[i].replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert all(torch.equal(a, b) for a, b in zip(outs[i], want[i]))


@pytest.mark.parametrize("options", [[], ["--head-dim", "64", "--block", "64", "--requests", "3", "--drafts", "1", "--kv-heads", "8"], ["--drafts", "0", "--steps", "3"]])
def test_example_serves_drafts(options):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "examples", "serve_drafts.py"), *options], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "kernel status 0" in r.stdout
