"""The paged 8-bit cache on the GPU: block tables, the quantiser and the attention against their plain 64-bit forms."""
import itertools
import math
import os
import subprocess
import sys

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from tests import _paged_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


# ------------------------------------------------------------------------------------------ block tables


def check_tables(cached, new, size, width, pool, num_free=None, extra=0, dtype=torch.int32, stride=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    batch = len(cached)
    order = torch.randperm(10 * pool + 1000, generator=g).to(torch.int32)
    free = order[:pool]
    num_free = pool if num_free is None else num_free
    table = torch.full((batch, width), -1, dtype=torch.int32)
    at = pool
    for b, c in enumerate(cached):
        n = min(-(-c // size), width)
        table[b, :n] = order[torch.arange(at, at + n) % order.numel()]
        at += n
    total = sum(new) + extra
    want = ref.tables(table, cached, new, free, num_free, size, total)
    wide = torch.full((max(batch, 1), stride or max(width, 1)), 77, dtype=torch.int32, device=DEV)
    mine = wide[:batch, :width]
    mine.copy_(table)
    slots, offsets, lens, left = G.build_block_tables(
        mine, torch.tensor(cached, dtype=dtype, device=DEV), torch.tensor(new, dtype=dtype, device=DEV), free.to(DEV), i32([num_free]), size, total)
    assert torch.equal(mine.cpu(), want[0])
    assert torch.equal(slots.cpu(), want[1])
    assert torch.equal(offsets.cpu().long(), want[2])
    assert torch.equal(lens.cpu().long(), want[3].long())
    assert int(left) == want[4]
    if stride:
        assert bool((wide[:, width:] == 77).all())


@pytest.mark.parametrize("size", [16, 32, 64, 128])
def test_tables_lengths(size):
    cached = [0, 0, 1, size - 1, size, size + 1, 5 * size, 3, 0, 700]
    new = [0, 1, 1, 1, 1, size - 1, 0, 400, 2 * size, 1]
    check_tables(cached, new, size, width=80, pool=120)
    check_tables(cached, new, size, width=80, pool=120, dtype=torch.int64, stride=91)


def test_tables_nothing():
    check_tables([], [], 16, width=4, pool=3)
    check_tables([0, 0], [0, 0], 16, width=0, pool=0)
    check_tables([5], [0], 16, width=2, pool=0, extra=7)


def test_tables_pool_runs_out():
    check_tables([0, 10, 0, 0], [100, 100, 1, 64], 16, width=9, pool=8)
    check_tables([0, 10, 0, 0], [100, 100, 1, 64], 16, width=9, pool=30, num_free=5)
    check_tables([0, 10], [100, 100], 16, width=9, pool=4, num_free=9)  # more than the stack can hold counts as all of it


def test_tables_full_rows():
    check_tables([100, 0, 64], [100, 200, 1], 16, width=4, pool=50)


@pytest.mark.parametrize("batch,most", [(1, 1), (1023, 3), (1025, 40), (8192, 2), (8193, 3), (20000, 1)])
def test_tables_many_requests(batch, most):
    g = torch.Generator().manual_seed(batch)
    cached = torch.randint(0, 60, (batch,), generator=g).tolist()
    new = torch.randint(0, most + 1, (batch,), generator=g).tolist()
    check_tables(cached, new, 16, width=8, pool=batch * 4 + 8)


def test_tables_refusals():
    ok = dict(block_tables=torch.zeros(2, 3, dtype=torch.int32, device=DEV), cached_lens=i32([1, 2]), new_lens=i32([1, 1]),
              free_blocks=i32([0, 1]), num_free=i32([2]), block_size=16, total_new=2)
    G.build_block_tables(**ok)
    for change, error in [
        (dict(block_size=24), NotImplementedError), (dict(total_new=-1), ValueError), (dict(new_lens=i32([1])), ValueError),
        (dict(new_lens=torch.tensor([1, 1], device=DEV)), TypeError), (dict(cached_lens=torch.tensor([1., 2.], device=DEV)), TypeError),
        (dict(num_free=i32([1, 1])), ValueError), (dict(free_blocks=torch.tensor([0, 1], device=DEV)), TypeError),
        (dict(block_tables=torch.zeros(3, 3, dtype=torch.int32, device=DEV)), ValueError), (dict(block_tables=torch.zeros(2, 3, device=DEV)), TypeError),
        (dict(block_tables=torch.zeros(3, 2, dtype=torch.int32, device=DEV).t()), ValueError), (dict(num_free=torch.zeros(1, dtype=torch.int32)), RuntimeError),
        (dict(cached_lens=torch.zeros(2, dtype=torch.int32)), Exception),
    ]:
        with pytest.raises(error):
            G.build_block_tables(**{**ok, **change})


# ------------------------------------------------------------------------------------------ new keys and values


def new_cache(blocks, size, heads, dim, seed=0, fill=0x7F, layout="rows"):
    """Byte-filled caches (0x7F: NaN everywhere) and scales; "heads" has the heads before the rows in memory."""
    def one():
        if layout == "heads":
            return torch.full((blocks, heads, size, dim), fill, dtype=torch.uint8, device=DEV).transpose(1, 2)
        return torch.full((blocks, size, heads, dim), fill, dtype=torch.uint8, device=DEV)

    return one(), one(), torch.full((blocks, heads), math.nan, device=DEV), torch.full((blocks, heads), math.nan, device=DEV)


def check_append(x, slots, cache):
    k, v, ks, vs = cache
    want = []
    for t, c, s in ((x[0], k, ks), (x[1], v, vs)):
        c, s = c.cpu().contiguous(), s.cpu().double()
        ref.append(t.detach().cpu(), c, s, slots)
        want.append((c, s))
    G.append_kv_cache_fp8(x[0], x[1], k.view(torch.float8_e4m3fn), v.view(torch.float8_e4m3fn), ks, vs, slots.to(DEV))
    touched = torch.unique(slots[(slots >= 0) & (slots < k.shape[0] * k.shape[1])] // k.shape[1])
    for (c, s), mine, scale in ((want[0], k, ks), (want[1], v, vs)):
        assert torch.equal(scale.cpu()[touched].double(), s[touched])
        got, c = mine.cpu().contiguous(), c.contiguous()
        nan = lambda b: (b & 0x7F) == 0x7F  # noqa: E731  (a NaN's sign says nothing)
        assert torch.equal(torch.where(nan(got), 0x7F, got), torch.where(nan(c), 0x7F, c))


def values(tokens, heads, dim, dtype, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return [(torch.randn(tokens, heads, dim, generator=g) * std).to(dtype).to(DEV) for _ in range(2)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("dim,size", [(64, 16), (64, 128), (128, 16), (128, 128)])
def test_append_runs(dtype, dim, size):
    # whole blocks, a block begun, a block ended, single tokens, skipped tokens between runs, slots beyond the cache
    cache = new_cache(9, size, 3, dim)
    first = torch.cat([torch.arange(4 * size, 5 * size), torch.arange(0, size // 2), torch.arange(2 * size, 3 * size), torch.tensor([7 * size])])
    check_append(values(len(first), 3, dim, dtype, 1), first, cache)
    second = torch.cat([torch.arange(size // 2, size), torch.tensor([7 * size + 1, 7 * size + 2, -1, 9 * size, 10 ** 12]), torch.arange(8 * size, 8 * size + 3)])
    check_append(values(len(second), 3, dim, dtype, 2, std=30.0), second, cache)  # ten times larger: the scales grow
    third = torch.tensor([8 * size + 3, 7 * size + 3])
    check_append(values(2, 3, dim, dtype, 3, std=0.01), third, cache)  # smaller: they stay


@pytest.mark.parametrize("tokens", [1, 31, 32, 33, 300])
def test_append_one_token_each(tokens):
    size = 16
    cache = new_cache(tokens, size, 2, 128)
    order = torch.randperm(tokens, generator=torch.Generator().manual_seed(tokens))
    for row in range(3):
        check_append(values(tokens, 2, 128, torch.bfloat16, row, std=2.0 ** row), order * size + row, cache)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_append_odd_values(dtype):
    size, dim = 16, 64
    k, v = values(8 * size, 1, dim, dtype, 5)
    big = 3.0e38
    k[0 * size:1 * size] = 0
    k[1 * size, 0, 3], k[1 * size + 1, 0, 4] = math.inf, -math.inf
    k[2 * size + 2, 0, 5] = math.nan
    k[3 * size:4 * size] = math.nan
    k[4 * size:5 * size] *= 1e-36
    k[5 * size, 0, 0] = big
    k[6 * size:7 * size] = 448.0
    k[7 * size:8 * size] = -0.0
    v[0 * size:1 * size] = torch.arange(size)[:, None, None].to(dtype) * 1.75
    check_append([k, v], torch.arange(8 * size), new_cache(8, size, 1, dim))


def test_append_strided_and_long_runs():
    # K and V interleaved along the last dimension, heads before rows in the cache, runs that cross windows of 32 tokens
    size, dim, heads, tokens = 128, 128, 2, 517
    kv = torch.randn(tokens, heads, 2 * dim, generator=torch.Generator().manual_seed(0)).bfloat16().to(DEV)
    cache = new_cache(7, size, heads, dim, layout="heads")
    check_append([kv[:, :, :dim], kv[:, :, dim:]], torch.arange(tokens) + 37, cache)


def test_append_token_by_token_is_append_at_once():
    size, dim, tokens = 32, 64, 40
    k, v = values(tokens, 2, dim, torch.bfloat16, 9, std=3.0)
    a, b = new_cache(2, size, 2, dim), new_cache(2, size, 2, dim)
    slots = torch.arange(tokens, device=DEV)
    args = lambda c: (c[0].view(torch.float8_e4m3fn), c[1].view(torch.float8_e4m3fn), c[2], c[3])  # noqa: E731
    G.append_kv_cache_fp8(k, v, *args(a), slots)
    for t in range(tokens):
        G.append_kv_cache_fp8(k[t:t + 1], v[t:t + 1], *args(b), slots[t:t + 1])
    assert torch.equal(a[2], b[2]) and torch.equal(a[3], b[3])
    for x, y, s in ((a[0], b[0], a[2]), (a[1], b[1], a[3])):
        x, y = (t.reshape(-1, 2, dim)[:tokens].view(torch.float8_e4m3fn).double() for t in (x, y))
        assert float((x - y).abs().max()) <= 2.0 ** -9  # one step of e4m3's subnormals, in units of the scale


def test_append_far_into_a_large_cache():
    # more than 2^32 bytes from the cache's first block
    size, heads, dim, blocks = 128, 4, 128, 66000
    k8 = torch.empty(blocks, size, heads, dim, dtype=torch.uint8, device=DEV)
    scales = torch.ones(blocks, heads, device=DEV)
    k, v = values(130, heads, dim, torch.bfloat16)
    slots = torch.arange(130) + (blocks - 2) * size
    v8, vs = k8.clone(), scales.clone()
    G.append_kv_cache_fp8(k, v, k8.view(torch.float8_e4m3fn), v8.view(torch.float8_e4m3fn), scales, vs, slots.to(DEV))
    tail, s = torch.zeros(2, size, heads, dim, dtype=torch.uint8), torch.ones(2, heads, dtype=torch.float64)
    ref.append(k.cpu(), tail, s, torch.arange(130))
    assert torch.equal(k8[-2:].reshape(-1, heads, dim)[:130].cpu(), tail.reshape(-1, heads, dim)[:130])
    # and the attention that reads it there
    q = values(2, heads, dim, torch.bfloat16, 3)[0]
    table = i32([[blocks - 2, blocks - 1]])
    o = G.generalized_dot_product_attention_paged_fp8(q, k8.view(torch.float8_e4m3fn), v8.view(torch.float8_e4m3fn), scales, vs, table, i32([0, 2]),
                                                      i32([130]), 2, qk_scale=0.1)
    want, tol = ref.attend(q.cpu(), k8[-2:].cpu(), v8[-2:].cpu(), scales[-2:].cpu(), vs[-2:].cpu(), torch.tensor([[0, 1]]), [0, 2], [130], 0.1, "softmax")
    assert bool(((o.cpu().double() - want).abs() <= tol).all())


def test_append_refusals():
    k, v = values(4, 2, 64, torch.bfloat16)
    c = new_cache(3, 16, 2, 64)
    f8 = torch.float8_e4m3fn
    ok = dict(key=k, value=v, k_cache=c[0].view(f8), v_cache=c[1].view(f8), k_scales=c[2], v_scales=c[3], slot_mapping=torch.arange(4, device=DEV))
    G.append_kv_cache_fp8(**ok)
    for change, error in [
        (dict(key=k.half()), TypeError), (dict(value=v.float()), TypeError), (dict(key=k[:3]), ValueError), (dict(key=k[:, :1], value=v[:, :1]), ValueError),
        (dict(key=k.transpose(1, 2).contiguous().transpose(1, 2)), ValueError), (dict(k_cache=c[0]), TypeError),
        (dict(k_cache=c[0].view(f8)[:, :8], v_cache=c[1].view(f8)[:, :8]), NotImplementedError), (dict(v_cache=c[1].view(f8)[:2]), ValueError),
        (dict(k_scales=c[2].double()), TypeError), (dict(k_scales=c[2][:2]), ValueError), (dict(v_scales=c[3].cpu()), RuntimeError),
        (dict(slot_mapping=i32([0, 1, 2, 3])), TypeError), (dict(slot_mapping=torch.arange(3, device=DEV)), ValueError),
        (dict(k_cache=c[0].view(f8)[..., :32], v_cache=c[1].view(f8)[..., :32]), NotImplementedError),
    ]:
        with pytest.raises(error):
            G.append_kv_cache_fp8(**{**ok, **change})
    old = G.set_offset_validation(True)
    try:
        G.append_kv_cache_fp8(**ok)
        with pytest.raises(ValueError):  # two runs of one block
            G.append_kv_cache_fp8(**{**ok, "slot_mapping": torch.tensor([0, 1, 16, 2], device=DEV)})
    finally:
        G.set_offset_validation(old)


# ------------------------------------------------------------------------------------------ attention


class Case:
    """Requests with caches of random values whose unused rows, blocks and scales are NaN."""

    def __init__(self, lens, q_lens, heads, kv_heads, dim, size, seed=0, q_std=1.0, block_std=0.3, layout="rows", spare_width=0):
        g = torch.Generator().manual_seed(seed)
        self.lens, self.dim, self.size = lens, dim, size
        n_blocks = [-(-n // size) for n in lens]
        blocks = sum(n_blocks) + 2
        order = torch.randperm(blocks, generator=g)
        self.table = torch.full((len(lens), max(n_blocks + [1]) + spare_width), -1, dtype=torch.int32)
        self.k = torch.full((blocks, size, kv_heads, dim), 0x7F, dtype=torch.uint8)
        self.v = self.k.clone()
        self.ks = torch.full((blocks, kv_heads), math.nan)
        self.vs = self.ks.clone()
        at = 0
        for b, n in enumerate(lens):
            for j in range(n_blocks[b]):
                blk = int(order[at])
                at += 1
                self.table[b, j] = blk
                rows = min(size, n - j * size)
                for c, s in ((self.k, self.ks), (self.v, self.vs)):
                    x = torch.randn(rows, kv_heads, dim, generator=g) * torch.exp(block_std * torch.randn(1, kv_heads, 1, generator=g))
                    for h in range(kv_heads):
                        s[blk, h] = ref.least_scale(x[:, h])
                    c[blk, :rows] = ref.e4m3_bytes(x.double() / s[blk].double()[None, :, None])
        self.offsets = [0] + list(itertools.accumulate(q_lens))
        self.max_q = max(q_lens + [0])
        self.q = (torch.randn(self.offsets[-1], heads, dim, generator=g) * q_std).bfloat16()
        self.layout = layout

    def device(self, cache):
        if self.layout == "heads":
            return cache.transpose(1, 2).contiguous().to(DEV).transpose(1, 2).view(torch.float8_e4m3fn)
        return cache.to(DEV).view(torch.float8_e4m3fn)

    def run(self, scale, activation, causal=False, window=None, q=None, dtype=torch.int32, max_q=None):
        q = self.q.to(DEV) if q is None else q
        return G.generalized_dot_product_attention_paged_fp8(
            q, self.device(self.k), self.device(self.v), self.ks.to(DEV), self.vs.to(DEV), self.table.to(DEV),
            torch.tensor(self.offsets, dtype=dtype, device=DEV), torch.tensor(self.lens, dtype=dtype, device=DEV), max_q or self.max_q, qk_scale=scale,
            activation=activation, is_causal=causal, window_size=window)

    def want(self, scale, activation, causal=False, window=None):
        return ref.attend(self.q, self.k, self.v, self.ks, self.vs, self.table, self.offsets, self.lens, scale, activation, causal, window)

    def check(self, scale, activation, causal=False, window=None, **how):
        o = self.run(scale, activation, causal, window, **how).cpu().double()
        assert G.kernel_status() == 0
        want, tol = self.want(scale, activation, causal, window)
        assert bool(torch.isfinite(o).all())
        over = (o - want).abs() - tol
        assert float(over.max() if over.numel() else 0) <= 0, f"{int((over > 0).sum())} of {over.numel()} elements too far, worst by {float(over.max()):.3g}"
        return o


@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_one_token(dim, size):
    lens = [0, 1, 15, 16, 17, 127, 128, 129, 255, 300, 1000, 1]
    Case(lens, [1] * len(lens), 8, 2, dim, size).check(dim ** -0.5, "softmax")


@pytest.mark.parametrize("heads,kv_heads", [(1, 1), (3, 1), (10, 2), (8, 8), (16, 1), (17, 1), (32, 1), (48, 1)])
def test_attend_head_groups(heads, kv_heads):
    Case([70, 400], [1, 1], heads, kv_heads, 64, 32).check(0.125, "softmax")
    Case([70, 400], [3, 2], heads, kv_heads, 64, 32, seed=1).check(0.125, "softmax", causal=True)


@pytest.mark.parametrize("activation", sorted(ref.ACT))
@pytest.mark.parametrize("dim", [64, 128])
def test_attend_activations(activation, dim):
    Case([300, 129, 1], [1, 1, 1], 4, 2, dim, 64).check(1 / 300, activation)
    Case([300, 129, 60], [30, 129, 70], 4, 2, dim, 64, q_std=0.5).check(1 / 300, activation)


@pytest.mark.parametrize("activation", ["softmax", "silu"])
@pytest.mark.parametrize("q_lens", [[0, 5, 1], [16, 17, 15], [64, 0, 33], [128, 130, 7], [300, 1, 257]])
def test_attend_many_queries(q_lens, activation):
    scale = 0.1 if activation == "softmax" else 1 / 500
    Case([500, 129, 31], q_lens, 4, 2, 128, 32).check(scale, activation)
    Case([500, 129, 31], q_lens, 4, 2, 64, 32, seed=1).check(scale, activation)


@pytest.mark.parametrize("dim", [64, 128])
def test_attend_many_queries_over_long_histories(dim):
    # items of more tiles than the kernels have stages, one after another in a CTA
    Case([3000, 2500, 1700], [130, 257, 100], 4, 2, dim, 64).check(0.1, "softmax", causal=True)
    Case([2000] * 3, [40, 64, 33], 32, 32, dim, 128).check(1 / 2000, "relu")


@pytest.mark.parametrize("tokens", [1, 64, 129, 300, 640, 1000])
def test_attend_less_work_than_ctas(tokens):
    # items whose tiles go to as many CTAs, with CTAs over that have none
    for q, dim in ((70, 128), (300, 64)):
        Case([tokens], [q], 1, 1, dim, 16).check(0.1, "softmax")
        Case([tokens, 1], [q, 90], 2, 1, dim, 128).check(0.01, "silu", causal=True)
    Case([tokens], [1], 1, 1, 128, 16).check(0.1, "softmax")
    Case([tokens], [20], 1, 1, 64, 16).check(0.1, "softmax")


def test_attend_growing_scores():
    # references that have to move again and again, by a little and past any of the formats' ranges; V scales far apart
    for q_len, dim in ((1, 128), (3, 64), (90, 128), (150, 64)):
        case = Case([1500], [q_len], 2, 1, dim, 16, seed=q_len)
        blocks = case.table[0, : -(-1500 // 16)].long()
        case.ks[blocks, 0] *= torch.exp2(torch.arange(len(blocks)) // 24).to(case.ks.dtype)
        case.vs[blocks, 0] *= torch.exp2(torch.arange(len(blocks)) % 5 * 4 - 8).to(case.vs.dtype)
        case.check(0.05, "softmax")
        case.check(0.05, "softmax", causal=True)
        case.check(1e-4, "relu_square")
        case.check(1e-4, "silu")


@pytest.mark.parametrize("window", [None, 0, 1, 100, 128, 5000])
@pytest.mark.parametrize("causal", [False, True])
def test_attend_masks(causal, window):
    # more queries than keys: rows without keys, and whole row tiles without them
    lens, q_lens = [600, 40, 1, 0, 257], [5, 90, 3, 4, 257]
    for dim, activation in ((128, "softmax"), (64, "softmax"), (128, "silu")):
        case = Case(lens, q_lens, 4, 2, dim, 16, seed=dim)
        o = case.check(0.1 if activation == "softmax" else 0.01, activation, causal, window)
        if causal:
            assert bool((o[5:5 + 50] == 0).all())  # positions before the first key
    Case(lens, [1] * 5, 4, 2, 128, 64).check(0.1, "softmax", causal, window)
    Case(lens, [4, 3, 2, 1, 4], 4, 2, 64, 128).check(0.1, "softmax", causal, window)


def test_attend_layouts_and_types():
    case = Case([300, 129], [3, 40], 4, 2, 128, 64, layout="heads", spare_width=3)
    case.check(0.1, "softmax", causal=True)
    case.check(0.1, "softmax", causal=True, dtype=torch.int64)
    packed = torch.zeros(43, 4, 384, dtype=torch.bfloat16, device=DEV)
    packed[:, :, 128:256] = case.q.to(DEV)
    case.check(0.1, "softmax", q=packed[:, :, 128:256])
    case.check(0.1, "softmax", max_q=1000)
    # the table as a slice of a wider one
    wide = torch.zeros(2, 50, dtype=torch.int32)
    wide[:, 7:7 + case.table.shape[1]] = case.table
    plain = case.run(0.1, "softmax")
    case.table = wide[:, 7:7 + case.table.shape[1]]
    sliced = G.generalized_dot_product_attention_paged_fp8(
        case.q.to(DEV), case.device(case.k), case.device(case.v), case.ks.to(DEV), case.vs.to(DEV), wide.to(DEV)[:, 7:7 + case.table.shape[1]],
        i32(case.offsets), i32(case.lens), case.max_q, qk_scale=0.1)
    assert torch.equal(plain, sliced)


def test_attend_split_over_many_ctas():
    # one head: every CTA has a piece of the one item; then a few heads, whose pieces end inside tiles of others
    Case([30000], [1], 8, 1, 128, 128).check(0.3, "softmax")
    Case([20000, 300], [2, 1], 4, 1, 64, 16).check(0.3, "softmax", causal=True)
    Case([5000, 9000, 3], [1, 1, 1], 4, 2, 128, 64).check(1 / 9000, "silu")
    Case([5000, 700], [100, 60], 2, 1, 128, 64).check(0.2, "softmax", causal=True)


@pytest.mark.parametrize("q_lens", [[1, 1], [40, 40]])
def test_attend_rising_scores(q_lens):
    # every tile holds larger scores than the ones before, then smaller: the reference of the rows moves at each, then stays
    case = Case([900, 900], q_lens, 4, 2, 128, 32, block_std=0.0)
    direction = torch.randn(128, generator=torch.Generator().manual_seed(3))
    case.q = (direction + 0.05 * torch.randn(case.q.shape, generator=torch.Generator().manual_seed(4))).bfloat16()
    for b in range(2):
        for j in range(900):
            blk, row = int(case.table[b, j // 32]), j % 32
            amount = (j if b == 0 else 900 - j) / 900
            x = direction * amount * 0.7
            case.ks[blk] = 2.0 ** -8
            case.k[blk, row] = ref.e4m3_bytes(x.double() / 2.0 ** -8)
    case.check(0.5, "softmax")
    case.check(0.01, "relu_square")


@pytest.mark.parametrize("q_lens", [[1, 1], [40, 30]])
def test_attend_uneven_scales(q_lens):
    # blocks whose values differ by powers of ten, rows of Q too
    case = Case([700, 300], q_lens, 4, 2, 128, 32, block_std=6.0)
    case.ks = torch.where(case.ks.isnan(), case.ks, torch.full_like(case.ks, 2.0 ** -8))
    case.check(0.1, "softmax")
    case.check(0.01, "relu")
    case.q[::2] *= 1024.0
    case.check(0.0001, "softmax")
    case.check(0.01, "raw")


def test_attend_missing_blocks():
    # a block that the table has not takes no part, as if its tokens were not there
    case = Case([200, 130], [1, 40], 4, 2, 64, 16)
    whole = case.table.clone()
    case.table[0, 3] = -1
    case.table[0, 5] = 10 ** 6
    case.table[1, 0] = -5
    got = case.run(0.2, "softmax").cpu().double()
    for b, gone in ((0, (3, 5)), (1, (0,))):
        keep = [j for j in range(-(-case.lens[b] // 16)) if j not in gone]
        n = case.lens[b] - 16 * len(gone)
        lo, hi = case.offsets[b], case.offsets[b + 1]
        want, tol = ref.attend(case.q[lo:hi], case.k, case.v, case.ks, case.vs, whole[b:b + 1, keep], [0, hi - lo], [n], 0.2, "softmax")
        assert bool(((got[lo:hi] - want).abs() <= tol).all())
    assert G.kernel_status() == 0


@pytest.mark.parametrize("activation", ["softmax", "silu"])
def test_attend_nan_stays_where_it_is(activation):
    case = Case([200, 200], [20, 20], 4, 2, 128, 64)
    clean = case.run(0.1, activation, causal=True)
    blk = int(case.table[0, 190 // 64])
    case.v[blk, 190 % 64, 0, 5] = 0x7F  # V of position 190, K / V head 0: queries 10 .. 19 of request 0, heads 0 and 1
    dirty = case.run(0.1, activation, causal=True)
    assert torch.equal(dirty[:10], clean[:10]) and torch.equal(dirty[20:], clean[20:]) and torch.equal(dirty[:, 2:], clean[:, 2:])
    assert bool(dirty[10:20, :2, 5].isnan().all())
    case.v[blk, 190 % 64, 0, 5] = 0
    case.k[blk, 190 % 64, 0, 5] = 0xFF
    dirty = case.run(0.1, activation, causal=True)
    assert torch.equal(dirty[:10], clean[:10]) and torch.equal(dirty[20:], clean[20:]) and torch.equal(dirty[:, 2:], clean[:, 2:])
    assert bool(dirty[10:20, :2].isnan().all())


def test_attend_odd_queries():
    case = Case([200, 100], [3, 40], 4, 2, 128, 64)
    clean = case.run(0.1, "softmax")
    case.q[1, 2, 7] = math.nan
    case.q[10, 0, 0] = math.inf
    case.q[20] = 0
    dirty = case.run(0.1, "softmax")
    rows = torch.ones(43, 4, dtype=torch.bool)
    rows[1, 2] = rows[10, 0] = False
    assert bool(dirty[1, 2].isnan().all()) and bool(dirty[10, 0].isnan().all())
    rows[20] = False
    assert torch.equal(dirty[rows], clean[rows])
    case.q[1, 2, 7] = case.q[10, 0, 0] = 1.0
    case.check(0.1, "softmax")


def test_attend_many_short_requests():
    g = torch.Generator().manual_seed(0)
    lens = torch.randint(0, 40, (3000,), generator=g).tolist()
    Case(lens, torch.randint(0, 3, (3000,), generator=g).tolist(), 2, 1, 64, 16).check(0.2, "softmax", causal=True)


def test_attend_twice_is_the_same_and_streams():
    case = Case([3000, 10, 700], [1, 1, 1], 8, 2, 128, 64)
    args = (case.q.to(DEV), case.device(case.k), case.device(case.v), case.ks.to(DEV), case.vs.to(DEV), case.table.to(DEV), i32(case.offsets), i32(case.lens))
    first = G.generalized_dot_product_attention_paged_fp8(*args, 1, qk_scale=0.1)
    for _ in range(20):
        assert torch.equal(first, G.generalized_dot_product_attention_paged_fp8(*args, 1, qk_scale=0.1))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    for i in range(12):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(G.generalized_dot_product_attention_paged_fp8(*args, 1, qk_scale=0.1))
    torch.cuda.synchronize()
    assert all(torch.equal(first, o) for o in outs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = G.generalized_dot_product_attention_paged_fp8(*args, 1, qk_scale=0.1)
    for _ in range(3):
        out.zero_()
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(first, out)
    assert G.kernel_status() == 0


def test_attend_nothing():
    q = torch.zeros(0, 4, 64, dtype=torch.bfloat16, device=DEV)
    c = new_cache(2, 16, 2, 64)
    f8 = torch.float8_e4m3fn
    empty = torch.zeros(0, 3, dtype=torch.int32, device=DEV)
    o = G.generalized_dot_product_attention_paged_fp8(q, c[0].view(f8), c[1].view(f8), c[2], c[3], empty, i32([0]), i32([]), 0)
    assert o.shape == (0, 4, 64)
    # no block at all, and a table without columns
    q = torch.ones(2, 4, 64, dtype=torch.bfloat16, device=DEV)
    o = G.generalized_dot_product_attention_paged_fp8(q, c[0][:0].view(f8), c[1][:0].view(f8), c[2][:0], c[3][:0],
                                                      torch.zeros(1, 0, dtype=torch.int32, device=DEV), i32([0, 2]), i32([5]), 2)
    assert bool((o == 0).all()) and G.kernel_status() == 0


def test_attend_refusals():
    case = Case([40, 3], [1, 2], 4, 2, 64, 16)
    f8 = torch.float8_e4m3fn
    ok = dict(query=case.q.to(DEV), k_cache=case.device(case.k), v_cache=case.device(case.v), k_scales=case.ks.to(DEV), v_scales=case.vs.to(DEV),
              block_tables=case.table.to(DEV), query_offset=i32(case.offsets), seq_lens=i32(case.lens), max_seq_len_q=2)
    run = G.generalized_dot_product_attention_paged_fp8
    run(**ok)
    for change, error in [
        (dict(query=ok["query"].float()), TypeError), (dict(query=ok["query"][:, :3].contiguous()), ValueError), (dict(query=ok["query"][:, :, ::2]), ValueError),
        (dict(query=torch.zeros(3, 4, 128, dtype=torch.bfloat16, device=DEV)), ValueError), (dict(query=case.q), Exception),
        (dict(k_cache=ok["k_cache"].view(torch.uint8)), TypeError), (dict(v_scales=ok["v_scales"].cpu()), RuntimeError),
        (dict(block_tables=ok["block_tables"].long()), TypeError), (dict(block_tables=ok["block_tables"][:1]), ValueError),
        (dict(query_offset=i32([0, 1])), ValueError), (dict(seq_lens=ok["seq_lens"].float()), TypeError), (dict(max_seq_len_q=-1), ValueError),
        (dict(activation="nonsense"), ValueError), (dict(k_cache=torch.zeros(4, 24, 2, 64, dtype=torch.uint8, device=DEV).view(f8),
                                                         v_cache=torch.zeros(4, 24, 2, 64, dtype=torch.uint8, device=DEV).view(f8)), NotImplementedError),
    ]:
        with pytest.raises(error):
            run(**{**ok, **change})
    old = G.set_offset_validation(True)
    try:
        run(**ok)
        with pytest.raises(ValueError):
            run(**{**ok, "seq_lens": i32([40, -1])})
        with pytest.raises(ValueError):
            run(**{**ok, "query_offset": i32([0, 2, 9])})
    finally:
        G.set_offset_validation(old)
    q = ok["query"].clone().requires_grad_(True)
    o = run(**{**ok, "query": q})
    if o.requires_grad:
        with pytest.raises(RuntimeError):
            o.sum().backward()


def test_malformed_lengths_stay_inside():
    # values of such requests are unspecified; the others' are right and nothing outside the tensors is touched
    case = Case([300, 129, 60], [1, 1, 1], 4, 2, 64, 16)
    good = case.run(0.1, "softmax")
    case.lens = [300, 1 << 30, -7]
    o = case.run(0.1, "softmax")
    assert torch.equal(o[0], good[0]) and bool((o[2] == 0).all()) and G.kernel_status() == 0


# ------------------------------------------------------------------------------------------ all together


def test_cache_steps_and_release():
    torch.manual_seed(0)
    heads, kv_heads, dim, size, batch = 8, 2, 64, 16, 5
    cache = G.PagedKVCache(40, size, kv_heads, dim, batch, 128)
    cpu = dict(k=[[] for _ in range(batch)], v=[[] for _ in range(batch)])
    steps = [[20, 0, 33, 1, 16], [1, 5, 1, 1, 1], [1, 1, 1, 1, 1]]
    for new in steps:
        q, k, v = (torch.randn(sum(new), h, dim, device=DEV).bfloat16() for h in (heads, kv_heads, kv_heads))
        o = cache.step(q, k, v, i32(new), max(new), qk_scale=0.125)
        offsets = [0] + list(itertools.accumulate(new))
        lens = cache.seq_lens.tolist()
        want, tol = ref.attend(q.cpu(), cache.k_cache.view(torch.uint8).cpu(), cache.v_cache.view(torch.uint8).cpu(), cache.k_scales.cpu(), cache.v_scales.cpu(),
                               cache.block_tables.cpu(), offsets, lens, 0.125, "softmax", causal=True)
        assert bool(((o.cpu().double() - want).abs() <= tol).all())
        for b in range(batch):
            cpu["k"][b].append(k[offsets[b]:offsets[b + 1]].cpu())
    # what the cache holds is what was put in, to e4m3's precision (2^-4 of a value, a 2^-10 of the scale below its normal values)
    for b in range(batch):
        k = torch.cat(cpu["k"][b]).double()
        x, s = ref.gather(cache.k_cache.view(torch.uint8).cpu(), cache.k_scales.cpu(), cache.block_tables[b].cpu(), len(k))
        assert bool(((x * s[..., None] - k).abs() <= 2.0 ** -4 * k.abs() + 2.0 ** -9 * s[..., None]).all())
    used = sum(-(-n // size) for n in cache.seq_lens.tolist())
    assert int(cache.num_free) == 40 - used
    held = set(cache.block_tables[[0, 2]].flatten().tolist()) - {-1}
    cache.release([0, 2])
    free = set(cache.free_blocks[: int(cache.num_free)].tolist())
    assert len(free) == int(cache.num_free) == 40 - used + len(held) and held <= free
    assert cache.seq_lens.tolist()[0] == 0 and bool((cache.block_tables[[0, 2]] == -1).all())
    new = [40, 1, 50, 1, 1]
    q, k, v = (torch.randn(sum(new), h, dim, device=DEV).bfloat16() for h in (heads, kv_heads, kv_heads))
    cache.step(q, k, v, i32(new), max(new))
    table = cache.block_tables[cache.block_tables >= 0].tolist()
    assert len(table) == len(set(table)) == 40 - int(cache.num_free)


def test_operators_trace():
    case = Case([40, 3], [1, 2], 4, 2, 64, 16)
    args = (case.q.to(DEV), case.device(case.k), case.device(case.v), case.ks.to(DEV), case.vs.to(DEV), case.table.to(DEV), i32(case.offsets), i32(case.lens), 2,
            0.1, 100, True, -1)
    # (test_schema multiplies its arguments, which torch cannot for e4m3)
    torch.library.opcheck(torch.ops.gdpa.generalized_dot_product_attention_paged_fp8.default, args, test_utils=("test_faketensor",))
    tables = (torch.full((2, 3), -1, dtype=torch.int32, device=DEV), i32([1, 2]), i32([1, 30]), i32([0, 1, 2, 3]), i32([4]), 16, 31)
    torch.library.opcheck(torch.ops.gdpa.build_block_tables.default, tables, test_utils=("test_schema", "test_faketensor"))


@pytest.mark.parametrize("options", [[], ["--activation", "silu", "--head-dim", "64", "--block", "16", "--requests", "5", "--most-tokens", "300"]])
def test_example_serves(options):
    # one bound on the error for both: uniform rounding of four significant bits leaves 2^-4 / sqrt(12) of a key's or value's size, 0.03 together
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, os.path.join(root, "examples", "serve_paged.py"), *options], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "kernel status 0" in r.stdout
