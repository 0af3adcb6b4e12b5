"""Edges of the paged 8-bit cache on the GPU: batches and values at which its operators can go wrong."""
import os
import subprocess
import sys

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from ads_model_kernel_library_b200.gdpa import ops
from tests import _paged_oracle as ref
from tests._paged_batches import Batch

pytestmark = pytest.mark.gpu
DEV = "cuda"


# ------------------------------------------------------------------------------------------ requests without keys


def lengths(batch, most, empty, seed):
    lens = torch.randint(1, most + 1, (batch,), generator=torch.Generator().manual_seed(seed)).tolist()
    for b in empty:
        lens[b] = 0
    return lens


def check_empty_requests(lens, q_lens, heads, kv_heads, dim, size, **options):
    batch = Batch(lens, q_lens, heads, kv_heads, dim, size)
    o = batch.check(0.1, **options)
    for b, n in enumerate(lens):
        if n == 0:
            assert bool((o[batch.offsets[b]:batch.offsets[b + 1]] == 0).all())


@pytest.mark.parametrize("empty", [[0], [100], [255], [0, 1, 2, 3, 4], [7, 100, 101, 102, 254], [251, 252, 253, 254, 255]])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 8, 128), (4, 4, 64)])
def test_empty_requests_in_a_large_batch(heads, kv_heads, dim, empty):
    # an empty request has an item without keys for each of its K / V heads, one after the other, behind items with keys in the same CTA
    check_empty_requests(lengths(256, 4096 if dim == 64 else 1500, empty, len(empty)), [1] * 256, heads, kv_heads, dim, 64)


@pytest.mark.parametrize("queries", [1, 5, 40])
@pytest.mark.parametrize("dim", [64, 128])
def test_runs_of_empty_requests(dim, queries):
    # between requests of some 400 tokens runs of 1 to 8 without a key, whose queries are there; row tiles of 16, 64 and 256
    lens, q_lens = [], []
    for i in range(300):
        lens += [300 + i % 200] + [0] * (i % 9)
        q_lens += [queries] + [1 + i % queries] * (i % 9)
    check_empty_requests(lens, q_lens, 16, 8, dim, 32)


@pytest.mark.parametrize("queries", [1, 20])
def test_positions_before_the_first_key(queries):
    # causal, more queries than tokens: whole row tiles without a key in requests that have some
    lens = [(50 * b) % 700 for b in range(200)]
    check_empty_requests(lens, [queries if n % 100 else 64 for n in lens], 4, 4, 64, 16, causal=True)


# ------------------------------------------------------------------------------------------ tensors that share their memory


def test_expanded_inputs_are_refused():
    f8, tokens, heads, dim = torch.float8_e4m3fn, 6, 4, 64
    cache = [torch.zeros(2, 16, heads, dim, dtype=torch.uint8, device=DEV).view(f8) for _ in range(2)] + [torch.ones(2, heads, device=DEV) for _ in range(2)]
    slots = torch.arange(tokens, device=DEV)
    full = torch.randn(tokens, heads, dim, device=DEV).bfloat16()
    row = torch.randn(tokens * heads * dim, device=DEV).bfloat16()
    shared = [full[:, :1].expand(-1, heads, -1),                            # one head for all
              full[:1].expand(tokens, -1, -1),                              # one token for all
              full[:1, :1].expand(tokens, heads, -1),
              torch.as_strided(row, (tokens, heads, dim), (heads * dim, dim // 2, 1))]  # heads that overlap
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    attend = lambda q: G.generalized_dot_product_attention_paged_fp8(q, *cache, i32([[0, 1]]), i32([0, tokens]), i32([20]), tokens)  # noqa: E731
    for x in shared:
        for key, value in ((x, full), (full, x)):
            with pytest.raises(ValueError):
                G.append_kv_cache_fp8(key, value, *cache, slots)
        with pytest.raises(ValueError):
            attend(x)
        assert torch.isfinite(attend(x.contiguous())).all()
    # a dimension of one entry has no stride that matters
    one = full[:1, :1].expand(1, 1, dim)
    narrow = [c[:, :, :1] for c in cache[:2]] + [c[:, :1].contiguous() for c in cache[2:]]
    G.append_kv_cache_fp8(one, one, *narrow, slots[:1])
    # the heads before the tokens in memory
    swapped = full.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(attend(swapped), attend(full))


def test_a_shared_table_is_read_but_not_written():
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    table = i32([[0, 1, -1]]).expand(3, -1)
    with pytest.raises(ValueError):
        G.build_block_tables(table, i32([5, 5, 5]), i32([1, 1, 1]), i32([2, 3]), i32([2]), 16, 3)
    batch = Batch([30], [2], 4, 2, 64, 16)
    alone = batch.run(0.1)
    batch.lens, batch.offsets, batch.q, batch.table = [30] * 3, [0, 2, 4, 6], batch.q.repeat(3, 1, 1), batch.table.expand(3, -1)
    assert torch.equal(batch.run(0.1), alone.repeat(3, 1, 1))


# ------------------------------------------------------------------------------------------ one key far ahead of the others


def peaked(gap, tokens, queries, heads, kv_heads, dim, seed=0, tail=None):
    """A batch of one request whose token `tokens // 3` is `gap` (a softmax's scale included) ahead of the others' mean, with values of zero; the
    others' scores are normal, or all the same, and their values positive."""
    batch = Batch([tokens], [queries], heads, kv_heads, dim, 64, seed=seed)
    g = torch.Generator(device=DEV).manual_seed(seed + 1)
    u = torch.randint(0, 2, (dim,), generator=g, device=DEV) * 2.0 - 1
    batch.q = (u + 0.02 * torch.randn(batch.q.shape, generator=g, device=DEV)).bfloat16()
    batch.v = (batch.v & 0x7F) if tail is None else torch.full_like(batch.v, 0x38)  # |v|, or ones (times the scale)
    if tail is not None:
        batch.k[:] = 0
    at = tokens // 3
    blk, row = int(batch.table[0, at // 64]), at % 64
    batch.k[blk, row] = (u * gap / dim ** 0.5 * 64).to(torch.float8_e4m3fn).view(torch.uint8)
    batch.v[blk, row] = 0
    return batch


def check_copies(batch, copies, scale, activation="softmax"):
    """One request many times over, so that a CTA goes through a whole history (one alone is cut into pieces, each with a reference of its own)."""
    want, tol = batch.want(scale, activation)
    queries = len(batch.q)
    batch.lens, batch.offsets = batch.lens * copies, [queries * i for i in range(copies + 1)]
    batch.q, batch.table = batch.q.repeat(copies, 1, 1), batch.table.expand(copies, -1)
    o = batch.run(scale, activation).double().view(copies, *want.shape)
    assert G.kernel_status() == 0
    assert bool(torch.isfinite(o).all())
    over = ((o - want).abs() - tol).amax(0)
    assert float(over.max()) <= 0, (f"{int((over > 0).sum())} of {over.numel()} elements too far, worst by {float((over / tol).max()):.3g} tolerances; "
                                    f"the row's output off by {float(((o - want).norm(dim=3) / want.norm(dim=2)).max()):.3g} of it")


@pytest.mark.parametrize("queries,heads,kv_heads", [(1, 8, 2), (5, 16, 2), (70, 4, 2)])
@pytest.mark.parametrize("gap,tokens", [(8, 4096), (10, 4096), (11, 4096), (12, 4096), (13, 4096), (11, 32768), (12, 32768), (13, 32768), (14, 32768)])
def test_the_tail_of_a_peaked_softmax(gap, tokens, queries, heads, kv_heads):
    for dim in (64, 128):
        check_copies(peaked(gap, tokens, queries, heads, kv_heads, dim), 250, dim ** -0.5)
        peaked(gap, tokens, queries, heads, kv_heads, dim).check(dim ** -0.5)


@pytest.mark.parametrize("queries", [1, 12, 70])
@pytest.mark.parametrize("gap,tokens", [(11.25, 32768), (12, 100000), (12, 200000), (14, 200000)])
def test_a_tail_of_equal_scores(gap, tokens, queries):
    # all P of the tail are rounded the same way
    for dim in (64, 128):
        check_copies(peaked(gap, tokens, queries, 4, 1, dim, tail="equal"), 250, dim ** -0.5)


@pytest.mark.parametrize("queries", [1, 5, 70])
@pytest.mark.parametrize("activation", ["relu_square", "raw", "silu"])
def test_one_product_far_ahead(activation, queries):
    for dim in (64, 128):
        batch = peaked(12, 4096, queries, 8, 2, dim)
        blk = int(batch.table[0, (4096 // 3) // 64])
        batch.ks[blk] *= 256  # the scores of that block
        check_copies(batch, 250, 1 / 4096, activation)


def test_a_peak_that_comes_late():
    # the row's reference moves at the last tile, and everything before it with the reference
    for queries in (1, 12, 70):
        batch = peaked(12, 8192, queries, 4, 1, 128)
        batch.table = batch.table.roll(128 - 8192 // 3 // 64 - 1, 1).contiguous()
        check_copies(batch, 250, 128 ** -0.5)


# ------------------------------------------------------------------------------------------ scales of V


@pytest.mark.parametrize("queries", [1, 12, 70])
@pytest.mark.parametrize("activation", ["softmax", "silu", "relu"])
def test_blocks_with_a_scale_of_zero(activation, queries):
    # their values are zeros; their tokens take part like any others (a softmax's sum has them)
    for dim in (64, 128):
        batch = Batch([700, 64, 130, 1000], [queries] * 4, 4, 2, dim, 32, seed=queries)
        for b, j in ((0, 0), (0, 3), (0, 21), (1, 0), (1, 1), (2, 4), (3, 0), (3, 1), (3, 2), (3, 3), (3, 4)):
            batch.vs[int(batch.table[b, j])] = 0.0
        batch.vs[int(batch.table[0, 5]), 1] = 0.0
        scale = 0.1 if activation == "softmax" else 1e-3
        o = batch.check(scale, activation)
        assert bool((o[batch.offsets[1]:batch.offsets[2]] == 0).all())
        batch.check(scale, activation, causal=True)


@pytest.mark.parametrize("queries", [1, 12, 70])
@pytest.mark.parametrize("power", [0, 24, 60, 100])
def test_scales_far_apart(power, queries):
    # a token whose values are large is 8 ahead of 4095 whose values are zeros (so that their scale is the least there is): these have 0.58 of the weight
    for dim in (64, 128):
        batch = peaked(8, 4096, queries, 4, 2, dim)
        blk = int(batch.table[0, (4096 // 3) // 64])
        batch.v[:], batch.vs[:] = 0, 2.0 ** -100
        batch.v[blk, 4096 // 3 % 64], batch.vs[blk] = 0x40, 2.0 ** power
        batch.check(dim ** -0.5)


@pytest.mark.parametrize("queries", [1, 12, 70])
def test_products_of_zero_with_large_scales(queries):
    # no score above zero in the first tiles, or anywhere
    for dim in (64, 128):
        batch = Batch([500], [queries], 4, 2, dim, 64)
        batch.q, batch.vs[:] = batch.q.abs(), 2.0 ** 60
        batch.k |= 0x80
        assert bool((batch.check(1e-3, "relu") == 0).all())
        batch.k[int(batch.table[0, 6])] &= 0x7F
        batch.k[int(batch.table[0, 6])] &= 0x5F  # (a byte of 0x7F is NaN)
        batch.check(1e-3, "relu")
        batch.check(1e-3, "relu_square")


@pytest.mark.parametrize("queries", [1, 12, 70])
def test_a_nan_scale_stays_where_it_is(queries):
    for dim, activation in ((64, "softmax"), (128, "silu")):
        batch = Batch([300, 300], [queries] * 2, 4, 2, dim, 64)
        clean = batch.run(0.1, activation, causal=True)
        batch.vs[int(batch.table[0, 4]), 1] = float("nan")  # tokens 256 .. 299
        dirty = batch.run(0.1, activation, causal=True)
        sees = torch.zeros(2 * queries, 4, dtype=torch.bool, device=DEV)
        sees[max(0, queries - 44):queries, 2:] = True
        assert bool(dirty[sees].isnan().all()) and torch.equal(dirty[~sees], clean[~sees])
        assert G.kernel_status() == 0


# ------------------------------------------------------------------------------------------ NaN in V


@pytest.mark.parametrize("queries", [1, 6, 30, 70, 300])
@pytest.mark.parametrize("activation", ["softmax", "silu"])
@pytest.mark.parametrize("causal,window", [(False, None), (True, None), (True, 40), (False, 0), (False, 700)])
def test_a_nan_in_v_is_its_column_s(causal, window, activation, queries):
    # whether the tile it lies in has a mask or not, whether the item is cut or not: the element is NaN for the queries that see the token, and
    # nothing else changes
    for dim, lens in ((64, [900, 400, 130]), (128, [300, 5000, 64])):
        batch = Batch(lens, [queries] * 3, 4, 2, dim, 32, seed=queries)
        clean = batch.run(0.1, activation, causal, window)
        bad = torch.zeros(clean.shape, dtype=torch.bool, device=DEV)
        for b, pos, head, column in ((0, 5, 0, 3), (0, lens[0] - 1, 1, 40), (0, lens[0] - 1, 1, dim - 1), (1, lens[1] - 2, 0, 31), (1, 250, 1, 0), (2, 60, 0, 17)):
            batch.v[int(batch.table[b, pos // 32]), pos % 32, head, column] = 0x7F if column % 2 else 0xFF
            for i in range(queries):
                p = lens[b] - queries + i
                if (not causal or pos <= p) and (window is None or abs(pos - p) <= window):
                    bad[batch.offsets[b] + i, 2 * head:2 * head + 2, column] = True
        dirty = batch.run(0.1, activation, causal, window)
        assert G.kernel_status() == 0
        assert torch.equal(dirty.isnan(), bad)
        assert torch.equal(dirty[~bad], clean[~bad])


# ------------------------------------------------------------------------------------------ a wait that ran out


def test_a_wait_that_ran_out_is_said_by_the_next_call():
    batch = Batch([100], [2], 4, 2, 64, 16)
    clean = batch.run(0.1)
    word = ops._status_word(torch.device("cuda", torch.cuda.current_device()))
    torch.cuda.synchronize()
    word[0] = 0x1703  # what a kernel writes
    with pytest.raises(RuntimeError, match="wait ran out .*0x1703"):
        batch.run(0.1)
    assert torch.equal(batch.run(0.1), clean) and G.kernel_status() == 0


_TRACED = """
import torch
import ads_model_kernel_library_b200.gdpa as G
from ads_model_kernel_library_b200.gdpa import ops
from tests import _paged_oracle as ref
from tests._paged_batches import Batch
b = Batch([100], [2], 4, 2, 64, 16)
args = (b.q, b.k.view(torch.float8_e4m3fn), b.v.view(torch.float8_e4m3fn), b.ks, b.vs, b.table, b.int32(b.offsets), b.int32(b.lens))
step = torch.compile(lambda *a: G.generalized_dot_product_attention_paged_fp8(*a, 2, qk_scale=0.1), backend="aot_eager")
first = step(*args)
torch.cuda.synchronize()
ops._status_word(torch.device("cuda", 0))[0] = 0x1703
try:
    step(*args)
except RuntimeError as e:
    assert "0x1703" in str(e), e
    assert torch.equal(step(*args), first) and G.kernel_status() == 0
    print("said")
"""


def test_a_traced_call_has_the_status_word_too():
    # in a process of its own, in which no call was made before the traced one
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    r = subprocess.run([sys.executable, "-c", _TRACED], capture_output=True, text=True, timeout=300, cwd=root)
    assert r.returncode == 0 and "said" in r.stdout, r.stdout + r.stderr


# ------------------------------------------------------------------------------------------ a cache's steps


def test_a_step_and_a_release_do_not_wait_for_the_gpu():
    cache = G.PagedKVCache(40, 16, 2, 64, 5, 128)
    new = torch.tensor([20, 1, 0, 33, 5], dtype=torch.int32, device=DEV)
    q, kv = torch.randn(59, 4, 64, device=DEV).bfloat16(), torch.randn(59, 2, 64, device=DEV).bfloat16()
    cache.step(q, kv, kv, new, 33)
    cache.release([2])
    torch.cuda.synchronize()
    mode = torch.cuda.get_sync_debug_mode()
    torch.cuda.set_sync_debug_mode("error")
    try:
        cache.step(q, kv, kv, new, 33)
        cache.release([0, 3])
        cache.step(q, kv, kv, new, 33)
    finally:
        torch.cuda.set_sync_debug_mode(mode)
    assert cache.seq_lens.tolist() == [20, 3, 0, 33, 15]
    assert int(cache.num_free) == 40 - 2 - 1 - 0 - 3 - 1
    table = cache.block_tables[cache.block_tables >= 0].tolist()
    assert len(set(table) | set(cache.free_blocks[:int(cache.num_free)].tolist())) == 40
    with pytest.raises(IndexError):
        cache.release([5])


# ------------------------------------------------------------------------------------------ block tables


@pytest.mark.parametrize("batch", [5, 300, 9000])
@pytest.mark.parametrize("share", [0.0, 0.3, 0.99])
def test_tables_with_fewer_slots_than_tokens(batch, share):
    # the tables, lengths and offsets are the same; the slots are the first ones
    g = torch.Generator().manual_seed(batch)
    cached, new = torch.randint(0, 60, (batch,), generator=g).tolist(), torch.randint(0, 90, (batch,), generator=g).tolist()
    free, table = torch.randperm(batch * 8, generator=g).int(), torch.full((batch, 8), -1, dtype=torch.int32)
    at = 0
    for b, c in enumerate(cached):
        n = -(-c // 16)
        table[b, :n] = torch.arange(at, at + n) + 10 ** 6
        at += n
    total, short = sum(new), int(sum(new) * share)
    want = ref.tables(table, cached, new, free, len(free) - 3, 16, total)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    mine = table.to(DEV)
    slots, offsets, lens, left = G.build_block_tables(mine, i32(cached), i32(new), free.to(DEV), i32([len(free) - 3]), 16, short)
    assert torch.equal(mine.cpu(), want[0]) and torch.equal(slots.cpu(), want[1][:short])
    assert torch.equal(offsets.cpu().long(), want[2]) and torch.equal(lens.cpu().long(), want[3].long()) and int(left) == want[4]


@pytest.mark.parametrize("batch", [6, 400, 3000])
@pytest.mark.parametrize("length", [2 ** 30, 2 ** 31 - 1, 2 ** 40])
def test_tables_of_lengths_that_are_nonsense(batch, length):
    # what they say is unspecified; the call ends, writes nothing but its outputs, and the first request's tokens have their slots
    dtype = torch.int64 if length > 2 ** 31 else torch.int32
    wide = torch.full((batch, 9), 77, dtype=torch.int32, device=DEV)
    free = torch.arange(100, dtype=torch.int32, device=DEV)
    new = torch.full((batch,), length, dtype=dtype, device=DEV)
    slots, offsets, lens, left = G.build_block_tables(wide[:, :4], torch.zeros_like(new), new, free, torch.tensor([100], dtype=torch.int32, device=DEV), 16, 40)
    torch.cuda.synchronize()
    assert bool((wide[:, 4:] == 77).all()) and wide[0, :4].tolist() == [99, 98, 97, 96]
    assert slots.tolist() == [(99 - i // 16) * 16 + i % 16 for i in range(40)]
    assert bool(((wide[:, :4] >= -1) & (wide[:, :4] < 100)).all())


# ------------------------------------------------------------------------------------------ requests longer than their tables


@pytest.mark.parametrize("queries,more", [(1, 1), (1, 300), (12, 5), (12, 12), (12, 400), (100, 30), (100, 700)])
@pytest.mark.parametrize("causal,window", [(True, None), (True, 50), (False, 0), (False, 200), (False, None)])
def test_attend_past_the_end_of_the_table(causal, window, queries, more):
    # tokens without a place take no part; the queries keep their positions
    for dim in (64, 128):
        batch = Batch([320, 64, 192], [queries] * 3, 4, 2, dim, 32)
        batch.lens[0] += more  # the table is as wide as the first needs
        batch.check(0.1, causal=causal, window=window)
        batch.check(1e-3, "silu", causal=causal, window=window)


def test_a_cache_that_is_full_goes_on():
    # the second step brings tokens that the first request has no place for
    cache = G.PagedKVCache(20, 16, 2, 64, 2, 64)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=DEV)  # noqa: E731
    q, kv = torch.randn(70, 4, 64, device=DEV).bfloat16(), torch.randn(70, 2, 64, device=DEV).bfloat16()
    cache.step(q, kv, kv, i32([60, 10]), 60)
    o = cache.step(q[:12], kv[:12], kv[:12], i32([10, 2]), 10, qk_scale=0.1)
    assert cache.seq_lens.tolist() == [70, 12] and G.kernel_status() == 0
    seen = Batch([70], [10], 4, 2, 64, 16)
    seen.q, seen.table, seen.k, seen.v, seen.ks, seen.vs = (q[:10], cache.block_tables[:1], cache.k_cache.view(torch.uint8), cache.v_cache.view(torch.uint8),
                                                           cache.k_scales, cache.v_scales)
    want, tol = seen.want(0.1, causal=True)
    assert bool(((o[:10].double() - want).abs() <= tol).all())


# ------------------------------------------------------------------------------------------ traced


def test_the_append_traces():
    f8 = torch.float8_e4m3fn
    cache = [torch.zeros(2, 16, 2, 64, dtype=torch.uint8, device=DEV).view(f8) for _ in range(2)] + [torch.ones(2, 2, device=DEV) for _ in range(2)]
    kv = torch.randn(5, 2, 64, device=DEV).bfloat16()
    torch.library.opcheck(torch.ops.gdpa.append_kv_cache_fp8.default, (kv, kv, *cache, torch.arange(5, device=DEV)), test_utils=("test_faketensor",))


def test_a_compiled_step_is_the_step():
    f8 = torch.float8_e4m3fn

    def step(q, k, v, k8, v8, ks, vs, table, cached, new, free, num_free):
        slots, offsets, lens, left = G.build_block_tables(table, cached, new, free, num_free, 16, q.shape[0])
        G.append_kv_cache_fp8(k * 2, v + 1, k8, v8, ks, vs, slots)
        return G.generalized_dot_product_attention_paged_fp8(q, k8, v8, ks, vs, table, offsets, lens, 30, qk_scale=0.1, is_causal=True) * 3, lens, left

    def state():
        cache = [torch.zeros(12, 16, 2, 64, dtype=torch.uint8, device=DEV).view(f8) for _ in range(2)] + [torch.ones(12, 2, device=DEV) for _ in range(2)]
        return [*cache, torch.full((3, 8), -1, dtype=torch.int32, device=DEV), torch.zeros(3, dtype=torch.int32, device=DEV),
                torch.arange(12, dtype=torch.int32, device=DEV), torch.tensor([12], dtype=torch.int32, device=DEV)]

    compiled = torch.compile(step, backend="aot_eager", fullgraph=True)
    mine, theirs = state(), state()
    for new in ([20, 3, 30], [1, 1, 1], [0, 2, 1]):
        q, k, v = (torch.randn(sum(new), h, 64, device=DEV).bfloat16() for h in (4, 2, 2))
        new = torch.tensor(new, dtype=torch.int32, device=DEV)
        results = []
        for f, s in ((step, mine), (compiled, theirs)):
            o, s[5], s[7] = f(q, k, v, *s[:5], s[5], new, s[6], s[7])
            results.append(o)
        assert torch.equal(*results)
        assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(mine, theirs))
    assert G.kernel_status() == 0
