"""Edges of the paged 8-bit cache on the GPU: batches and values at which its operators can go wrong."""
import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
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
