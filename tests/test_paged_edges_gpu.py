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
