"""What of the paged cache's edges needs no GPU."""
import os
import subprocess
import sys

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def in_a_process_of_its_own(code):
    r = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert r.returncode == 0 and "ok" in r.stdout, r.stdout + r.stderr


def test_a_step_traces_as_one_graph_before_any_other_call():
    in_a_process_of_its_own("""
import torch
from torch._subclasses.fake_tensor import FakeTensorMode
import ads_model_kernel_library_b200.gdpa as G

def step(q, k, v, k8, v8, ks, vs, table, cached, new, free, num_free):
    slots, offsets, lens, left = G.build_block_tables(table, cached, new, free, num_free, 16, q.shape[0])
    G.append_kv_cache_fp8(k, v, k8, v8, ks, vs, slots)
    return G.generalized_dot_product_attention_paged_fp8(q, k8, v8, ks, vs, table, offsets, lens, 2, is_causal=True), lens, left

calls = []
def backend(graph, inputs):
    calls.append([str(n.target) for n in graph.graph.nodes if n.op == "call_function" and "gdpa" in str(n.target)])
    return graph.forward

with FakeTensorMode(allow_non_fake_inputs=True):
    i = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")
    x = lambda h: torch.zeros(3, h, 64, dtype=torch.bfloat16, device="cuda")
    f8 = lambda: torch.zeros(8, 16, 2, 64, dtype=torch.float8_e4m3fn, device="cuda")
    s = lambda: torch.ones(8, 2, device="cuda")
    out, lens, left = torch.compile(step, backend=backend, fullgraph=True)(x(4), x(2), x(2), f8(), f8(), s(), s(), i(2, 4), i(2), i(2), i(8), i(1))
assert out.shape == (3, 4, 64) and out.dtype == torch.bfloat16 and lens.shape == (2,) and left.shape == (1,)
assert calls == [["gdpa.build_block_tables.default", "gdpa.append_kv_cache_fp8.default", "gdpa.generalized_dot_product_attention_paged_fp8.default"]], calls
print("ok")
""")


def test_first_calls_of_several_threads_load_the_operators_once():
    in_a_process_of_its_own("""
import threading
import ads_model_kernel_library_b200.gdpa as G
paged = G.paged
paged._operators = None  # as on an import that could not load them
made, meet, errors = [], threading.Barrier(8), []
init = paged._Operators.__init__
def counted(self):
    made.append(self)
    threading.Event().wait(0.05)
    init(self)
paged._Operators.__init__ = counted
def first():
    meet.wait()
    try:
        assert paged._operators or paged._load()
    except Exception as e:
        errors.append(e)
threads = [threading.Thread(target=first) for _ in range(8)]
[t.start() for t in threads], [t.join() for t in threads]
assert not errors and len(made) == 1, (errors, len(made))
print("ok")
""")


def held_cache():
    """A cache of five requests on the CPU, of which the first four hold 1 to 4 blocks."""
    cache = G.PagedKVCache(20, 16, 1, 64, 5, 128, device="cpu")
    for b in range(4):
        n = b + 1
        cache.block_tables[b, :n] = cache.free_blocks[int(cache.num_free) - n:int(cache.num_free)]
        cache.seq_lens[b], cache.num_free = 16 * n - 3, cache.num_free - n
    return cache


def free(cache):
    return sorted(cache.free_blocks[:int(cache.num_free)].tolist())


@pytest.mark.parametrize("requests", [[5], [-6], [0, 99], [2 ** 40], [1, -1000]])
def test_release_of_a_request_that_is_not_there(requests):
    cache = held_cache()
    before = [t.clone() for t in (cache.block_tables, cache.seq_lens, cache.free_blocks, cache.num_free)]
    with pytest.raises(IndexError, match="is not one of this cache's 5"):
        cache.release(requests)
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.block_tables, cache.seq_lens, cache.free_blocks, cache.num_free)))
    with pytest.raises(TypeError):
        cache.release([1.5])


def test_release_of_a_request_by_two_names():
    cache = held_cache()
    cache.release([3, -2, 3, 1])  # 3 and -2 are the same one
    assert int(cache.num_free) == 16 and len(set(free(cache))) == 16
    assert cache.seq_lens.tolist() == [13, 0, 45, 0, 0] and cache.block_tables[[1, 3]].eq(-1).all()
    cache.release([])
    cache.release([0, 1, 2, 3, 4])
    assert free(cache) == list(range(20))


@pytest.mark.parametrize("slots,good", [
    ([], True), ([-1, -1], True), ([3], True), ([14, 15, 16, 17], True), ([0, 1, -1, 32, 33], True), ([-1, 4, 5, -1], True), ([10 ** 12, 0, 1], True),
    ([48, 49, 10 ** 12, 0], True), ([63, 64, 65], True),
    ([5, -1, 6], False), ([5, 10 ** 12, 6], False), ([5, 64, 6], False), ([-1, 5, -1, 6, -1], False), ([0, 1, 16, 2], False), ([1, 0], False), ([3, 3], False),
])
def test_what_the_check_of_slots_says(slots, good):
    # of a cache of four blocks of 16
    cache = torch.zeros(4, 16, 1, 64, dtype=torch.uint8)
    if good:
        G.paged._check_slots(torch.tensor(slots, dtype=torch.int64), cache)
    else:
        with pytest.raises(ValueError):
            G.paged._check_slots(torch.tensor(slots, dtype=torch.int64), cache)


def test_tokens_that_are_refused_are_not_counted(monkeypatch):
    cache = held_cache()
    monkeypatch.setattr(G.paged, "build_block_tables", lambda tables, cached, new, *args: (torch.zeros(3), torch.zeros(6), cached + new, torch.zeros(1)))
    monkeypatch.setattr(G.paged, "append_kv_cache_fp8", lambda *args: (_ for _ in ()).throw(ValueError("refused")))
    lens, left = cache.seq_lens.tolist(), int(cache.num_free)
    with pytest.raises(ValueError, match="refused"):
        cache.append(torch.zeros(3, 1, 64), torch.zeros(3, 1, 32), torch.tensor([1, 1, 1, 0, 0], dtype=torch.int32))
    assert cache.seq_lens.tolist() == lens and int(cache.num_free) == left
    monkeypatch.setattr(G.paged, "append_kv_cache_fp8", lambda *args: None)
    cache.append(torch.zeros(3, 1, 64), torch.zeros(3, 1, 64), torch.tensor([1, 1, 1, 0, 0], dtype=torch.int32))
    assert cache.seq_lens.tolist() == [14, 30, 46, 61, 0] and int(cache.num_free) == 0
