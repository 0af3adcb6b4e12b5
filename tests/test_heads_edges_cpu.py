"""Calls of the operators on either side of the attention that are easily got wrong and need no GPU."""
import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode

import ads_model_kernel_library_b200.gdpa as G
from ads_model_kernel_library_b200.gdpa import _cabi
from tests.test_paged_cache_cpu import BAD_ARG, OK, fields


def empty(*shape, dtype=torch.bfloat16):
    return torch.empty(shape, dtype=dtype, device="cuda")


def rotary_arguments():
    """query, key, query_weight, key_weight, inv_freq, positions"""
    return [empty(7, 4, 128), empty(7, 2, 128), empty(128, dtype=torch.float32), empty(128, dtype=torch.float32), empty(64, dtype=torch.float64),
            empty(7, dtype=torch.int32)]


@pytest.mark.parametrize("which", range(5))
@pytest.mark.parametrize("grad", ["wanted", "not wanted", "off"])
def test_tangents_are_refused(which, grad):
    """No forward-mode derivative: a call with a tangent raises, as the other operators' do; it does not return results without one."""
    with FakeTensorMode(), forward_ad.dual_level(), torch.set_grad_enabled(grad != "off"):
        args = rotary_arguments()
        if grad == "wanted":
            args[:4] = [t.requires_grad_() for t in args[:4]]
        args[which] = forward_ad.make_dual(args[which], torch.ones_like(args[which]))
        with pytest.raises(RuntimeError):
            G.qk_norm_rotary(args[0], args[1], args[4], args[5], query_weight=args[2], key_weight=args[3])


def test_tangents_of_a_functional_call_are_refused():
    with FakeTensorMode():
        q, k, _, _, f, p = rotary_arguments()
        with pytest.raises(RuntimeError):
            torch.func.jvp(lambda x: G.qk_norm_rotary(x, k, f, p)[0], (q,), (q,))


# ------------------------------------------------------------------------------------------ a step that is refused


@pytest.mark.parametrize("rotary", [None, dict(inv_freq=torch.ones(32))])
def test_a_step_whose_attention_is_refused_counts_no_tokens(monkeypatch, rotary):
    cache, calls = G.PagedKVCache(8, 16, 1, 64, 2, 64, device="cpu"), []
    new, x = torch.tensor([3, 1], dtype=torch.int32), torch.zeros(4, 1, 64, dtype=torch.bfloat16)
    monkeypatch.setattr(G.paged, "build_block_tables",
                        lambda tables, cached, new, *args: (torch.zeros(4), torch.tensor([0, 3, 4]), cached + new, torch.tensor([6], dtype=torch.int32)))
    monkeypatch.setattr(G.paged, "append_kv_cache_fp8", lambda *args: calls.append("append"))
    monkeypatch.setattr(G.paged, "append_rotated_kv_cache_fp8", lambda query, *args, **options: calls.append("append") or query)
    attended = []

    def attend(query, *args, **options):
        attended.append(args[6].tolist())  # the lengths that it is given: the new tokens counted
        if options.get("activation") == "unknown":
            raise ValueError("refused")
        return query

    monkeypatch.setattr(G.paged, "generalized_dot_product_attention_paged_fp8", attend)
    with pytest.raises(TypeError, match="query"):  # the attention takes bf16: nothing is stored before it says so
        cache.step(x.float(), x.float(), x.float(), new, 3, rotary=rotary)
    assert calls == [] and cache.seq_lens.tolist() == [0, 0] and int(cache.num_free) == 8
    with pytest.raises(ValueError, match="refused"):
        cache.step(x, x, x, new, 3, rotary=rotary, activation="unknown")
    assert calls == ["append"] and cache.seq_lens.tolist() == [0, 0] and int(cache.num_free) == 8
    assert torch.equal(cache.step(x, x, x, new, 3, rotary=rotary), x)
    assert attended == [[3, 1]] * 2 and cache.seq_lens.tolist() == [3, 1] and int(cache.num_free) == 6


# ------------------------------------------------------------------------------------------ lengths that are updated in place


def drop_call(**change):
    """Refused calls only: the addresses are made up."""
    good = dict(block_size=16, block_tables=0x10000, table_stride=4, table_width=4, batch=2, seq_lens=0x20000, dropped=0x30000, free_blocks=0x40000, free_capacity=4,
                num_free=0x50000, seq_lens_after=0x60000, num_free_after=0x70000)
    return _cabi.lib.gdpa_drop_cached_tokens(C.byref(fields(_cabi.GdpaDropParams, **{**good, **change})), None)


@pytest.mark.parametrize("change", [
    dict(seq_lens_after=0x20000), dict(seq_lens_after=0x30000), dict(seq_lens_after=0x20004), dict(seq_lens_after=0x20008, lens_are_int64=1),
    dict(seq_lens_after=0x2fffc), dict(seq_lens_after=0x3000c, dropped_is_int64=1), dict(seq_lens_after=0x10010), dict(seq_lens_after=0x40000),
    dict(seq_lens_after=0x50000), dict(seq_lens_after=0x6fffc, num_free_after=0x70000), dict(num_free_after=0x20004), dict(num_free_after=0x3000c, dropped_is_int64=1),
    dict(num_free_after=0x50000), dict(num_free_after=0x4000c), dict(num_free_after=0x1001c), dict(free_blocks=0x10010), dict(free_blocks=0x4fff4)])
def test_drop_refuses_outputs_over_its_inputs(change):
    assert drop_call(**change) == BAD_ARG


@pytest.mark.parametrize("change", [dict(block_size=8), dict(batch=-1), dict(table_width=-1), dict(table_stride=-1), dict(free_capacity=-1), dict(table_width=1 << 27),
                                    dict(num_free=0), dict(num_free_after=0), dict(seq_lens=0), dict(dropped=0), dict(seq_lens_after=0), dict(block_tables=0),
                                    dict(free_blocks=0)])
def test_drop_refusals_with_memory_of_their_own(change):
    assert drop_call(**change) == BAD_ARG


@pytest.mark.skipif(torch.cuda.is_available(), reason="made-up addresses: only where no kernel can be launched")
@pytest.mark.parametrize("change", [{}, dict(seq_lens_after=0x20008), dict(seq_lens_after=0x1fff8), dict(seq_lens_after=0x20010, lens_are_int64=1),
                                    dict(seq_lens_after=0x10020), dict(num_free_after=0x60008), dict(free_blocks=0x4fff0), dict(seq_lens_after=0x30008)])
def test_drop_takes_neighbours(change):
    assert drop_call(**change) not in (BAD_ARG, OK)  # the arguments are good, there is no device
