"""Calls of the operators on either side of the attention that are easily got wrong and need no GPU."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad
from torch._subclasses.fake_tensor import FakeTensorMode

import ads_model_kernel_library_b200.gdpa as G


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
