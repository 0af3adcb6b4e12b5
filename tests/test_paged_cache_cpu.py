"""What of the paged cache needs no GPU: the C entry points' refusals, the operators' refusal of CPU tensors, the plain forms."""
import ctypes as C
import math

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from ads_model_kernel_library_b200.gdpa import _cabi
from tests import _paged_oracle as ref

OK, BAD_ARG, DIM, ACT, MISALIGNED = 0, 1, 2, 4, 5


def fields(cls, **values):
    p = cls()
    p.struct_size = C.sizeof(cls)
    for name, v in values.items():
        if isinstance(v, (list, tuple)):
            for i, x in enumerate(v):
                getattr(p, name)[i] = x
        else:
            setattr(p, name, v)
    return p


def refused(fn, cls, good, change):
    return fn(C.byref(fields(cls, **{**good, **change})), None)


def test_null_and_struct_sizes():
    for fn, cls in ((_cabi.lib.gdpa_build_block_tables, _cabi.GdpaBlockTableParams), (_cabi.lib.gdpa_append_kv_cache_fp8, _cabi.GdpaCacheAppendParams),
                    (_cabi.lib.gdpa_fwd_paged_fp8, _cabi.GdpaPagedParams)):
        assert fn(None, None) == BAD_ARG
        p = cls()
        p.struct_size = C.sizeof(cls) - 4
        assert fn(C.byref(p), None) == BAD_ARG


def test_block_table_refusals():
    good = dict(cached_lens=16, new_lens=16, batch=2, block_size=16, block_tables=16, table_stride=4, table_width=4, free_blocks=16, free_capacity=4,
                num_free=16, total_new=3, slots=16, query_offset=16, seq_lens=16, num_free_after=32)
    fn, cls = _cabi.lib.gdpa_build_block_tables, _cabi.GdpaBlockTableParams
    for change in (dict(block_size=8), dict(block_size=0), dict(batch=-1), dict(table_width=-1), dict(total_new=-1), dict(total_new=1 << 31),
                   dict(free_capacity=-1), dict(table_width=1 << 27), dict(num_free=0), dict(query_offset=0), dict(num_free_after=0), dict(num_free_after=16),
                   dict(slots=0), dict(cached_lens=0), dict(new_lens=0), dict(seq_lens=0), dict(block_tables=0), dict(free_blocks=0), dict(table_stride=-1)):
        assert refused(fn, cls, good, change) == BAD_ARG, change


def test_append_refusals():
    good = dict(key=16, value=16, k_cache=16, v_cache=16, k_scales=16, v_scales=16, slot_mapping=16, tokens=4, num_blocks=4, block_size=16, kv_heads=2,
                head_dim=64)
    fn, cls = _cabi.lib.gdpa_append_kv_cache_fp8, _cabi.GdpaCacheAppendParams
    for change, code in ((dict(block_size=20), BAD_ARG), (dict(tokens=-1), BAD_ARG), (dict(num_blocks=-1), BAD_ARG), (dict(kv_heads=0), BAD_ARG),
                         (dict(head_dim=96), DIM), (dict(key=0), BAD_ARG), (dict(value=0), BAD_ARG), (dict(k_cache=0), BAD_ARG), (dict(k_scales=0), BAD_ARG),
                         (dict(slot_mapping=0), BAD_ARG), (dict(key=8), MISALIGNED), (dict(v_cache=24), MISALIGNED), (dict(key_strides=(4, 64)), MISALIGNED),
                         (dict(key_strides=(-8, 64)), BAD_ARG), (dict(k_cache_strides=(2048, 128, 8)), MISALIGNED), (dict(v_cache_strides=(-16, 0, 0)), BAD_ARG)):
        assert refused(fn, cls, good, change) == code, change
    assert refused(fn, cls, good, dict(tokens=0)) == OK


def test_attention_refusals():
    good = dict(activation=100, q=16, o=16, k_cache=16, v_cache=16, k_scales=16, v_scales=16, block_tables=16, table_stride=4, table_width=4, block_size=16,
                num_blocks=4, q_offsets=16, seq_lens=16, batch=1, heads=4, kv_heads=2, head_dim=64, total_q=2, max_seq_len_q=2, qk_scale=1.0, workspace=16)
    fn, cls = _cabi.lib.gdpa_fwd_paged_fp8, _cabi.GdpaPagedParams
    for change, code in ((dict(activation=55), ACT), (dict(head_dim=32), DIM), (dict(block_size=48), BAD_ARG), (dict(batch=-1), BAD_ARG), (dict(heads=3), BAD_ARG),
                         (dict(kv_heads=0), BAD_ARG), (dict(total_q=-1), BAD_ARG), (dict(max_seq_len_q=-1), BAD_ARG), (dict(max_seq_len_q=1 << 30), BAD_ARG),
                         (dict(table_width=1 << 27), BAD_ARG), (dict(num_blocks=1 << 31), BAD_ARG), (dict(window_plus_one=-1), BAD_ARG),
                         (dict(q=0), BAD_ARG), (dict(o=0), BAD_ARG), (dict(workspace=0), BAD_ARG), (dict(seq_lens=0), BAD_ARG), (dict(block_tables=0), BAD_ARG),
                         (dict(k_cache=0), BAD_ARG), (dict(v_scales=0), BAD_ARG), (dict(q=24), MISALIGNED), (dict(workspace=20), MISALIGNED),
                         (dict(q_strides=(4, 64)), MISALIGNED), (dict(k_cache_strides=(0, 0, 72)), MISALIGNED)):
        assert refused(fn, cls, good, change) == code, change
    assert refused(fn, cls, good, dict(total_q=0)) == OK and refused(fn, cls, good, dict(batch=0)) == OK


def test_cpu_tensors_are_refused():
    f8 = torch.zeros(2, 16, 1, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s, i = torch.ones(2, 1), torch.zeros(1, dtype=torch.int32)
    x = torch.zeros(1, 1, 64, dtype=torch.bfloat16)
    with pytest.raises((RuntimeError, NotImplementedError)):
        G.build_block_tables(torch.zeros(1, 2, dtype=torch.int32), i, i, i, i, 16, 1)
    with pytest.raises((RuntimeError, NotImplementedError)):
        G.append_kv_cache_fp8(x, x, f8, f8, s, s, torch.zeros(1, dtype=torch.int64))
    with pytest.raises((RuntimeError, NotImplementedError)):
        G.generalized_dot_product_attention_paged_fp8(x, f8, f8, s, s, i.view(1, 1), torch.zeros(2, dtype=torch.int32), i, 1)


def test_plain_e4m3_is_torch_s():
    x = torch.cat([torch.randn(20000) * 2.0 ** k for k in range(-14, 9)]).clamp(-448, 448)
    assert torch.equal(ref.e4m3_bytes(x), x.to(torch.float8_e4m3fn).view(torch.uint8))
    assert ref.least_scale(torch.tensor([448.0])) == 1.0 and ref.least_scale(torch.tensor([448.1])) == 2.0
    assert ref.least_scale(torch.tensor([0.0])) == ref.least_scale(torch.tensor([math.inf])) == 2.0 ** -100


def test_plain_tables_small():
    table = torch.tensor([[5, -1, -1], [-1, -1, -1]], dtype=torch.int32)
    t, slots, off, lens, left = ref.tables(table, [14, 0], [4, 1], [7, 8, 9], 3, 16, 6)
    assert t.tolist() == [[5, 9, -1], [8, -1, -1]] and slots.tolist() == [94, 95, 144, 145, 128, -1]
    assert off.tolist() == [0, 4, 5] and lens.tolist() == [18, 1] and left == 1
