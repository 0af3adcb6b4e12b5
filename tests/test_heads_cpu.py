"""What of the operators on either side of the attention needs no GPU: refusals, traced shapes, the plain forms."""
import ctypes as C

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from ads_model_kernel_library_b200.gdpa import _cabi
from tests import _heads_oracle as ref
from tests.test_paged_cache_cpu import ACT, BAD_ARG, DIM, MISALIGNED, OK, fields  # noqa: F401

ENTRIES = {"gdpa_qk_norm_rotary": "GdpaRotaryParams", "gdpa_qk_norm_rotary_bwd": "GdpaRotaryParams",
           "gdpa_append_rotated_kv_cache_fp8": "GdpaRotatedAppendParams", "gdpa_read_kv_cache_fp8": "GdpaCacheReadParams",
           "gdpa_verify_draft_tokens": "GdpaVerifyParams", "gdpa_drop_cached_tokens": "GdpaDropParams"}


def nested(cls, values):
    """A structure with the values of "a.b" in its member a."""
    p = cls()
    p.struct_size = C.sizeof(cls)
    for name, v in values.items():
        at, *rest = name.split(".")
        to = getattr(p, at) if rest else p
        name = rest[0] if rest else at
        if isinstance(v, (list, tuple)):
            for i, x in enumerate(v):
                getattr(to, name)[i] = x
        else:
            setattr(to, name, v)
    return p


def call(name, good, change):
    return getattr(_cabi.lib, name)(C.byref(nested(getattr(_cabi, ENTRIES[name]), {**good, **change})), None)


@pytest.mark.parametrize("name", ENTRIES)
def test_null_and_struct_sizes(name):
    fn, cls = getattr(_cabi.lib, name), getattr(_cabi, ENTRIES[name])
    assert fn(None, None) == BAD_ARG
    p = cls()
    p.struct_size = C.sizeof(cls) - 4
    assert fn(C.byref(p), None) == BAD_ARG


ROTARY = {"head_dim": 128, "rotary.inv_freq": 16, "rotary.pairs": 64, "rotary.axes": 1, "rotary.norm": 1, "rotary.eps": 1e-6}
for _t in ("query", "key"):
    ROTARY.update({f"{_t}.x": 16, f"{_t}.y": 16, f"{_t}.dy": 16, f"{_t}.heads": 2, f"{_t}.tokens": 3, f"{_t}.positions": 16})


@pytest.mark.parametrize("backward", [False, True])
def test_rotary_refusals(backward):
    name = "gdpa_qk_norm_rotary_bwd" if backward else "gdpa_qk_norm_rotary"
    for change, code in (({"head_dim": 96}, DIM), ({"rotary.pairs": 12}, BAD_ARG), ({"rotary.pairs": 72}, BAD_ARG), ({"rotary.pairs": -8}, BAD_ARG),
                         ({"rotary.axes": 0}, BAD_ARG), ({"rotary.axes": 5}, BAD_ARG), ({"rotary.inv_freq": 0}, BAD_ARG), ({"rotary.eps": -1.0}, BAD_ARG),
                         ({"rotary.eps": float("nan")}, BAD_ARG), ({"rotary.axes": 2, "rotary.section_ends": (32, 60)}, BAD_ARG),
                         ({"rotary.axes": 3, "rotary.section_ends": (32, 16, 64)}, BAD_ARG), ({"query.tokens": -1}, BAD_ARG), ({"key.tokens": 1 << 30}, BAD_ARG),
                         ({"key.heads": -1}, BAD_ARG), ({"query.x": 0}, BAD_ARG), ({"key.y": 0}, BAD_ARG), ({"query.positions": 0}, BAD_ARG),
                         ({"key.position_stride": -1}, BAD_ARG), ({"query.x": 8}, MISALIGNED), ({"key.y": 24}, MISALIGNED),
                         ({"query.x_strides": (260, 128)}, MISALIGNED), ({"query.x_strides": (-256, 128)}, BAD_ARG)):
        assert call(name, ROTARY, change) == code, change
    nothing = {"query.tokens": 0, "key.tokens": 0}
    assert call(name, ROTARY, nothing) == OK
    if backward:
        assert call(name, ROTARY, {"query.dy": 0}) == BAD_ARG
        assert call(name, ROTARY, {"key.dy": 8}) == MISALIGNED
        assert call(name, ROTARY, {"query.dweight": 16}) == BAD_ARG  # no workspace
        assert call(name, ROTARY, {"query.dweight": 16, "workspace": 8}) == MISALIGNED


def test_rotated_append_refusals():
    good = {"heads": 4, "cache.struct_size": C.sizeof(_cabi.GdpaCacheAppendParams), "cache.key": 16, "cache.value": 16, "cache.k_cache": 16, "cache.v_cache": 16,
            "cache.k_scales": 16, "cache.v_scales": 16, "cache.slot_mapping": 16, "cache.tokens": 4, "cache.num_blocks": 4, "cache.block_size": 16,
            "cache.kv_heads": 2, "cache.head_dim": 64, "rotary.inv_freq": 16, "rotary.pairs": 32, "rotary.axes": 1, "rotary.norm": 1, "rotary.eps": 1e-6,
            "query": 16, "query_out": 16, "batch": 1, "q_offsets": 16, "seq_lens": 16}
    name = "gdpa_append_rotated_kv_cache_fp8"
    for change, code in (({"cache.struct_size": 8}, BAD_ARG), ({"cache.block_size": 20}, BAD_ARG), ({"cache.head_dim": 96}, DIM), ({"cache.key": 0}, BAD_ARG),
                         ({"cache.v_cache": 24}, MISALIGNED), ({"rotary.pairs": 40}, BAD_ARG), ({"heads": 0}, BAD_ARG), ({"query": 0}, BAD_ARG),
                         ({"query_out": 0}, BAD_ARG), ({"query": 8}, MISALIGNED), ({"query_strides": (4, 64)}, MISALIGNED), ({"batch": -1}, BAD_ARG),
                         ({"seq_lens": 0}, BAD_ARG), ({"q_offsets": 0}, BAD_ARG), ({"cache.tokens": 1 << 30}, BAD_ARG), ({"position_stride": -1}, BAD_ARG)):
        assert call(name, good, change) == code, change
    assert call(name, good, {"cache.tokens": 0}) == OK


def test_read_refusals():
    good = dict(k_cache=16, v_cache=16, k_scales=16, v_scales=16, block_tables=16, table_stride=4, table_width=4, block_size=16, num_blocks=4, offsets=16, batch=1,
                kv_heads=2, head_dim=64, total=3, key=16, value=16)
    name = "gdpa_read_kv_cache_fp8"
    for change, code in ((dict(head_dim=32), DIM), (dict(block_size=48), BAD_ARG), (dict(batch=-1), BAD_ARG), (dict(kv_heads=0), BAD_ARG), (dict(total=-1), BAD_ARG),
                         (dict(table_width=1 << 27), BAD_ARG), (dict(num_blocks=1 << 31), BAD_ARG), (dict(key=0), BAD_ARG), (dict(value=0), BAD_ARG),
                         (dict(offsets=0), BAD_ARG), (dict(block_tables=0), BAD_ARG), (dict(k_scales=0), BAD_ARG), (dict(v_cache=8), MISALIGNED),
                         (dict(key=8), MISALIGNED), (dict(k_cache_strides=(0, 0, 72)), MISALIGNED), (dict(k_cache_strides=(-16, 0, 0)), BAD_ARG)):
        assert call(name, good, change) == code, change
    assert call(name, good, dict(total=0)) == OK


def test_verify_refusals():
    good = dict(target=16, draft=16, target_stride=100, draft_stride=100, rows=4, drafts=3, vocab=100, tokens=16, row_offsets=16, draft_offsets=16, batch=1,
                accept=16, sample=16, max_drafts=3, out_tokens=16, accepted=16, refused=16)
    name = "gdpa_verify_draft_tokens"
    for change in (dict(vocab=0), dict(vocab=(1 << 20) + 1), dict(batch=-1), dict(rows=-1), dict(drafts=-1), dict(max_drafts=-1), dict(target_stride=-1),
                   dict(target=0), dict(tokens=0), dict(accept=0), dict(sample=0), dict(row_offsets=0), dict(draft_offsets=0), dict(out_tokens=0),
                   dict(accepted=0), dict(refused=0)):
        assert call(name, good, change) == BAD_ARG, change
    assert call(name, good, dict(batch=0)) == OK


def test_drop_refusals():
    good = dict(block_size=16, block_tables=16, table_stride=4, table_width=4, batch=2, seq_lens=16, dropped=16, free_blocks=16, free_capacity=4, num_free=16,
                seq_lens_after=16, num_free_after=32)
    for change in (dict(block_size=8), dict(batch=-1), dict(table_width=-1), dict(table_stride=-1), dict(free_capacity=-1), dict(table_width=1 << 27),
                   dict(num_free=0), dict(num_free_after=0), dict(num_free_after=16), dict(seq_lens=0), dict(dropped=0), dict(seq_lens_after=0),
                   dict(block_tables=0), dict(free_blocks=0)):
        assert call("gdpa_drop_cached_tokens", good, change) == BAD_ARG, change


def test_cpu_tensors_are_refused():
    x, f, i = torch.zeros(2, 1, 64, dtype=torch.bfloat16), torch.ones(32), torch.zeros(2, dtype=torch.int32)
    f8, s = torch.zeros(2, 16, 1, 64, dtype=torch.uint8).view(torch.float8_e4m3fn), torch.ones(2, 1)
    table, slots = torch.zeros(1, 2, dtype=torch.int32), torch.zeros(2, dtype=torch.int64)
    for call_it in (lambda: G.qk_norm_rotary(x, x, f, i), lambda: G.append_rotated_kv_cache_fp8(x, x, x, f8, f8, s, s, slots, i, i[:1], f),
                    lambda: G.read_kv_cache_fp8(f8, f8, s, s, table, i, 0), lambda: G.drop_cached_tokens(table, i[:1], i[:1], i, i[:1], 16),
                    lambda: G.verify_draft_tokens(torch.ones(1, 4), None, i[:0], i, i, f[:0], f[:1], 0)):
        with pytest.raises((RuntimeError, NotImplementedError)):
            call_it()


def test_shapes_are_traced():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        e = lambda *s, dtype=torch.bfloat16: torch.empty(s, dtype=dtype, device="cuda")  # noqa: E731
        i32 = lambda *s: e(*s, dtype=torch.int32)  # noqa: E731
        q, k, w = e(7, 4, 128).requires_grad_(), e(7, 2, 128).requires_grad_(), e(128, dtype=torch.float32).requires_grad_()
        a, b = G.qk_norm_rotary(q, k, e(64, dtype=torch.float64), i32(7), query_weight=w)
        assert a.shape == q.shape and b.shape == k.shape
        assert a.requires_grad and b.requires_grad and type(a.grad_fn).__name__ == type(b.grad_fn).__name__
        with torch.no_grad():  # the engine would want the device itself
            g = torch.ops.gdpa.qk_norm_rotary_backward(a, b, q, k, e(64, dtype=torch.float64), i32(7), i32(7), w, None, 1e-6, True, False, [], True)
        assert [t.shape for t in g] == [q.shape, k.shape, w.shape, (0,)] and g[2].dtype == torch.float32
        cache, scales = e(4, 16, 2, 128, dtype=torch.float8_e4m3fn), e(4, 2, dtype=torch.float32)
        out = G.append_rotated_kv_cache_fp8(e(7, 4, 128), e(7, 2, 128), e(7, 2, 128), cache, cache, scales, scales, e(7, dtype=torch.int64), i32(3), i32(2),
                                            e(64, dtype=torch.float64))
        assert out.shape == (7, 4, 128) and out.dtype == torch.bfloat16
        key, value = G.read_kv_cache_fp8(cache, cache, scales, scales, i32(2, 3), i32(3), 9, dtype=torch.float32)
        assert key.shape == value.shape == (9, 2, 128) and key.dtype == torch.float32
        tokens, accepted, refused = G.verify_draft_tokens(e(7, 50), None, e(5, dtype=torch.int64), i32(3), i32(3), e(5, dtype=torch.float32),
                                                          e(2, dtype=torch.float32), 4)
        assert tokens.shape == (2, 5) and tokens.dtype == torch.int64 and accepted.shape == refused.shape == (2,)
        lens, left = G.drop_cached_tokens(i32(2, 3), i32(2), i32(2), i32(8), i32(1), 16)
        assert lens.shape == (2,) and left.shape == (1,) and lens.dtype == torch.int32


@pytest.mark.parametrize("interleaved", [False, True])
def test_plain_gradient_is_autograd_s(interleaved):
    g = torch.Generator().manual_seed(1)
    x, dy, w = (torch.randn(*s, generator=g, dtype=torch.float64) for s in ((5, 3, 64), (5, 3, 64), (64,)))
    angle = ref.angles(100.0 ** -torch.rand(16, generator=g), torch.tensor([0, 3, 9, 10, 100000]))
    xg, wg = x.clone().requires_grad_(), w.clone().requires_grad_()
    n = xg * torch.rsqrt(xg.pow(2).mean(-1, keepdim=True) + 1e-6) * wg
    a, b = ref.pairs_of(16, interleaved)
    z = torch.complex(n[..., a], n[..., b]) * torch.polar(torch.ones_like(angle), angle)[:, None]
    y = n.index_copy(-1, a, z.real).index_copy(-1, b, z.imag)
    torch.testing.assert_close(ref.norm_rotary(x, w, 1e-6, True, angle, interleaved)[0], y.detach())
    dx, dw = torch.autograd.grad(y, (xg, wg), dy)
    (got, _), (got_w, _) = ref.norm_rotary_grad(x, dy, w, 1e-6, True, angle, interleaved)
    torch.testing.assert_close(got, dx)
    torch.testing.assert_close(got_w, dw)


def test_plain_verification_small():
    p = torch.tensor([[0.5, 0.25, 0.25], [0.1, 0.9, 0.0], [0.2, 0.3, 0.5]])
    q = torch.tensor([[0.25, 0.5, 0.25], [0.8, 0.1, 0.1]])
    tokens = torch.tensor([0, 0])
    args = ([0, 3], [0, 2])
    # the first is surely accepted, the second if u 0.8 < 0.1; what is left then is 0.8 for token 1
    assert ref.verify(p, q, tokens, *args, torch.tensor([0.99, 0.12]), torch.tensor([0.6]), 2) == ([[0, 0, 2]], [2], [0])
    assert ref.verify(p, q, tokens, *args, torch.tensor([0.99, 0.13]), torch.tensor([0.0]), 3) == ([[0, 1, -1, -1]], [1], [1])
    assert ref.verify(p, None, tokens, *args, torch.tensor([0.6, 0.0]), torch.tensor([0.5]), 2) == ([[2, -1, -1]], [0], [2])


def test_plain_drop_small():
    table = torch.tensor([[4, 7, 9], [3, -1, 6]])
    assert ref.drop(table, [40, 48], [30, 100], [1, 2, 0, 0, 0, 0, 0], 2, 16) == ([10, 0], 6, [1, 2, 7, 9, 3, 6, 0])
