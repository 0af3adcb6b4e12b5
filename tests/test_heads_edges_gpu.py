"""Calls of the operators on either side of the attention that are easily got wrong, on the GPU."""
import ctypes as C
import threading

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from ads_model_kernel_library_b200.gdpa import _cabi
from tests import _heads_oracle as ref
from tests.test_heads_cpu import nested
from tests.test_heads_gpu import BF, DEV, F32, frequencies, weights

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------ norm and rotation

# gradients as a result's uses leave them: (function of the result, what of it a gradient in plain form is)
USES = {
    "sum": lambda y, r: y.sum(),
    "sum of heads": lambda y, r: (y.sum(1) * r[:, 0]).sum(),
    "mean of tokens": lambda y, r: (y.mean(0) * r[0]).sum(),
    "values first": lambda y, r: (y.permute(2, 0, 1) * r.permute(2, 0, 1).contiguous()).sum(),
    "heads first": lambda y, r: (y.transpose(0, 1) * r.transpose(0, 1).contiguous()).sum(),
    "beside another": lambda y, r: (torch.cat((r[..., :1], y), -1) * torch.cat((r[..., :1], r), -1)).sum(),
    "one head": lambda y, r: (y[:, 1] * r[:, 1]).sum(),
}


@pytest.mark.parametrize("use", USES)
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("dim", [64, 128])
def test_gradients_of_any_strides(use, norm, dtype, dim):
    g = torch.Generator().manual_seed(3)
    x = [torch.randn(9, h, dim, generator=g).to(dtype) for h in (4, 2)]
    r = [torch.randn(9, h, dim, generator=g).to(dtype) for h in (4, 2)]
    w = weights(dim, g)
    f, p = frequencies(dim // 2), torch.arange(9) * 7
    angle = ref.angles(f, p)
    # the gradient of each result as autograd makes it, in its type
    dy = []
    for y, t in zip(x, r):
        y = y.clone().requires_grad_()
        dy.append(torch.autograd.grad(USES[use](y, t), y)[0])
    leaves = [t.to(DEV).requires_grad_() for t in x]
    out = G.qk_norm_rotary(*leaves, f.to(DEV), p.to(DEV), query_weight=w.to(DEV), key_weight=w.to(DEV), norm=norm)
    got = torch.autograd.grad(sum(USES[use](y, t.to(DEV)) for y, t in zip(out, r)), leaves)
    for name, d, t, v in zip("qk", got, x, dy):
        assert d.is_contiguous()
        ref.check_close(d, *ref.norm_rotary_grad(t, v, w, 1e-6, norm, angle, False)[0], "d" + name)
    # one of the two alone: the other's gradient is zeros
    out = G.qk_norm_rotary(*leaves, f.to(DEV), p.to(DEV), query_weight=w.to(DEV), key_weight=w.to(DEV), norm=norm)
    got = torch.autograd.grad(USES[use](out[1], r[1].to(DEV)), leaves, materialize_grads=True)
    assert not got[0].any()
    ref.check_close(got[1], *ref.norm_rotary_grad(x[1], dy[1], w, 1e-6, norm, angle, False)[0], "dk alone")


@pytest.mark.parametrize("norm", [False, True])
def test_gradient_refusals(norm):
    x, f, p = torch.zeros(4, 2, 64, device=DEV, dtype=BF), frequencies(32).to(DEV), torch.arange(4, device=DEV)

    def call(gq, gk, q=x, k=x):
        return torch.ops.gdpa.qk_norm_rotary_backward(gq, gk, q, k, f, p, p, None, None, 1e-6, norm, False, [], True)

    assert [t.shape for t in call(x, x)] == [x.shape, x.shape, (0,), (0,)]
    for args, error in (((x.float(), x), TypeError), ((x, x.cpu()), RuntimeError), ((x[:3], x), ValueError), ((x, x[:, :1]), ValueError),
                        ((x[..., :32], x), ValueError), ((x[0], x), ValueError), ((x, x, x.half(), x), TypeError), ((x, x, x[0], x), ValueError)):
        with pytest.raises(error):
            call(*args)


# ------------------------------------------------------------------------------------------ two threads


def calls_of_two_threads(fn, params, repeats=20000):
    """The return codes other than 0 of two host threads that call the same entry point, each with parameters and a stream of its own."""
    codes, begin = [[], []], threading.Barrier(2)
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()

    def work(i):
        torch.cuda.set_device(0)
        ref_to, stream = C.byref(params[i]), C.c_void_p(streams[i].cuda_stream)
        begin.wait()
        for n in range(repeats):  # the call gives up Python's lock
            code = fn(ref_to, stream)
            if code != 0:
                codes[i].append(code)
            if n % 200 == 0:
                streams[i].synchronize()

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return codes


@pytest.mark.parametrize("dim,is_fp32", [(64, 0), (128, 0), (64, 1), (128, 1)])
def test_two_threads_gradients_with_and_without_the_weights(dim, is_fp32):
    dtype = F32 if is_fp32 else BF
    f, p = frequencies(dim // 2).to(DEV), torch.arange(4, device=DEV)
    hold, params = [], []
    for with_weights in (True, False):
        x = {n: [torch.randn(4, 1, dim, device=DEV).to(dtype) for _ in range(3)] for n in ("query", "key")}
        w = torch.ones(dim, device=DEV)
        dw, workspace = torch.zeros(2, dim, device=DEV), torch.empty(_cabi.lib.gdpa_rotary_workspace_bytes(dim), dtype=torch.uint8, device=DEV)
        values = {"head_dim": dim, "is_fp32": is_fp32, "rotary.inv_freq": f.data_ptr(), "rotary.inv_freq_is_fp64": 1, "rotary.pairs": dim // 2, "rotary.axes": 1,
                  "rotary.norm": 1, "rotary.eps": 1e-6, "workspace": workspace.data_ptr(), "workspace_bytes": workspace.numel()}
        for i, (name, (a, y, dy)) in enumerate(x.items()):
            values.update({f"{name}.x": a.data_ptr(), f"{name}.y": y.data_ptr(), f"{name}.dy": dy.data_ptr(), f"{name}.weight": w.data_ptr(), f"{name}.heads": 1,
                           f"{name}.tokens": 4, f"{name}.positions": p.data_ptr(), f"{name}.positions_are_int64": 1})
            if with_weights:
                values[f"{name}.dweight"] = dw[i].data_ptr()
        hold.append((x, w, dw, workspace))
        params.append(nested(_cabi.GdpaRotaryParams, values))
    assert calls_of_two_threads(_cabi.lib.gdpa_qk_norm_rotary_bwd, params) == [[], []]


@pytest.mark.parametrize("is_fp32", [0, 1])
def test_two_threads_appends_to_blocks_of_two_sizes(is_fp32):
    dtype, dim, tokens = F32 if is_fp32 else BF, 64, 32
    f, p, slots = frequencies(dim // 2).to(DEV), torch.arange(tokens, device=DEV), torch.arange(tokens, device=DEV)
    hold, params = [], []
    for size in (16, 32):
        q, k, v, out = (torch.randn(tokens, 1, dim, device=DEV).to(dtype) for _ in range(4))
        caches, scales = torch.zeros(2, 64, 1, dim, dtype=torch.uint8, device=DEV), torch.ones(2, 64, device=DEV)
        hold.append((q, k, v, out, caches, scales))
        params.append(nested(_cabi.GdpaRotatedAppendParams, {
            "heads": 1, "cache.struct_size": C.sizeof(_cabi.GdpaCacheAppendParams), "cache.x_is_fp32": is_fp32, "cache.key": k.data_ptr(), "cache.value": v.data_ptr(),
            "cache.k_cache": caches[0].data_ptr(), "cache.v_cache": caches[1].data_ptr(), "cache.k_scales": scales[0].data_ptr(), "cache.v_scales": scales[1].data_ptr(),
            "cache.slot_mapping": slots.data_ptr(), "cache.tokens": tokens, "cache.num_blocks": 64 // size, "cache.block_size": size, "cache.kv_heads": 1,
            "cache.head_dim": dim, "rotary.inv_freq": f.data_ptr(), "rotary.inv_freq_is_fp64": 1, "rotary.pairs": dim // 2, "rotary.axes": 1, "rotary.norm": 1,
            "rotary.eps": 1e-6, "query": q.data_ptr(), "query_out": out.data_ptr(), "positions": p.data_ptr(), "positions_are_int64": 1}))
    assert calls_of_two_threads(_cabi.lib.gdpa_append_rotated_kv_cache_fp8, params) == [[], []]


# ------------------------------------------------------------------------------------------ a step that is refused


@pytest.mark.parametrize("rotated", [False, True])
def test_a_refused_step_can_be_made_again(rotated):
    g = torch.Generator().manual_seed(6)
    q, k, v = (torch.randn(2, 40, h, 64, generator=g).bfloat16().to(DEV) for h in (4, 2, 2))
    new = torch.tensor([[30, 10], [10, 30]], dtype=torch.int32, device=DEV)
    rotary = dict(inv_freq=frequencies(32).to(DEV)) if rotated else None

    def serve(refused):
        cache, outs = G.PagedKVCache(12, 16, 2, 64, 2, 64), []
        for x, y, z, n in zip(q, k, v, new):
            if refused:
                lens, left = cache.seq_lens.tolist(), int(cache.num_free)
                for args, options, error in (((x.float(), y.float(), z.float()), {}, TypeError), ((x[:, :3].contiguous(), y, z), {}, ValueError),
                                             ((x, y, z), dict(activation="none of them"), (KeyError, ValueError))):
                    with pytest.raises(error):
                        cache.step(*args, n, 30, rotary=rotary, **options)
                    assert cache.seq_lens.tolist() == lens and int(cache.num_free) == left
            outs.append(cache.step(x, y, z, n, 30, rotary=rotary, qk_scale=0.125))
        return (*outs, cache.seq_lens, cache.num_free, cache.block_tables, cache.k_cache.view(torch.uint8), cache.v_cache.view(torch.uint8), cache.k_scales,
                cache.v_scales)

    assert all(torch.equal(a, b) for a, b in zip(serve(False), serve(True)))


# ------------------------------------------------------------------------------------------ fp32 as near as its roundings
#
# With u = 2^-24, each fp32 rounding's share.  A sum of D squares: 4 in a lane's chain, the two halves, 4 over lanes: 9 u; with eps 10, so 5 of its root's inverse, and 4
# of rsqrt itself (2 units in the last place): r 9 u, x r w 11 u.  Sine and cosine 2 u each, of which 1.3 are the reduced angle's and the result's own
# rounding.  Two products and their sum: 2 u.  A value of a pair: (11 + 2 + 2) u (|n_a| + |n_b|), so
FORWARD = 16 * 2.0 ** -24
# Backwards dn = R^T dy is 4 u off (of both values' magnitudes), g = dn w 5 u; mean(g x) 5 + 9 u, times r^2 18 + 2 more: 34 u; g r 14 u; x r times that mean 10 + 34 + 1 u;
# their sum 1 u: 46 u of r (|g| + |u| mean |g u|) at most, so
BACKWARD = 48 * 2.0 ** -24
# A weight's gradient sums products that are 4 + 10 u off, one after the other: 18 of an item's heads and tokens, the item's into the warp's 1, 16 warps' heads, 14 rows of
# CTAs, 32 of these: 95 u, so
WEIGHTS = 128 * 2.0 ** -24


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("norm", [False, True])
@pytest.mark.parametrize("tokens,far,pairs", [(200, 5000, None), (200, 4 * 10 ** 6, 16), (3000, 5000, None), (1, 9, 24)])
def test_fp32_is_as_near_as_its_roundings(dim, interleaved, norm, tokens, far, pairs):
    g = torch.Generator().manual_seed(8)
    pairs = dim // 2 if pairs is None else pairs
    x, dy = ([torch.randn(tokens, h, dim, generator=g) for h in (5, 3)] for _ in range(2))
    w = [weights(dim, g) for _ in range(2)]
    f, p = frequencies(pairs), torch.randint(0, far, (tokens,), generator=g)
    angle = ref.angles(f, p)
    leaves = [t.to(DEV).requires_grad_() for t in (*x, *w)]
    out = G.qk_norm_rotary(*leaves[:2], f.to(DEV), p.to(DEV), query_weight=leaves[2], key_weight=leaves[3], norm=norm, interleaved=interleaved)
    got = torch.autograd.grad(out, leaves[:4 if norm else 2], [t.to(DEV) for t in dy])
    for i, name in enumerate("qk"):
        want, tol = ref.norm_rotary(x[i], w[i], 1e-6, norm, angle, interleaved)
        ref.check_close(out[i], want, tol * (2.0 ** 16 * FORWARD), name)
        (dx, tol), of_weight = ref.norm_rotary_grad(x[i], dy[i], w[i], 1e-6, norm, angle, interleaved)
        ref.check_close(got[i], dx, tol * (2.0 ** 15 * BACKWARD if norm else 2.0 ** 16 * FORWARD), "d" + name)
        if norm:
            ref.check_close(got[2 + i], of_weight[0], of_weight[1] * (2.0 ** 15 * WEIGHTS), "dw of " + name)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("lens", [[1] * 9, [70, 1, 200]])
def test_fp32_queries_of_an_append_are_as_near_as_their_roundings(dim, lens):
    g = torch.Generator().manual_seed(9)
    n, before = sum(lens), 3000
    q, k, v = (torch.randn(n, h, dim, generator=g) for h in (5, 3, 3))
    w, f = weights(dim, g), frequencies(dim // 2)
    p = torch.cat([before + torch.arange(m) for m in lens])
    offsets = torch.tensor([sum(lens[:b]) for b in range(len(lens) + 1)], dtype=torch.int32, device=DEV)
    cache, scales = torch.zeros(2, 1, 16, 3, dim, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.ones(2, 1, 3, device=DEV)
    out = G.append_rotated_kv_cache_fp8(q.to(DEV), k.to(DEV), v.to(DEV), cache[0], cache[1], scales[0], scales[1], torch.full((n,), -1, device=DEV), offsets,
                                        torch.tensor([before + m for m in lens], dtype=torch.int32, device=DEV), f.to(DEV), query_weight=w.to(DEV))
    want, tol = ref.norm_rotary(q, w, 1e-6, True, ref.angles(f, p), False)
    ref.check_close(out, want, tol * (2.0 ** 16 * FORWARD))
    assert not cache.view(torch.uint8).any()
