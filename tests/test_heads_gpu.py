"""The operators on either side of the attention on the GPU, against their plain 64-bit forms (tests/_heads_oracle.py)."""
import math

import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from tests import _heads_oracle as ref

pytestmark = pytest.mark.gpu
DEV = "cuda"
BF, F32 = torch.bfloat16, torch.float32


def i32(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def frequencies(pairs, base=10000.0, dtype=torch.float64):
    return (base ** -(torch.arange(pairs, dtype=torch.float64) / max(pairs, 1))).to(dtype)


def weights(dim, gen, dtype=F32):
    return (1 + 0.3 * torch.randn(dim, generator=gen)).to(dtype)


# ------------------------------------------------------------------------------------------ norm and rotation


def check_rotary(tokens, heads, dim, dtype, pairs=None, interleaved=False, sections=None, norm=True, weight=F32, kv=None, far=5000, packed=False, pos=torch.int64,
                 freq=torch.float64, grad=True, seed=0, edit=None, eps=1e-6):
    g = torch.Generator().manual_seed(seed)
    kv_tokens, kv_heads = kv or (tokens, max(1, heads // 2))
    pairs = dim // 2 if pairs is None else pairs
    inv = frequencies(pairs, dtype=freq)
    axes = () if sections is None else (len(sections),)
    qp, kp = (torch.randint(0, far, (*axes, n), generator=g).to(pos) for n in (tokens, kv_tokens))
    if packed:
        whole = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g).to(dtype)
        q, k, _ = whole.split([heads, kv_heads, kv_heads], 1)
        qd, kd, _ = whole.to(DEV).split([heads, kv_heads, kv_heads], 1)
        kp = qp
    else:
        q, k = torch.randn(tokens, heads, dim, generator=g).to(dtype), torch.randn(kv_tokens, kv_heads, dim, generator=g).to(dtype)
        if edit:
            edit(q, k)
        qd, kd = q.to(DEV), k.to(DEV)
    w = [None if weight is None else weights(dim, g, weight) for _ in range(2)]
    wd = [None if t is None else t.to(DEV).requires_grad_(grad) for t in w]
    qd, kd = qd.requires_grad_(grad), kd.requires_grad_(grad)
    options = dict(query_weight=wd[0], key_weight=wd[1], eps=eps, norm=norm, interleaved=interleaved, sections=sections)
    out = G.qk_norm_rotary(qd, kd, inv.to(DEV), qp.to(DEV), None if packed else kp.to(DEV), **options)
    angle = [ref.angles(inv, p, sections) for p in (qp, kp)]
    for name, x, y, v, a in zip("qk", (q, k), out, w, angle):
        assert y.is_contiguous() and y.dtype == dtype and y.shape == x.shape
        ref.check_close(y, *ref.norm_rotary(x, v, eps, norm, a, interleaved), name)
    if not grad:
        assert not out[0].requires_grad
        return
    dy = [torch.randn(y.shape, generator=g).to(dtype) for y in out]
    leaves = [qd, kd] + ([t for t in wd if t is not None] if norm else [])
    got = torch.autograd.grad(out, leaves, [t.to(DEV) for t in dy])
    want = [ref.norm_rotary_grad(x, d, v, eps, norm, a, interleaved) for x, d, v, a in zip((q, k), dy, w, angle)]
    for name, d, (dx, _) in zip("qk", got, want):
        ref.check_close(d, *dx, "d" + name)
    for name, d, (_, dw) in zip("qk", got[2:], want):
        ref.check_close(d, *dw, "dw of " + name)


@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("part", ["all", "half", 8, 24])
def test_rotary_heads(dim, dtype, interleaved, part):
    pairs = {"all": dim // 2, "half": dim // 4}.get(part, part)
    check_rotary(77, 5, dim, dtype, pairs, interleaved)
    check_rotary(3, 1, dim, dtype, pairs, interleaved, weight=BF, seed=1)


@pytest.mark.parametrize("tokens,heads,kv", [(1, 1, (1, 1)), (1, 32, (1, 4)), (0, 4, (3, 2)), (3, 4, (0, 2)), (513, 3, (40, 7)), (2500, 12, (9000, 1)),
                                             (300, 128, (300, 128))])
def test_rotary_sizes(tokens, heads, kv):
    check_rotary(tokens, heads, 128, BF, kv=kv)
    check_rotary(tokens, heads, 64, F32, kv=kv, interleaved=True, seed=3)


@pytest.mark.parametrize("options", [
    dict(sections=(8, 12, 12), pos=torch.int32), dict(sections=(32, 0)), dict(sections=(8, 8, 8, 8), interleaved=True), dict(sections=(3, 29), freq=F32),
    dict(norm=False), dict(norm=False, weight=None, interleaved=True), dict(weight=None), dict(pairs=0), dict(pairs=0, norm=False), dict(packed=True),
    dict(far=10 ** 6 * 4, pos=torch.int32), dict(far=1 << 40), dict(eps=0.0), dict(eps=100.0), dict(grad=False), dict(weight=BF, packed=True)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_options(options, dtype):
    check_rotary(200, 6, 64, dtype, **options)


def test_rotary_negative_positions_turn_back():
    x = torch.randn(4, 2, 64, device=DEV)
    f, p = frequencies(32).to(DEV), torch.tensor([5, 1000, 123456, 7], device=DEV)
    y, _ = G.qk_norm_rotary(x, x, f, p, norm=False)
    z, _ = G.qk_norm_rotary(y, y, f, -p, norm=False)
    assert float((z - x).abs().max()) < 2.0 ** -16 * 8  # two turns, each off by 2^-16 of values below 6


@pytest.mark.parametrize("dtype", [BF, F32])
def test_rotary_special_values_stay_in_their_head(dtype):
    def edit(q, k):
        q[1, 0, 3], q[2, 1, 70], k[0, 1, 5], k[4, 0] = math.inf, math.nan, -math.inf, 0.0
        q[5], k[5] = 0.0, 1e-30

    check_rotary(8, 4, 128, dtype, pairs=16, edit=edit, grad=False)
    check_rotary(8, 4, 128, dtype, pairs=64, edit=edit, grad=False)


def test_rotary_without_norm_special_values_stay_in_their_pair():
    def edit(q, k):
        q[1, 0, 100], q[1, 0, 101], k[2, 0, 40] = math.inf, math.nan, math.nan

    for interleaved in (False, True):
        check_rotary(4, 2, 128, BF, pairs=16, interleaved=interleaved, norm=False, edit=edit, grad=False)


def test_rotary_one_gradient_of_two_and_expanded_ones():
    g = torch.Generator().manual_seed(5)
    q, k = torch.randn(9, 4, 64, generator=g).bfloat16(), torch.randn(9, 2, 64, generator=g).bfloat16()
    w = weights(64, g)
    f, p = frequencies(32), torch.arange(9)
    qd, kd, wd = q.to(DEV).requires_grad_(), k.to(DEV), w.to(DEV).requires_grad_()
    a, b = G.qk_norm_rotary(qd, kd, f.to(DEV), p.to(DEV), query_weight=wd, key_weight=wd.detach())
    a.sum().backward()  # a gradient that is one value, expanded
    dx, dw = ref.norm_rotary_grad(q, torch.ones_like(q), w, 1e-6, True, ref.angles(f, p), False)
    ref.check_close(qd.grad, *dx)
    ref.check_close(wd.grad, *dw)
    # a weight that queries and keys share: the sum of both
    qd.grad = wd.grad = None
    kd.requires_grad_()
    a, b = G.qk_norm_rotary(qd, kd, f.to(DEV), p.to(DEV), query_weight=wd, key_weight=wd)
    (a.float().sum() + b.float().sum()).backward()
    _, dk = ref.norm_rotary_grad(k, torch.ones_like(k), w, 1e-6, True, ref.angles(f, p), False)
    ref.check_close(wd.grad, dw[0] + dk[0], dw[1] + dk[1])


def test_rotary_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    x, dy, w = torch.randn(3, 2, 64, generator=g), torch.randn(3, 2, 64, generator=g), weights(64, g)
    f, p = frequencies(32).to(DEV), torch.tensor([0, 17, 90000], device=DEV)

    def value(x, w):  # in 64 bits from the kernel's fp32 outputs
        return float((G.qk_norm_rotary(x, x, f, p, query_weight=w, key_weight=w)[0].double() * dy.to(DEV).double()).sum())

    xd, wd = x.to(DEV).requires_grad_(), w.to(DEV).requires_grad_()
    y, _ = G.qk_norm_rotary(xd, xd.detach(), f, p, query_weight=wd)
    dx, dw = torch.autograd.grad(y, (xd, wd), dy.to(DEV))
    step = 2.0 ** -6
    for grad, at, of in ((dx, (2, 1, 40), "x"), (dx, (0, 0, 0), "x"), (dw, (33,), "w"), (dw, (2,), "w")):
        ends = []
        for s in (step, -step):
            x2, w2 = x.clone(), w.clone()
            (x2 if of == "x" else w2)[at] += s
            ends.append(value(x2.to(DEV), w2.to(DEV)))
        # outputs below 8 are off by 2^-21 each, some hundred of them with random signs; the third derivative is below 1
        assert abs((ends[0] - ends[1]) / (2 * step) - float(grad[at])) < 2.0 ** -21 * 8 * 400 ** 0.5 / step + step ** 2


def test_rotary_gradients_are_the_same_every_time():
    q, k = torch.randn(3000, 8, 128, device=DEV).bfloat16(), torch.randn(3000, 8, 128, device=DEV).bfloat16()
    w, f, p = torch.ones(128, device=DEV), frequencies(64).to(DEV), torch.arange(3000, device=DEV)

    def grads():
        leaves = [t.clone().requires_grad_() for t in (q, k, w)]
        out = G.qk_norm_rotary(leaves[0], leaves[1], f, p, query_weight=leaves[2], key_weight=leaves[2])
        return torch.autograd.grad(out, leaves, (k, q))

    first = grads()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, grads()))


def test_rotary_long_batches_offsets_pass_32_bits():
    tokens, heads = 1 << 18, 72  # 2^18 * 72 * 128 = 2.4e9 values
    x = torch.randn(1, heads, 128, device=DEV).bfloat16().expand(tokens, heads, 128).contiguous()
    k, w = x[:, :1], torch.ones(128, device=DEV)
    p = torch.arange(tokens, device=DEV)
    f = frequencies(64).to(DEV)
    y, _ = G.qk_norm_rotary(x, k, f, p, query_weight=w)
    at = torch.tensor([0, 1, 99999, tokens - 2, tokens - 1])
    ref.check_close(y[at.to(DEV)], *ref.norm_rotary(x[:5].cpu(), None, 1e-6, True, ref.angles(f.cpu(), at), False))
    del y
    dx, _, dw, _ = torch.ops.gdpa.qk_norm_rotary_backward(x, k, x, k, f, p, p, w, None, 1e-6, True, False, [], True)
    want, _ = ref.norm_rotary_grad(x[:5].cpu(), x[:5].cpu(), None, 1e-6, True, ref.angles(f.cpu(), at), False)
    ref.check_close(dx[at.to(DEV)], *want)
    assert bool(torch.isfinite(dw).all())


def test_rotary_refusals():
    x, f, p = torch.zeros(4, 2, 64, device=DEV, dtype=BF), frequencies(32).to(DEV), i32([0, 1, 2, 3])
    for args, options, error in (
            ((x.half(), x.half(), f, p), {}, TypeError), ((x, x.float(), f, p), {}, TypeError), ((x[0], x, f, p), {}, ValueError),
            ((x[:, :, ::2], x, f, p), {}, ValueError), ((x, x[..., :32], f, p), {}, NotImplementedError), ((x, x[:3], f, p), {}, ValueError),
            ((x, x, f[:12], p), {}, NotImplementedError), ((x, x, torch.cat([f, f]), p), {}, ValueError), ((x, x, f.half(), p), {}, TypeError),
            ((x, x, f.cpu(), p), {}, RuntimeError), ((x, x, f, p.float()), {}, TypeError), ((x, x, f, p[:3]), {}, ValueError),
            ((x, x, f, p[None]), {}, ValueError), ((x, x, f, p), dict(sections=(16, 16)), ValueError),
            ((x, x, f, torch.stack([p, p])), dict(sections=(16, 15)), ValueError), ((x, x, f, torch.stack([p, p])), dict(sections=(40, -8)), ValueError),
            ((x, x, f, torch.stack([p] * 5)), dict(sections=(8, 8, 8, 8, 0)), ValueError), ((x, x, f, p), dict(eps=-1.0), ValueError),
            ((x, x, f, p), dict(eps=math.nan), ValueError), ((x, x, f, p), dict(query_weight=f[:5]), TypeError),
            ((x, x, f, p), dict(key_weight=torch.ones(63, device=DEV)), ValueError), ((x[:1].expand(4, 2, 64), x, f, p), {}, ValueError),
            ((x.requires_grad_(), x, f.clone().requires_grad_(), p), {}, RuntimeError)):
        with pytest.raises(error):
            G.qk_norm_rotary(*args, **options)
    a, _ = G.qk_norm_rotary(x, x.detach(), f, p)
    (g,) = torch.autograd.grad(a, x, torch.ones_like(a), create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.float().sum(), x)


def test_rotary_replays_from_a_graph_and_on_another_stream():
    q, k = torch.randn(50, 4, 128, device=DEV).bfloat16(), torch.randn(50, 2, 128, device=DEV).bfloat16()
    w, f, p = weights(128, torch.Generator().manual_seed(0)).to(DEV), frequencies(64).to(DEV), torch.arange(50, device=DEV)
    still = [t.clone() for t in (q, k, w)]

    def step():
        leaves = [t.detach().requires_grad_() for t in still]
        out = G.qk_norm_rotary(leaves[0], leaves[1], f, p, query_weight=leaves[2])
        return (*out, *torch.autograd.grad(out, leaves, out))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        eager = step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for scale in (1, 3):
        still[0].copy_(q * scale)
        still[2].copy_(w * scale)
        graph.replay()
        torch.cuda.synchronize()
        again = step()
        assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(outs, again))
        if scale == 1:
            assert all(torch.equal(a.detach(), b.detach()) for a, b in zip(eager, again))


@pytest.mark.filterwarnings("ignore")
def test_rotary_compiles():
    q, k = torch.randn(20, 4, 64, device=DEV).bfloat16(), torch.randn(20, 2, 64, device=DEV).bfloat16()
    w, f, p = torch.ones(64, device=DEV), frequencies(32).to(DEV), torch.arange(20, device=DEV)

    def fn(q, k, w):
        a, b = G.qk_norm_rotary(q, k, f, p, query_weight=w)
        return a * 2, b

    res = []
    for f_ in (fn, torch.compile(fn, backend="aot_eager", fullgraph=True)):
        leaves = [t.clone().requires_grad_() for t in (q, k, w)]
        a, b = f_(*leaves)
        res.append((a, b, *torch.autograd.grad((a, b), leaves, (a.detach(), b.detach()))))
    assert all(torch.equal(x, y) for x, y in zip(*res))


# ------------------------------------------------------------------------------------------ with the append


def check_append(before, new, heads, kv_heads, dim, dtype, size, pairs=None, interleaved=False, sections=None, norm=True, weight=F32, given=False, seed=0, missing=(),
                 lens=torch.int32, edit=None, head_major=False, loud=1.0):
    g = torch.Generator().manual_seed(seed)
    pairs, batch, tokens = dim // 2 if pairs is None else pairs, len(new), sum(new)
    held = [-(-(b + n) // size) for b, n in zip(before, new)]
    blocks = sum(held) + 3
    order = torch.randperm(blocks, generator=g)
    table, at = torch.full((batch, max(held + [1])), -1, dtype=torch.int64), 0
    slots, positions, offsets = [], [], [0]
    for b, n in enumerate(held):
        table[b, :n] = order[at:at + n]
        at += n
        for p in range(before[b], before[b] + new[b]):
            slots.append(-1 if len(slots) in missing else int(table[b, p // size]) * size + p % size)
            positions.append(p)
        offsets.append(offsets[-1] + new[b])
    slots, positions = torch.tensor(slots, dtype=torch.int64), torch.tensor(positions, dtype=torch.int64)
    if given:
        axes = () if sections is None else (len(sections),)
        positions = torch.randint(-100, 10000, (*axes, tokens), generator=g)
    elif sections is not None:
        positions = positions.expand(len(sections), -1)
    whole = torch.randn(tokens, heads + 2 * kv_heads, dim, generator=g) * loud
    if edit:
        edit(whole)
    whole = whole.to(dtype)
    q, k, v = whole.split([heads, kv_heads, kv_heads], 1)
    caches = [torch.randint(0, 120, (blocks, size, kv_heads, dim), generator=g, dtype=torch.uint8) for _ in range(2)]
    scales = [2.0 ** torch.randint(-9, -5, (blocks, kv_heads), generator=g).float() for _ in range(2)]

    def stored(c):
        c = c.to(DEV)
        return (c.transpose(1, 2).contiguous().transpose(1, 2) if head_major else c).view(torch.float8_e4m3fn)

    cd, sd = [stored(c) for c in caches], [s.to(DEV) for s in scales]
    w = [None if weight is None else weights(dim, g, weight) for _ in range(2)]
    inv = frequencies(pairs)
    ends = torch.tensor([b + n for b, n in zip(before, new)], dtype=lens)
    out = G.append_rotated_kv_cache_fp8(
        *whole.to(DEV).split([heads, kv_heads, kv_heads], 1), *cd, *sd, slots.to(DEV), torch.tensor(offsets, dtype=lens, device=DEV), ends.to(DEV), inv.to(DEV),
        positions=positions.to(DEV) if given else None, query_weight=None if w[0] is None else w[0].to(DEV), key_weight=None if w[1] is None else w[1].to(DEV),
        norm=norm, interleaved=interleaved, sections=sections)
    angle = ref.angles(inv, positions, sections)
    ref.check_close(out, *ref.norm_rotary(q, w[0], 1e-6, norm, angle, interleaved), "query")
    keys, tol = ref.norm_rotary(k, w[1], 1e-6, norm, angle, interleaved)
    got = [c.view(torch.uint8).cpu() for c in cd]
    ref.check_append(keys, tol, caches[0], scales[0], got[0], sd[0].cpu(), slots, "keys")
    ref.check_append(v.double(), torch.zeros_like(tol), caches[1], scales[1], got[1], sd[1].cpu(), slots, "values")


@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_ragged(size, dim, dtype):
    # single tokens, drafts, ends inside blocks, whole blocks, a prompt over several
    check_append([0, 5, size - 1, size, 3, 0, 40], [1, 1, 1, 2, 0, 3 * size + 5, size], 4, 2, dim, dtype, size)
    check_append([7] * 40, [1] * 40, 4, 3, dim, dtype, size, seed=1)  # single tokens
    check_append([size - 2] * 9, [4] * 9, 2, 1, dim, dtype, size, seed=2, interleaved=True)  # drafts over the blocks' ends
    check_append([0], [1], 1, 1, dim, dtype, size, seed=3)
    check_append([size // 2] * 2, [2 * size, 11], 6, 2, dim, dtype, size, seed=4, weight=BF)


@pytest.mark.parametrize("size,dim,dtype", [(16, 64, BF), (64, 128, BF), (128, 128, BF), (128, 64, F32), (64, 128, F32)])
@pytest.mark.parametrize("given", [False, True])
def test_append_prompts_among_single_tokens(size, dim, dtype, given):
    """Runs of every length in the same windows, where single tokens are most of the requests and where they are not."""
    before = [size - 3, 0, 5, 2 * size, 11, size - 1, 40, 0, 7]
    new = [1, 2, 9, 70, 3, 40, 200, 1, 17]
    check_append(before * 3, [1] * 18 + new, 3, 2, dim, dtype, size, given=given)
    check_append(before, new, 3, 2, dim, dtype, size, seed=1, given=given, loud=1e3 if size == 64 else 1.0)
    check_append(before, list(reversed(new)), 1, 1, dim, dtype, size, seed=2, given=given)


@pytest.mark.parametrize("options", [
    dict(given=True), dict(given=True, sections=(16, 24, 24)), dict(sections=(32, 32)), dict(norm=False), dict(norm=False, given=True, interleaved=True),
    dict(pairs=8), dict(pairs=0), dict(pairs=24, interleaved=True), dict(weight=None), dict(lens=torch.int64), dict(head_major=True), dict(loud=1e4, norm=False),
    dict(loud=1e-30, norm=False)])
def test_append_options(options):
    check_append([0, 20, 0, 63, 5], [33, 1, 70, 1, 3], 4, 2, 128, BF, 64, **options)
    check_append([0, 20, 0, 63, 5] * 6, [1, 1, 2, 3, 1] * 6, 2, 4, 128, F32, 16, seed=1, **options)


def test_append_tokens_without_a_slot():
    check_append([0, 20, 0, 63, 5] * 6, [1, 1, 2, 3, 1] * 6, 2, 4, 128, F32, 16, seed=1, missing=(0, 3, 4, 40, 41, 42, 43))
    check_append([0, 20, 0, 63, 5], [33, 1, 70, 1, 3], 4, 2, 128, BF, 64, missing=(0, 1, 31, 32, 33, 34, 107))
    # one in the middle of a block's tokens makes two runs of them, which the append does not take: said with validation on
    old = G.set_offset_validation(True)
    try:
        with pytest.raises(ValueError):
            check_append([0, 20, 0, 63, 5], [33, 1, 70, 1, 3], 4, 2, 128, BF, 64, missing=(0, 3, 4, 40, 41, 42, 43, 90))
    finally:
        G.set_offset_validation(old)


def test_append_many_requests_without_tokens_between():
    new = ([0] * 50 + [1]) * 30 + [0] * 70 + [2, 0, 5]
    check_append([3] * len(new), new, 2, 1, 64, BF, 16)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_append_special_values(dtype):
    def edit(whole):
        whole[0, 2, 5], whole[1, 3, 9], whole[2, 4, 3], whole[40, 5, 0] = math.inf, math.nan, math.inf, -math.inf
        whole[3], whole[70] = 0.0, 0.0

    # rows with an infinity: keys of 2 and 3 are NaN and 0 after the norm, values keep it at the largest
    check_append([0, 5, 16, 0], [70, 1, 1, 20], 2, 2, 64, dtype, 16, edit=edit)
    check_append([0] * 80, [1] * 80, 2, 2, 64, dtype, 16, edit=edit)
    check_append([0, 5, 16, 0], [70, 1, 1, 20], 2, 2, 64, dtype, 64, edit=edit, norm=False, pairs=8)


def test_append_with_offsets_that_are_none_ends():
    """Offsets that are not in order: positions are unspecified, norms hold, nothing else is written."""
    g = torch.Generator().manual_seed(0)
    for offsets in ([0, 900, 900] + [0] * 97 + [70], [50] * 60 + [0] * 40 + [5], list(range(2000, 1899, -1))):
        for tokens in (70, 4000):
            q = torch.randn(tokens, 2, 64, generator=g).to(DEV)
            c = [torch.zeros(4, 16, 1, 64, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
            s = [torch.ones(4, 1, device=DEV) for _ in range(2)]
            slots = torch.full((tokens,), -1, device=DEV)
            y = G.append_rotated_kv_cache_fp8(q, q[:, :1], q[:, 1:], *c, *s, slots, i32(offsets), i32([5] * 100), frequencies(32).to(DEV))
            # a rotation keeps each pair's length: 2^-16 as in the oracle
            want = q * torch.rsqrt(q.pow(2).mean(-1, keepdim=True) + 1e-6)
            a, b = (x[..., :32].hypot(x[..., 32:]) for x in (y, want))
            assert float(((a - b).abs() - 2.0 ** -16 * b).max()) <= 0
            assert all(int(x.view(torch.uint8).sum()) == 0 for x in c)


def test_append_nothing():
    check_append([], [], 2, 1, 64, BF, 16)
    check_append([3, 0], [0, 0], 2, 1, 64, BF, 16)
    check_append([0, 0], [5, 6], 2, 1, 64, BF, 16, missing=range(11))


def test_append_into_a_cache_without_blocks():
    x = torch.randn(3, 2, 64, device=DEV).bfloat16()
    c, s = torch.zeros(0, 16, 2, 64, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn), torch.zeros(0, 2, device=DEV)
    f = frequencies(32)
    out = G.append_rotated_kv_cache_fp8(x, x, x, c, c.clone(), s, s.clone(), torch.full((3,), -1, device=DEV), i32([0, 3]), i32([3]), f.to(DEV))
    ref.check_close(out, *ref.norm_rotary(x.cpu(), None, 1e-6, True, ref.angles(f, torch.arange(3)), False))


def test_append_long_strides_and_offsets():
    """A cache whose later blocks lie past 2^32 bytes, two tokens in its first and last."""
    blocks, size = 300000, 128
    c = [torch.zeros(blocks, size, 1, 128, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn) for _ in range(2)]
    s = [torch.ones(blocks, 1, device=DEV) for _ in range(2)]
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 128, generator=g).bfloat16()
    f = frequencies(64)
    slots = torch.tensor([5 * size, (blocks - 1) * size])
    q, k, v = x.to(DEV).split(1, 1)
    G.append_rotated_kv_cache_fp8(q, k, v, *c, *s, slots.to(DEV), i32([0, 1, 2]), i32([1, 1]), f.to(DEV))
    want, tol = ref.norm_rotary(x[:, 1:2], None, 1e-6, True, ref.angles(f, torch.zeros(2)), False)
    for i, b in enumerate((5, blocks - 1)):
        for name, cache, scale, y, t in (("k", c[0], s[0], want, tol), ("v", c[1], s[1], x[:, 2:].double(), 0 * tol)):
            ref.check_append(y[i:i + 1], t[i:i + 1], torch.zeros(1, size, 1, 128, dtype=torch.uint8), torch.ones(1, 1), cache[b:b + 1].view(torch.uint8).cpu(),
                             scale[b:b + 1].cpu(), torch.tensor([0]), name)
    table = i32([[5, blocks - 1]])
    key, value = G.read_kv_cache_fp8(*c, *s, table, i32([0, size + 1]), size + 1)
    for packed, cache, scale in ((key, c[0], s[0]), (value, c[1], s[1])):
        assert torch.equal(packed[0].float(), cache[5, 0].float() * scale[5, 0]) and torch.equal(packed[-1].float(), cache[-1, 0].float() * scale[-1, 0])


# ------------------------------------------------------------------------------------------ read back


def check_read(lens, first, heads, dim, size, dtype, width=None, extra=0, seed=0, head_major=False, holes=(), ints=torch.int32, powers=True, without_first=False):
    g = torch.Generator().manual_seed(seed)
    held = [-(-(n + f) // size) for n, f in zip(lens, first)]
    blocks, batch = sum(held) + 2, len(lens)
    width = max(held + [1]) if width is None else width
    order, at = torch.randperm(blocks, generator=g), 0
    table = torch.full((batch, width), -1, dtype=torch.int32)
    for b, n in enumerate(held):
        n = min(n, width)
        table[b, :n] = order[at:at + n]
        at += n
    for b, j, value in holes:
        table[b, j] = value
    caches = [torch.randint(0, 256, (blocks, size, heads, dim), generator=g, dtype=torch.uint8) for _ in range(2)]
    for c in caches:
        c[(c & 127) == 127] = 0x37  # no NaN: they are looked at by themselves
    scales = [2.0 ** torch.randint(-12, 3, (blocks, heads), generator=g).float() if powers else torch.rand(blocks, heads, generator=g) for _ in range(2)]
    offsets = [0]
    for n in lens:
        offsets.append(offsets[-1] + n)
    total = offsets[-1] + extra
    want = [ref.read(c, s, table, offsets, [0] * batch if without_first else first, total) for c, s in zip(caches, scales)]
    cd = [(c.to(DEV).transpose(1, 2).contiguous().transpose(1, 2) if head_major else c.to(DEV)).view(torch.float8_e4m3fn) for c in caches]
    got = G.read_kv_cache_fp8(*cd, *(s.to(DEV) for s in scales), table.to(DEV), torch.tensor(offsets, dtype=ints, device=DEV), total,
                              first_tokens=None if without_first else torch.tensor(first, dtype=ints, device=DEV), dtype=dtype)
    for y, x in zip(got, want):
        assert y.dtype == dtype and y.shape == (total, heads, dim) and y.is_contiguous()
        assert torch.equal(y.cpu(), x.float().to(dtype))  # the product in fp32, then rounded


@pytest.mark.parametrize("size", [16, 32, 64, 128])
@pytest.mark.parametrize("dim", [64, 128])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_read(size, dim, dtype):
    check_read([1, 0, 100, 0, 0, 3, size, 2 * size + 1], [0, 4, 30, 0, 7, size - 1, size, 5], 3, dim, size, dtype)
    check_read([5, 70], [0, 0], 1, dim, size, dtype, without_first=True, powers=False)


@pytest.mark.parametrize("options", [dict(extra=40), dict(width=2), dict(width=0), dict(holes=((1, 0, -1), (1, 2, 10 ** 6), (0, 0, -5))), dict(head_major=True),
                                     dict(ints=torch.int64)])
def test_read_options(options):
    check_read([20, 90, 33], [3, 0, 50], 2, 128, 16, BF, **options)


def test_read_nothing_and_many():
    check_read([], [], 2, 64, 16, BF)
    check_read([], [], 2, 64, 16, BF, extra=5)
    check_read([0, 0, 0], [0, 1, 2], 2, 64, 16, F32)
    check_read([i % 3 for i in range(3000)], [i % 7 for i in range(3000)], 1, 64, 16, BF)


def test_read_nan_and_what_lies_behind():
    c = torch.full((2, 16, 1, 64), 0x7f, dtype=torch.uint8, device=DEV)  # NaN everywhere but in three rows
    c[1, :3] = 0x38
    s = torch.ones(2, 1, device=DEV)
    c = c.view(torch.float8_e4m3fn)
    key, value = G.read_kv_cache_fp8(c, c, s, s, i32([[1, 0]]), i32([0, 4]), 6)
    assert torch.equal(key[:3].float(), torch.ones(3, 1, 64, device=DEV)) and bool(torch.isnan(key[3].float()).all())
    assert torch.equal(key[4:].float(), torch.zeros(2, 1, 64, device=DEV)) and torch.equal(value[:3], key[:3])


def test_cache_refusals():
    x = torch.zeros(4, 2, 64, device=DEV, dtype=BF)
    c = torch.zeros(3, 16, 2, 64, dtype=torch.uint8, device=DEV).view(torch.float8_e4m3fn)
    s, f, slots = torch.ones(3, 2, device=DEV), frequencies(32).to(DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    o, n, t = i32([0, 4]), i32([4]), i32([[0, 1]])
    good = [x, x, x, c, c.clone(), s, s.clone(), slots, o, n, f]
    for at, bad, error in ((0, x.half(), TypeError), (1, x.float(), TypeError), (2, x[:3], ValueError), (0, x[:3], ValueError), (1, x[:, :1], ValueError),
                           (3, c.view(torch.uint8), TypeError), (5, s.double(), TypeError), (7, slots.int(), TypeError), (7, slots[:3], ValueError),
                           (8, o[:1], ValueError), (9, n.float(), TypeError), (10, f[:5], NotImplementedError), (10, torch.cat([f, f]), ValueError),
                           (2, x[:, :1].expand(4, 2, 64), ValueError)):
        with pytest.raises(error):
            G.append_rotated_kv_cache_fp8(*good[:at], bad, *good[at + 1:])
    for options, error in ((dict(positions=o), ValueError), (dict(sections=(16, 16), positions=slots), ValueError), (dict(eps=-1), ValueError),
                           (dict(query_weight=f), TypeError), (dict(key_weight=torch.ones(32, device=DEV)), ValueError)):
        with pytest.raises(error):
            G.append_rotated_kv_cache_fp8(*good, **options)
    good = [c, c, s, s, t, o, 4]
    for at, bad, error in ((0, c.view(torch.uint8), TypeError), (2, s[:2], ValueError), (4, t.long(), TypeError), (4, t.expand(2, 2), ValueError),
                           (5, o.float(), TypeError), (5, o[:0], ValueError), (6, -1, ValueError)):
        with pytest.raises(error):
            G.read_kv_cache_fp8(*good[:at], bad, *good[at + 1:])
    for options, error in ((dict(first_tokens=o), ValueError), (dict(dtype=torch.float16), TypeError)):
        with pytest.raises(error):
            G.read_kv_cache_fp8(*good, **options)
    with pytest.raises(RuntimeError):
        G.read_kv_cache_fp8(c, c, s.clone().requires_grad_(), s, t, o, 4)[0].float().sum().backward()
