"""Calls of the operators on either side of the attention that are easily got wrong, on the GPU."""
import pytest
import torch

import ads_model_kernel_library_b200.gdpa as G
from tests import _heads_oracle as ref
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
