"""The gradient of the trunk recurrence's decay keeps its float32 digits: from the operator's gradient of `scale` to the parameters' there are no roundings but float32's.

a = exp(-softplus(d) exp(l)), da/dl = -a softplus(d) exp(l).  Float32: two exponentials and a logarithm (2 units each, of arguments below 4, whose own rounding they
pass on: 4 more each), four products: below 32 units of 2^-24."""
import pytest
import torch

from kfold_b200 import functional as F
from kfold_b200 import trunk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, dtype)


@pytest.mark.parametrize("c, dtype", [(128, BF), (128, F32), (64, BF)])
def test_decay(c, dtype):
    mod = trunk.ParcaeRecurrence(c).to(DEV)
    with torch.no_grad():
        mod.parcae_log_a.add_(_randn(6, c, scale=0.3))
        mod.parcae_log_delta.add_(_randn(7, c, scale=0.3))
    z, u, dout = (_randn(i, 1, 21, 21, c, dtype=dtype) for i in (1, 2, 3))
    z.requires_grad_()
    with torch.autocast("cuda", dtype=BF, enabled=dtype == F32):
        out = mod(z, u)
        a, _ = mod.dynamics(z.device)
    out.backward(dout)
    g = F.residual_norm_backward(dout, None, out.detach(), torch.empty(out.shape, dtype=BF, device=DEV), None, z.detach(), a)
    assert torch.equal(z.grad, g.x)                       # (the decay itself is inference's)
    delta, rate = torch.nn.functional.softplus(mod.parcae_log_delta.detach().double()), torch.exp(mod.parcae_log_a.detach().double())
    want = g.scale.double() * -torch.exp(-delta * rate) * delta * rate
    assert mod.parcae_log_a.grad.dtype == F32
    assert ((mod.parcae_log_a.grad.double() - want).abs() <= 32 * 2.0 ** -24 * want.abs()).all()
