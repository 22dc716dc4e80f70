"""Gradients of a residual stream without a norm, u and x kept in 8 bits: against 64-bit arithmetic at the values that are kept.

Widths whose rows have other than a multiple of four groups of 32 channels, so that exponents come one by one, and ones that come in words; exponents that start between
two words.  Tolerances of the operator are those of test_gpu_residual_norm.py (256 roundings of float32 and one more for each term of a sum over samples or rows), of the
modules those of test_gpu_conditioned_training.py."""
import pytest
import torch

import plain_residual as R
import plain_training as P
import test_gpu_conditioned_training as T
from kfold_b200 import _lib as L
from kfold_b200 import autograd as A
from kfold_b200 import functional as F
from kfold_b200 import modules as M
from kfold_b200 import trunk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
TYPES = {"bf16": (BF, BF), "f32": (F32, F32), "mixed": (F32, BF)}


@pytest.fixture(autouse=True)
def _status():
    yield
    assert L.device_status() == 0


def _randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, dtype)


def _near(got, ref, size, steps, what):
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    far = (got.double() - ref).abs() - (P.HALF_STEP[got.dtype] * (ref.abs() + steps * P.U32 * size) + steps * P.U32 * size)
    assert (far <= 1e-37).all(), f"{what}: {far.max().item():.3e} beyond its room"


def _case(samples, c, types, gate, scale, l=13):
    st, ct = TYPES[types]
    # (magnitudes of groups that differ, so that another group's or tensor's exponent shows)
    spread = torch.exp2(torch.arange(c, device=DEV).div(32, rounding_mode="floor") % 5 - 2.0)
    x, u = (_randn(1, 2 * samples, l, c) * spread).to(st), (_randn(2, 2 * samples, l, c) / spread).to(ct)
    return x, u, _randn(3, 2, l, c, dtype=ct) if gate else None, 1 + 0.2 * _randn(4, c) if scale else None, _randn(5, 2 * samples, l, c, dtype=st, scale=0.1)


def _check(x, u, gate, scale, dr, samples, keep=F.compress):
    r, _ = F.residual_norm(x, u, gate, scale, samples=samples, norm=False)
    u8, x8 = keep(u), keep(x)
    g = F.residual_norm_backward(dr, None, r, u8, gate, x8, scale, samples=samples)
    ref = R.residual_norm_gradient(dr, None, r, F.expand(u8), gate, F.expand(x8), scale, None, None, samples, 1e-5)
    rows = r.numel() // r.shape[-1]
    for name, there, more in (("x", True, 0), ("u", True, 0), ("gate", gate is not None, samples), ("scale", scale is not None, rows)):
        if there:
            _near(getattr(g, name), *ref[name], 256 + more, name)
        else:
            assert getattr(g, name) is None


@pytest.mark.parametrize("c", [8, 32, 64, 96, 100, 128, 136, 160, 192, 256, 320, 384, 520, 672, 768, 1000])
@pytest.mark.parametrize("gate, scale", [(True, False), (False, True), (True, True)], ids=["gate", "scale", "gate and scale"])
@pytest.mark.parametrize("samples", [1, 4])
@pytest.mark.parametrize("types", list(TYPES))
def test_widths(c, gate, scale, samples, types):
    _check(*_case(samples, c, types, gate, scale), samples)


def _between_words(t):
    k = F.compress(t)
    e = torch.empty(k.exponents.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(k.exponents.shape)
    return F.Compressed(k.values, e.copy_(k.exponents), k.dtype)


@pytest.mark.parametrize("samples", [1, 4])
def test_exponents_between_two_words(samples):
    case = _case(samples, 128, "bf16", True, True)
    assert _between_words(case[0]).exponents.data_ptr() % 4
    _check(*case, samples, keep=_between_words)


@pytest.mark.parametrize("c", [64, 160, 128])
@pytest.mark.parametrize("samples", [1, 4])
def test_nothing_came_back_through_the_norm(c, samples):
    x, u, gate, scale, dr = _case(samples, c, "bf16", True, True)
    leaves = [t.requires_grad_() for t in (x, u, gate, scale)]
    weight = (1 + 0.1 * _randn(6, c)).requires_grad_()
    with A.compressed():
        r, _ = A.residual_norm(x, u, gate, scale, weight, samples=samples)
    r.backward(dr)
    u8, x8 = (F.expand(F.compress(t.detach())) for t in (u, x))
    ref = R.residual_norm_gradient(dr, None, r.detach(), u8, gate.detach(), x8, scale.detach(), None, None, samples, 1e-5)
    for t, name, more in zip(leaves, ("x", "u", "gate", "scale"), (0, 0, samples, r.numel() // c)):
        _near(t.grad, *ref[name], 256 + more, name)
    assert weight.grad is None


@pytest.mark.parametrize("c", [64, 160, 320])
@pytest.mark.parametrize("lead, own", [((1, 1, 7), 1), ((2, 3, 33), 1), ((2, 3, 33), 3)], ids=["one sample", "shared", "own conditioning"])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_conditioned_transition(c, lead, own, dtype):
    mod = T._filled(M.ConditionedTransitionBlock(c, 64), 3)
    a, s = _randn(1, *lead, c, dtype=dtype).requires_grad_(), _randn(2, lead[0], own, lead[2], 64, dtype=dtype).requires_grad_()
    with A.compressed():
        out = mod(a, s, residual=True)
    dout = _randn(4, *out.shape, dtype=dtype, scale=0.1)
    out.backward(dout)
    w, m = T._weights(mod, dtype)
    ad, sd = a.detach().double().requires_grad_(), s.detach().double().requires_grad_()
    T._plain_transition(ad, sd, w, m, True).backward(dout.double())
    for got, want, name in ((a.grad, ad.grad, "da"), (s.grad, sd.grad, "ds"), *((q.grad, w[n].grad, n) for n, q in mod.named_parameters())):
        T._near(got, want, 2.5e-2, name)


@pytest.mark.parametrize("c", [64, 160])
@pytest.mark.parametrize("autocast", [False, True])
def test_recurrence_of_the_trunk(c, autocast):
    mod = trunk.ParcaeRecurrence(c).to(DEV)
    with torch.no_grad():
        mod.parcae_log_a.add_(_randn(6, c, scale=0.1))
    z, u = (_randn(i, 1, 21, 21, c, dtype=F32 if autocast else BF).requires_grad_() for i in (1, 2))
    with torch.autocast("cuda", dtype=BF, enabled=autocast), A.compressed():
        out = mod(z, u)
    dout = _randn(3, *out.shape, dtype=out.dtype, scale=0.1)
    out.backward(dout)
    w = {n: q.detach().double().requires_grad_() for n, q in mod.named_parameters()}
    zd, ud = z.detach().double().requires_grad_(), u.detach().double().requires_grad_()
    delta = torch.nn.functional.softplus(w["parcae_log_delta"])
    un = T._norm(ud) * w["layernorm_z.weight"] + w["layernorm_z.bias"]
    (torch.exp(-delta * torch.exp(w["parcae_log_a"])) * zd + un @ (delta[:, None] * w["parcae_b_cont"]).t()).backward(dout.double())
    for got, want, name in ((z.grad, zd.grad, "dz"), (u.grad, ud.grad, "du"), *((q.grad, w[n].grad, n) for n, q in mod.named_parameters())):
        T._near(got, want, 2.5e-2, name)
