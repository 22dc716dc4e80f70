"""Gates of float32 logits keep their float32 digits, forward and backward, however far open or shut.

With u = 2^-24: an exponential within a unit (2 u), 1 + e, its reciprocal, their product and 1 - q of an open gate one rounding each (u): 6 u; the product with what is gated
one more: 8 u with room.  A slope q - q^2 of q below a half passes q's error on at most once, one rounding for the difference and two for products: 12 u.  Where a
number is compared with the same call's at a logit of zero (one half, a quarter: exact), that call's own products are rounded too: 16 u."""
import pytest
import torch

from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
U = 2.0 ** -24


def _randn(seed, *shape):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV)


def _logits(c, l):
    """From -40 to 40, small ones among them."""
    t = torch.linspace(-40, 40, l * c, device=DEV).view(l, c)
    t[: l // 3] *= 0.05
    return t


def _within(got, want, units, what):
    off = ((got.double() - want).abs() / (want.abs() * U).clamp(min=1e-300)).max()
    assert off <= units, f"{what}: {off.item():.1f} units"


def _slope(a):
    return torch.sigmoid(a) * torch.sigmoid(-a)


@pytest.mark.parametrize("c", [128, 1000, 99])
@pytest.mark.parametrize("samples", [1, 3, 40])
def test_output_gate(c, samples):
    l = 12
    a, u, dr = _logits(c, l)[None], _randn(1, samples, l, c), _randn(2, samples, l, c)
    at = a.double()
    r, _ = F.residual_norm(None, u, a, samples=samples, norm=False)
    _within(r, torch.sigmoid(at) * u.double(), 8, "r")
    g, zero = (F.residual_norm_backward(dr, None, r, u, t, samples=samples) for t in (a, torch.zeros_like(a)))
    _within(g.u, torch.sigmoid(at) * dr.double(), 8, "du")
    _within(g.gate, zero.gate.double() * 4 * _slope(at), 16, "dgate")


@pytest.mark.parametrize("c", [128, 1000, 99])
@pytest.mark.parametrize("samples", [1, 3, 40])
def test_gates_of_the_norm(c, samples):
    l = 12
    a, x, dy = _logits(c, l)[None], _randn(1, samples, l, c), _randn(2, samples, l, c)
    at, none = a.double(), torch.zeros_like(a)
    table, half = torch.cat((a, none), -1), torch.cat((none, none), -1)
    y, at_half = (F.residual_norm(x, gate_shift=t, samples=samples)[1] for t in (table, half))
    _within(y, at_half.double() * 2 * torch.sigmoid(at), 8, "y")
    g, zero = (F.residual_norm_backward(None, dy, x, gate_shift=t, samples=samples) for t in (table, half))
    _within(g.gate_shift[..., :c], zero.gate_shift[..., :c].double() * 4 * _slope(at), 16, "dg")
    assert torch.equal(g.gate_shift[..., c:], zero.gate_shift[..., c:])


def test_ends():
    inf = float("inf")
    a = torch.tensor([inf, -inf, 200.0, -200.0, 3e38, -3e38, 88.0, -86.0], device=DEV).view(1, 1, 8)
    u, dr = _randn(1, 1, 1, 8), _randn(2, 1, 1, 8)
    r, _ = F.residual_norm(None, u, a, norm=False)
    g = F.residual_norm_backward(dr, None, r, u, a)
    open_ = torch.tensor([1, 0, 1, 0, 1, 0, 1], device=DEV).view(1, 1, 7)
    assert torch.equal(r[..., :7], open_ * u[..., :7]) and torch.equal(g.u[..., :7], open_ * dr[..., :7]) and not g.gate[..., :6].any()
    _within(g.u[..., 7:], torch.sigmoid(a[..., 7:].double()) * dr[..., 7:].double(), 8, "du")
    assert torch.isfinite(g.gate).all()
