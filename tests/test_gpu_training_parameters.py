"""Parameters of a LayerNorm in every shape that its forward pass takes."""
import pytest
import torch

from kfold_b200 import _lib as L
from kfold_b200 import autograd as A
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _status():
    yield
    assert L.device_status() == 0


def _randn(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


@pytest.mark.parametrize("weight, bias", [((64,), (64,)), ((1, 64), (64,)), ((64,), (1, 64)), ((1, 64), (1, 1, 64)), ((64, 1), (64,)), (None, (1, 64)),
                                          ((1, 64), None)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_a_gradient_has_its_parameters_shape(weight, bias, dtype):
    """The same numbers as of parameters (C,)."""
    x, dy = _randn(1, 5, 64, dtype=dtype).requires_grad_(), _randn(2, 5, 64, dtype=dtype)
    make = lambda seed, shape: None if shape is None else (1 + 0.1 * _randn(seed, *shape)).to(dtype).requires_grad_()
    flat = lambda t: None if t is None else t.detach().view(-1).clone().requires_grad_()
    w, b = make(3, weight), make(4, bias)
    x1, w1, b1 = x.detach().clone().requires_grad_(), flat(w), flat(b)
    y, y1 = A.layer_norm(x, w, b), A.layer_norm(x1, w1, b1)
    assert torch.equal(y, y1)
    y.backward(dy)
    y1.backward(dy)
    for t, t1 in ((x, x1), (w, w1), (b, b1)):
        assert t is None or (t.grad.shape == t.shape and t.grad.dtype == t.dtype and torch.equal(t.grad.view(-1), t1.grad.view(-1)))


def test_gradient_of_a_strided_parameter():
    """A parameter that is a column of a wider table."""
    x, dy, table = _randn(1, 5, 64), _randn(2, 5, 64), (1 + 0.1 * _randn(3, 64, 3)).requires_grad_()
    A.layer_norm(x, table[:, 1], table[:, 2]).backward(dy)
    w, b = (table.detach()[:, i].contiguous().requires_grad_() for i in (1, 2))
    A.layer_norm(x, w, b).backward(dy)
    assert torch.equal(table.grad[:, 1], w.grad) and torch.equal(table.grad[:, 2], b.grad) and not table.grad[:, 0].any()


def test_shapes_of_the_plain_call():
    x, dy = _randn(1, 5, 64), _randn(2, 5, 64)
    dx, dw, db = F.layer_norm_backward(dy, x, _randn(3, 1, 64))
    assert dw.shape == (1, 64) and db.shape == (64,)
    for bad in (_randn(3, 1, 32), _randn(3, 2, 64), _randn(3, 1)):
        with pytest.raises(ValueError, match="layer_norm_backward"):
            F.layer_norm_backward(dy, x, bad)
