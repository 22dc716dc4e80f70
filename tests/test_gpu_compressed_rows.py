"""Rows in 8 bits: every byte is determined, so values and exponents have to be equal."""
import pytest
import torch

import plain_residual as R
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _randn(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def _check(x):
    c = F.compress(x)
    value, byte = R.kept(x)
    assert c.shape == x.shape and c.dtype == x.dtype and c.values.dtype == torch.int8 and torch.equal(c.exponents, byte)
    for dtype in (None, BF, F32):
        back = F.expand(c, dtype)
        assert back.dtype == (dtype or x.dtype) and torch.equal(torch.nan_to_num(back.double(), nan=1e300), torch.nan_to_num(value, nan=1e300))
    assert (c.values > -128).all()
    return c


@pytest.mark.parametrize("c", [1, 5, 8, 24, 31, 32, 33, 40, 64, 100, 128, 250, 256, 768, 1025, 1500, 4096])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_widths(c, dtype):
    _check(_randn(c, 37, c, dtype=dtype) * torch.exp2(4 * _randn(c + 1, c)).to(dtype))


@pytest.mark.parametrize("shape", [(64,), (1, 64), (3, 5, 7, 96), (40001, 64), (0, 64), (5, 0, 64), (2, 300000)])
def test_shapes(shape):
    if shape[-1] > 65536:
        with pytest.raises(ValueError, match="65536|channels"):
            F.compress(torch.zeros(shape, device=DEV))
    else:
        _check(_randn(1, *shape, dtype=BF))


@pytest.mark.parametrize("dtype", [BF, F32])
def test_borders(dtype):
    """Largest magnitudes around the border at which they would round to 128, ties, zeros, the smallest and the largest numbers, signs."""
    step = 2.0 ** -7 if dtype == BF else 2.0 ** -23
    tops = [1.0, 1 + step, 2 - step, 1.9921875, 1.9921875 - step, 1.9921875 + (0 if dtype == BF else step), 0.0, -0.0, 127.5, 127.0, 126.5, 2.0 ** -119, 2.0 ** -119 * (1 - step),
            2.0 ** -118, 2.0 ** -120, 2.0 ** -126, 2.0 ** -133, 2.0 ** 127, 2.0 ** 127 * (2 - step), 2.0 ** 127 * 1.9921875, 2.0 ** 121]
    x = torch.zeros(len(tops), 64, dtype=torch.float64)
    for i, t in enumerate(tops):
        x[i, 3], x[i, 40], x[i, 41] = t, -t, t / 2
        x[i, 4:32] = t * torch.linspace(-1, 1, 28, dtype=torch.float64)
        x[i, 42:64] = t * (torch.arange(22) - 11 + 0.5) / 128
    _check(x.to(DEV, dtype))


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("bad", [float("nan"), float("inf"), -float("inf")])
def test_what_is_not_finite_takes_its_group(bad, dtype):
    x = _randn(3, 9, 100, dtype=dtype)
    x[2, 33], x[5, 99], x[7, 0] = bad, bad, bad
    c = _check(x)
    back = F.expand(c)
    assert torch.isnan(back[2, 32:64]).all() and torch.isnan(back[5, 96:]).all() and torch.isnan(back[7, :32]).all()
    assert int(torch.isnan(back).sum()) == 32 + 4 + 32


def test_halves_go_to_the_even_number():
    x = torch.zeros(1, 32)
    x[0, 0] = 100.0
    x[0, 1:9] = torch.tensor([0.5, 1.5, 2.5, -0.5, -1.5, -2.5, 99.5, -99.5])
    c = F.compress(x.to(DEV))
    assert int(c.exponents) == 133 and c.values[0, 1:9].tolist() == [0, 2, 2, 0, -2, -2, 100, -100]


def test_off_by_half_a_step_of_the_largest():
    x = _randn(5, 1000, 256)
    off = (F.expand(F.compress(x)) - x).abs().unflatten(-1, (-1, 32)).amax(-1)
    assert (off <= 2.0 ** -7 * 1.004 * x.abs().unflatten(-1, (-1, 32)).amax(-1)).all()


def test_views_and_odd_addresses():
    wide = _randn(1, 40, 300, dtype=BF)
    for x in (wide[:, 3:131], wide[:, 8:136], wide.t(), torch.full((), 0.3, device=DEV).expand(5, 64), _randn(2, 20 * 64 + 1)[1:].view(20, 64)):
        a, b = F.compress(x), F.compress(x.contiguous().clone())
        assert torch.equal(a.values, b.values) and torch.equal(a.exponents, b.exponents) and torch.equal(F.expand(a), F.expand(b))
    flat, e = F.compress(_randn(3, 20 * 64 + 3).view(1, -1)), F.compress(_randn(4, 20, 64))
    v = flat.values.flatten()[3:].view(20, 64)
    assert v.data_ptr() % 8 and torch.equal(F.expand(F.Compressed(v, e.exponents, F32)), F.expand(F.Compressed(v.clone(), e.exponents, F32)))


def test_more_than_2_to_31_elements():
    n, c = (1 << 24) + 3, 128
    x = torch.empty(n, c, dtype=BF, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1))
    k = F.compress(x)
    back = F.expand(k)
    for part in (slice(0, 3), slice((1 << 24) - 2, n)):
        ref = F.compress(x[part])
        assert torch.equal(k.values[part], ref.values) and torch.equal(k.exponents[part], ref.exponents) and torch.equal(back[part], F.expand(ref))


def test_compressed_inputs_of_the_gradients():
    """The gradients at the values that are kept."""
    x, dy, w = _randn(1, 300, 128, dtype=BF), _randn(2, 300, 128, dtype=BF), 1 + 0.1 * _randn(3, 128)
    k = F.compress(x)
    got, ref = F.layer_norm_backward(dy, k, w), F.residual_norm_backward(None, dy, F.expand(k), weight=w)
    assert torch.equal(got[0], ref.x) and torch.equal(got[1], ref.weight) and torch.equal(got[2], ref.bias)
    w_in, w_out = _randn(4, 512, 128, dtype=BF) / 11, _randn(5, 128, 256, dtype=BF) / 16
    for a, b in zip(F.gated_feed_forward_backward(dy, k, w_in, w_out), F.gated_feed_forward_backward(dy, F.expand(k), w_in, w_out)):
        assert torch.equal(a, b)
    for a, b in zip(F.fused_linear_backward(dy, k, w_in[:128], w, "silu"), F.fused_linear_backward(dy, F.expand(k), w_in[:128], w, "silu")):
        assert torch.equal(a, b)


def test_refusals():
    x = _randn(1, 4, 64)
    k = F.compress(x)
    for bad in (lambda: F.compress(x.half()), lambda: F.compress(x.double()), lambda: F.compress(torch.zeros((), device=DEV)), lambda: F.compress(x[:, :0]),
                lambda: F.expand(k, torch.float16), lambda: F.Compressed(k.values, k.exponents[:, :1], F32), lambda: F.Compressed(x, k.exponents, F32),
                lambda: F.Compressed(k.values, k.exponents.cpu(), F32), lambda: F.Compressed(k.values.t(), k.exponents, F32), lambda: F.Compressed(k.values, k.exponents, torch.int8)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        F.expand(F.Compressed(k.values.cpu(), k.exponents.cpu(), F32))
