"""LayerNorm's gradient and dropout against 64-bit arithmetic.

Tolerances.  A result is rounded once to its type (half a step of the value) after float32 arithmetic.  A float32 sum of n terms is off by
at most n u (sum of the magnitudes), u = 2^-24, in whatever order; the width-wise sums here add at most 32 terms in a lane and 5 across
lanes, and a gradient passes through four of them (mean, variance, two of the products) and less than 30 single roundings or
approximated functions of 2 u: 4 * 37 + 60 < 256 u of the magnitudes that `plain_training` sums up.  Sums over rows add `rows`.
"""
import pytest
import torch

import plain_training as P
from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


def _randn(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def _near(got, ref, size, steps, what):
    assert torch.isfinite(got).all(), what
    room = P.HALF_STEP[got.dtype] * ref.abs() + steps * P.U32 * size
    far = (got.double() - ref).abs() - room
    assert (far <= 0).all(), f"{what}: {far.max().item():.3e} beyond its room of {room.flatten()[far.argmax()].item():.3e}"


def _check_norm(x, dy, w, eps=1e-5, need_bias=True):
    dx, dw, db = F.layer_norm_backward(dy, x, w, eps, need_bias=need_bias)
    (rx, rw, rb), (sx, sw, sb) = P.layer_norm_gradient(dy, x, w, eps)
    rows = rx.shape[0]
    assert dx.dtype == x.dtype and dx.shape == x.shape
    _near(dx.reshape(rx.shape), rx, sx, 256, "dx")
    assert (dw is None) == (w is None) and (db is None) == (not need_bias)
    if dw is not None:
        _near(dw, rw, sw, 256 + rows, "dweight")
    if db is not None:
        _near(db, rb, sb, 256 + rows, "dbias")


@pytest.mark.parametrize("c", [1, 2, 7, 32, 33, 64, 100, 128, 200, 255, 256, 260, 384, 505, 512, 516, 768, 1000, 1023, 1024])
@pytest.mark.parametrize("x_dtype, dy_dtype", [(BF, BF), (F32, F32), (F32, BF), (BF, F32)], ids=["bf16", "f32", "f32 from bf16", "bf16 from f32"])
def test_layer_norm_gradient_widths_and_types(c, x_dtype, dy_dtype):
    rows = 67
    x = _randn(c, rows, c, dtype=x_dtype) * 2 + _randn(c + 1, c, dtype=x_dtype)
    _check_norm(x, _randn(c + 2, rows, c, dtype=dy_dtype), 1 + 0.2 * _randn(c + 3, c))


@pytest.mark.parametrize("rows", [1, 2, 3, 15, 31, 33, 257, 4099, 40001])
@pytest.mark.parametrize("c, dtype", [(128, BF), (256, BF), (384, F32), (99, BF)])
def test_layer_norm_gradient_rows(rows, c, dtype):
    _check_norm(_randn(rows, rows, c, dtype=dtype), _randn(rows + 1, rows, c, dtype=dtype), 1 + 0.2 * _randn(7, c))


@pytest.mark.parametrize("with_weight, need_bias", [(False, False), (False, True), (True, False)])
def test_layer_norm_gradient_without_scale_or_offset(with_weight, need_bias):
    x, dy = _randn(1, 5, 33, 128, dtype=BF), _randn(2, 5, 33, 128, dtype=BF)
    _check_norm(x, dy, 1 + 0.1 * _randn(3, 128) if with_weight else None, need_bias=need_bias)


def test_layer_norm_gradient_of_no_rows():
    dx, dw, db = F.layer_norm_backward(_randn(1, 0, 64), _randn(1, 0, 64), _randn(2, 64))
    assert dx.shape == (0, 64) and not dw.any() and not db.any() and dw.shape == db.shape == (64,)


def test_layer_norm_gradient_of_views_and_broadcast_gradients():
    """Rows at a stride, a transposed gradient, one value for all of it, tensors that start between two pieces of 16 bytes."""
    wide, w = _randn(1, 40, 300, dtype=BF), 1 + 0.1 * _randn(2, 128)
    x, dy = wide[:, 3:131], _randn(3, 128, 40, dtype=BF).t()
    _check_norm(x, dy, w)
    _check_norm(x, torch.full((), 0.25, device=DEV, dtype=BF).expand(40, 128), w)
    flat, g = _randn(4, 40 * 128 + 3, dtype=BF), _randn(5, 40 * 128 + 1, dtype=F32)
    _check_norm(flat[3:].view(40, 128), g[1:].view(40, 128), _randn(6, 129)[1:])


def test_layer_norm_gradient_constant_rows_and_no_epsilon():
    """A row without spread has z = 0 and dx = (g - mean g) / sqrt(eps); with eps = 0 rows with spread stay finite beside what no row fills."""
    x = _randn(1, 5, 64)
    x[2] = 3.0
    _check_norm(x, _randn(2, 5, 64), None)
    _check_norm(_randn(3, 5, 64), _randn(4, 5, 64), 1 + 0.1 * _randn(5, 64), eps=0.0)


def test_layer_norm_gradient_same_bits_every_time():
    x, dy, w = _randn(1, 30011, 128, dtype=BF), _randn(2, 30011, 128, dtype=BF), 1 + 0.1 * _randn(3, 128)
    a, b = F.layer_norm_backward(dy, x, w), F.layer_norm_backward(dy, x, w)
    assert all(torch.equal(s, t) for s, t in zip(a, b))


def test_layer_norm_gradient_is_the_difference_quotient():
    """d/dt sum(dy y(x + t v)) against sum(dx v), float64 differences of the formula: step h^2 / 6 of the third derivative, here below 1e-6."""
    x, dy, v, w, b = _randn(1, 9, 96), _randn(2, 9, 96), _randn(3, 9, 96).double(), 1 + 0.1 * _randn(4, 96), _randn(5, 96)
    dx, dw, db = F.layer_norm_backward(dy, x, w)
    f = lambda x, w, b: (P.layer_norm(x, w, b, 1e-5) * dy.double()).sum()
    h = 1e-4
    x, w, b = x.double(), w.double(), b.double()
    slope = (f(x + h * v, w, b) - f(x - h * v, w, b)) / (2 * h)
    assert abs((dx.double() * v).sum() - slope) < 1e-4 * (dx.double() * v).abs().sum()
    u = v[0]
    assert abs((dw.double() * u).sum() - (f(x, w + h * u, b) - f(x, w - h * u, b)) / (2 * h)) < 1e-4 * (dw.double() * u).abs().sum()
    assert abs((db.double() * u).sum() - (f(x, w, b + h * u) - f(x, w, b - h * u)) / (2 * h)) < 1e-4 * (db.double() * u).abs().sum()


@pytest.mark.parametrize("c", [1, 3, 97, 505, 1023])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_layer_norm_of_odd_widths(c, dtype):
    """The forward pass of the widths that the kernels for pairs of channels do not take; the same bound as the gradient's z."""
    x, w, b = _randn(c, 37, c, dtype=dtype) + 1, 1 + 0.1 * _randn(2, c), _randn(3, c)
    y, ref = F.layer_norm(x, w, b), P.layer_norm(x, w, b, 1e-5)
    xd = x.double()
    r = 1.0 / torch.sqrt(xd.var(-1, keepdim=True, unbiased=False) + 1e-5)
    _near(y, ref, (r * (xd.abs() + xd.abs().mean(-1, keepdim=True)) + P.layer_norm(x, None, None, 1e-5).abs()) * w.double().abs() + b.double().abs(), 256, "y")


def test_layer_norm_of_a_tensor_that_starts_between_pairs():
    flat = _randn(1, 20 * 128 + 1, dtype=BF)
    x = flat[1:].view(20, 128)
    assert torch.equal(F.layer_norm(x, None, None), F.layer_norm(x.clone(), None, None)) or (
        F.layer_norm(x, None, None).double() - P.layer_norm(x, None, None, 1e-5)).abs().max() <= 2.0 ** -8 * 8


def test_norm_refusals():
    x = _randn(1, 4, 64)
    for bad in (lambda: F.layer_norm_backward(_randn(1, 4, 32), x, None), lambda: F.layer_norm_backward(x, x, _randn(1, 32)),
                lambda: F.layer_norm_backward(x.half(), x, None), lambda: F.layer_norm_backward(x, x.double(), None)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(L.KfbError, match="1024"):
        F.layer_norm_backward(_randn(1, 2, 1025), _randn(1, 2, 1025), None)


@pytest.mark.parametrize("which", ["weight", "bias"])
def test_norm_refuses_parameters_of_another_width_or_device(which):
    x, w = _randn(1, 4, 64), _randn(2, 64)
    norm = lambda t: F.layer_norm(x, **{"weight": w, "bias": w, which: t})
    for t in (_randn(3, 32), _randn(3, 65), _randn(3, 1)):
        with pytest.raises(ValueError, match="layer_norm"):
            norm(t)
    with pytest.raises(RuntimeError, match="CUDA"):
        norm(w.cpu())
    norm(w.view(1, 64))


# ------------------------------------------------------------------------------------------------ dropout
RNG = (0x0123456789ABCDEF, (1 << 63) + 12345)


def _check_dropout(x, p, rng, shared_dim, residual=None):
    got = F.dropout(x, p, rng if not isinstance(rng, list) else torch.tensor([L_ if L_ < 1 << 63 else L_ - (1 << 64) for L_ in rng], device=DEV),
                    shared_dim, residual)
    mask = P.kept(x.shape, shared_dim, p, tuple(rng)).to(DEV)
    zero = torch.zeros((), dtype=torch.float64, device=DEV)
    part = torch.where(mask, x.double() / (1 - p) if p < 1 else zero, zero)
    ref = part if residual is None else residual.double() + part
    assert got.dtype == (x.dtype if residual is None else residual.dtype) and got.shape == x.shape
    # the scale is rounded, the product and the sum are: 3 u of what they are made of
    _near(got, ref, part.abs() + (0 if residual is None else residual.double().abs()), 3, "out")
    if residual is None:
        dropped = ~mask.expand(x.shape)
        assert not got[dropped].any()
    return got


@pytest.mark.parametrize("shared_dim", [None, 0, 1, 2, -1])
@pytest.mark.parametrize("shape", [(3, 5, 64), (2, 7, 33), (4, 1, 20), (1, 9, 1), (5, 130, 8), (2, 3, 2048)])
@pytest.mark.parametrize("dtypes", [(BF, None), (F32, None), (BF, BF), (F32, F32), (BF, F32)], ids=lambda d: "+".join(str(t)[6:] for t in d if t))
def test_dropout_shapes_and_types(shape, shared_dim, dtypes):
    x = _randn(1, *shape, dtype=dtypes[0])
    _check_dropout(x, 0.3, RNG, shared_dim, None if dtypes[1] is None else _randn(2, *shape, dtype=dtypes[1]))


@pytest.mark.parametrize("n", [1, 2, 3, 4, 5, 1023, 4096, 4097, 1 << 20, (1 << 20) + 7])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_dropout_lengths(n, dtype):
    _check_dropout(_randn(n, n, dtype=dtype), 0.15, (n, 3), None, _randn(n + 1, n, dtype=dtype))


@pytest.mark.parametrize("p", [0.0, 2.0 ** -34, 0.5, 0.999, 1.0])
def test_dropout_probabilities(p):
    x = _randn(1, 64, 257)
    out = _check_dropout(x, p, (5, 6), None)
    if p < 2.0 ** -33:
        assert torch.equal(out, x)
    if p == 1.0:
        assert not out.any()


@pytest.mark.parametrize("rng", [(0, 0), (2 ** 64 - 1, 2 ** 64 - 1), (1, 2 ** 32), (2 ** 32, 1), RNG])
def test_dropout_seed_and_offset_as_numbers_and_in_device_memory(rng):
    x = _randn(1, 3, 50, 128, dtype=BF)
    for dim in (None, -3, -2):
        assert torch.equal(_check_dropout(x, 0.25, rng, dim), _check_dropout(x, 0.25, list(rng), dim))


def test_dropout_share_of_dropped_elements():
    """4 M elements at p = 0.25: the count's standard deviation is 866, and other offsets and seeds give other masks."""
    x = torch.ones(1 << 22, device=DEV)
    a, b, c = (F.dropout(x, 0.25, r) == 0 for r in ((1, 0), (1, 1), (2, 0)))
    for m in (a, b, c):
        assert abs(int(m.sum()) - (1 << 20)) < 6 * 887
    for m in (a & b, a & c, b & c):       # independent masks meet in 1 of 16
        assert abs(int(m.sum()) - (1 << 18)) < 6 * 496


def test_dropout_drops_infinities_and_nan():
    x = _randn(1, 4096)
    x[::3] = float("inf")
    x[1::3] = float("nan")
    out, mask = F.dropout(x, 0.4, (9, 9)), P.kept(x.shape, None, 0.4, (9, 9)).to(DEV)
    assert not out[~mask].any() and torch.equal(torch.isfinite(out), torch.isfinite(x) | ~mask)


def test_dropout_mask_does_not_hang_on_alignment_or_type():
    flat = _randn(1, 40 * 129 + 1)
    for x in (flat[1:].view(40, 129), flat[:-1].view(40, 129), flat[:40 * 128].view(40, 128), flat[1:40 * 128 + 1].view(40, 128)):
        _check_dropout(x, 0.2, RNG, None)
        _check_dropout(x.to(BF), 0.2, RNG, 0, x)


def test_dropout_in_place_through_the_library():
    """out may be x or the residual."""
    lib = L.lib()
    x, r = _randn(1, 9, 31, 64), _randn(2, 9, 31, 64)
    want = F.dropout(x, 0.25, (1, 2), shared_dim=1, residual=r)
    for out in (x.clone(), r.clone()):
        a, b = (out, r) if torch.equal(out, x) else (x, out)
        L.check(lib.kfb_dropout(L.ptr(a), L.ptr(b), L.ptr(out), 9, 31, 64, 1 << 30, 4.0 / 3.0, None, 1, 2, 1, 1, L.stream_ptr()))
        assert torch.equal(out, want)


def test_dropout_in_a_graph_draws_what_the_state_holds_at_replay():
    x, state = _randn(1, 33, 128, dtype=BF), torch.tensor([7, 0], device=DEV)
    with torch.cuda.stream(torch.cuda.Stream()):
        F.dropout(x, 0.5, state)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = F.dropout(x, 0.5, state)
    for offset in (0, 1, 1 << 40):
        state[1] = offset
        graph.replay()
        assert torch.equal(out, F.dropout(x, 0.5, (7, offset)))


def test_dropout_refusals():
    x = _randn(1, 4, 64)
    for bad in (lambda: F.dropout(x, -0.1, (1, 2)), lambda: F.dropout(x, 1.5, (1, 2)), lambda: F.dropout(x, float("nan"), (1, 2)),
                lambda: F.dropout(x, 0.1, (1 << 64, 2)), lambda: F.dropout(x, 0.1, (-1, 2)), lambda: F.dropout(x, 0.1, (1, 2), shared_dim=2),
                lambda: F.dropout(x, 0.1, (1, 2), residual=_randn(1, 64)), lambda: F.dropout(x, 0.1, (1, 2), residual=x.to(BF)),
                lambda: F.dropout(x, 0.1, torch.zeros(2, dtype=torch.int32, device=DEV)), lambda: F.dropout(x, 0.1, torch.zeros(2, dtype=torch.int64)),
                lambda: F.dropout(x.half(), 0.1, (1, 2))):
        with pytest.raises(ValueError):
            bad()


def test_empty_dropout():
    assert F.dropout(_randn(1, 0, 5), 0.1, (1, 2)).shape == (0, 5) and F.dropout(_randn(1, 3, 0, 5), 0.1, (1, 2), shared_dim=1).shape == (3, 0, 5)


def test_calls_on_another_stream_and_their_workspaces():
    x, dy, w = _randn(1, 5000, 256, dtype=BF), _randn(2, 5000, 256, dtype=BF), 1 + 0.1 * _randn(3, 256)
    want = F.layer_norm_backward(dy, x, w)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    got = []
    for s in streams * 4:
        with torch.cuda.stream(s):
            got.append(F.layer_norm_backward(dy, x, w))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
