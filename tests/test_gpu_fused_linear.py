"""A linear layer with its tail, and its gradient, against 64-bit arithmetic.

Tolerances.  A product's sum over K terms is cut off by the tensor core at every 16 of them, by 2^-23 of the terms' magnitudes: (8 + K / 16) 2^-23 of them
(float32 compute, whose operands are three bf16 parts each: (64 + K / 16) 2^-22).  f and f' follow z with slopes below 1.2 and 0.8 and are themselves off by
less than 32 u, u = 2^-24, of 1 + |z|.  bf16: dz is rounded once, by 2^-8 of itself, where an activation or a float32 dy makes it another value than what came in; dx, dW
carry that.  A result is rounded once to its type.
"""
import pytest
import torch

import plain_residual as R
import plain_training as P
from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
ACTIVATIONS = [None, "sigmoid", "silu", "gelu", "relu"]


@pytest.fixture(autouse=True)
def _status():
    yield
    assert L.device_status() == 0


def _randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, dtype)


def _case(rows, k, n, dtype=BF, bias=True, residual=False, weights=None, seed=0, out=None):
    lead = rows if isinstance(rows, tuple) else (rows,)
    return (_randn(seed, *lead, k, dtype=dtype), _randn(seed + 1, n, k, dtype=weights or dtype, scale=k ** -0.5), _randn(seed + 2, n) if bias else None,
            _randn(seed + 3, *lead, n, dtype=out or dtype) if residual else None, _randn(seed + 4, *lead, n, dtype=out or dtype, scale=0.1))


def _near(got, ref, room, what):
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    far = (got.double() - ref).abs() - (P.HALF_STEP[got.dtype] * (ref.abs() + room) + room)
    assert (far <= 1e-37).all(), f"{what}: {far.max().item():.2e} beyond its room"


def _check(x, w, bias, residual, dy, act):
    dt, k, n = x.dtype, x.shape[-1], w.shape[0]
    rows = x.numel() // k
    x2, dy2 = x.reshape(-1, k), dy.reshape(-1, n)
    wd = w.to(dt)
    sums = lambda terms: ((8 + terms / 16) * 2.0 ** -23) if dt == BF else (64 + terms / 16) * 2.0 ** -22
    (y, dx, dw, db), z = R.linear(x2, wd, bias, act, None if residual is None else residual.reshape(-1, n), dy2)
    dz_off = sums(k) * (x2.double().abs() @ wd.double().abs().t() + (0 if bias is None else bias.double().abs())) + 4 * P.U32 * z.abs()
    f_off = (0 if act is None else 32 * P.U32 * (1 + z.abs())) + 1.2 * dz_off
    got = F.fused_linear(x, w, bias, act, residual)
    assert got.dtype == (dt if residual is None else residual.dtype) and got.shape == dy.shape
    _near(got.reshape(-1, n), y, f_off + 2 * P.U32 * (0 if residual is None else residual.reshape(-1, n).double().abs()), "y")
    # gradients
    slope_off = 0 if act is None else 32 * P.U32 * (1 + z.abs()) + 0.8 * dz_off
    if act == "relu":                       # its slope jumps where z is nothing but rounding
        assert (z.abs() > 4 * dz_off).float().mean() > 0.98
        keep = (z.abs() > 4 * dz_off).double()
        slope_off = 1.0 - keep
    s = R.slope(z, act) if act else torch.ones_like(z)
    dz = dy2.double() * s
    once = P.HALF_STEP[BF] * dz.abs() if dt == BF and (act is not None or dy.dtype == F32) else 0
    off_db = dy2.double().abs() * slope_off
    off = off_db * (1 + P.HALF_STEP[BF]) + once
    off = off + torch.zeros_like(z)
    gx, gw, gb = F.fused_linear_backward(dy, x, w, bias, act)
    assert gx.dtype == dt and gx.shape == x.shape and gw.dtype == w.dtype and gw.shape == w.shape
    _near(gx.reshape(-1, k), dx, off @ wd.double().abs() + sums(n) * (dz.abs() @ wd.double().abs()), "dx")
    _near(gw, dw, off.t() @ x2.double().abs() + sums(rows) * (dz.abs().t() @ x2.double().abs()) + 16 * P.U32 * (dz.abs().t() @ x2.double().abs()), "dw")
    if bias is None:
        assert gb is None
    else:
        assert gb.dtype == F32
        _near(gb, db, (off_db + torch.zeros_like(z)).sum(0) + (16 + rows) * P.U32 * dz.abs().sum(0), "dbias")
    return got, gx, gw, gb


@pytest.mark.parametrize("rows", [1, 2, 7, 63, 64, 65, 127, 128, 129, 255, 257, 1000, 4097, 20001])
@pytest.mark.parametrize("k, n", [(128, 128), (384, 768), (256, 64)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_rows(rows, k, n, act):
    _check(*_case(rows, k, n, seed=rows), act)


@pytest.mark.parametrize("k, n", [(8, 8), (16, 24), (24, 16), (64, 8), (8, 64), (72, 136), (136, 72), (128, 520), (520, 128), (1024, 1000), (1000, 1024), (2048, 40), (40, 2048),
                                  (384, 1536), (1536, 384)])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_widths(k, n, dtype):
    _check(*_case(333, k, n, dtype, residual=True, seed=k), None)
    _check(*_case(67, k, n, dtype, seed=n), "gelu")


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype, weights, out", [(BF, BF, BF), (BF, F32, BF), (BF, BF, F32), (F32, F32, F32)], ids=["bf16", "f32 weights", "f32 residual", "f32"])
def test_every_tail(act, bias, residual, dtype, weights, out):
    if out == F32 and dtype == BF and not residual:
        residual = True
    for rows in (150, 3000):
        _check(*_case((2, rows // 2), 136, 200, dtype, bias, residual, weights, 3, out), act)


@pytest.mark.parametrize("act", ACTIVATIONS)
@pytest.mark.parametrize("dtype", [BF, F32])
def test_far_out_values_of_the_activations(act, dtype):
    """z from -60 to 60, and zero: slopes of shut and open gates."""
    x = torch.zeros(241, 8, device=DEV, dtype=dtype)
    x[:, 0] = torch.linspace(-60, 60, 241)
    w = torch.eye(8, device=DEV, dtype=dtype)
    dy = torch.ones(241, 8, device=DEV, dtype=dtype)
    got, dx, _, _ = F.fused_linear(x, w, None, act), *F.fused_linear_backward(dy, x, w, None, act)
    z = x[:, 0].double()
    f = R.FUNCTIONS[act](z)
    _near(got[:, 0], f, 64 * P.U32 * f.abs() * (1 + z.abs()) + 1e-30, "y")
    s = (R.slope(z, act) if act else torch.ones_like(z))
    tail = 64 * P.U32 * (s.abs() + z.abs() * torch.exp(-z.abs())) * (1 + z.abs()) + 1e-30
    if act == "gelu":                                    # two terms of opposite signs: each off by its own rounding
        tail = tail + 64 * P.U32 * (1 + z.square()) * (z.abs() * torch.exp(-0.5 * z * z) + 0.5 * torch.erfc(-z / 2 ** 0.5))
    keep = z != 0 if act == "relu" else z == z
    twice = (P.HALF_STEP[BF] * s.abs() + 0) if dtype == BF else 0
    _near(dx[keep, 0], s[keep], (tail + twice)[keep], "dx")


@pytest.mark.parametrize("rows, k, n, act", [(50001, 512, 256, "gelu"), (100000, 128, 128, None), (18432, 384, 1536, None), (30011, 768, 384, "sigmoid"), (400001, 64, 64, "silu"),
                                             (150000, 256, 1024, "relu")])
def test_many_rows(rows, k, n, act):
    """Sizes of the pair tensor, pieces of rows among them."""
    _check(*_case(rows, k, n, residual=act is None, seed=9), act)


@pytest.mark.parametrize("rows, k, n", [(30001, 264, 648), (20001, 776, 328), (5001, 1000, 1024), (4100, 2048, 2304), (10001, 512, 520), (9600, 512, 512), (19100, 512, 512)])
@pytest.mark.parametrize("act", [None, "silu"])
def test_weights_of_many_rows_and_odd_widths(rows, k, n, act):
    """Tiles of 256 columns that end inside, one piece of the rows and many, and both sides of where these tiles begin."""
    _check(*_case(rows, k, n, seed=k), act)


@pytest.mark.parametrize("rows, k, n", [(331, 256, 1024), (331, 2048, 64), (3000, 64, 64), (70, 24, 8)])
def test_the_float32_mode_is_float32(rows, k, n):
    """Root mean square of the errors: what is cut off at a step of the contraction is at most 2^-23 of an accumulator, 2^-24 on average, at k / 16 / 3 steps for each of
    three accumulators whose squares add up to the result's: 2^-24 k / 48 of it, and float32's own rounding and parts that are left out, 2^-23 together, twice over."""
    x, w, _, _, dy = _case(rows, k, n, F32, bias=False, seed=3)
    off = lambda got, ref: ((got.double() - ref).square().mean() / ref.square().mean()).sqrt().item()
    room = lambda terms: 2 * (2.0 ** -24 * terms / 48 + 2.0 ** -23)
    dx, dw, _ = F.fused_linear_backward(dy, x, w)
    assert off(F.fused_linear(x, w), x.double() @ w.double().t()) <= room(k)
    assert off(dx, dy.double() @ w.double()) <= room(n)
    assert off(dw, dy.double().t() @ x.double()) <= room(rows)


@pytest.mark.parametrize("rows, k, n", [(1999, 384, 1536), (4700, 512, 512), (4900, 512, 512), (2300, 768, 1000)])
def test_both_sides_of_where_pairs_begin(rows, k, n):
    """Half of the pairs of multiprocessors have a tile, or a few less."""
    _check(*_case(rows, k, n, residual=True, seed=n), "silu")


@pytest.mark.parametrize("rows", [30000, 900001])
def test_pieces_of_rows_in_float32(rows):
    """What a row keeps in the workspace is 6 (k + n) bytes, of which half a gigabyte is one piece."""
    k, n = (256, 384) if rows < 100000 else (40, 72)
    _check(*_case(rows, k, n, F32, residual=True, seed=4), "silu")


@pytest.mark.parametrize("rows, k, n, out", [(150001, 64, 2048, BF), (300001, 256, 1024, BF), (150001, 64, 2048, F32), (5000001, 8, 64, BF)])
def test_pieces_of_rows_in_bf16(rows, k, n, out):
    """2 n bytes a row; both ways of the products."""
    x, w, b, _, dy = _case(rows, k, n, seed=6, out=out)
    dx, dw, db = F.fused_linear_backward(dy, x, w, b, "silu")
    parts = [slice(i, min(i + 65536, rows)) for i in range(0, rows, 65536)]
    rw, rb, wsize, bsize = (torch.zeros(s, dtype=torch.float64, device=DEV) for s in ((n, k), (n,), (n, k), (n,)))
    for p in parts:
        (_, px, pw, pb), z = R.linear(x[p], w, b, "silu", None, dy[p])
        rw, rb = rw + pw, rb + pb
        dz = (dy[p].double() * R.slope(z, "silu")).abs()
        wsize, bsize = wsize + dz.t() @ x[p].double().abs(), bsize + dz.sum(0)
        room = 2.0 ** -7 * (dz @ w.double().abs())
        assert ((dx[p].double() - px).abs() <= P.HALF_STEP[BF] * px.abs() + room).all()
    assert ((dw.double() - rw).abs() <= P.HALF_STEP[BF] * rw.abs() + 2.0 ** -7 * wsize).all()
    assert ((db.double() - rb).abs() <= (2.0 ** -16 + rows * P.U32) * bsize).all()


def test_more_than_2_to_31_elements():
    """Element numbers that pass 32 bits: rows at the start, across the border and at the end as they are alone."""
    rows, k, n = (1 << 20) + 300, 64, 2048
    x, w = torch.empty(rows, k, dtype=BF, device=DEV).normal_(generator=torch.Generator(device=DEV).manual_seed(1)), _randn(2, n, k, dtype=BF, scale=0.1)
    y = F.fused_linear(x, w, None, "relu")
    dx = F.fused_linear_backward(y, x, w, None, None, True, False, False)[0]
    for p in (slice(0, 256), slice((1 << 20) - 256, (1 << 20) + 256), slice(rows - 256, rows)):
        assert torch.equal(y[p], F.fused_linear(x[p], w, None, "relu"))
        ref = y[p].double() @ w.double()
        assert ((dx[p].double() - ref).abs() <= 2.0 ** -8 * ref.abs() + (8 + n / 16) * 2.0 ** -23 * (y[p].double().abs() @ w.double().abs())).all()


@pytest.mark.parametrize("rows, k, n", [(300, 64, 72), (20000, 256, 264), (37000, 264, 520)])
@pytest.mark.parametrize("act", [None, "gelu"])
def test_what_lies_behind_the_rows_stays(rows, k, n, act):
    """The entry points write the rows they are given, of buffers that go on."""
    x, w, b, r, dy = _case(rows, k, n, residual=True)
    more = lambda c, rows=rows, dtype=BF: torch.full((rows + 200, c), 7.0, dtype=dtype, device=DEV)
    y, dx, dw, db = more(n), more(k), more(k, n), more(1, n, F32).view(-1)
    code, lib, stream = {None: 0, "gelu": 3}[act], L.lib(), L.raw_stream()
    size = max(lib.kfb_fused_linear_workspace_bytes(rows, k, n, code, 0, 0, wanted) for wanted in (0, 7))
    ws = torch.full((size + 4096,), 3, dtype=torch.uint8, device=DEV)
    L.check(lib.kfb_fused_linear_fwd(x.data_ptr(), w.data_ptr(), b.data_ptr(), r.data_ptr(), y.data_ptr(), ws.data_ptr(), size, rows, k, n, code, 0, 0, stream))
    L.check(lib.kfb_fused_linear_bwd(dy.data_ptr(), x.data_ptr(), w.data_ptr(), b.data_ptr(), dx.data_ptr(), dw.data_ptr(), db.data_ptr(), ws.data_ptr(), size, rows, k, n,
                                     code, 0, 0, 0, stream))
    assert torch.equal(y[:rows], F.fused_linear(x, w, b, act, r))
    for t, ref in zip((dx[:rows], dw[:n], db[:n]), F.fused_linear_backward(dy, x, w, b, act)):
        assert torch.equal(t, ref)
    assert (y[rows:] == 7).all() and (dx[rows:] == 7).all() and (dw[n:] == 7).all() and (db[n:] == 7).all() and (ws[size:] == 3).all()


@pytest.mark.parametrize("rows", [5, 30000])
def test_infinities_before_the_activation(rows):
    inf, nan = float("inf"), float("nan")
    x = torch.zeros(rows, 128, device=DEV, dtype=BF)
    x[0, 0], x[1, 0], x[2, 0], x[3, 0] = inf, -inf, nan, 1e30
    w = torch.zeros(128, 128, device=DEV, dtype=BF)
    w[0, 0] = 1
    zero = torch.zeros(rows, 128, device=DEV, dtype=BF)
    for act, want in (("relu", [inf, 0, nan, 1e30]), ("sigmoid", [1, 0, nan, 1]), ("gelu", [inf, 0, nan, 1e30]), ("silu", [inf, nan, nan, 1e30])):
        got = F.fused_linear(x, w, None, act)[:4, 0]
        assert torch.equal(torch.nan_to_num(got.float(), nan=-5.0), torch.nan_to_num(torch.tensor(want, device=DEV).to(BF).float(), nan=-5.0)), act
        assert torch.equal(F.fused_linear(x, w, None, act)[4:], F.fused_linear(zero, w, None, act)[4:])


def test_no_rows():
    x, w, b, r, dy = _case(0, 64, 128, residual=True)
    assert F.fused_linear(x, w, b, "gelu", r).shape == (0, 128)
    dx, dw, db = F.fused_linear_backward(dy, x, w, b, "gelu")
    assert dx.shape == (0, 64) and not dw.any() and not db.any() and dw.shape == w.shape and db.shape == b.shape


@pytest.mark.parametrize("act", [None, "silu"])
def test_only_what_is_asked_for(act):
    x, w, b, _, dy = _case(500, 128, 256)
    full = F.fused_linear_backward(dy, x, w, b, act)
    for want in range(8):
        need = [bool(want & 1 << i) for i in range(3)]
        for a, ref, asked in zip(F.fused_linear_backward(dy, x, w, b, act, *need), full, need):
            assert (a is None) if not asked else torch.equal(a, ref)


def test_views_and_odd_addresses():
    x, w, b, r, dy = _case(90, 64, 72, residual=True)
    ref = F.fused_linear(x, w, b, "silu", r), *F.fused_linear_backward(dy, x, w, b, "silu")
    odd = lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)
    turned = lambda t: t.t().contiguous().t()
    for f in (odd, turned):
        got = F.fused_linear(f(x), f(w), odd(b), "silu", f(r)), *F.fused_linear_backward(f(dy), f(x), f(w), odd(b), "silu")
        assert all(torch.equal(p, q) for p, q in zip(got, ref))
    one = torch.full((), 0.5, device=DEV, dtype=BF)
    assert torch.equal(F.fused_linear_backward(one.expand(90, 72), x, w)[0], F.fused_linear_backward(one.expand(90, 72).contiguous(), x, w)[0])


def test_rows_that_are_masked_do_not_reach_others():
    """NaN and infinities in some rows: the other rows' results are what they are without; a zero gradient for a finite row adds nothing to the weights'."""
    x, w, b, r, dy = _case(300, 128, 128, residual=True)
    clean = F.fused_linear(x, w, b, "gelu", r)
    bad = x.clone()
    bad[17], bad[200, 5] = float("nan"), float("inf")
    ok = torch.ones(300, dtype=torch.bool, device=DEV)
    ok[17] = ok[200] = False
    got = F.fused_linear(bad, w, b, "gelu", r)
    assert torch.equal(got[ok], clean[ok]) and torch.isnan(got[17]).all()
    dx = F.fused_linear_backward(dy, bad, w, b, "gelu")[0]
    assert torch.equal(dx[ok], F.fused_linear_backward(dy, x, w, b, "gelu")[0][ok])
    part = dy.clone()
    part[150:] = 0
    _, dw, db = F.fused_linear_backward(part, x, w, b, "gelu")
    (_, _, rw, rb), _ = R.linear(x[:150], w, b, "gelu", None, dy[:150])
    assert (dw.double() - rw).norm() < 4e-3 * rw.norm() and (db.double() - rb).norm() < 1e-4 * rb.norm()


def test_same_bits_every_time():
    x, w, b, _, dy = _case(30011, 384, 256)
    one, two = (F.fused_linear_backward(dy, x, w, b, "sigmoid") for _ in range(2))
    assert all(torch.equal(p, q) for p, q in zip(one, two))


def test_gradient_is_the_difference_quotient():
    x, w, b, _, dy = _case(37, 64, 40, F32)
    for act in ("sigmoid", "silu", "gelu"):
        grads = F.fused_linear_backward(dy, x, w, b, act)
        h = 1e-4
        for i, (t, g) in enumerate(zip((x, w, b), grads)):
            way = _randn(50 + i, *t.shape).double()
            args = [x.double(), w.double(), b.double()]
            value = []
            for sign in (1, -1):
                moved = list(args)
                moved[i] = moved[i] + sign * h * way
                value.append((R.FUNCTIONS[act](moved[0] @ moved[1].t() + moved[2]) * dy.double()).sum())
            terms = g.double() * way
            assert abs(terms.sum() - (value[0] - value[1]) / (2 * h)) < 1e-4 * terms.abs().sum()


def test_refusals():
    x, w, b, r, dy = _case(6, 64, 128, residual=True)
    for bad in (lambda: F.fused_linear(x, w[:, :32]), lambda: F.fused_linear(x, w[:12]), lambda: F.fused_linear(x[:, :12], w[:, :12]), lambda: F.fused_linear(x, w, b[:8]),
                lambda: F.fused_linear(x, w, b, "tanh"), lambda: F.fused_linear(x, w, b, None, r[:3]), lambda: F.fused_linear(x, w, b, None, r.half()),
                lambda: F.fused_linear(x.half(), w.half()), lambda: F.fused_linear(x, w.double()), lambda: F.fused_linear(x.float(), w), lambda: F.fused_linear(x, w[0]),
                lambda: F.fused_linear(x.float(), w.float(), b, None, r), lambda: F.fused_linear(torch.zeros((), device=DEV), w),
                lambda: F.fused_linear_backward(dy[:, :64], x, w), lambda: F.fused_linear_backward(dy.half(), x, w), lambda: F.fused_linear_backward(dy, x.float(), w.float())):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError, match="CUDA"):
        F.fused_linear(x, w, b.cpu())
    assert F.fused_linear_backward(dy, x, w, b, None, False, False, False) == (None, None, None)
