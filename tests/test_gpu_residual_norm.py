"""What lies between two blocks of a residual stream, and its gradient, against 64-bit arithmetic.

Tolerances.  A result is rounded once to its type (half a step of the value) after float32 arithmetic.  With u = 2^-24: a sum over a row's channels adds at most
8 values in a lane, 5 times across lanes and 3 across warps; a gradient passes through four of them and less than 30 single roundings: 4 * 16 + 60 < 128
u of the magnitudes that `plain_residual` sums up.  A gate's exponential is off by 2^-21 and by u |a| for its argument's rounding, its reciprocal by 2^-22: below
(16 + 2 |a|) u, for a slope twice that.  |a| < 8 here: 128 u is room for both; 256 together.  Sums over samples add a rounding for each, sums over rows one for
each row.  What is normalised, and what the gradient is taken at, is r as the call itself stored it.
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
TYPES = {"bf16": (BF, BF), "f32": (F32, F32), "mixed": (F32, BF)}


def _randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, dtype)


def _near(got, ref, size, steps, what):
    assert got.shape == ref.shape, what
    assert torch.isfinite(got).all(), what
    far = (got.double() - ref).abs() - (P.HALF_STEP[got.dtype] * (ref.abs() + steps * P.U32 * size) + steps * P.U32 * size)
    assert (far <= 1e-37).all(), f"{what}: {far.max().item():.3e} beyond its room"


def _case(groups, samples, l, c, types="bf16", gate=True, scale=False, norm="adaptive", seed=0, offset=True):
    st, ct = TYPES[types]
    shape = (groups * samples, l, c)
    d = dict(x=_randn(seed, *shape) * 2 + (_randn(seed + 1, c) if offset else 0), u=_randn(seed + 2, *shape, dtype=ct), gate=None, scale=None, weight=None, bias=None,
             gate_shift=None)
    d["x"] = d["x"].to(st)
    if gate:
        d["gate"] = _randn(seed + 3, groups, l, c, dtype=ct)
    if scale:
        d["scale"] = 1 + 0.2 * _randn(seed + 4, c)
    if norm == "adaptive":
        d["gate_shift"] = _randn(seed + 5, groups, l, 2 * c, dtype=ct)
    if norm == "affine":
        d["weight"], d["bias"] = 1 + 0.2 * _randn(seed + 6, c), _randn(seed + 7, c)
    return d, _randn(seed + 8, *shape, dtype=st, scale=0.1), _randn(seed + 9, *shape, dtype=ct, scale=0.1)


def _check(d, dr, dy, samples, eps=1e-5, norm=True, compress=False):
    r, y, *more = F.residual_norm(**d, samples=samples, eps=eps, norm=norm, compress=compress)
    base = d["u"] if d["x"] is None else d["x"]
    want, size = R.residual(d["x"], d["u"], d["gate"], d["scale"], samples)
    assert r.dtype == base.dtype and r.shape == base.shape
    _near(r, want, size, 8, "r")
    at = r
    if compress:
        at = more[0]
        value, byte = R.kept(r)
        assert torch.equal(at.exponents, byte) and torch.equal(F.expand(at).double(), value) and at.dtype == r.dtype
        at_value = F.expand(at)
    else:
        at_value = r
    if norm:
        z, _, dz = R.statistics(r, eps)
        m, v = R.norm_factor(r.shape, d["weight"], d["gate_shift"], samples)
        if d["bias"] is not None:
            v = d["bias"].double()
        _near(y, m * z + v, dz * abs(m) + abs(v) * torch.ones_like(z), 256, "y")
    else:
        assert y is None
    if not norm:
        dy = None
    g = F.residual_norm_backward(dr, dy, at, d["u"], d["gate"], d["x"], d["scale"], d["weight"], d["gate_shift"], samples, eps)
    ref = R.residual_norm_gradient(dr, dy, at_value, d["u"], d["gate"], d["x"], d["scale"], d["weight"], d["gate_shift"], samples, eps)
    rows = r.numel() // r.shape[-1]
    for name, more in (("x", 0), ("u", 0), ("gate", samples), ("scale", rows), ("weight", rows), ("bias", rows), ("gate_shift", samples)):
        got = getattr(g, name)
        like = d.get(name)
        if name == "bias" and dy is not None and d["gate_shift"] is None:
            assert got.shape == (r.shape[-1],)
        elif like is None or (dy is None and name in ("weight", "bias", "gate_shift")):
            assert got is None or name == "x", name
            continue
        if name in ("x", "u", "gate", "gate_shift"):
            assert got.dtype == like.dtype and got.shape == like.shape, name
        else:
            assert got.dtype == F32
        _near(got, *ref[name], 256 + more, name)
    return r, y, g


@pytest.mark.parametrize("c", [1, 2, 7, 8, 31, 32, 33, 40, 64, 100, 128, 200, 255, 256, 264, 384, 505, 512, 520, 768, 776, 1000, 1023, 1024])
@pytest.mark.parametrize("types", list(TYPES))
def test_widths_and_types(c, types):
    for samples in (1, 3):
        _check(*_case(2, samples, 11, c, types, seed=c), samples)
    _check(*_case(2, 1, 11, c, types, norm="affine", gate=False, scale=True, seed=c), 1, compress=True)


@pytest.mark.parametrize("groups, samples, l", [(1, 1, 1), (1, 5, 1), (1, 2, 3), (3, 4, 5), (1, 48, 2), (1, 48, 37), (7, 1, 33), (1, 5, 301), (2, 7, 130), (1, 3, 5000), (5, 1, 4000), (1, 3001, 2)])
@pytest.mark.parametrize("c", [64, 128, 768])
def test_rows_and_samples(groups, samples, l, c):
    """Gate rows that outnumber the teams, and too few of them: both ways of dividing the samples."""
    _check(*_case(groups, samples, l, c, seed=l), samples)


@pytest.mark.parametrize("gate", [False, True])
@pytest.mark.parametrize("scale", [False, True])
@pytest.mark.parametrize("norm", [None, "plain", "affine", "adaptive"])
@pytest.mark.parametrize("samples", [1, 4])
@pytest.mark.parametrize("types", list(TYPES))
def test_every_part_with_every_other(gate, scale, norm, samples, types):
    for c in (96, 99):
        d, dr, dy = _case(3, samples, 17, c, types, gate, scale, norm, seed=5)
        for compress in (False, True):
            _check(d, dr, dy, samples, norm=norm is not None, compress=compress)


@pytest.mark.parametrize("norm", ["plain", "affine", "adaptive"])
def test_the_norm_alone(norm):
    d, _, dy = _case(2, 3, 29, 128, norm=norm, gate=False)
    d["u"] = None
    r, y, g = _check(d, None, dy, 3)
    assert r is d["x"]
    if norm != "adaptive":
        ref = F.layer_norm_backward(dy, d["x"], d["weight"])
        for a, b, room in zip((g.x, g.weight, g.bias), ref, (2.0 ** -7, 1e-4, 1e-4)):       # (two roundings of one value)
            assert (a is None) == (b is None)
            if a is not None:
                assert (a.double() - b.double()).abs().max() <= room * b.double().abs().max()


def test_the_gate_alone():
    d, _, _ = _case(2, 3, 29, 128, norm=None)
    d["x"] = None
    dr = _randn(3, 6, 29, 128, dtype=BF)
    _check(d, dr, None, 3, norm=False)


def test_one_of_the_gradients():
    """Nothing came back through one of the results."""
    d, dr, dy = _case(2, 3, 29, 256)
    _check(d, None, dy, 3)
    r = F.residual_norm(**d, samples=3)[0]
    g = F.residual_norm_backward(dr, None, r, d["u"], d["gate"], samples=3, gate_shift=d["gate_shift"])
    ref = R.residual_norm_gradient(dr, None, r, d["u"], d["gate"], None, None, None, None, 3, 1e-5)
    assert g.gate_shift is None and torch.equal(g.x, dr)
    _near(g.u, *ref["u"], 256, "u")
    _near(g.gate, *ref["gate"], 260, "gate")


@pytest.mark.parametrize("samples", [1, 4])
def test_kept_branch_and_stream(samples):
    """u and x in 8 bits: the gradient at the values that these stand for."""
    d, dr, dy = _case(2, samples, 21, 136, scale=True)
    r, _, kept = F.residual_norm(**d, samples=samples, compress=True)
    u8, x8 = F.compress(d["u"]), F.compress(d["x"])
    g = F.residual_norm_backward(dr, dy, kept, u8, d["gate"], x8, d["scale"], None, d["gate_shift"], samples)
    h = F.residual_norm_backward(dr, dy, F.expand(kept), F.expand(u8), d["gate"], F.expand(x8), d["scale"], None, d["gate_shift"], samples)
    for a, b in zip(g, h):
        assert (a is None and b is None) or torch.equal(a, b)


@pytest.mark.parametrize("c", [64, 100, 128, 136, 505])
def test_the_same_kept_rows_in_two_places(c):
    d, dr, dy = _case(2, 3, 21, c, scale=True)
    d["u"] = d["x"].clone()
    kept = F.residual_norm(**d, samples=3, compress=True)[2]
    at = F.expand(kept)
    for gates in (3, 1):
        gate, gs = (t if gates == 3 else t.repeat_interleave(3, 0) for t in (d["gate"], d["gate_shift"]))
        g = F.residual_norm_backward(dr, dy, kept, kept, gate, kept, d["scale"], None, gs, gates)
        h = F.residual_norm_backward(dr, dy, at, at, gate, at, d["scale"], None, gs, gates)
        for a, b in zip(g, h):
            assert (a is None and b is None) or torch.equal(a, b)


def test_wide_rows_of_every_tensor_in_float32():
    """The widest rows with everything that they can bring: what does not fit the shared memory is read as it lies."""
    for c in (1023, 1021):
        for samples in (1, 2):
            d, dr, dy = _case(2, samples, 5, c, "f32", scale=True, seed=c)
            _check(d, dr, dy, samples)
            _check(d, dr, dy, samples, compress=True)


@pytest.mark.parametrize("c", [1016, 1024])
def test_wide_rows_of_seven_float32_tensors(c):
    """dr, dy, r, u, x, gate and the norm's gates, a row's own: more than a ring of two rows holds, with x as a tensor or in 8 bits."""
    d, dr, dy = _case(2, 1, 700, c, "f32", scale=True, seed=c)
    _check(d, dr, dy, 1)
    _check(d, dr, dy, 1, compress=True)
    r, y = F.residual_norm(**d)
    about = dict(scale=d["scale"], gate_shift=d["gate_shift"])
    x8 = F.compress(d["x"])
    a = F.residual_norm_backward(dr, dy, r, d["u"], d["gate"], x8, **about)
    b = F.residual_norm_backward(dr, dy, r, d["u"], d["gate"], F.expand(x8), **about)
    assert all((s is None and t is None) or torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("samples", [1, 4])
@pytest.mark.parametrize("c", [128, 100, 768])
@pytest.mark.parametrize("types", list(TYPES))
def test_the_stream_is_that_of_elementary_operations(samples, c, types):
    """Bit for bit, gates of every size among them; so are the rows in 8 bits."""
    d, _, _ = _case(2, samples, 500, c, types, norm=None, scale=types == "f32")
    d["gate"] = (d["gate"].float() * torch.linspace(0.1, 40, c, device=DEV)).to(d["gate"].dtype)
    r, _, kept = F.residual_norm(**d, samples=samples, compress=True)
    gate = 1.0 / (1.0 + torch.exp(-d["gate"].float())).repeat_interleave(samples, 0)
    x = d["x"].float() if d["scale"] is None else d["x"].float() * d["scale"]
    want = (x + gate * d["u"].float()).to(r.dtype)
    assert torch.equal(r, want)
    again = F.compress(want)
    assert torch.equal(kept.values, again.values) and torch.equal(kept.exponents, again.exponents)


def test_nothing_to_do():
    for groups, l in ((0, 5), (3, 0)):
        d, dr, dy = _case(max(groups, 1), 1, max(l, 1), 64, norm="affine", scale=True)
        cut = lambda t: t[:groups, :l]
        d.update(x=cut(d["x"]), u=cut(d["u"]), gate=cut(d["gate"]))
        r, y, kept = F.residual_norm(**d, compress=True)
        assert r.shape == y.shape == kept.shape == (groups, l, 64) or l == 0
        g = F.residual_norm_backward(cut(dr), cut(dy), r, d["u"], d["gate"], d["x"], d["scale"], d["weight"])
        assert not g.weight.any() and not g.bias.any() and not g.scale.any() and g.x.numel() == 0
    x = torch.zeros(0, 4, 64, device=DEV)
    assert F.residual_norm(x, x, gate=torch.zeros(0, 4, 64, device=DEV), samples=3)[0].shape == (0, 4, 64)


def test_one_row_without_leading_dims():
    x, u = _randn(1, 64), _randn(2, 64)
    r, y, kept = F.residual_norm(x, u, compress=True)
    assert torch.equal(r, x + u) and kept.exponents.shape == (2,)
    assert F.residual_norm_backward(r, y, kept, u).x.shape == (64,)


def test_views_strides_and_odd_addresses():
    """Columns of wider tables, rows at a stride, a broadcast gradient, tensors that start between two 16-byte boundaries."""
    c, l = 128, 40
    table = _randn(1, l, 7 * c, dtype=BF)
    d, dr, dy = _case(1, 2, l, c)
    want = F.residual_norm(**{**d, "gate": table[:, c:2 * c].contiguous()[None], "gate_shift": table[:, 3 * c:5 * c].contiguous()[None]}, samples=2)
    about = dict(gate=table[None, :, c:2 * c], gate_shift=table[None, :, 3 * c:5 * c], samples=2)
    got = F.residual_norm(d["x"], d["u"], **about)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    g = F.residual_norm_backward(dr, dy, got[0], d["u"], **about)
    h = F.residual_norm_backward(dr, dy, want[0], d["u"], gate=about["gate"].contiguous(), gate_shift=about["gate_shift"].contiguous(), samples=2)
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(g, h))
    turned = d["x"].transpose(0, 1).contiguous().transpose(0, 1)
    assert all(torch.equal(a, b) for a, b in zip(F.residual_norm(turned, d["u"], **about), want))
    one = torch.full((), 0.25, device=DEV, dtype=BF).expand(2, l, c)
    assert torch.equal(F.residual_norm_backward(one, one, got[0], d["u"], **about).x, F.residual_norm_backward(one.contiguous(), one.contiguous(), got[0], d["u"], **about).x)
    odd = lambda t: torch.cat((t.flatten()[:1], t.flatten()))[1:].view(t.shape)
    d2 = {k: None if v is None else odd(v) for k, v in d.items()}
    assert d2["x"].data_ptr() % 16
    _check(d2, odd(dr), odd(dy), 2, compress=True)


def test_masked_rows_and_extreme_gates():
    """Gates of the type's lowest value and of both infinities are shut or open, exactly; rows of zeros and rows without spread stay finite."""
    d, dr, dy = _case(1, 2, 12, 256, norm="affine")
    low, inf = torch.finfo(BF).min, float("inf")
    d["gate"][0, 0], d["gate"][0, 1], d["gate"][0, 2], d["gate"][0, 3], d["gate"][0, 4] = low, -inf, inf, -low, -120.0
    d["x"][:, 5], d["u"][:, 5], d["x"][:, 6], d["u"][:, 6] = 0, 0, 3.0, 0
    r, y = F.residual_norm(**d, samples=2)
    assert torch.equal(r[:, :2], d["x"][:, :2]) and torch.equal(r[:, 2:4], (d["x"][:, 2:4].float() + d["u"][:, 2:4].float()).to(BF)) and torch.equal(r[:, 4], d["x"][:, 4])
    g = F.residual_norm_backward(dr, dy, r, d["u"], d["gate"], weight=d["weight"], samples=2)
    assert all(torch.isfinite(t).all() for t in (r, y, g.x, g.u, g.gate, g.weight, g.bias))
    assert not g.u[:, :2].any() and torch.equal(g.u[:, 2:4], g.x[:, 2:4]) and not g.gate[0, :4].any()
    ref = R.residual_norm_gradient(dr, dy, r, d["u"], d["gate"], None, None, d["weight"], None, 2, 1e-5)
    _near(g.x, *ref["x"], 256, "x")


def test_infinities_and_nan_stay_in_their_rows():
    d, dr, dy = _case(1, 3, 9, 128)
    ok = F.residual_norm(**d, samples=3, compress=True)
    gok = F.residual_norm_backward(dr, dy, ok[2], d["u"], d["gate"], gate_shift=d["gate_shift"], samples=3)
    x = d["x"].clone()
    x[1, 4, 77], x[2, 6, 3] = float("nan"), float("inf")
    r, y, kept = F.residual_norm(**{**d, "x": x}, samples=3, compress=True)
    bad = torch.zeros(3, 9, dtype=torch.bool, device=DEV)
    bad[1, 4] = bad[2, 6] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], ok[1][~bad]) and torch.equal(r[~bad], ok[0][~bad])
    back = F.expand(kept)
    assert torch.isnan(back[1, 4, 64:96]).all() and torch.isnan(back[2, 6, :32]).all() and torch.isfinite(back[2, 6, 32:]).all()
    g = F.residual_norm_backward(dr, dy, kept, d["u"], d["gate"], gate_shift=d["gate_shift"], samples=3)
    assert torch.isnan(g.x[bad]).all() and torch.equal(g.x[~bad], gok.x[~bad]) and torch.equal(g.u[~bad], gok.u[~bad])
    rows = bad.any(0)
    assert torch.isnan(g.gate[0, rows]).all() and torch.equal(g.gate[0, ~rows], gok.gate[0, ~rows])


def test_no_epsilon():
    d, dr, dy = _case(1, 1, 33, 100, "f32", norm="affine")
    _check(d, dr, dy, 1, eps=0.0)
    d, dr, dy = _case(1, 5, 3, 60, "f32", scale=True)                # (lanes and teams without a row)
    _check(d, dr, dy, 5, eps=0.0)


@pytest.mark.parametrize("c", [128, 99])
@pytest.mark.parametrize("samples", [1, 5])
def test_what_lies_behind_the_rows_stays(c, samples):
    """The entry points write the rows they are given, of buffers that go on."""
    l, rows, g = 7, 7 * samples, c + 31 & ~31
    d, dr, dy = _case(1, samples, l, c)
    more = lambda n, c, dtype=BF: torch.full((n + 40, c), 7, dtype=dtype, device=DEV)
    r, y, kept, e = more(rows, c), more(rows, c), more(rows, c, torch.int8), more(rows, g // 32, torch.uint8)
    dx, du, dgate, dgs = more(rows, c), more(rows, c), more(l, c), more(l, 2 * c)
    lib, stream, p = L.lib(), L.raw_stream(), lambda t: t.data_ptr()
    L.check(lib.kfb_residual_norm_fwd(p(d["x"]), p(d["u"]), p(d["gate"]), c, None, None, None, p(d["gate_shift"]), 2 * c, p(r), p(y), p(kept), p(e), rows, c, samples, l, 1e-5, 2,
                                      0, 0, stream))
    size = lib.kfb_residual_norm_bwd_workspace_bytes(rows, c, samples, 0, 1)
    ws = torch.full((size + 4096,), 3, dtype=torch.uint8, device=DEV)
    L.check(lib.kfb_residual_norm_bwd(p(dr), p(dy), p(kept), p(e), p(d["u"]), None, None, None, p(d["gate"]), c, None, None, p(d["gate_shift"]), 2 * c, p(dx), p(du), p(dgate), p(dgs),
                                      None, None, None, p(ws), size, rows, c, samples, l, 1e-5, 2, 0, 0, stream))
    about = dict(gate=d["gate"], gate_shift=d["gate_shift"], samples=samples)
    want = F.residual_norm(d["x"], d["u"], compress=True, **about)
    grads = F.residual_norm_backward(dr, dy, want[2], d["u"], **about)
    for t, ref, n in ((r, want[0], rows), (y, want[1], rows), (kept, want[2].values, rows), (e, want[2].exponents, rows), (dx, grads.x, rows), (du, grads.u, rows),
                      (dgate, grads.gate, l), (dgs, grads.gate_shift, l)):
        assert torch.equal(t[:n], ref.reshape(n, -1)) and (t[n:] == 7).all()
    assert (ws[size:] == 3).all()


def test_long_rows_of_samples_same_bits_every_time():
    d, dr, dy = _case(1, 48, 61, 768, norm="affine")
    runs = [F.residual_norm_backward(dr, dy, F.residual_norm(**d, samples=48)[0], d["u"], d["gate"], weight=d["weight"], samples=48) for _ in range(2)]
    assert all((a is None and b is None) or torch.equal(a, b) for a, b in zip(*runs))


def test_more_than_2_to_31_elements():
    """Element numbers that pass 32 bits: rows at the start, across the border and at the end as they are alone."""
    c, n = 1024, (1 << 21) + 5
    gen = torch.Generator(device=DEV).manual_seed(1)
    x = torch.empty(n, c, dtype=BF, device=DEV).normal_(generator=gen)
    w = 1 + 0.1 * _randn(2, c)
    r, y, kept = F.residual_norm(x, x, weight=w, compress=True)
    g = F.residual_norm_backward(x, y, kept, weight=w)
    for part in (slice(0, 4), slice((1 << 21) - 3, n)):
        rp, yp, kp = F.residual_norm(x[part], x[part], weight=w, compress=True)
        assert torch.equal(r[part], rp) and torch.equal(y[part], yp) and torch.equal(kept.values[part], kp.values) and torch.equal(kept.exponents[part], kp.exponents)
        assert torch.equal(g.x[part], F.residual_norm_backward(x[part], yp, kp, weight=w).x)


def test_gradient_is_the_difference_quotient():
    """d/dt of sum(dr r + dy y) along a direction of every input, 64-bit differences of the formula: the step's error, h^2 / 6 of a third derivative, is
    below 1e-6 here, float32 arithmetic below 1e-5 of the terms."""
    d, dr, dy = _case(2, 3, 7, 72, "f32", scale=True)
    r, y = F.residual_norm(**d, samples=3)
    g = F.residual_norm_backward(dr, dy, r, d["u"], d["gate"], d["x"], d["scale"], None, d["gate_shift"], 3)

    def value(e):
        rr = R.residual(e["x"], e["u"], e["gate"], e["scale"], 3)[0]
        m, v = R.norm_factor(rr.shape, None, e["gate_shift"], 3)
        return (dr.double() * rr).sum() + (dy.double() * (m * R.statistics(rr, 1e-5)[0] + v)).sum()

    h = 1e-4
    for i, name in enumerate(("x", "u", "gate", "scale", "gate_shift")):
        way = _randn(70 + i, *d[name].shape).double()
        moved = [value({**{k: None if t is None else t.double() for k, t in d.items()}, name: d[name].double() + s * h * way}) for s in (1, -1)]
        terms = getattr(g, name).double() * way
        assert abs(terms.sum() - (moved[0] - moved[1]) / (2 * h)) < 1e-4 * terms.abs().sum(), name


def test_dx_and_du_may_be_one_tensor():
    d, dr, dy = _case(1, 1, 6, 64, gate=False)
    g = F.residual_norm_backward(dr, dy, F.residual_norm(**d)[0], d["u"], gate_shift=d["gate_shift"])
    assert g.x is g.u
    g = F.residual_norm_backward(dr, dy, F.residual_norm(**d)[0], d["u"], gate_shift=d["gate_shift"], need_x=False)
    assert g.x is None and g.u is not None


def test_refusals():
    d, dr, dy = _case(2, 3, 8, 64)
    x, u, gate, gs = (d[k] for k in ("x", "u", "gate", "gate_shift"))
    w = torch.ones(64, device=DEV)
    for bad in (lambda: F.residual_norm(None), lambda: F.residual_norm(x, gate=gate), lambda: F.residual_norm(None, u, scale=w), lambda: F.residual_norm(x, u[:, :4]),
                lambda: F.residual_norm(x, u.float()), lambda: F.residual_norm(x.half(), u.half()), lambda: F.residual_norm(x, u, gate=gate),
                lambda: F.residual_norm(x, u, gate=gate, samples=2), lambda: F.residual_norm(x, u, gate=gate, samples=0), lambda: F.residual_norm(x, u, gate=gate, samples=-3),
                lambda: F.residual_norm(x, u, gate=gate.float(), samples=3), lambda: F.residual_norm(x, u, gate=gate[..., :32], samples=3),
                lambda: F.residual_norm(x, gate_shift=gate, samples=3), lambda: F.residual_norm(x, gate_shift=gs, weight=w, samples=3),
                lambda: F.residual_norm(x, u, weight=torch.ones(32, device=DEV)), lambda: F.residual_norm(x, u, weight=w, norm=False),
                lambda: F.residual_norm(x, u, out_dtype=F32), lambda: F.residual_norm(x, out_dtype=F32), lambda: F.residual_norm(torch.zeros((), device=DEV)),
                lambda: F.residual_norm_backward(None, None, x), lambda: F.residual_norm_backward(dr, dy[:3], x), lambda: F.residual_norm_backward(dr.float(), dy, x),
                lambda: F.residual_norm_backward(dr, dy, x, gate=gate, samples=3), lambda: F.residual_norm_backward(dr, dy, x, scale=w),
                lambda: F.residual_norm_backward(dr, dy, x, weight=w, gate_shift=gs, samples=3), lambda: F.residual_norm_backward(dr, dy, x, u, gate, samples=5),
                lambda: F.layer_norm_backward(dy.float(), F.compress(x), w)):
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(L.KfbError, match="1024"):
        F.residual_norm(_randn(1, 2, 1025))
    with pytest.raises(RuntimeError, match="CUDA"):
        F.residual_norm(x, u.cpu())
