"""The gated feed-forward and its gradient against 64-bit arithmetic.

Tolerances.  bf16: h, da and db are rounded once as operands, by at most 2^-8 of themselves, and sigmoid(a), taken as tanh.approx(a / 2) / 2 + 1 / 2
with an error of at most 2^-11 of tanh, is off by less than 2^-11; `plain_training.feed_forward_pass` carries both through to every
element, and the element's own rounding comes on top.  a, b and dh are sums over the channels that the tensor core cuts off at every 16 terms, by
2^-23 of the terms' magnitudes: (8 + c / 16) 2^-23 of them, carried through likewise.  Over a whole output the
root mean square is far smaller: a rounding is off by 2^-8 / sqrt(3) of the value in the root mean square at the worst place of a binade, the
errors of a sum's terms are independent and add like the terms do: sqrt(2) * 2^-8 / sqrt(3) = 3.2e-3 with the output's own rounding, and below 1e-3
from the sigmoid: 4e-3 of the output's root mean square.
Float32: three bf16 parts hold 24 bits and the six products leave out 2^-24 each; the other sums over k are cut off in the
same way: (64 + k / 16) 2^-22 of the magnitudes for an element; 2e-5 of the root mean square.
"""
import pytest
import torch

import plain_training as P
from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
RMS = {BF: 4e-3, F32: 2e-5}


@pytest.fixture(autouse=True)
def _status():
    yield
    assert L.device_status() == 0


def _randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, dtype)


def _case(rows, c, hidden, dtype=BF, seed=0, weights=None):
    lead = rows if isinstance(rows, tuple) else (rows,)
    w = dict(dtype=weights or dtype)
    return (_randn(seed, *lead, c, dtype=dtype), _randn(seed + 1, 2 * hidden, c, scale=c ** -0.5, **w), _randn(seed + 2, c, hidden, scale=hidden ** -0.5, **w),
            _randn(seed + 3, *lead, c, dtype=dtype, scale=0.1))


def _near(got, ref, room, dtype, what):
    assert got.shape == ref.shape and torch.isfinite(got).all(), what
    d = (got.double() - ref).abs()
    rms = float(ref.square().mean().sqrt()) + 1e-30
    off = float(d.square().mean().sqrt())
    assert off <= RMS[dtype] * rms, f"{what}: {off / rms:.2e} of its root mean square"
    far = d - (P.HALF_STEP[got.dtype] * (ref.abs() + room) + room)
    assert (far <= 1e-30).all(), f"{what}: an element is {far.max().item():.2e} beyond its room"


def _plain(x, w_in, w_out, dy=None):
    k = max(x.numel() // x.shape[-1], 2 * w_out.shape[1], x.shape[-1])
    operand, gate = (2.0 ** -8 + 2.0 ** -16, 2.0 ** -11) if x.dtype == BF else ((64 + k / 16) * 2.0 ** -22, 2.0 ** -22)
    return P.feed_forward_pass(x, w_in.to(x.dtype), w_out.to(x.dtype), dy, operand, gate, (8 + x.shape[-1] / 16) * 2.0 ** -23)


def _check(x, w_in, w_out, dy):
    dt = x.dtype
    want = _plain(x, w_in, w_out, dy)
    got = (F.gated_feed_forward(x, w_in, w_out), *F.gated_feed_forward_backward(dy, x, w_in, w_out))
    for g, r, room, name, like in zip(got, want[:4], want[4:], ("y", "dx", "dw_in", "dw_out"), (x, x, w_in, w_out)):
        assert g.dtype == like.dtype and g.shape == like.shape
        _near(g, r, room, dt, name)
    return got[1:]


@pytest.mark.parametrize("rows", [1, 2, 7, 63, 64, 65, 127, 128, 129, 255, 257, 300, 1000, 4097])
@pytest.mark.parametrize("c, hidden", [(128, 512), (256, 1024), (384, 1536)])
def test_rows(rows, c, hidden):
    _check(*_case(rows, c, hidden, seed=rows))


@pytest.mark.parametrize("c, hidden", [(8, 8), (16, 24), (64, 256), (72, 136), (128, 64), (128, 128), (128, 192), (128, 520), (128, 1024), (136, 512),
                                       (256, 64), (256, 192), (256, 512), (256, 1000), (512, 512), (768, 1536), (1024, 136)])
def test_widths(c, hidden):
    _check(*_case(333, c, hidden, seed=c + hidden))


@pytest.mark.parametrize("rows, c, hidden", [(20000, 128, 512), (33333, 256, 256), (16385, 384, 64), (50001, 128, 128), (40000, 256, 1024), (37890, 128, 512)])
def test_many_rows(rows, c, hidden):
    _check(*_case(rows, c, hidden, seed=5))


@pytest.mark.parametrize("rows, c, hidden", [(7200, 128, 16384), (9600, 256, 16384), (1, 64, 65536), (3, 65536, 8), (200, 4096, 64)])
def test_largest_widths(rows, c, hidden):
    _check(*_case(rows, c, hidden))


@pytest.mark.parametrize("rows", [7103, 7104, 7105, 7167, 7169, 7231, 7295, 7297, 9471, 9472, 9473, 9535, 9537, 9599, 9601, 18943, 18945, 19072, 19201, 37889])
@pytest.mark.parametrize("c, hidden", [(128, 128), (256, 128)])
def test_rows_around_the_tiles_of_many(rows, c, hidden):
    """From 7 104 rows (128 channels) and 9 472 (256) on other kernels take them: tiles that end inside a tile, a warp, a pair; one, two and more a CTA."""
    _check(*_case(rows, c, hidden, seed=rows))


@pytest.mark.parametrize("c, hidden", [(128, 8), (128, 64), (128, 192), (128, 448), (128, 1024), (128, 2048), (256, 64), (256, 192), (256, 448), (256, 576), (256, 2048)])
def test_widths_with_many_rows(c, hidden):
    """One chunk of hidden channels, odd numbers of them, more than the device has multiprocessors for."""
    _check(*_case(19333, c, hidden, seed=hidden))


@pytest.mark.parametrize("c", [128, 256])
def test_only_some_gradients_of_many_rows(c):
    x, w_in, w_out, dy = _case(10001, c, 256)
    want = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True), (False, False, False)):
        got = F.gated_feed_forward_backward(dy, x, w_in, w_out, *need)
        for g, w, n in zip(got, want, need):
            assert (g is None) == (not n) and (g is None or torch.equal(g, w))


@pytest.mark.parametrize("c", [128, 256])
def test_rows_behind_the_last_of_many_are_left_alone(c):
    rows, hidden = 9601, 192
    x, w_in, w_out, dy = _case(rows, c, hidden)
    out, dx = (torch.full((rows + 300, c), 7.0, dtype=BF, device=DEV) for _ in range(2))
    dwi, dwo = torch.empty_like(w_in), torch.empty_like(w_out)
    lib = L.lib()
    need = [lib.kfb_feed_forward_workspace_bytes(rows, c, hidden, 0, b) for b in (0, 1)]
    ws = torch.full((max(need) + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    L.check(lib.kfb_feed_forward_fwd(L.ptr(x), L.ptr(w_in), L.ptr(w_out), L.ptr(out), L.ptr(ws), need[0], rows, c, hidden, 0, L.stream_ptr()))
    L.check(lib.kfb_feed_forward_bwd(L.ptr(dy), L.ptr(x), L.ptr(w_in), L.ptr(w_out), L.ptr(dx), L.ptr(dwi), L.ptr(dwo), L.ptr(ws), need[1], rows, c,
                                     hidden, 0, 0, L.stream_ptr()))
    assert (out[rows:] == 7).all() and (dx[rows:] == 7).all() and (ws[max(need):] == 0xA5).all()
    want = _plain(x, w_in, w_out, dy)
    _near(out[:rows], want[0], want[4], BF, "y")
    _near(dx[:rows], want[1], want[5], BF, "dx")


# The kernels of many rows: from 64 rows a multiprocessor on (9 472 on 148 of them), and as many more as hidden channels are fewer than 4 C.
@pytest.mark.parametrize("rows", [9471, 9472, 9473, 9535, 9537, 9599, 9601, 18943, 18945, 19072, 19201, 37889])
@pytest.mark.parametrize("c, hidden", [(128, 512), (256, 1024)])
def test_rows_around_the_tiles_of_the_kernels_of_many(rows, c, hidden):
    _check(*_case(rows, c, hidden, seed=rows))


@pytest.mark.parametrize("rows, c, hidden", [(75777, 128, 64), (37887, 128, 128), (37889, 128, 128), (25301, 128, 192), (10901, 128, 448), (9473, 128, 576), (9473, 128, 2048),
                                             (151601, 256, 64), (75777, 256, 128), (50601, 256, 192), (21701, 256, 448), (16901, 256, 576), (9473, 256, 2048)])
def test_widths_of_the_kernels_of_many_rows(rows, c, hidden):
    _check(*_case(rows, c, hidden, seed=hidden))


@pytest.mark.parametrize("c", [128, 256])
def test_only_some_gradients_by_the_kernels_of_many_rows(c):
    x, w_in, w_out, dy = _case(10001, c, 4 * c)
    want = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, False, True), (False, False, False)):
        got = F.gated_feed_forward_backward(dy, x, w_in, w_out, *need)
        for g, w, n in zip(got, want, need):
            assert (g is None) == (not n) and (g is None or torch.equal(g, w))


@pytest.mark.parametrize("rows, c, hidden", [(9601, 128, 512), (9601, 256, 1024), (3001, 256, 1024), (1001, 384, 1536)])
def test_nothing_is_written_behind_the_last_row_or_the_workspace(rows, c, hidden):
    x, w_in, w_out, dy = _case(rows, c, hidden)
    want = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    dx, dwi, dwo = (torch.full((n + 300, k), 7.0, dtype=BF, device=DEV) for n, k in ((rows, c), (2 * hidden, c), (c, hidden)))
    lib = L.lib()
    need = lib.kfb_feed_forward_workspace_bytes(rows, c, hidden, 0, 1)
    ws = torch.full((need + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    L.check(lib.kfb_feed_forward_bwd(L.ptr(dy), L.ptr(x), L.ptr(w_in), L.ptr(w_out), L.ptr(dx), L.ptr(dwi), L.ptr(dwo), L.ptr(ws), need, rows, c, hidden, 0, 0,
                                     L.stream_ptr()))
    assert (ws[need:] == 0xA5).all()
    for g, w in zip((dx, dwi, dwo), want):
        assert (g[w.shape[0]:] == 7).all() and torch.equal(g[:w.shape[0]], w)


@pytest.mark.parametrize("rows, c, hidden", [(5000, 128, 512), (10000, 128, 512), (4000, 256, 1024), (10000, 256, 1024), (1000, 384, 1536), (300, 72, 64)])
def test_what_the_scratch_memory_holds_does_not_matter(rows, c, hidden):
    x, w_in, w_out, dy = _case(rows, c, hidden)
    call = lambda: (F.gated_feed_forward(x, w_in, w_out), *F.gated_feed_forward_backward(dy, x, w_in, w_out))
    want = call()
    for fill in (0xFF, 0x7F):
        F._call_workspace(x.device, L.lib().kfb_feed_forward_workspace_bytes(rows, c, hidden, 0, 1)).fill_(fill)
        assert all(torch.equal(a, b) for a, b in zip(call(), want))


@pytest.mark.parametrize("rows, c, hidden, dtype", [(30001, 64, 8192, BF), (47000, 128, 8192, BF), (23000, 256, 8192, BF), (9000, 72, 8192, BF), (5000, 8, 8192, F32)])
def test_rows_in_several_pieces(rows, c, hidden, dtype):
    """More rows than a workspace holds at once, the last piece a short one."""
    _check(*_case(rows, c, hidden, dtype=dtype, seed=3))


@pytest.mark.parametrize("rows, c, hidden", [(1, 128, 512), (200, 128, 512), (129, 256, 1024), (65, 72, 136), (777, 384, 1536), (17000, 64, 64)])
def test_float32(rows, c, hidden):
    _check(*_case(rows, c, hidden, dtype=F32, seed=9))


def test_float32_parameters_with_bf16_rows():
    """Parameters that an optimizer holds in float32: rounded for the products, their gradients float32."""
    got = _check(*_case((3, 50), 128, 512, weights=F32))
    assert got[1].dtype == got[2].dtype == F32 and got[0].dtype == BF


def test_rows_without_gradient_and_rows_of_zero():
    """Padding: rows whose dy is zero get dx = 0 and add nothing; rows of x that are zero have h = 0."""
    x, w_in, w_out, dy = _case(500, 128, 512)
    dy[300:] = 0
    x[::7] = 0
    dx, dwi, dwo = _check(x, w_in, w_out, dy)
    assert not dx[300:].any()
    y = F.gated_feed_forward(x, w_in, w_out)
    assert not y[::7].any()


def test_large_activations():
    """Gates far in either saturation: silu(a) = a or 0, its derivative 1 or 0."""
    x, w_in, w_out, dy = _case(300, 128, 256)
    _check(x * 64, w_in, w_out, dy)


def test_only_some_gradients():
    x, w_in, w_out, dy = _case(1300, 128, 512)
    want = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    for need in ((True, False, False), (False, True, False), (False, False, True), (False, True, True), (True, True, False), (False, False, False)):
        got = F.gated_feed_forward_backward(dy, x, w_in, w_out, *need)
        for g, w, n in zip(got, want, need):
            assert (g is None) == (not n) and (g is None or torch.equal(g, w))


def test_no_rows():
    x, w_in, w_out, dy = _case(0, 128, 512)
    assert F.gated_feed_forward(x, w_in, w_out).shape == (0, 128)
    dx, dwi, dwo = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    assert dx.shape == (0, 128) and not dwi.any() and not dwo.any()


def test_views_and_broadcast_gradients():
    x, w_in, w_out, dy = _case(96, 128, 512)
    wide = _randn(7, 96, 300, dtype=BF)
    _check(wide[:, 3:131], w_in, w_out, dy)
    _check(x, w_in, w_out, dy.t().contiguous().t())
    _check(x, w_in.t().contiguous().t(), w_out.t().contiguous().t(), torch.full((), 0.25, device=DEV, dtype=BF).expand(96, 128))


@pytest.mark.parametrize("c, hidden", [(128, 512), (256, 512), (72, 64)])
def test_same_bits_every_time(c, hidden):
    x, w_in, w_out, dy = _case(20011, c, hidden)
    a = (F.gated_feed_forward(x, w_in, w_out), *F.gated_feed_forward_backward(dy, x, w_in, w_out))
    for _ in range(3):
        b = (F.gated_feed_forward(x, w_in, w_out), *F.gated_feed_forward_backward(dy, x, w_in, w_out))
        assert all(torch.equal(s, t) for s, t in zip(a, b))


@pytest.mark.parametrize("c", [128, 256, 96])
def test_rows_behind_the_last_are_left_alone(c):
    """Through the library: outputs with more room than rows, and a workspace with more than it asks for."""
    rows, hidden = 201, 4 * c
    x, w_in, w_out, dy = _case(rows, c, hidden)
    out, dx = (torch.full((rows + 300, c), 7.0, dtype=BF, device=DEV) for _ in range(2))
    dwi, dwo = torch.empty_like(w_in), torch.empty_like(w_out)
    lib = L.lib()
    need = [lib.kfb_feed_forward_workspace_bytes(rows, c, hidden, 0, b) for b in (0, 1)]
    ws = torch.full((max(need) + 4096,), 0xA5, dtype=torch.uint8, device=DEV)
    L.check(lib.kfb_feed_forward_fwd(L.ptr(x), L.ptr(w_in), L.ptr(w_out), L.ptr(out), L.ptr(ws), need[0], rows, c, hidden, 0, L.stream_ptr()))
    L.check(lib.kfb_feed_forward_bwd(L.ptr(dy), L.ptr(x), L.ptr(w_in), L.ptr(w_out), L.ptr(dx), L.ptr(dwi), L.ptr(dwo), L.ptr(ws), need[1], rows, c,
                                     hidden, 0, 0, L.stream_ptr()))
    assert (out[rows:] == 7).all() and (dx[rows:] == 7).all() and (ws[max(need):] == 0xA5).all()
    want = _plain(x, w_in, w_out, dy)
    _near(out[:rows], want[0], want[4], BF, "y")
    _near(dx[:rows], want[1], want[5], BF, "dx")


def test_workspace_contents_do_not_matter():
    x, w_in, w_out, dy = _case(5000, 128, 512)
    want = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    for fill in (0xFF, 0x7F):
        F._workspace(x.device, 1 << 20).fill_(fill)
        assert all(torch.equal(a, b) for a, b in zip(F.gated_feed_forward_backward(dy, x, w_in, w_out), want))


def test_gradient_is_the_difference_quotient():
    """Float32 mode against float64 central differences of the formula along random directions."""
    x, w_in, w_out, dy = _case(40, 64, 128, dtype=F32)
    grads = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    at, h = [t.double() for t in (x, w_in, w_out)], 1e-4
    for i, g in enumerate(grads):
        v = _randn(20 + i, *g.shape).double()
        moved = lambda t: [a + t * v if k == i else a for k, a in enumerate(at)]
        f = lambda t: (P.feed_forward(*moved(t)) * dy.double()).sum()
        assert abs((g.double() * v).sum() - (f(h) - f(-h)) / (2 * h)) <= 1e-4 * (g.double() * v).norm()


def test_streams_and_graph():
    x, w_in, w_out, dy = _case(3001, 128, 512)
    call = lambda: (F.gated_feed_forward(x, w_in, w_out), *F.gated_feed_forward_backward(dy, x, w_in, w_out))
    want = call()
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in range(2)]
    for s in streams * 3:
        with torch.cuda.stream(s):
            got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))
    from kfold_b200.graphs import GraphedCall
    graphed = GraphedCall(lambda x, dy: (F.gated_feed_forward(x, w_in, w_out), *F.gated_feed_forward_backward(dy, x, w_in, w_out)), x, dy)
    x2, dy2 = _randn(77, 3001, 128, dtype=BF), _randn(78, 3001, 128, dtype=BF)
    out = graphed(x2, dy2)
    again = (F.gated_feed_forward(x2, w_in, w_out), *F.gated_feed_forward_backward(dy2, x2, w_in, w_out))
    assert all(torch.equal(a, b) for a, b in zip(out, again))


def test_refusals():
    x, w_in, w_out, dy = _case(5, 128, 512)
    for bad in (lambda: F.gated_feed_forward(x, w_in[:-1], w_out), lambda: F.gated_feed_forward(x, w_in, w_out[:, :-8]),
                lambda: F.gated_feed_forward(x[:, :64], w_in, w_out), lambda: F.gated_feed_forward(x.half(), w_in, w_out),
                lambda: F.gated_feed_forward(x, w_in.float(), w_out), lambda: F.gated_feed_forward(x.float(), w_in, w_out),
                lambda: F.gated_feed_forward_backward(dy[:4], x, w_in, w_out), lambda: F.gated_feed_forward_backward(dy.float(), x, w_in, w_out),
                lambda: F.gated_feed_forward(*_case(5, 12, 16)[:3]), lambda: F.gated_feed_forward(*_case(5, 16, 12)[:3])):
        with pytest.raises(ValueError):
            bad()
