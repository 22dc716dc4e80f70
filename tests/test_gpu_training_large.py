"""Training operators on tensors whose element numbers pass 32 bits, checked where they are largest (tens of gigabytes, a few milliseconds)."""
import numpy as np
import pytest
import torch

import plain_training as P
from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _room():
    free, _ = torch.cuda.mem_get_info()
    if free < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    yield
    torch.cuda.empty_cache()
    assert L.device_status() == 0


def _randn(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, BF)


def test_dropout_of_more_than_two_to_the_34_elements():
    """There the generator's block number takes its upper half.  In place, through the library."""
    n, p, rng = (1 << 34) + 24, 0.25, (77, 5)
    x = torch.ones(n, dtype=BF, device=DEV)
    L.check(L.lib().kfb_dropout(L.ptr(x), None, L.ptr(x), 1, 1, n, 1 << 30, 4.0 / 3.0, None, rng[0], rng[1], 0, 0, L.stream_ptr()))
    for first in (0, (1 << 31) - 8, (1 << 32) - 8, (1 << 33) - 8, (1 << 34) - 16, n - 24):
        words = P.philox(np.arange(first // 4, first // 4 + 6, dtype=np.uint64), rng[1], rng[0]).reshape(-1)
        assert torch.equal((x[first:first + 24] != 0).cpu(), torch.from_numpy(words >= np.uint64(1 << 30))), first


def test_shared_dropout_of_more_than_two_to_the_31_elements():
    x = torch.ones(1, (1 << 31) // 4096 + 3, 4096, dtype=BF, device=DEV)
    out = F.dropout(x, 0.5, (1, 2), shared_dim=1)
    mask = P.kept(x.shape, 1, 0.5, (1, 2)).to(DEV)
    for row in (0, 1, x.shape[1] // 2, x.shape[1] - 1):
        assert torch.equal(out[0, row] != 0, mask[0, 0])


def test_layer_norm_gradient_of_more_than_two_to_the_31_elements():
    rows, c, last = (1 << 31) // 128 + 77, 128, 300
    x, dy = torch.zeros(rows, c, dtype=BF, device=DEV), torch.zeros(rows, c, dtype=BF, device=DEV)
    x[-last:], dy[-last:] = _randn(1, last, c), _randn(2, last, c)
    w = 1 + 0.1 * torch.randn(c, generator=torch.Generator().manual_seed(3)).to(DEV)
    dx, dw, db = F.layer_norm_backward(dy, x, w)
    (rx, rw, rb), (sx, sw, sb) = P.layer_norm_gradient(dy[-last:], x[-last:], w, 1e-5)
    assert ((dx[-last:].double() - rx).abs() <= 2.0 ** -8 * rx.abs() + 256 * P.U32 * sx).all()
    assert ((dw - rw).abs() <= (256 + last) * P.U32 * sw).all() and ((db - rb).abs() <= (256 + last) * P.U32 * sb).all()
    assert not dx[:-last].any()


@pytest.mark.parametrize("c, hidden", [(128, 128), (256, 256)])
def test_feed_forward_of_more_than_two_to_the_31_elements(c, hidden):
    rows, last = (1 << 31) // c + 77, 300
    x, dy = torch.zeros(rows, c, dtype=BF, device=DEV), torch.zeros(rows, c, dtype=BF, device=DEV)
    x[-last:], dy[-last:] = _randn(1, last, c), _randn(2, last, c, scale=0.1)
    w_in, w_out = _randn(3, 2 * hidden, c, scale=c ** -0.5), _randn(4, c, hidden, scale=hidden ** -0.5)
    y = F.gated_feed_forward(x, w_in, w_out)
    ref = P.feed_forward_pass(x[-last:], w_in, w_out, dy[-last:])[:4]
    near = lambda got, want: float((got.double() - want).square().mean().sqrt() / want.square().mean().sqrt()) < 4e-3     # (see the feed-forward's tests)
    assert near(y[-last:], ref[0]) and not y[:-last].any()
    del y
    dx, dwi, dwo = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    assert near(dx[-last:], ref[1]) and near(dwi, ref[2]) and near(dwo, ref[3]) and not dx[:-last].any()
