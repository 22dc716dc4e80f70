"""Ways through the training operators that need unusual sizes: several units a block, the forward pass in several pieces, rows that start between two pairs.

Tolerances as in test_gpu_training_feed_forward.py (its `_plain` and `_near`) and test_gpu_training_norm_dropout.py."""
import pytest
import torch

import plain_training as P
import test_gpu_training_feed_forward as T
from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _status():
    yield
    F.release_workspaces()
    assert L.device_status() == 0


@pytest.mark.parametrize("rows, hidden", [(9473, 9536), (9600, 16384)])
def test_weights_gradients_of_more_chunks_than_multiprocessors(rows, hidden):
    """128 channels: a block takes 64 hidden channels after other 64, whose weights and sums take their place."""
    assert L.lib().kfb_feed_forward_call_bytes(rows, 128, hidden, 0, 6) <= 3 * hidden * 128 * 4 + 512      # (one plane each and nothing kept: that kernel)
    T._check(*T._case(rows, 128, hidden, seed=rows))


@pytest.mark.parametrize("rows, border, c, hidden, dtype", [(9000, 8192, 64, 65536, BF), (66000, 65536, 384, 8192, BF), (14000, 13312, 72, 8192, BF), (9600, 9472, 8, 8192, F32)])
def test_forward_in_several_pieces(rows, border, c, hidden, dtype):
    """More rows than a workspace holds at once: rows of the first piece, around the border and of the last one.  Rows do not depend on one another."""
    x, w_in, w_out, _ = T._case(rows, c, hidden, dtype=dtype, seed=11)
    whole = L.lib().kfb_feed_forward_call_bytes(rows, c, hidden, 0 if dtype == BF else 2, 0)
    assert whole == L.lib().kfb_feed_forward_call_bytes(rows + 1000, c, hidden, 0 if dtype == BF else 2, 0)
    y = F.gated_feed_forward(x, w_in, w_out)
    assert torch.isfinite(y).all()
    for at in (slice(0, 200), slice(border - 150, border + 150), slice(rows - 200, rows)):
        want, room = T._plain(x[at], w_in, w_out)
        T._near(y[at], want, room, dtype, f"rows {at.start} to {at.stop}")


@pytest.mark.parametrize("c", [64, 128, 256, 384])
@pytest.mark.parametrize("dtype", [BF, F32])
def test_layer_norm_of_rows_that_start_between_pairs(c, dtype):
    """Every element to a rounding of its own and the float32 sums' errors (256 u of what they are made of, as for odd widths)."""
    flat = (torch.randn(20 * c + 1, generator=torch.Generator().manual_seed(c)) + 1).to(DEV, dtype)
    x, w, b = flat[1:].view(20, c), (1 + 0.2 * torch.randn(c, device=DEV)), torch.randn(c, device=DEV)
    ref, xd = P.layer_norm(x, w, b, 1e-5), x.double()
    r = 1.0 / torch.sqrt(xd.var(-1, keepdim=True, unbiased=False) + 1e-5)
    size = (r * (xd.abs() + xd.abs().mean(-1, keepdim=True)) + P.layer_norm(x, None, None, 1e-5).abs()) * w.double().abs() + b.double().abs()
    far = (F.layer_norm(x, w, b).double() - ref).abs() - (P.HALF_STEP[dtype] * ref.abs() + 256 * P.U32 * size)
    assert (far <= 0).all()
    # an offset and a scale that start between two pairs of floats
    wide = torch.cat((w[:1], w)), torch.cat((b[:1], b))
    assert torch.equal(F.layer_norm(x, wide[0][1:], wide[1][1:]), F.layer_norm(x, w, b))
