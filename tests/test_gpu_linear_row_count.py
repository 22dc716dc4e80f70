"""A linear layer of nearly 2^31 rows: the rows of a launch are counted in 32 bits, so the call takes them in pieces.

x is zeros but for a few rows at its ends and around the border between the pieces; 34 GB, and as much for a result."""
import pytest
import torch

from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


def test_nearly_all_rows():
    torch.cuda.empty_cache()
    if torch.cuda.mem_get_info()[0] < 80 << 30:
        pytest.skip("80 GB of device memory")
    rows, gen = (1 << 31) - 1, torch.Generator(device=DEV).manual_seed(1)
    random = lambda *shape: torch.randn(shape, generator=gen, device=DEV)
    w, bias, at = random(8, 8).to(BF), random(8), [slice(0, 200), slice((1 << 30) - 150, (1 << 30) + 150), slice(rows - 333, rows)]
    x = torch.zeros(rows, 8, dtype=BF, device=DEV)
    for s in at:
        x[s] = random(s.stop - s.start, 8).to(BF)
    y = F.fused_linear(x, w, bias, "relu")
    for s in at:
        assert torch.equal(y[s], F.fused_linear(x[s].clone(), w, bias, "relu"))
    assert torch.equal(y[1 << 29], torch.relu(bias).to(BF)) and torch.equal(y[3 << 29], torch.relu(bias).to(BF))
    del y
    # (the gradient that comes back is x itself)
    dx, dw, db = F.fused_linear_backward(x, x, w, bias)
    few = torch.cat([x[s] for s in at])
    for s in at:
        assert torch.equal(dx[s], F.fused_linear_backward(x[s].clone(), x[s].clone(), w, bias)[0])
    assert not dx[1 << 29].any() and not dx[3 << 29].any()
    few = few.double()
    # (833 float32 additions, and the rounding of dw to bf16)
    size = few.abs().t() @ few.abs()
    assert ((dw.double() - few.t() @ few).abs() <= 833 * 2.0 ** -24 * size + 2.0 ** -8 * (few.t() @ few).abs()).all()
    assert ((db.double() - few.sum(0)).abs() <= 833 * 2.0 ** -24 * few.abs().sum(0)).all()
    del x, dx, few
    torch.cuda.empty_cache()
    assert L.device_status() == 0
