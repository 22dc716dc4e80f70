"""LayerNorm's gradient from rows in 8 bits has the shapes that it has from a tensor: dweight the weight's, dbias (C,)."""
import pytest
import torch

from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.parametrize("shape", [None, (64,), (1, 64), (8, 8), (64, 1, 1)])
def test_shapes(shape):
    gen = torch.Generator(device=DEV).manual_seed(1)
    x, dy = (torch.randn(7, 5, 64, device=DEV, generator=gen, dtype=torch.bfloat16) for _ in range(2))
    weight = None if shape is None else torch.rand(shape, device=DEV, generator=gen) + 0.5
    kept = F.compress(x)
    got, want = F.layer_norm_backward(dy, kept, weight), F.layer_norm_backward(dy, F.expand(kept), weight)
    assert got[2].shape == want[2].shape == (64,) and got[2].dtype == want[2].dtype == torch.float32
    assert (got[1] is None) == (want[1] is None) == (shape is None) and (shape is None or got[1].shape == want[1].shape == shape)
    for a, b in zip(got[1:], want[1:]):
        assert a is None or (a - b).abs().max() <= 1e-4 * b.abs().max()
    assert all(t is None for t in F.layer_norm_backward(dy, kept, weight, need_weight=False, need_bias=False)[1:])
