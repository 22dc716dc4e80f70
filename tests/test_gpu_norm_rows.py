"""LayerNorm of many short rows: the launch has blocks enough for a long walk."""
import pytest
import torch

from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def _us(calls, rounds=9, each=10):
    """Median time of one call of each, in turn (graph replays: the GPU alone)."""
    graphs = []
    for call in calls:
        side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        with torch.cuda.stream(side):
            call()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph, stream=side):
            for _ in range(each):
                call()
        graphs.append(graph)
    times = [[] for _ in graphs]
    for _ in range(rounds):
        for graph, t in zip(graphs, times):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            graph.replay()
            b.record()
            torch.cuda.synchronize()
            t.append(a.elapsed_time(b) * 1e3 / each)
    return [sorted(t)[rounds // 2] for t in times]


def test_time_grows_with_the_rows():
    """1 048 576 rows of 64 bf16 channels against 262 144: 3.7 to 4.3 times as long by 16 blocks an SM, 5.5 by four."""
    x, w = torch.randn(1 << 20, 64, device=DEV).to(torch.bfloat16), torch.ones(64, device=DEV)
    long, short = _us([lambda: F.layer_norm(x, w, w), lambda: F.layer_norm(x[:1 << 18], w, w)])
    assert long < 4.8 * short, (long, short)
    assert L.device_status() == 0


@pytest.mark.parametrize("c, dtype, out", [(64, torch.bfloat16, None), (128, torch.float32, torch.bfloat16), (384, torch.float32, None)])
def test_the_result_does_not_hang_on_the_number_of_rows(c, dtype, out):
    """Rows of a launch of few blocks an SM and of one of many: equal bits."""
    x, w, b = torch.randn(80011, c, device=DEV).to(dtype), torch.randn(c, device=DEV), torch.randn(c, device=DEV)
    many, few = F.layer_norm(x, w, b, out_dtype=out), torch.cat([F.layer_norm(t, w, b, out_dtype=out) for t in x.split(15000)])
    assert torch.equal(many, few)
