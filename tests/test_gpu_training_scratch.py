"""Scratch memory of training calls on a GPU."""
import threading

import pytest
import torch

from kfold_b200 import _lib as L
from kfold_b200 import autograd as A
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF = torch.bfloat16


@pytest.fixture(autouse=True)
def _clean():
    F.release_workspaces()
    yield
    F.release_workspaces()
    assert L.device_status() == 0


def _randn(seed, *shape, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, BF)


def _case(rows, c, hidden):
    return _randn(1, rows, c), _randn(2, 2 * hidden, c, scale=c ** -0.5), _randn(3, c, hidden, scale=hidden ** -0.5), _randn(4, rows, c)


def test_autograd_keeps_its_threads_scratch_from_step_to_step():
    x, w_in, w_out, dy = _case(2000, 128, 512)
    params = [t.requires_grad_() for t in (x, w_in, w_out)]
    kept = []
    for _ in range(3):
        torch.autograd.grad(A.gated_feed_forward(*params), params, dy)
        kept.append({key: ws.data_ptr() for key, ws in F._workspaces.items()})
    assert kept[0] == kept[1] == kept[2] and kept[0]


def test_threads_that_ended_hold_no_memory():
    x, w_in, w_out, dy = _case(2000, 128, 512)
    want = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    torch.cuda.synchronize()
    before, got = set(F._workspaces), []
    for _ in range(4):
        gate = threading.Barrier(3)

        def work():
            try:
                got.append(F.gated_feed_forward_backward(dy, x, w_in, w_out))
            finally:
                gate.wait(timeout=60)

        threads = [threading.Thread(target=work) for _ in range(3)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
    assert set(F._workspaces) == before
    torch.cuda.synchronize()
    assert len(got) == 12 and all(torch.equal(a, b) for g in got for a, b in zip(g, want))
