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


def _beyond_outputs(call):
    """Bytes that a call takes beyond its outputs."""
    F.release_workspaces()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    out = call()
    torch.cuda.synchronize()
    outputs = sum(t.numel() * t.element_size() for t in (out if isinstance(out, tuple) else (out,)) if t is not None)
    return torch.cuda.max_memory_allocated() - before - outputs


@pytest.mark.parametrize("c, hidden", [(128, 512), (256, 1024)])
def test_kernels_that_keep_nothing_are_given_nothing(c, hidden):
    """The forward pass of many rows, their dx alone, and no gradient at all.  (Blocks of the allocator are multiples of 512 bytes.)"""
    x, w_in, w_out, dy = _case(20000, c, hidden)
    assert _beyond_outputs(lambda: F.gated_feed_forward(x, w_in, w_out)) <= 512
    assert _beyond_outputs(lambda: F.gated_feed_forward_backward(dy, x, w_in, w_out, True, False, False)) <= 512
    assert _beyond_outputs(lambda: F.gated_feed_forward_backward(dy, x, w_in, w_out, False, False, False)) == 0
    assert not F._workspaces


SIZES = [(9601, 128, 512, BF), (700, 128, 512, BF), (47000, 128, 8192, BF), (9601, 256, 1024, BF), (700, 256, 1024, BF), (23000, 256, 8192, BF), (33000, 256, 8192, BF),
         (1001, 384, 1536, BF), (30001, 64, 8192, BF), (300, 72, 64, BF), (9000, 72, 8192, BF), (300, 72, 64, torch.float32), (5000, 8, 8192, torch.float32)]


@pytest.mark.parametrize("rows, c, hidden, dtype", SIZES, ids=lambda v: str(v).replace("torch.", ""))
def test_a_call_of_some_gradients_keeps_to_its_own_workspace(rows, c, hidden, dtype):
    """Through the library: exactly the bytes that the call asks for, poisoned, and what lies behind them; a gradient has the same bits whoever else is asked
    for, and a byte less is refused."""
    x, w_in, w_out, dy = (t.to(dtype) for t in _case(rows, c, hidden))
    lib, code = L.lib(), 0 if dtype == BF else 2
    need = [lib.kfb_feed_forward_call_bytes(rows, c, hidden, code, w) for w in range(8)]
    most = [lib.kfb_feed_forward_workspace_bytes(rows, c, hidden, code, b) for b in (0, 1)]
    assert need[0] <= most[0] and max(need[1:]) == need[7] == most[1]
    want = F.gated_feed_forward_backward(dy, x, w_in, w_out)
    y = F.gated_feed_forward(x, w_in, w_out)
    ws = torch.empty(max(need) + 4096, dtype=torch.uint8, device=DEV)
    for wanted in range(8):
        ws.fill_(0xA5)
        at = L.ptr(ws) if need[wanted] else None
        outs = [torch.full_like(t, float("nan")) for t in ((y,) if wanted == 0 else want)]
        if wanted == 0:
            call = lambda size: lib.kfb_feed_forward_fwd(L.ptr(x), L.ptr(w_in), L.ptr(w_out), L.ptr(outs[0]), at, size, rows, c, hidden, code, L.stream_ptr())
        else:
            grads = [L.ptr(t) if wanted >> i & 1 else None for i, t in enumerate(outs)]
            call = lambda size: lib.kfb_feed_forward_bwd(L.ptr(dy), L.ptr(x), L.ptr(w_in), L.ptr(w_out), *grads, at, size, rows, c, hidden, code, code and 1,
                                                         L.stream_ptr())
        if need[wanted]:
            assert call(need[wanted] - 1) == 1
        L.check(call(need[wanted]))
        assert (ws[need[wanted]:] == 0xA5).all(), wanted
        for i, (got, ref) in enumerate(zip(outs, (y,) if wanted == 0 else want)):
            if wanted == 0 or wanted >> i & 1:
                assert torch.equal(got, ref), (wanted, i)
            else:
                assert torch.isnan(got).all(), (wanted, i)
