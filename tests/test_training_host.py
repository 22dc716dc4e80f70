"""What the training operators refuse, and the generator the dropout's mask comes from (no GPU)."""
import ctypes

import numpy as np
import pytest
import torch

import plain_training as P
from kfold_b200 import functional as F


@pytest.fixture(scope="module")
def library():
    from kfold_b200 import _lib, build
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("block, offset, seed, words", [
    (0, 0, 0, (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
    (2 ** 64 - 1, 2 ** 64 - 1, 2 ** 64 - 1, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
    (0x85A308D3243F6A88, 0x0370734413198A2E, 0x299F31D0A4093822, (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1)),
])
def test_generator_gives_the_published_words(block, offset, seed, words):
    """The known answers that the method's authors publish."""
    assert tuple(P.philox(np.array([block], dtype=np.uint64), offset, seed)[0].tolist()) == words


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    for call in (lambda: F.layer_norm_backward(x, x, None), lambda: F.dropout(x, 0.1, (1, 2))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_layernorm_bwd_refuses_before_any_cuda_call(library):
    vp, some = ctypes.c_void_p, 256
    need = library.kfb_layernorm_bwd_workspace_bytes(64)
    call = lambda dy=some, x=some, dx=some, dw=some, ws=some, size=need, rows=3, c=64, dt=0: library.kfb_layernorm_bwd(
        vp(dy), vp(x), None, vp(dx), vp(dw), None, vp(ws), size, rows, c, 1e-5, dt, 0, None)
    assert call(dy=None) == call(x=None) == call(dx=None) == 1
    assert call(rows=-1) == call(c=0) == call(dt=2) == call(dt=7) == 1
    assert call(ws=None) == call(size=need - 1) == call(ws=some + 8) == 1
    assert b"aligned" in library.kfb_last_error()
    assert call(c=1025, size=1 << 30) == 2


def test_dropout_refuses_before_any_cuda_call(library):
    vp, some = ctypes.c_void_p, 256
    call = lambda x=some, out=some, n=8, below=1 << 30, xt=0, ot=0: library.kfb_dropout(vp(x), None, vp(out), 1, 1, n, below, 1.5, None, 1, 2, xt, ot, None)
    assert call(x=None) == call(out=None) == call(n=-1) == 1
    assert call(below=-1) == call(below=(1 << 32) + 1) == 1
    assert call(xt=1, ot=0) == call(xt=2) == call(ot=5) == 1
    assert call(n=0) == 0


def test_feed_forward_refuses_before_any_cuda_call(library):
    vp, some, big = ctypes.c_void_p, 256, 1 << 40
    fwd = lambda x=some, wi=some, out=some, ws=some, size=big, rows=3, c=64, h=128, dt=0: library.kfb_feed_forward_fwd(
        vp(x), vp(wi), vp(some), vp(out), vp(ws), size, rows, c, h, dt, None)
    bwd = lambda dy=some, wi=some, dx=some, ws=some, size=big, rows=3, c=64, h=128, dt=0, gt=0: library.kfb_feed_forward_bwd(
        vp(dy), vp(some), vp(wi), vp(some), vp(dx), vp(some), vp(some), vp(ws), size, rows, c, h, dt, gt, None)
    for call in (fwd, bwd):
        assert call(wi=None) == call(ws=None) == call(size=16) == call(ws=some + 16) == 1
        assert call(rows=-1) == call(rows=1 << 31) == call(c=0) == call(c=60) == call(h=100) == call(h=-8) == call(dt=1) == call(dt=9) == 1
        assert call(wi=some + 8) == 1
        assert b"16-byte" in library.kfb_last_error()
    assert fwd(x=None) == fwd(out=None) == bwd(dy=None) == bwd(gt=2) == bwd(dt=2, gt=0) == 1
    assert fwd(rows=0) == 0


def test_feed_forward_workspace_stops_growing(library):
    need = library.kfb_feed_forward_workspace_bytes
    for c in (128, 256, 384):
        for dt in (0, 2):
            for backward in (0, 1):
                sizes = [need(r, c, 4 * c, dt, backward) for r in (1, 1000, 1 << 20, 1 << 22, (1 << 31) - 1)]
                assert sizes == sorted(sizes) and sizes[-1] == sizes[-2] == sizes[-3] and sizes[0] > 0
    assert need(0, 128, 512, 0, 0) == need(5, 0, 512, 0, 0) == 0


@pytest.mark.parametrize("c, hidden", [(8, 2 ** 31 - 8), (2 ** 31 - 8, 8), (2 ** 31 - 8, 2 ** 31 - 8), (65544, 8), (8, 65544), (12, 8), (8, -8)])
def test_feed_forward_refuses_widths_out_of_range(library, c, hidden):
    vp, some, big = ctypes.c_void_p, 256, 1 << 60
    for dt in (0, 2):
        for rows in (1, 1000, (1 << 31) - 1):
            assert library.kfb_feed_forward_workspace_bytes(rows, c, hidden, dt, 0) == library.kfb_feed_forward_workspace_bytes(rows, c, hidden, dt, 1) == 0
            assert library.kfb_feed_forward_fwd(vp(some), vp(some), vp(some), vp(some), vp(some), big, rows, c, hidden, dt, None) == 1
            assert library.kfb_feed_forward_bwd(vp(some), vp(some), vp(some), vp(some), vp(some), vp(some), vp(some), vp(some), big, rows, c, hidden, dt, 1,
                                                None) == 1
            assert b"multiples of 8" in library.kfb_last_error()
    assert library.kfb_feed_forward_bwd(None, None, None, None, None, vp(some), vp(some), None, 0, 0, c, hidden, 0, 0, None) == 1


def test_feed_forward_refuses_cpu_tensors():
    x, wi, wo = torch.zeros(4, 8), torch.zeros(32, 8), torch.zeros(8, 16)
    for call in (lambda: F.gated_feed_forward(x, wi, wo), lambda: F.gated_feed_forward_backward(x, x, wi, wo)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_modules_refuse_cpu_tensors_while_recording():
    from kfold_b200 import modules as M
    x = torch.zeros(3, 64)
    for call in (lambda: M.LayerNorm(64)(x), lambda: M.Transition(64, 2)(x), lambda: M.Dropout(0.5)(x)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(ValueError):
        M.Dropout(1.5)
    assert M.Dropout(0.5).eval()(x) is x and M.Dropout(0.0)(x) is x


def test_transition_keeps_its_parameters_names():
    from kfold_b200 import modules as M
    assert sorted(M.Transition(64, 2).state_dict()) == ["layernorm.bias", "layernorm.weight", "linear_out.weight", "swiglu.linear.weight"]
    assert not M.Dropout(0.1).state_dict()


@pytest.mark.parametrize("name", ["layer_norm", "layer_norm_backward", "gated_feed_forward", "gated_feed_forward_backward", "dropout"])
def test_another_current_device_than_the_tensors(monkeypatch, name):
    """The library is called with the tensors' device current, and the caller's is current again afterwards.  (CPU tensors that say they are on GPU 0.)"""
    current, seen = [1], []

    class OnDevice:
        def __init__(self, device):
            pass

        def __enter__(self):
            self.before, current[0] = current[0], 0

        def __exit__(self, *exc):
            current[0] = self.before

    class Library:
        def __getattr__(self, entry):
            return lambda *args: seen.append((entry, current[0])) or (4096 if entry.endswith("bytes") else 0)

    F._feed_forward_bytes.cache_clear()
    monkeypatch.setattr(F, "_one_gpu", lambda *a: 0)
    monkeypatch.setattr(F, "_workspace", lambda device, nbytes, *a: torch.empty(nbytes, dtype=torch.uint8))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for what, fake in (("current_device", lambda: current[0]), ("on_device", OnDevice), ("lib", Library), ("raw_stream", lambda at=None: 7)):
        monkeypatch.setattr(F.L, what, fake)
    x, w, w_in, w_out = torch.zeros(4, 8), torch.zeros(8), torch.zeros(32, 8), torch.zeros(8, 16)
    call = getattr(F, name)
    args = {"layer_norm": (x, w, w), "layer_norm_backward": (x, x, w), "gated_feed_forward": (x, w_in, w_out),
            "gated_feed_forward_backward": (x, x, w_in, w_out), "dropout": (x, 0.1, (1, 2))}[name]
    for device in (1, 0):
        current[0] = device
        seen.clear()
        call(*args)
        assert seen and all(d == 0 for _, d in seen) and current[0] == device
    F._feed_forward_bytes.cache_clear()
