"""What the operators of a residual stream, of a linear layer with its tail and of rows in 8 bits refuse, before any CUDA call (no GPU)."""
import ctypes

import pytest
import torch

from kfold_b200 import functional as F

VP, SOME, BIG = ctypes.c_void_p, 256, 1 << 60


@pytest.fixture(scope="module")
def library():
    from kfold_b200 import _lib, build
    build.build()
    return _lib.lib()


def test_residual_norm_refuses(library):
    def call(x=SOME, u=SOME, gate=SOME, gate_ld=64, scale=None, w=None, b=None, gs=None, gs_ld=0, r=SOME, y=SOME, kept=None, ke=None, rows=12, c=64, samples=2, l=3,
             norm=1, st=0, ct=0):
        return library.kfb_residual_norm_fwd(VP(x), VP(u), VP(gate), gate_ld, VP(scale), VP(w), VP(b), VP(gs), gs_ld, VP(r), VP(y), VP(kept), VP(ke), rows, c, samples, l, 1e-5,
                                             norm, st, ct, None)
    for bad in (dict(x=None, u=None, gate=None), dict(u=None), dict(gate_ld=63), dict(r=None), dict(y=None), dict(kept=SOME), dict(ke=SOME), dict(rows=-1), dict(rows=1 << 31),
                dict(rows=13), dict(c=0), dict(c=-4), dict(samples=0), dict(l=0), dict(norm=3), dict(norm=-1), dict(norm=2), dict(norm=0, w=SOME), dict(norm=0, b=SOME),
                dict(gs=SOME, gs_ld=128), dict(norm=2, gs=SOME, gs_ld=127), dict(norm=2, gs=SOME, gs_ld=128, w=SOME), dict(st=2), dict(ct=1), dict(st=1, ct=2), dict(st=0, ct=1)):
        assert call(**bad) == 1, bad
        assert b"residual_norm" in library.kfb_last_error()
    assert call(c=1025, gate_ld=1025) == 2
    assert call(rows=0) == call(rows=0, x=None, u=None, gate=None, r=None, y=None) == 0


def test_residual_norm_gradient_refuses(library):
    need = library.kfb_residual_norm_bwd_workspace_bytes(12, 64, 2, 1, 1)

    def call(dr=SOME, dy=SOME, r=SOME, u=SOME, x=None, gate=SOME, gate_ld=64, w=None, gs=None, gs_ld=0, dx=SOME, du=SOME, dgate=SOME, dgs=None, dw=None, db=SOME, ds=None, ws=SOME,
             size=need, rows=12, c=64, samples=2, l=3, norm=1, st=0, ct=0):
        return library.kfb_residual_norm_bwd(VP(dr), VP(dy), VP(r), None, VP(u), None, VP(x), None, VP(gate), gate_ld, None, VP(w), VP(gs), gs_ld, VP(dx), VP(du), VP(dgate), VP(dgs),
                                             VP(dw), VP(db), VP(ds), VP(ws), size, rows, c, samples, l, 1e-5, norm, st, ct, None)
    for bad in (dict(dy=None), dict(r=None), dict(norm=0, db=None, dr=None), dict(norm=0), dict(u=None), dict(gate=None), dict(ds=SOME), dict(ws=None), dict(size=need - 1),
                dict(ws=SOME + 8), dict(dgs=SOME), dict(norm=2, db=None), dict(norm=2, gs=SOME, gs_ld=128), dict(gate_ld=8), dict(rows=-1), dict(rows=1 << 31), dict(rows=11),
                dict(c=0), dict(samples=-1), dict(l=0), dict(st=2), dict(st=0, ct=1), dict(norm=4)):
        assert call(**bad) == 1, bad
        assert b"residual_norm_bwd" in library.kfb_last_error()
    assert call(c=1025, gate_ld=2000, size=BIG) == 2
    assert call(rows=0, db=None) == 0
    room = library.kfb_residual_norm_bwd_workspace_bytes
    assert room(12, 0, 2, 1, 1) == room(12, -3, 2, 1, 1) == room(0, 64, 2, 1, 1) == room(12, 64, 0, 1, 1) == room(12, 64, 2, 0, 0) == room(12, 64, 1, 0, 1) == 0
    for c in (1, 64, 128, 768, 1024):
        sizes = [room(n, c, 4, 1, 1) for n in (4, 400, 1 << 20, (1 << 31) - 4)]
        assert sizes == sorted(sizes) and sizes[-1] == sizes[-2] < 64 << 20


def test_rows_in_8_bits_refuse(library):
    for f in (library.kfb_compress, library.kfb_expand):
        call = lambda a=SOME, b=SOME, d=SOME, rows=3, c=64, dt=0: f(VP(a), VP(b), VP(d), rows, c, dt, None)
        assert call(a=None) == call(b=None) == call(d=None) == call(rows=-1) == call(rows=1 << 40) == call(c=0) == call(c=65537) == call(dt=2) == call(dt=-1) == 1
        assert b"compress" in library.kfb_last_error() or b"expand" in library.kfb_last_error()
        assert call(rows=0, a=None) == 0


def test_linear_refuses(library):
    fwd = lambda x=SOME, w=SOME, res=None, out=SOME, ws=SOME, size=BIG, rows=3, k=64, n=128, act=0, dt=0, ot=0: library.kfb_fused_linear_fwd(
        VP(x), VP(w), None, VP(res), VP(out), VP(ws), size, rows, k, n, act, dt, ot, None)
    bwd = lambda dy=SOME, x=SOME, w=SOME, dx=SOME, dw=SOME, db=SOME, ws=SOME, size=BIG, rows=3, k=64, n=128, act=0, dt=0, dyt=0, dwt=0: library.kfb_fused_linear_bwd(
        VP(dy), VP(x), VP(w), None, VP(dx), VP(dw), VP(db), VP(ws), size, rows, k, n, act, dt, dyt, dwt, None)
    for call in (fwd, bwd):
        for bad in (dict(w=None), dict(x=None), dict(rows=-1), dict(rows=1 << 31), dict(k=0), dict(k=12), dict(n=100), dict(n=-8), dict(k=65544), dict(n=2 ** 31 - 8), dict(act=5),
                    dict(act=-1), dict(dt=1), dict(dt=7), dict(w=SOME + 8), dict(x=SOME + 2)):
            assert call(**bad) == 1, bad
            assert b"fused_linear" in library.kfb_last_error()
    for bad in (dict(out=None), dict(ot=2), dict(dt=2, ot=0), dict(res=SOME + 4)):
        assert fwd(**bad) == 1, bad
    for bad in (dict(dy=None), dict(dyt=2), dict(dwt=5), dict(dt=2, dyt=0, dwt=1), dict(dt=2, dyt=1, dwt=0), dict(dy=SOME + 8), dict(ws=SOME + 16), dict(ws=None), dict(size=16)):
        assert bwd(**bad) == 1, bad
    assert fwd(rows=0, x=None) == 0 and bwd(dx=None, dw=None, db=None) == 0


def test_linear_workspace(library):
    need = library.kfb_fused_linear_workspace_bytes
    for k, n in ((128, 128), (384, 1536), (2048, 64)):
        for act in (0, 3):
            for dt, dyt in ((0, 0), (0, 1), (2, 1)):
                for wanted in range(8):
                    sizes = [need(r, k, n, act, dt, dyt, wanted) for r in (1, 1000, 1 << 20, 1 << 24, (1 << 31) - 1)]
                    assert sizes == sorted(sizes) and sizes[-1] == sizes[-2] < 1 << 31
    for rows, k, n in ((0, 64, 64), (1, 0, 64), (1, 64, -8), (1, 2 ** 31 - 8, 2 ** 31 - 8), (1 << 31, 64, 64)):
        assert need(rows, k, n, 0, 0, 0, 7) == 0


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(4, 8), torch.zeros(8, 8)
    kept = F.Compressed(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8), torch.float32)
    for call in (lambda: F.residual_norm(x), lambda: F.residual_norm_backward(x, x, x), lambda: F.residual_norm_backward(None, x, kept), lambda: F.compress(x), lambda: F.expand(kept),
                 lambda: F.fused_linear(x, w), lambda: F.fused_linear_backward(x, x, w), lambda: F.fused_linear_backward(x, kept, w), lambda: F.layer_norm_backward(x, kept, None)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_modules_refuse_cpu_tensors_while_recording():
    from kfold_b200 import modules as M
    from kfold_b200 import trunk
    a, s = torch.zeros(1, 2, 5, 64), torch.zeros(1, 1, 5, 32)
    z = torch.zeros(1, 4, 4, 64, dtype=torch.bfloat16)
    for call in (lambda: M.AdaLN(64, 32)(a, s), lambda: M.ConditionedTransitionBlock(64, 32)(a, s), lambda: M.Linear(64, 64)(a), lambda: trunk.ParcaeRecurrence(64)(z, z)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
        with torch.no_grad(), pytest.raises(RuntimeError, match="CUDA"):
            call()


def test_rows_in_8_bits_are_what_they_say():
    v, e = torch.zeros(2, 3, 40, dtype=torch.int8), torch.zeros(2, 3, 2, dtype=torch.uint8)
    k = F.Compressed(v, e, torch.bfloat16)
    assert k.shape == (2, 3, 40) and k.device == v.device and "bfloat16" in repr(k)
    for bad in ((v.float(), e, torch.bfloat16), (v, e.int(), torch.bfloat16), (v, e[..., :1], torch.bfloat16), (v, e, torch.float16), (v.transpose(0, 1), e, torch.bfloat16),
                (torch.zeros((), dtype=torch.int8), e, torch.bfloat16)):
        with pytest.raises(ValueError):
            F.Compressed(*bad)


@pytest.mark.parametrize("name", ["residual_norm", "residual_norm_backward", "compress", "expand", "fused_linear", "fused_linear_backward"])
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

    F._fused_linear_bytes.cache_clear()
    monkeypatch.setattr(F, "_one_gpu", lambda *a: 0)
    monkeypatch.setattr(F, "_workspace", lambda device, nbytes, *a: torch.empty(nbytes, dtype=torch.uint8))
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    for what, fake in (("current_device", lambda: current[0]), ("on_device", OnDevice), ("lib", Library), ("raw_stream", lambda at=None: 7)):
        monkeypatch.setattr(F.L, what, fake)
    x, w, v = torch.zeros(4, 8), torch.zeros(8, 8), torch.zeros(8)
    kept = F.Compressed(torch.zeros(4, 8, dtype=torch.int8), torch.zeros(4, 1, dtype=torch.uint8), torch.float32)
    args = {"residual_norm": (x, x), "residual_norm_backward": (x, x, x, x, None, None, None, v), "compress": (x,), "expand": (kept,), "fused_linear": (x, w, v),
            "fused_linear_backward": (x, kept, w, v)}[name]
    for device in (1, 0):
        current[0] = device
        seen.clear()
        getattr(F, name)(*args)
        assert seen and all(d == 0 for _, d in seen) and current[0] == device
    F._fused_linear_bytes.cache_clear()


@pytest.mark.parametrize("bad", [dict(samples=3, gate=(3, 4, 8)), dict(gate=(6, 4, 16)), dict(gate_shift=(6, 4, 8)), dict(u=(6, 4, 16)), dict(weight=(4,)),
                                 dict(samples=0), dict(samples=7, gate=(1, 4, 8))])
def test_shapes_are_refused_before_the_library_is_called(monkeypatch, bad):
    monkeypatch.setattr(F, "_one_gpu", lambda *a: 0)
    monkeypatch.setattr(F.L, "current_device", lambda: 0)
    monkeypatch.setattr(F.L, "lib", lambda: pytest.fail("called"))
    more = {k: v if k == "samples" else torch.zeros(v) for k, v in bad.items()}
    x = torch.zeros(6, 4, 8)
    with pytest.raises(ValueError, match="residual_norm"):
        F.residual_norm(x, more.pop("u", x), **more)
