"""Dropout of element counts that no piece of 16 bytes divides, every element by itself."""
import pytest
import torch

import plain_training as P
from kfold_b200 import _lib as L
from kfold_b200 import functional as F

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32
TYPES = [(BF, None), (F32, None), (BF, BF), (F32, F32), (BF, F32)]
IDS = ["+".join(str(t)[6:] for t in d if t) for d in TYPES]
RNG = (0x0123456789ABCDEF, (1 << 63) + 12345)


@pytest.fixture(autouse=True)
def _status():
    yield
    assert L.device_status() == 0


def _randn(seed, *shape, dtype=F32):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed)).to(DEV, dtype)


def _in_turn(calls, rounds=9, each=10):
    """Median us of one call of each (graph replays: the GPU alone)."""
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


@pytest.mark.parametrize("dtype, resid", [(BF, False), (BF, True), (F32, False), (F32, True)])
def test_an_odd_count_costs_what_its_neighbour_does(dtype, resid):
    n = 384 * 384 * 128
    x = _randn(1, n + 1, dtype=dtype)
    r = x.clone() if resid else None
    even, odd = _in_turn([lambda n=n: F.dropout(x[:n], 0.25, (1, 2), residual=None if r is None else r[:n]) for n in (n, n + 1)])
    assert odd < 1.6 * even, (odd, even)


@pytest.mark.parametrize("types", TYPES, ids=IDS)
@pytest.mark.parametrize("n", [1, 3, 7, 9, 15, 1023, 2047, 2049, 4093, 4097, 4103, 8191, 8193, 8199, 3 * 8192 + 5, (1 << 20) + 4, 2000003])
def test_every_element_once_and_none_behind_the_last(n, types):
    """The last piece, a block's last and the first of a block: out has more room than elements."""
    x, r = _randn(n, n, dtype=types[0]), None if types[1] is None else _randn(n + 1, n, dtype=types[1])
    dtype = types[1] or types[0]
    p, scale = 0.25, 4.0 / 3.0
    mask = P.kept((n,), None, p, RNG).to(DEV)
    part = torch.where(mask, x.double() * scale, torch.zeros((), dtype=torch.float64, device=DEV))
    ref = part if r is None else r.double() + part
    # the scale is rounded, the product and the sum are: 3 u of what they are made of, and the result to its type
    room = P.HALF_STEP[dtype] * ref.abs() + 3 * P.U32 * (part.abs() + (0 if r is None else r.double().abs()))
    state = torch.tensor([RNG[0], RNG[1] - (1 << 64)], device=DEV)
    codes = [{BF: 0, F32: 1}[t] for t in (types[0], dtype)]
    for rng in (None, L.ptr(state)):
        out = torch.full((n + 64,), 7.0, dtype=dtype, device=DEV)
        L.check(L.lib().kfb_dropout(L.ptr(x), L.ptr(r), L.ptr(out), 1, 1, n, 1 << 30, scale, rng, RNG[0], RNG[1] - (1 << 64), *codes, L.stream_ptr()))
        assert (out[n:] == 7).all()
        assert ((out[:n].double() - ref).abs() <= room).all()
        if r is None:
            assert not out[:n][~mask].any()


@pytest.mark.parametrize("n", [4099, 8197])
def test_in_place(n):
    """out may be x or the residual."""
    for dtype, code in ((BF, 0), (F32, 1)):
        x, r = _randn(1, n, dtype=dtype), _randn(2, n, dtype=dtype)
        want = F.dropout(x, 0.25, (1, 2), residual=r)
        for which in range(2):
            a, b = x.clone(), r.clone()
            L.check(L.lib().kfb_dropout(L.ptr(a), L.ptr(b), L.ptr((a, b)[which]), 1, 1, n, 1 << 30, 4.0 / 3.0, None, 1, 2, code, code, L.stream_ptr()))
            assert torch.equal((a, b)[which], want)
        a = x.clone()
        L.check(L.lib().kfb_dropout(L.ptr(a), None, L.ptr(a), 1, 1, n, 1 << 30, 4.0 / 3.0, None, 1, 2, code, code, L.stream_ptr()))
        assert torch.equal(a, F.dropout(x, 0.25, (1, 2)))


def test_infinities_behind_the_last_whole_piece():
    x = torch.full((4103,), float("inf"), device=DEV)
    x[1::2] = float("nan")
    mask = P.kept(x.shape, None, 0.4, (9, 9)).to(DEV)
    out = F.dropout(x, 0.4, (9, 9))
    assert not out[~mask].any() and not torch.isfinite(out[mask]).any()
