"""The conditioned modules and the trunk's recurrence in training, with and without rows in 8 bits: against float64 autograd of the formulas, and as a training
program runs them (graphs, streams, threads, checkpoints).

Tolerances: between the roundings of a chain's results (2^-8 / sqrt(3) = 2.3e-3 of a value in the root mean square at the worst place of a binade) there are,
in a conditioned transition, the normalised conditioning, the gate and shift rows, the normalised stream, the feed-forward's output with its own 4e-3, the output gate, the result,
and on the way back as many again: sqrt(14 * 2.3^2 + 2 * 4^2) e-3 = 1.03e-2 of the root mean square of each result.  Float32 compute: 1e-4.  In 8 bits a
value is off by at most 2^-7 of its group's largest, which for 32 normal numbers is near 2.5 of their root mean square: 2^-7 * 2.5 / sqrt(12) * 2 = 1.1e-2 for each of the up
to four tensors kept, 2.2e-2 together, beside the other roundings: 2.5e-2.
"""
import threading

import pytest
import torch

import plain_residual as R
from kfold_b200 import _lib as L
from kfold_b200 import autograd as A
from kfold_b200 import functional as F
from kfold_b200 import modules as M
from kfold_b200 import trunk

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF, F32 = torch.bfloat16, torch.float32


@pytest.fixture(autouse=True)
def _status():
    yield
    assert L.device_status() == 0


def _randn(seed, *shape, dtype=F32, scale=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(DEV, dtype)


def _near(got, ref, bound, what):
    got = got.detach()
    off = float((got.double() - ref).square().mean().sqrt()) / (float(ref.square().mean().sqrt()) + 1e-30)
    assert got.shape == ref.shape and off <= bound, f"{what}: {off:.2e}"


def _filled(mod, seed=0):
    mod = mod.to(DEV)
    with torch.no_grad():
        for i, (name, p) in enumerate(sorted(mod.named_parameters())):
            p.copy_(_randn(seed + i, *p.shape, scale=p.shape[-1] ** -0.5 if p.dim() == 2 else 0.1))
            if name.endswith("layernorm_s.weight"):
                p.add_(1.0)
    return mod


def _norm(x, w=None):
    z = (x - x.mean(-1, keepdim=True)) / torch.sqrt(x.var(-1, unbiased=False, keepdim=True) + 1e-5)
    return z if w is None else z * w


def _weights(mod, compute):
    w = {n: q.detach().double().requires_grad_() for n, q in mod.named_parameters()}
    rounded = lambda n: w[n] + (w[n].detach().to(compute).double() - w[n].detach())
    return w, rounded


def _plain_adaln(a, s, w, m, p=""):
    sn = _norm(s, w[p + "layernorm_s.weight"])
    return torch.sigmoid(sn @ m(p + "linear_g.weight").t() + w[p + "linear_g.bias"]) * _norm(a) + sn @ m(p + "linear_bias.weight").t()


def _plain_transition(a, s, w, m, residual):
    h, g = (_plain_adaln(a, s, w, m, "adaln.") @ m("swiglu.linear.weight").t()).chunk(2, -1)
    u = (h * torch.sigmoid(h) * g) @ m("linear_out.weight").t()
    out = torch.sigmoid(s @ m("linear_g.weight").t() + w["linear_g.bias"]) * u
    return a + out if residual else out


CASES = [((1, 1, 7), 1), ((2, 3, 33), 1), ((2, 3, 33), 3), ((1, 48, 61), 1)]


@pytest.mark.parametrize("lead, own", CASES, ids=["one sample", "shared", "own conditioning", "many samples"])
@pytest.mark.parametrize("dtype, autocast", [(BF, False), (F32, True), (F32, False)], ids=["bf16", "autocast", "f32"])
@pytest.mark.parametrize("small", [False, True], ids=["", "8 bits"])
@pytest.mark.parametrize("which", ["adaln", "transition", "residual transition"])
def test_conditioned_modules(lead, own, dtype, autocast, small, which):
    c, cs = 128, 64
    b, samples, l = lead
    mod = _filled(M.AdaLN(c, cs) if which == "adaln" else M.ConditionedTransitionBlock(c, cs), 3)
    a, s = _randn(1, *lead, c, dtype=dtype).requires_grad_(), _randn(2, b, own, l, cs, dtype=dtype).requires_grad_()
    compute = BF if autocast else dtype
    more = {"residual": True} if which == "residual transition" else {}
    with torch.autocast("cuda", dtype=BF, enabled=autocast), A.compressed(small):
        out = mod(a, s, **more)
    dout = _randn(4, *out.shape, dtype=out.dtype, scale=0.1)
    out.backward(dout)
    w, m = _weights(mod, compute)
    ad, sd = a.detach().double().requires_grad_(), s.detach().double().requires_grad_()
    ref = _plain_adaln(ad, sd, w, m) if which == "adaln" else _plain_transition(ad, sd, w, m, bool(more))
    ref.backward(dout.double())
    bound = 1.03e-2 if compute == BF else 1e-4
    _near(out, ref.detach(), bound, "out")
    assert out.dtype == (compute if which == "adaln" else dtype)
    bound = 2.5e-2 if small else bound
    _near(a.grad, ad.grad, bound, "da")
    _near(s.grad, sd.grad, bound, "ds")
    for n, q in mod.named_parameters():
        assert q.grad.dtype == q.dtype and q.grad.shape == q.shape
        _near(q.grad, w[n].grad, bound, n)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_training_and_inference_agree(dtype):
    mod, a, s = _filled(M.ConditionedTransitionBlock(128, 64)), _randn(1, 2, 3, 40, 128, dtype=dtype), _randn(2, 2, 1, 40, 64, dtype=dtype)
    for m, bound in ((mod, 1.03e-2), (mod.adaln, 1.03e-2)):
        with torch.no_grad():
            ref = m(a, s)
        _near(m(a, s), ref.double(), bound if dtype == BF else 1e-4, "out")


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("small", [False, True], ids=["", "8 bits"])
def test_recurrence_of_the_trunk(autocast, small):
    c, shape = 128, (1, 21, 21)
    mod = trunk.ParcaeRecurrence(c).to(DEV)
    with torch.no_grad():
        mod.parcae_b_cont.add_(_randn(5, c, c, scale=0.02))
        mod.parcae_log_a.add_(_randn(6, c, scale=0.1))
    z, u = (_randn(i, *shape, c, dtype=F32 if autocast else BF).requires_grad_() for i in (1, 2))
    with torch.autocast("cuda", dtype=BF, enabled=autocast), A.compressed(small):
        out = mod(z, u)
        with torch.no_grad():
            assert out.dtype == z.dtype
            _near(out, mod(z, u).double(), 1.03e-2, "as in inference")
    dout = _randn(3, *out.shape, dtype=out.dtype, scale=0.1)
    out.backward(dout)
    w = {n: q.detach().double().requires_grad_() for n, q in mod.named_parameters()}
    zd, ud = z.detach().double().requires_grad_(), u.detach().double().requires_grad_()
    delta = torch.nn.functional.softplus(w["parcae_log_delta"])
    a = torch.exp(-delta * torch.exp(w["parcae_log_a"]))
    ref = a * zd + (_norm(ud) * w["layernorm_z.weight"] + w["layernorm_z.bias"]) @ (delta[:, None] * w["parcae_b_cont"]).t()
    ref.backward(dout.double())
    bound = 2.5e-2 if small else 1.03e-2
    _near(out, ref.detach(), bound, "out")
    for got, want, name in ((z.grad, zd.grad, "dz"), (u.grad, ud.grad, "du"), *((q.grad, w[n].grad, n) for n, q in mod.named_parameters())):
        _near(got, want, bound, name)


def test_linear_module():
    for mod, dtype in ((M.Linear(64, 128), F32), (M.LinearNoBias(64, 128), BF)):
        mod = _filled(mod)
        x, r = _randn(1, 3, 50, 64, dtype=dtype).requires_grad_(), _randn(2, 3, 50, 128, dtype=dtype).requires_grad_()
        out = mod(x, "gelu", residual=r)
        dout = _randn(3, *out.shape, dtype=dtype)
        out.backward(dout)
        dx, dw, db = F.fused_linear_backward(dout, x.detach(), mod.weight.detach(), None if mod.bias is None else mod.bias.detach(), "gelu")
        assert torch.equal(x.grad, dx) and torch.equal(mod.weight.grad, dw) and torch.equal(r.grad, dout)
        assert mod.bias is None or torch.equal(mod.bias.grad, db)
        with torch.no_grad():
            assert torch.equal(mod(x, "gelu", residual=r), out)
        with torch.autocast("cuda", dtype=BF):
            assert mod(x).dtype == BF
    with pytest.raises(NotImplementedError):
        mod(x.detach().half())


@pytest.mark.parametrize("small", [False, True], ids=["", "8 bits"])
def test_residual_norm_records(small):
    """Results of which one, the other or both are used; leaves that are given twice; inputs that need no gradient."""
    shape, c = (4, 9, 96), 96
    make = lambda: [t.requires_grad_() for t in (_randn(1, *shape, dtype=BF), _randn(2, *shape, dtype=BF), _randn(3, 2, 9, c, dtype=BF), 1 + 0.1 * _randn(4, c), 1 + 0.1 * _randn(5, c),
                                                 _randn(6, c))]
    dr, dy = _randn(7, *shape, dtype=BF), _randn(8, *shape, dtype=BF)
    for use in ("r", "y", "both"):
        x, u, gate, scale, w, b = make()
        with A.compressed(small):
            r, y = A.residual_norm(x, u, gate, scale, w, b, samples=2)
        torch.autograd.backward([t for t, k in ((r, "r"), (y, "y")) if use in (k, "both")], [t for t, k in ((dr, "r"), (dy, "y")) if use in (k, "both")])
        keep = (lambda t: F.compress(t.detach())) if small else (lambda t: t.detach())
        g = F.residual_norm_backward(dr if use != "y" else None, dy if use != "r" else None, keep(r), keep(u), gate.detach(), keep(x), scale.detach(), w.detach(), samples=2)
        for t, want in zip((x, u, gate, scale, w, b), g):
            assert (t.grad is None and want is None) or torch.equal(t.grad, want)
    x, u, gate, scale, w, b = make()
    r, y = A.residual_norm(x, x, weight=w, bias=b)                 # the same leaf twice
    torch.autograd.backward([r, y], [dr, dy])
    g = F.residual_norm_backward(dr, dy, r.detach(), x.detach(), weight=w.detach())
    assert torch.equal(x.grad, g.x + g.u)
    x.grad = None
    r, y = A.residual_norm(x, u.detach(), gate.detach(), samples=2)
    y.backward(dy)
    assert x.grad is not None and u.grad is None and gate.grad is None
    x, u, *_ = make()
    r, y = A.residual_norm(x, u, norm=False)
    assert y is None
    r.backward(dr)
    x.grad += 1                                                    # neither gradient is the other's memory
    assert torch.equal(u.grad, dr)
    r, y = A.residual_norm(x, weight=w)
    assert r is x
    (g,) = torch.autograd.grad(y.square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_what_8_bits_hold_is_what_is_kept():
    """The inputs themselves are not: the memory between the passes is that of the bytes."""
    n, c = 1 << 16, 256
    mod, x = M.Transition(c, 2).to(DEV), _randn(1, n, c, dtype=BF)
    held = {}
    for small in (False, True):
        t = x.clone().requires_grad_()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        with A.compressed(small):
            y = mod(t * 1.0)
        held[small] = torch.cuda.memory_allocated() - before - y.numel() * 2
        y.backward(torch.ones_like(y))
        assert torch.isfinite(t.grad).all()
        del y, t
    # (the input and the normalised rows; a result's allocation is rounded up to 2 MB)
    assert held[False] >= 2 * 2 * n * c and held[True] <= 2 * 33 / 32 * n * c + (8 << 20)


def test_compressed_is_of_the_thread_and_of_the_block():
    seen = []
    with A.compressed():
        assert A._compressing()
        t = threading.Thread(target=lambda: seen.append(A._compressing()))
        t.start()
        t.join()
        with A.compressed(False):
            assert not A._compressing()
        with pytest.raises(KeyError):
            with A.compressed(False):
                raise KeyError
        assert A._compressing()
    assert not A._compressing() and seen == [False]


def test_forward_results_do_not_hang_on_what_is_kept():
    mod, a, s = _filled(M.ConditionedTransitionBlock(128, 64)), _randn(1, 2, 3, 40, 128, dtype=BF), _randn(2, 2, 1, 40, 64, dtype=BF)
    with A.compressed():
        one = mod(a, s, residual=True)
    assert (one.double() - mod(a, s, residual=True).double()).norm() <= 4e-3 * one.double().norm()


def test_under_checkpointing():
    from torch.utils.checkpoint import checkpoint
    mod = _filled(M.ConditionedTransitionBlock(128, 64))
    grads = []
    for through in (lambda f, *t: f(*t), lambda f, *t: checkpoint(f, *t, use_reentrant=False)):
        a, s = _randn(1, 2, 3, 40, 128, dtype=BF).requires_grad_(), _randn(2, 2, 1, 40, 64, dtype=BF)
        through(lambda p, q: mod(p, q, residual=True), a, s).sum().backward()
        grads.append(a.grad)
    assert torch.equal(*grads)


@pytest.mark.parametrize("small", [False, True], ids=["", "8 bits"])
def test_captured_step_of_a_conditioned_block(small):
    """Forward and backward pass in one graph: every replay gives the gradients of its inputs.  (No eager graph of the same parameters is alive while the step is
    captured: its accumulation nodes belong to another stream.)"""
    mod = _filled(M.ConditionedTransitionBlock(128, 64))
    params = list(mod.parameters())
    a, s = torch.zeros(2, 5, 50, 128, dtype=BF, device=DEV, requires_grad=True), torch.zeros(2, 1, 50, 64, dtype=BF, device=DEV, requires_grad=True)
    dout = torch.zeros(2, 5, 50, 128, dtype=BF, device=DEV)

    def step(a, s, dout):
        with A.compressed(small):
            out = mod(a, s, residual=True)
        return (out.detach(), *torch.autograd.grad(out, [a, s, *params], dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(a, s, dout)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(a, s, dout)
    for i in range(3):
        with torch.no_grad():
            a.copy_(_randn(30 + i, *a.shape))
            s.copy_(_randn(40 + i, *s.shape))
            dout.copy_(_randn(50 + i, *a.shape, scale=0.1))
        graph.replay()
        want = step(a.detach().clone().requires_grad_(), s.detach().clone().requires_grad_(), dout)
        for got, ref in zip(outs, want):
            assert torch.equal(got, ref)


def _step(x, u, gate, w, dy):
    r, y, kept = F.residual_norm(x, u, gate, weight=w, samples=2, compress=True)
    g = F.residual_norm_backward(None, y, kept, F.compress(u), gate, weight=w, samples=2)
    z = F.fused_linear(y, dy, w, "silu", r)
    return (r, y, *(t for t in g if t is not None), z, *F.fused_linear_backward(z, F.compress(y), dy, w, "silu"))


def _data(i, l=700, c=256):
    return (_randn(10 + i, 4, l, c, dtype=BF), _randn(20 + i, 4, l, c, dtype=BF), _randn(30 + i, 2, l, c, dtype=BF), 1 + 0.1 * _randn(40 + i, c),
            _randn(50 + i, c, c, dtype=BF, scale=c ** -0.5))


def test_two_graphs_replayed_at_once():
    """Each has its own scratch memory: replays on two streams do not meet."""
    data = [_data(i) for i in range(2)]
    want = [_step(*d) for d in data]
    graphs = []
    for d in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = _step(*d)
        graphs.append((g, out))
    streams = [torch.cuda.Stream() for _ in data]
    torch.cuda.synchronize()
    for _ in range(20):
        for s, (g, _) in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for (_, out), ref in zip(graphs, want):
        assert all(torch.equal(a, b) for a, b in zip(out, ref))


def test_host_threads_and_streams():
    data = [_data(i, 300) for i in range(4)]
    want = [_step(*d) for d in data]
    torch.cuda.synchronize()
    start, wrong = threading.Barrier(len(data)), []

    def run(i):
        own = torch.cuda.Stream() if i % 2 else torch.cuda.current_stream()
        start.wait()
        with torch.cuda.stream(own):
            for _ in range(30):
                got = _step(*data[i])
                own.synchronize()
                if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                    wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(data))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_steps_of_an_optimizer():
    """Parameters that change in place: the next training pass and the packed inference weights both follow."""
    mod, a, s = _filled(M.ConditionedTransitionBlock(128, 64)), _randn(1, 2, 3, 40, 128, dtype=BF), _randn(2, 2, 1, 40, 64, dtype=BF)
    opt = torch.optim.SGD(mod.parameters(), lr=0.5)
    for _ in range(2):
        opt.zero_grad()
        out = mod(a, s)
        out.float().square().mean().backward()
        opt.step()
        with torch.no_grad():
            inference = mod(a, s)
        after = mod(a, s)
        assert not torch.equal(after, out)
        _near(after, inference.double(), 1.03e-2, "after the step")
