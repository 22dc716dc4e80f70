"""The training operators together, as a training step uses them: z + dropout(Transition(z)) under autograd, against float64 autograd of the
formulas with the same mask.

Tolerances: bf16 stores the normalised rows, the feed-forward's output, their gradients and dx, five roundings of 2^-8 / sqrt(3) of a value in the
root mean square each, and the feed-forward's own 4e-3 (see its tests) for y and again for its gradients: sqrt(5 * 2.3^2 + 2 * 4^2) e-3 = 7.6e-3
of the root mean square of each result at most.  Float32 parameters' gradients add up bf16 products: the same.  Float32 compute: 4e-5.
"""
import threading

import pytest
import torch

import plain_training as P
from kfold_b200 import _lib as L
from kfold_b200 import autograd as A
from kfold_b200 import functional as F
from kfold_b200 import modules as M

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


def _transition(c, factor=4, seed=0):
    mod = M.Transition(c, factor).to(DEV)
    with torch.no_grad():
        for i, (name, p) in enumerate(mod.named_parameters()):
            p.copy_(_randn(seed + i, *p.shape, scale=p.shape[-1] ** -0.5 if p.dim() == 2 else 0.1))
            if name == "layernorm.weight":
                p.add_(1.0)
    return mod


def _plain(mod, z, p, rng, shared_dim, dout, compute):
    """Float64: result and the gradients of z and the parameters (weights rounded as the products take them)."""
    z = z.double().detach().requires_grad_()
    w = {n: q.detach().double().requires_grad_() for n, q in mod.named_parameters()}
    rounded = lambda t: t + (t.detach().to(compute).double() - t.detach())
    xn = P.layer_norm(z, w["layernorm.weight"], w["layernorm.bias"], mod.layernorm.eps)
    a, b = (xn @ rounded(w["swiglu.linear.weight"]).t()).chunk(2, -1)
    y = (a * torch.sigmoid(a) * b) @ rounded(w["linear_out.weight"]).t()
    mask = P.kept(z.shape, shared_dim, p, rng).to(DEV)
    out = z + torch.where(mask, y / (1 - p), torch.zeros((), dtype=y.dtype, device=DEV))
    out.backward(dout.double())
    return out.detach(), z.grad, {n: q.grad for n, q in w.items()}


@pytest.mark.parametrize("c, shape, shared_dim", [(128, (1, 37, 37), -3), (256, (2, 20, 20), -2), (384, (3, 65), None), (128, (1, 150, 150), -3)])
@pytest.mark.parametrize("dtype, autocast", [(BF, False), (F32, True), (F32, False)], ids=["bf16", "autocast", "f32"])
def test_residual_update_of_a_block(c, shape, shared_dim, dtype, autocast):
    mod, rng, p = _transition(c), (11, 22), 0.25
    z, dout = _randn(1, *shape, c, dtype=dtype).requires_grad_(), _randn(2, *shape, c, dtype=dtype, scale=0.1)
    with torch.autocast("cuda", dtype=BF, enabled=autocast):
        out = A.dropout(mod(z), p, rng, shared_dim=shared_dim, residual=z)
    out.backward(dout)
    compute = BF if autocast else dtype
    ref, dz, grads = _plain(mod, z, p, rng, shared_dim, dout, compute)
    bound = 7.6e-3 if compute == BF else 4e-5
    assert out.dtype == z.grad.dtype == dtype
    _near(out, ref, bound, "out")
    _near(z.grad, dz, bound, "dz")
    for n, q in mod.named_parameters():
        assert q.grad.dtype == q.dtype
        _near(q.grad, grads[n], bound, n)


@pytest.mark.parametrize("dtype", [BF, F32])
def test_training_and_inference_agree(dtype):
    """The same module with and without autograd: other kernels, the same arithmetic up to the roundings in between."""
    mod, x = _transition(128), _randn(3, 2, 61, 61, 128, dtype=dtype)
    for residual in (False, True):
        with torch.no_grad():
            ref = mod(x, residual=residual)
        _near(mod(x, residual=residual).detach(), ref.double(), 7.6e-3 if dtype == BF else 4e-5, "out")


def test_steps_of_an_optimizer():
    """Parameters that change in place: the next training pass and the packed inference weights both follow."""
    mod = _transition(128)
    x, target = _randn(5, 300, 128, dtype=BF), _randn(6, 300, 128)
    opt = torch.optim.SGD(mod.parameters(), lr=0.5)
    for step in range(3):
        opt.zero_grad()
        out = mod(x)
        (out.float() - target).square().sum(-1).mean().backward()
        opt.step()
        with torch.no_grad():
            inference = mod(x)
        after = mod(x)
        assert not torch.equal(after, out)
        _near(after, inference.double(), 7.6e-3, "after the step")


def test_only_what_needs_a_gradient():
    mod = _transition(128)
    x = _randn(1, 90, 128, dtype=BF)
    mod.swiglu.linear.weight.requires_grad_(False)
    mod.layernorm.bias.requires_grad_(False)
    mod(x).float().sum().backward()
    assert mod.swiglu.linear.weight.grad is None and mod.layernorm.bias.grad is None
    assert mod.linear_out.weight.grad is not None and mod.layernorm.weight.grad is not None
    y = x.clone().requires_grad_()
    for q in mod.parameters():
        q.requires_grad_(False)
    mod(y).float().sum().backward()
    assert y.grad is not None and torch.isfinite(y.grad).all()


def test_layer_norm_module_records():
    mod, x = M.LayerNorm(200).to(DEV), _randn(1, 33, 200).requires_grad_()
    dy = _randn(2, 33, 200)
    mod(x).backward(dy)
    dx, dw, db = F.layer_norm_backward(dy, x.detach(), mod.weight.detach())
    assert torch.equal(x.grad, dx) and torch.equal(mod.weight.grad, dw) and torch.equal(mod.bias.grad, db)
    plain = M.LayerNorm(200, create_scale=False, create_offset=False).to(DEV)
    x.grad = None
    plain(x).backward(dy)
    assert torch.equal(x.grad, F.layer_norm_backward(dy, x.detach(), None, need_bias=False)[0])


def test_second_derivatives_are_refused():
    x = _randn(1, 8, 64).requires_grad_()
    (g,) = torch.autograd.grad(A.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_dropout_module():
    x, r = _randn(1, 1, 40, 40, 128, dtype=BF).requires_grad_(), _randn(2, 1, 40, 40, 128, dtype=BF).requires_grad_()
    mod = M.Dropout(0.25, shared_dim=-3).to(DEV)
    torch.manual_seed(7)
    a = mod(x, residual=r)
    b = mod(x, residual=r)
    torch.manual_seed(7)
    assert torch.equal(a, mod(x, residual=r)) and not torch.equal(a, b)
    dy = _randn(3, 1, 40, 40, 128, dtype=BF)
    a.backward(dy)
    dropped = (a == r).all(dim=1, keepdim=True)          # a whole column of the mask
    assert torch.equal(r.grad, dy)
    assert not x.grad[dropped.expand_as(x)].any() and 0.2 < float(dropped.float().mean()) < 0.3
    kept = ~dropped.expand_as(x)
    assert torch.equal(x.grad[kept], (dy.float() * (1 / 0.75)).to(BF)[kept])
    mod.eval()
    assert mod(x) is x and torch.equal(mod(x, residual=r), (x.float() + r.float()).to(BF))


def test_dropout_under_checkpointing():
    """A recomputed forward pass draws the mask of the first one."""
    from torch.utils.checkpoint import checkpoint
    mod, tr = M.Dropout(0.3), _transition(128)
    x, dy = _randn(1, 70, 128, dtype=BF), _randn(2, 70, 128, dtype=BF)
    grads = []
    for through in (lambda f, t: f(t), lambda f, t: checkpoint(f, t, use_reentrant=False)):
        torch.manual_seed(3)
        t = x.clone().requires_grad_()
        through(lambda u: mod(tr(u), residual=u), t).backward(dy)
        grads.append(t.grad)
    assert torch.equal(*grads)


def test_dropout_state_moved_on_before_the_backward_pass():
    x, rng = torch.ones(64, 128, device=DEV).requires_grad_(), torch.tensor([5, 0], device=DEV)
    y = A.dropout(x, 0.5, rng)
    rng[1] += 1
    y.backward(torch.ones_like(y))
    assert torch.equal(x.grad, y.detach())


def test_dropout_module_in_a_graph_wants_a_state():
    x, mod = _randn(1, 64, 128), M.Dropout(0.5)
    rng = torch.tensor([1, 0], device=DEV)
    with torch.no_grad():
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = mod(x, rng=rng)
            rng[1] += 1
        seen = []
        for _ in range(3):
            graph.replay()
            seen.append(out.clone())
    assert not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_two_graphs_replayed_at_once():
    """Each has its own scratch memory: replays on two streams do not meet."""
    n, c, hidden = 4000, 256, 1024
    w_in, w_out = _randn(1, 2 * hidden, c, dtype=BF, scale=c ** -0.5), _randn(2, c, hidden, dtype=BF, scale=hidden ** -0.5)
    ln = 1 + 0.1 * _randn(3, c)
    data = [(_randn(10 + i, n, c, dtype=BF), _randn(20 + i, n, c, dtype=BF, scale=0.1)) for i in range(2)]
    step = lambda x, dy: (*F.gated_feed_forward_backward(dy, x, w_in, w_out), *F.layer_norm_backward(dy, x, ln))
    want = [step(*d) for d in data]
    graphs = []
    for d in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*d)
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


def test_blocks_stay_inference_only():
    blk = M.TriangularBlock(128).to(DEV)
    with pytest.raises(RuntimeError, match="inference-only"):
        blk(_randn(1, 1, 24, 24, 128, dtype=BF), torch.ones(1, 24, 24, dtype=torch.bool, device=DEV))


def test_cpu_tensors_are_refused_while_recording():
    with pytest.raises(RuntimeError, match="CUDA"):
        M.Transition(64, 2)(torch.zeros(3, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        M.LayerNorm(64)(torch.zeros(3, 64))


def test_host_threads_that_share_a_stream():
    """Their calls' launches mix on the stream; each thread has scratch memory of its own."""
    c, hidden, n = 256, 1024, 1500
    w_in, w_out = _randn(1, 2 * hidden, c, dtype=BF, scale=c ** -0.5), _randn(2, c, hidden, dtype=BF, scale=hidden ** -0.5)
    ln = 1 + 0.1 * _randn(3, c)
    data = [(_randn(10 + i, n, c, dtype=BF), _randn(20 + i, n, c, dtype=BF, scale=0.1)) for i in range(4)]
    step = lambda x, dy: (F.gated_feed_forward(x, w_in, w_out), *F.gated_feed_forward_backward(dy, x, w_in, w_out), *F.layer_norm_backward(dy, x, ln))
    want = [step(*d) for d in data]
    torch.cuda.synchronize()
    start, wrong, places = threading.Barrier(len(data)), [], []

    def run(i):
        start.wait()
        places.append(F._call_workspace(data[i][0].device, 1 << 16))      # (held, or a freed one's address comes again)
        for _ in range(40):
            got = step(*data[i])
            torch.cuda.current_stream().synchronize()
            if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                wrong.append(i)

    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(data))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong and len({t.data_ptr() for t in places}) == len(data)


@pytest.mark.parametrize("rng", [(1, 2), None], ids=["numbers", "device memory"])
@pytest.mark.parametrize("dtypes", [(BF, BF), (F32, F32), (BF, F32)], ids=lambda d: "+".join(str(t)[6:] for t in d))
def test_residual_sum_without_dropout(dtypes, rng):
    """p = 0 adds, and its gradient goes to both sides as it is."""
    x, res = (_randn(1 + i, 5, 64, dtype=t).requires_grad_() for i, t in enumerate(dtypes))
    out = A.dropout(x, 0.0, torch.tensor([1, 2], device=DEV) if rng is None else rng, residual=res)
    dy = _randn(3, 5, 64, dtype=dtypes[1])
    out.backward(dy)
    assert torch.equal(out, (x.float() + res.float()).to(dtypes[1]))
    assert torch.equal(x.grad, dy.to(dtypes[0])) and torch.equal(res.grad, dy)
    x.grad += 1                                            # neither gradient is the other's memory
    assert torch.equal(res.grad, dy)


def test_captured_step_of_modules():
    """Forward and backward pass of LayerNorm, Transition and Dropout in one graph: every replay gives the gradients of its inputs and its mask.
    (No eager graph of the same parameters is alive while the step is captured: its accumulation nodes belong to another stream.)"""
    c, p = 128, 0.25
    mod, drop, norm = _transition(c), M.Dropout(p), M.LayerNorm(c).to(DEV)
    params = [*mod.parameters(), *norm.parameters()]
    z, dy = torch.zeros(3, 50, c, dtype=BF, device=DEV, requires_grad=True), torch.zeros(3, 50, c, dtype=BF, device=DEV)
    rng = torch.tensor([9, 0], device=DEV)

    def step(z, dy, rng):
        out = norm(drop(mod(z), residual=z, rng=rng))
        return (out.detach(), *torch.autograd.grad(out, [z, *params], dy))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(z, dy, rng)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(z, dy, rng)
        rng[1] += 1
    rng[1] = 0
    for i in range(3):
        with torch.no_grad():
            z.copy_(_randn(30 + i, *z.shape))
            dy.copy_(_randn(40 + i, *z.shape, scale=0.1))
        graph.replay()
        want = step(z.detach().clone().requires_grad_(), dy, torch.tensor([9, i], device=DEV))
        assert int(rng[1]) == i + 1
        for got, ref in zip(outs, want):
            assert torch.equal(got, ref)
