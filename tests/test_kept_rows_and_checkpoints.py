"""Rows kept in 8 bits under torch.utils.checkpoint, whose repeated forward pass runs on another thread than the first."""
import threading

import pytest
import torch
from torch.utils.checkpoint import CheckpointError, checkpoint

import test_gpu_conditioned_training as T
from kfold_b200 import autograd as A
from kfold_b200 import modules as M

DEV = "cuda:0"
BF = torch.bfloat16


class _Double(torch.autograd.Function):
    """Keeps its input as one tensor or as two, as the operators do."""
    chosen = []

    @staticmethod
    def forward(ctx, x):
        small = A._compressing()
        _Double.chosen.append(small)
        ctx.save_for_backward(*((x.to(torch.int8), x[:1].to(torch.uint8)) if small else (x,)))
        return 2 * x

    @staticmethod
    def backward(ctx, dy):
        assert len(ctx.saved_tensors) in (1, 2)
        return 2 * dy


def _on_another_thread(f):
    out = []

    def run():
        try:
            f()
        except Exception as e:
            out.append(e)

    t = threading.Thread(target=run)
    t.start()
    t.join()
    if out:
        raise out[0]


@pytest.mark.parametrize("small", [False, True])
def test_the_repeated_pass_keeps_rows_as_the_first(small):
    """Backward passes on another thread than the forward pass, two of them, under another choice than the first's."""
    x = torch.arange(4.0, requires_grad=True)
    _Double.chosen.clear()
    with A.compressed(small):
        y = checkpoint(lambda t: _Double.apply(t), x, use_reentrant=False, context_fn=A.checkpoint_contexts)
        assert A._compressing() == small
    def twice():
        with A.compressed(not small):
            y.sum().backward(retain_graph=True)
            y.sum().backward()
            assert A._compressing() != small
    _on_another_thread(twice)
    assert _Double.chosen == [small] * 3 and torch.equal(x.grad, torch.full((4,), 4.0)) and not A._compressing()


def test_the_choice_inside_the_function():
    x = torch.arange(4.0, requires_grad=True)

    @A.compressed()
    def block(t):
        return _Double.apply(t)

    _Double.chosen.clear()
    y = checkpoint(block, x, use_reentrant=False)
    _on_another_thread(lambda: y.sum().backward())
    assert _Double.chosen == [True] * 2 and not A._compressing()


def test_without_either_torch_says_so():
    x = torch.arange(4.0, requires_grad=True)
    with A.compressed():
        y = checkpoint(lambda t: _Double.apply(t), x, use_reentrant=False)
    with pytest.raises(CheckpointError):
        _on_another_thread(lambda: y.sum().backward())


def test_one_manager_entered_again_and_from_two_threads():
    small, seen, both = A.compressed(), [], threading.Barrier(2)
    with small, A.compressed(False), small:
        assert A._compressing()
    assert not A._compressing()

    def run():
        with small:
            both.wait()
            with A.compressed(False):
                both.wait()
            seen.append(A._compressing())
        seen.append(A._compressing())

    threads = [threading.Thread(target=run) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert sorted(seen) == [False, False, True, True]


@pytest.mark.gpu
@pytest.mark.parametrize("inside", [False, True])
@pytest.mark.parametrize("c", [128, 64])
def test_conditioned_block(inside, c):
    mod = T._filled(M.ConditionedTransitionBlock(c, 64))
    grads = []
    for again in (False, True):
        a, s = T._randn(1, 2, 3, 40, c, dtype=BF).requires_grad_(), T._randn(2, 2, 1, 40, 64, dtype=BF).requires_grad_()
        mod.zero_grad()

        def block(p, q):
            with A.compressed(True if inside else A._compressing()):
                return mod(p, q, residual=True)

        with A.compressed(not inside):
            if again:
                y = checkpoint(block, a, s, use_reentrant=False, **({} if inside else {"context_fn": A.checkpoint_contexts}))
            else:
                y = block(a, s)
        y.sum().backward()
        grads.append([a.grad, s.grad, *(p.grad.clone() for p in mod.parameters())])
    assert all(torch.equal(p, q) for p, q in zip(*grads))
