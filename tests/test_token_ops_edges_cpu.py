"""What the 8-bit context leaves alone, and forward-mode tangents: decided in Python, checked without a GPU."""
import gc
import weakref

import pytest
import torch


def kept_by(f):
    """the tensors that autograd keeps while f runs -> [(tensor, is it taken for a weight)]"""
    from movedepth_amd import ops

    seen = []
    with torch.autograd.graph.saved_tensors_hooks(lambda t: (seen.append((t, ops._is_weight(t))), t.detach())[1], lambda t: t):
        f()
    return seen


def weights_of(seen, shape):
    return [w for t, w in seen if sorted(t.shape) == sorted(shape)]


@pytest.mark.parametrize("frozen", [False, True])
@pytest.mark.parametrize("autocast", [False, True])
def test_a_modules_weights_are_told_from_activations(frozen, autocast):
    lin, conv = torch.nn.Linear(8, 6), torch.nn.Conv2d(3, 5, 2)
    x, im = torch.randn(4, 8, requires_grad=True), torch.randn(1, 3, 9, 9, requires_grad=True)
    for m in (lin, conv):
        m.requires_grad_(not frozen)

    def run():
        with torch.autocast("cpu", torch.bfloat16, enabled=autocast):
            lin(x * 1.0)
            conv((im * 1.0).contiguous(memory_format=torch.channels_last))

    seen = kept_by(run)
    for shape in ((8, 6), (3, 5, 2, 2)):
        w = weights_of(seen, shape)
        # (the autocast copy of a frozen weight has no graph: the context's `weights` is for it)
        assert w and all(w) is not (frozen and autocast)
    if not frozen:
        for shape in ((4, 8), (1, 3, 9, 9)):
            a = weights_of(seen, shape)
            assert a and not any(a)


def test_activations_that_custom_functions_make_are_not_weights():
    class Double(torch.autograd.Function):
        @staticmethod
        def forward(ctx, x, w):
            ctx.save_for_backward(x, w, x * 2, x.view(-1), w.view(-1))
            return x * 2 * w

        @staticmethod
        def backward(ctx, g):
            return g, g

    x, w = torch.randn(4, 8, requires_grad=True), torch.nn.Parameter(torch.randn(4, 8))
    assert [b for _, b in kept_by(lambda: Double.apply(torch.relu(x), w))][-5:] == [False, True, False, False, True]
    assert [b for _, b in kept_by(lambda: Double.apply(x, w))][-5:] == [True, True, False, True, True]      # x is a leaf that requires grad


def test_the_context_is_told_of_weights_by_shape():
    from movedepth_amd import ops

    left = ops._left_alone([torch.empty(6, 8), torch.empty(5, 3, 2, 2)])
    assert left(torch.empty(8, 6)) and left(torch.empty(5, 2, 2, 3)) and not left(torch.empty(48)) and not left(torch.empty(8, 7))


def test_tensors_left_alone_are_checked_for_changes():
    from movedepth_amd import ops

    x = torch.randn(5, 7, requires_grad=True)
    with ops.saved_act8(min_numel=1):
        a = x * 1.0
        y = a * a
    a.add_(1)
    with pytest.raises(RuntimeError, match="modified"):
        y.sum().backward()


def test_outputs_left_alone_do_not_keep_themselves_alive():
    """an operator that keeps its own result: the graph must not hold the tensor that holds the graph"""
    from movedepth_amd import ops

    x = torch.randn(5, 7, requires_grad=True)
    with ops.saved_act8(min_numel=1):
        y = torch.sigmoid(x * 1.0)
    r = weakref.ref(y)
    del y
    gc.collect()
    assert r() is None


def test_second_derivatives_through_tensors_left_alone():
    from movedepth_amd import ops

    x = torch.randn(5, 7, dtype=torch.float64, requires_grad=True)

    def f(t):
        with ops.saved_act8(min_numel=1):
            return torch.sigmoid(t * t) * t

    assert torch.autograd.gradgradcheck(f, (x,))


def test_tangents_are_seen():
    import torch.autograd.forward_ad as fw

    from movedepth_amd import _lib, ops

    x = torch.randn(3)
    ops._refuse_tangents("op", x, None)
    with fw.dual_level():
        ops._refuse_tangents("op", x, None)
        d = fw.make_dual(x, x)
        for ts in ((d,), (None, x, d)):
            with pytest.raises(_lib.MovedepthHipError, match="op.*forward"):
                ops._refuse_tangents("op", *ts)
        with torch.no_grad(), pytest.raises(_lib.MovedepthHipError):
            ops._refuse_tangents("op", d)
    with pytest.raises(_lib.MovedepthHipError):
        torch.func.jvp(lambda t: (ops._refuse_tangents("op", t), t)[1], (x,), (x,))
