"""CPU: what deepshift_amd.training.gated_linear refuses, and the library's own checks."""
import pytest
import torch

from deepshift_amd import _lib, training

X, W = torch.ones(3, 4), torch.ones(6, 4)


def test_tensors_are_refused_before_anything_runs():
    for call in (lambda: training.gated_linear(X, W), lambda: training.gated_linear(X, W.clone().requires_grad_()),
                 lambda: training.GatedLinear(4, 3)(X), lambda: training.GatedShift(4, 3)(X)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for kind in ("tanh", None, 0):
        with pytest.raises(ValueError, match="activation"):
            training.gated_linear(X, W, activation=kind)
        with pytest.raises(ValueError, match="activation"):
            training.GatedLinear(4, 3, activation=kind)
    with pytest.raises(ValueError, match="shift_type"):
        training.GatedShift(4, 3, shift_type="X")
    with pytest.raises(TypeError, match="float32"):
        training.gated_linear(X.double(), W.double())
    with pytest.raises(ValueError, match="resolve_neg"):
        training.gated_linear(X, torch._neg_view(W))


def test_forward_mode_and_tracing_are_refused():
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward"):
            training.gated_linear(X, forward_ad.make_dual(W, torch.ones_like(W)))
    with pytest.raises(NotImplementedError, match="trac"):
        torch.jit.trace(lambda x: training.gated_linear(x, W), (X,))
    with pytest.raises(NotImplementedError, match="trac"):
        make_fx(lambda x: training.gated_linear(x, W))(X)


def test_the_library_checks_sizes_and_pointers():
    L = _lib.lib()
    at = X.data_ptr()
    assert L.ds_gated_workspace_bytes(at, 4, at, 4, 3, 4, 3, 3, 1) == 0
    assert L.ds_gated_workspace_bytes(at, 4, at, 4, 3, 4, 3, 0, 3) == 0
    assert L.ds_gated_workspace_bytes(at, 4, at, 4, -1, 4, 3, 0, 1) == 0

    def forward(x=at, ldx=4, w=at, ldw=4, activation=0, T=3, D=4, F=3, dtype=0, out=at):
        return L.ds_gated_forward(x, ldx, w, ldw, None, activation, T, D, F, dtype, out, None, None, 0, None)

    assert forward() == -4     # nothing wrong but that there is no workspace
    for wrong in (dict(x=None), dict(w=None), dict(ldx=3), dict(ldw=3), dict(activation=4), dict(activation=-1), dict(T=-1),
                  dict(dtype=3), dict(out=None)):
        assert forward(**wrong) == -1, wrong
    for large in (dict(D=2000000, ldx=2000000, ldw=2000000), dict(ldw=2000001), dict(T=2 ** 31), dict(F=2 ** 30)):
        assert forward(**large) == -5, large

    def backward(halves=at, grad=at, ldg=3, activation=0):
        return L.ds_gated_backward(at, 4, at, 4, halves, grad, ldg, activation, 3, 4, 3, 0, at, at, at, None, 0, None)

    assert backward(halves=None) == -1 and backward(grad=None) == -1 and backward(ldg=2) == -1 and backward(activation=9) == -1
