"""CPU: what deepshift_amd.training.gated_recurrence refuses, and the library's own checks."""
import pytest
import torch

from deepshift_amd import _lib, training

X = torch.zeros(2, 3, 4)


def test_tensors_are_refused_before_anything_runs():
    for call in (lambda: training.gated_recurrence(X, X), lambda: training.gated_recurrence(X, X, torch.zeros(2, 4)),
                 lambda: training.gated_recurrence(X.clone().requires_grad_(), X)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    with pytest.raises(TypeError, match="float32"):
        training.gated_recurrence(X.double(), X.double())
    with pytest.raises(TypeError, match="tensor"):
        training._recur(X, [1.0], None, None, False)
    with pytest.raises(ValueError, match="resolve_neg"):
        training.gated_recurrence(torch._neg_view(X), X)


def test_forward_mode_and_tracing_are_refused():
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward"):
            training.gated_recurrence(X, forward_ad.make_dual(X, torch.ones_like(X)))
    with pytest.raises(NotImplementedError, match="trac"):
        torch.jit.trace(lambda x: training.gated_recurrence(x, x), (X,))
    with pytest.raises(NotImplementedError, match="trac"):
        make_fx(lambda x: training.gated_recurrence(x, x))(X)


def test_the_library_checks_sizes_and_pointers():
    L = _lib.lib()
    assert [L.ds_recur_blocks(T) for T in (0, 1, 8, 9, 32, 33, 64, 65, 129)] == [0, 1, 1, 1, 1, 1, 1, 2, 3]
    assert L.ds_recur_workspace_bytes(2, 3, 4, 7) == 0 and L.ds_recur_workspace_bytes(-1, 3, 4, 0) == 0
    at = X.data_ptr()

    def forward(B=2, T=3, D=4, dtype=0, lengths=None, length_bytes=0, x=at, last=at):
        return L.ds_recur_forward(x, 12, 4, at, 12, 4, None, lengths, length_bytes, at, last, None, B, T, D, dtype, None, 0, None)

    assert forward(T=-1) == -1 and forward(dtype=3) == -1 and forward(lengths=at, length_bytes=2) == -1
    assert forward(x=None) == -1 and forward(last=None) == -1
    assert forward(B=2 ** 31) == -5 and forward(D=2 ** 31) == -5 and forward(B=2 ** 20, D=2 ** 20) == -5
    assert forward(T=2 ** 41) == -5
    assert forward(B=0) == 0 and forward(D=0) == 0

    def backward(T=3, kept=at, lengths=None, length_bytes=0):
        return L.ds_recur_backward(at, 12, 4, at, 12, 4, at, 12, 4, None, lengths, length_bytes, kept, at, at, at, 2, T, 4, 0,
                                   None, 0, None)

    assert backward(kept=None) == -1 and backward(T=-1) == -1 and backward(lengths=at, length_bytes=3) == -1
