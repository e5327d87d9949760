"""CPU: what deepshift_amd.training.linear_distillation refuses, and the library's own checks."""
import pytest
import torch

from deepshift_amd import _lib, training

H, W, IDS, LOGITS = torch.ones(3, 4), torch.ones(6, 4), torch.zeros(3, 2, dtype=torch.int64), torch.zeros(3, 2)


def test_tensors_are_refused_before_anything_runs():
    for call in (lambda: training.linear_distillation(H, W, IDS, LOGITS), lambda: training.linear_distillation_grad(H, W, IDS, LOGITS),
                 lambda: training.linear_distillation(H.clone().requires_grad_(), W, IDS, LOGITS),
                 lambda: training.LinearCrossEntropy(4, 6).distill(H, IDS, LOGITS)):
        with pytest.raises(ValueError, match="GPU"):
            call()
    for f in (training.linear_distillation, training.linear_distillation_grad):
        for temperature in (0.0, -1.0, float("inf"), float("nan"), 2.0 ** 21):
            with pytest.raises(ValueError, match="temperature"):
                f(H, W, IDS, LOGITS, temperature=temperature)
        with pytest.raises(ValueError, match="reduction"):
            f(H, W, IDS, LOGITS, reduction="max")
    with pytest.raises(TypeError, match="float32"):
        training.linear_distillation(H.double(), W.double(), IDS, LOGITS)


def test_forward_mode_and_tracing_are_refused():
    import torch.autograd.forward_ad as forward_ad
    from torch.fx.experimental.proxy_tensor import make_fx
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward"):
            training.linear_distillation(H, forward_ad.make_dual(W, torch.ones_like(W)), IDS, LOGITS)
    with pytest.raises(NotImplementedError, match="trac"):
        torch.jit.trace(lambda x: training.linear_distillation(x, W, IDS, LOGITS), (H,))
    with pytest.raises(NotImplementedError, match="trac"):
        make_fx(lambda x: training.linear_distillation(x, W, IDS, LOGITS))(H)


def test_the_library_checks_sizes_and_pointers():
    L = _lib.lib()
    at = H.data_ptr()
    for words, dtype, what, T in ((0, 0, 1, 3), (1025, 0, 1, 3), (2, 3, 1, 3), (2, 0, 4, 3), (2, 0, 0, 3), (2, 0, 1, -1)):
        assert L.ds_distill_workspace_bytes(at, 4, at, 4, T, 4, 6, dtype, words, what) == 0

    def loss(h=at, ldh=4, ids=at, id_bytes=8, logits=at, logits_type=0, words=2, temperature=1.0, T=3, D=4, V=6, dtype=0, reduction=0,
             rows=at, lse=at, total=at):
        return L.ds_distill_loss(h, ldh, at, 4, None, ids, id_bytes, logits, logits_type, words, temperature, T, D, V, dtype,
                                 reduction, rows, lse, total, None, 0, None)

    assert loss() == -4      # nothing wrong but that there is no workspace
    for wrong in (dict(h=None), dict(ldh=3), dict(ids=None), dict(id_bytes=2), dict(logits=None), dict(logits_type=5), dict(words=0),
                  dict(words=1025), dict(temperature=0.0), dict(temperature=float("nan")), dict(temperature=2.0 ** 21), dict(T=-1),
                  dict(V=0), dict(dtype=3), dict(reduction=3), dict(rows=None), dict(lse=None), dict(reduction=2, total=None)):
        assert loss(**wrong) == -1, wrong
    for large in (dict(T=2 ** 31), dict(V=2 ** 31), dict(ldh=2000001), dict(T=2 ** 24, words=1024)):
        assert loss(**large) == -5, large
    assert L.ds_distill_loss_grad(at, 4, at, 4, None, at, 8, at, 0, 2, 1.0, 3, 4, 6, 0, None, None, None, None, at, at, at, None, 0,
                                  None) == -1
    assert L.ds_distill_loss_grad(at, 4, at, 4, None, at, 8, at, 0, 2, 1.0, 3, 4, 6, 0, at, at, at, None, at, at, at, None, 0,
                                  None) == -1
