"""CPU: what deepshift_amd.training refuses rather than answer wrongly."""
import itertools

import pytest
import torch

from deepshift_amd import _lib, training

IDS, X, W = torch.zeros(3, dtype=torch.int64), torch.ones(3, 4), torch.ones(5, 4)


def test_whether_tensors_meet_is_told_exactly():
    # against the bytes themselves
    base = torch.zeros(6, 9)
    half = base.view(torch.bfloat16)

    def touched(t):
        at = torch.zeros((), dtype=torch.int64)
        for n, stride in zip(t.shape, t.stride()):
            at = at[..., None] + torch.arange(n) * stride
        start = t.data_ptr() - base.data_ptr()
        return {start + int(i) * t.element_size() + k for i in at.flatten() for k in range(t.element_size())}

    views = [base[:, 2:5], base[:, 5:], base[:, 1], base.t()[3:6], base[::2, ::3], base[1::2, 1::3], base.flatten()[7:12],
             base[2:4, 4:5], half[:, ::2], half[:, 1::2], half[3:, 6:8], base.as_strided((3, 4), (5, 7), 2), base[0, 0]]
    for a, b in itertools.product(views, views):
        assert training._meet(a, b) == bool(touched(a) & touched(b)), (a.shape, a.stride(), b.shape, b.stride())
    with pytest.raises(ValueError, match="share"):
        training._check_apart([base[:, 2:5], base[:, 4:]])
    with pytest.raises(ValueError, match="share"):
        training._check_apart([base[:, :1].expand(6, 4)])
    training._check_apart([base[:, 2:5], base[:, 5:], base[:, :2].t(), base[:0]])


def test_forward_mode_is_refused():
    import torch.autograd.forward_ad as forward_ad
    with forward_ad.dual_level():
        w, x = forward_ad.make_dual(W, torch.ones_like(W)), forward_ad.make_dual(X, torch.ones_like(X))
        for call in (lambda: training.embedding(IDS, w), lambda: training.embedding_grad(IDS, x, 5),
                     lambda: training.linear_cross_entropy(x, W, IDS), lambda: training.linear_cross_entropy_grad(X, w, IDS),
                     lambda: training.gradient_norm([x, X]), lambda: training.clip_gradients_([x], 1.0, out=[X])):
            with pytest.raises(NotImplementedError, match="forward"):
                call()


def test_tracing_is_refused():
    from torch.fx.experimental.proxy_tensor import make_fx
    for call, arg in ((lambda w: training.embedding(IDS, w), W), (lambda x: training.embedding_grad(IDS, x, 5), X),
                      (lambda x: training.linear_cross_entropy(x, W, IDS), X),
                      (lambda x: training.linear_cross_entropy_grad(x, W, IDS)[:3], X),
                      (lambda x: training.linear_cross_entropy(x, W.clone().requires_grad_(), IDS), X),
                      (lambda x: training.gradient_norm([x]), X), (lambda x: training.clip_gradients_([x], 1.0), X)):
        with pytest.raises(NotImplementedError, match="trac"):
            torch.jit.trace(call, (arg,))
        with pytest.raises(NotImplementedError, match="trac"):
            make_fx(call)(arg)
    with pytest.raises(ValueError, match="GPU"):
        training.embedding(IDS, W)      # and afterwards it is as before


def test_lazily_negated_tensors_are_refused():
    w = torch._neg_view(W)
    with pytest.raises(ValueError, match="resolve_neg"):
        training.embedding(IDS, w)
    with pytest.raises(ValueError, match="resolve_neg"):
        training.clip_gradients_([w], 1.0)


def test_a_wrong_padding_idx_is_refused_without_gradients_too():
    for padding in (5, -6):
        with pytest.raises(ValueError, match="padding_idx"):
            training.embedding(IDS, W, padding_idx=padding)


@pytest.mark.parametrize("scale", [1e39, -1e39, float("inf"), float("nan")])
def test_scales_beyond_float32_are_refused(scale):
    with pytest.raises(ValueError, match="scale"):
        training.embedding(IDS, W, scale)
    with pytest.raises(ValueError, match="scale"):
        training.embedding_grad(IDS, X, 5, scale)


@pytest.mark.parametrize("norm_type", [1, 1.0, float("inf"), 0, "fro"])
def test_norms_other_than_the_second_are_refused(norm_type):
    p = torch.nn.Parameter(torch.ones(3))
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match="norm_type"):
        training.clip_grad_norm_([p], 1.0, norm_type)
    with pytest.raises(ValueError, match="norm_type"):
        training.clip_grad_norm_([p], 1.0, norm_type=norm_type)


def test_a_size_that_has_no_grid_is_refused_before_anything_is_written():
    # more slices of columns than a launch has along y
    assert _lib.lib().ds_embed_grad(4096, 8, 4096, 1 << 25, 4096, 4, 8, 1 << 25, -1, 1.0, 0, 4096, 1 << 62, None) == -5
    assert _lib.lib().ds_embed_grad(4096, 8, 4096, 1 << 30, 4096, 4, 8, 1 << 30, -1, 1.0, 1, 4096, 1 << 62, None) == -5
