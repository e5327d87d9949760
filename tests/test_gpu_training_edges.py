"""GPU: what deepshift_amd.training does at the edges of its definition.

Bounds are those of test_gpu_training.py, but for what each test says.
"""
import math

import pytest
import torch

from deepshift_amd import training
from tests.conftest import Tune
from tests.test_gpu_training import DEV, E, TINY, TYPES, U, _gen, _head, _head_check, _rand, _within

pytestmark = pytest.mark.gpu


def _softmax(h, w, b):
    """Logits, probabilities, and how far off float32 may have them, in 64 bits."""
    H, W = h.double(), w.double()
    s, size = H @ W.t(), H.abs() @ W.abs().t()
    if b is not None:
        s, size = s + b.double(), size + b.double().abs()
    d = ((h.shape[1] + 8) * E * size).amax(1, keepdim=True)
    p = s.softmax(1)
    return p, p * (2 * d + (4 * s.abs().amax(1, keepdim=True) + 16) * E)


def _own_rows(h, w, b, y, g, dh, roundings=2):
    """``dh`` against 64 bits, each row by the size of its own gradient ``g``."""
    dtype, V, g = h.dtype, w.shape[0], g.double()[:, None]
    p, off = _softmax(h, w, b)
    p = p.scatter_add(1, y[:, None], torch.full_like(g, -1.0))
    off = (off + p.abs() * roundings * U[dtype] + TINY[dtype] * 2.0 ** -14) * g.abs()
    W = w.double()
    want, off = (p * g) @ W, off @ W.abs()
    _within(dh, want, off + (V + 16) * E * ((p * g).abs() @ W.abs()) + (U[dtype] + 4 * E) * (want.abs() + off) + TINY[dtype], "dhidden")


def _backward(h, w, b, y, up, **kw):
    """Gradients of hidden, weight and bias under autograd."""
    leaves = [x.detach().requires_grad_() for x in (h, w) + (() if b is None else (b,))]
    loss = training.linear_cross_entropy(leaves[0], leaves[1], y, *leaves[2:], **kw)
    return torch.autograd.grad(loss, leaves, up)


# ---- gradients of rows ------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")], ids=str)
def test_a_rows_gradient_that_is_no_number_stays_in_its_row(dtype, bad):
    for T, D, V in [(6, 40, 200), (70, 48, 300), (20, 1024, 8200), (300, 64, 513)]:
        print(T, D, V, flush=True)
        g = _gen(T, D, V, 71)
        h, w, b, y = _head(T, D, V, dtype, True, g)
        up = _rand(g, T)
        up[3] = bad
        dh, dw, db = _backward(h, w, b, y, up, reduction="none")
        fine = torch.arange(T, device=DEV) != 3
        assert not dh[3].isfinite().any() and not dw.isfinite().any() and not db.isfinite().any()
        _own_rows(h[fine], w, b, y[fine], up[fine], dh[fine])
        # the only gradient that is not 0
        up = torch.where(fine, 0.0, up)
        dh, dw, db = _backward(h, w, b, y, up, reduction="none")
        assert not dh[3].isfinite().any() and (dh[fine] == 0).all()
        # of a token that does not count
        y[3], up[0] = -100, 0.5
        dh, dw, db = _backward(h, w, b, y, up, reduction="none")
        assert (dh[1:] == 0).all() and dw.isfinite().all() and db.isfinite().all()
        _own_rows(h[:1], w, b, y[:1], up[:1], dh[:1])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bad", [float("inf"), -float("inf"), float("nan")], ids=str)
def test_a_losss_gradient_that_is_no_number_leaves_tokens_that_do_not_count(dtype, bad):
    up = torch.tensor(bad, device=DEV)
    for T, D, V in [(6, 40, 200), (70, 48, 300), (20, 1024, 8200), (300, 64, 513)]:
        print(T, D, V, flush=True)
        g = _gen(T, D, V, 79)
        h, w, b, y = _head(T, D, V, dtype, True, g)
        y[2::5] = -100
        for reduction in ("sum", "mean"):
            dh, dw, db = _backward(h, w, b, y, up, reduction=reduction)
            assert (dh[2::5] == 0).all() and not dh[y != -100].isfinite().any()
            assert not dw.isfinite().any() and not db.isfinite().any()
            # nothing counts
            for grad in _backward(h, w, b, torch.full_like(y, -100), up, reduction=reduction):
                assert (grad == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_of_rows_far_apart_keep_their_bits(dtype):
    # many words and large weights: by 2^-26 of the largest gradient most probabilities are below 2^-39, and what a row of 2^-17
    # gets is inside float16 all the same
    for T, D, V, kb in [(70, 48, 20000, 1 << 20), (300, 200, 15000, 1 << 20), (40, 64, 20000, 200)]:
        print(T, D, V, kb, flush=True)
        g = _gen(T, D, V, 72)
        h, w = _rand(g, T, D, dtype=dtype, scale=0.125 / math.sqrt(D)), _rand(g, V, D, dtype=dtype, scale=16.0)
        b, y = _rand(g, V, dtype=dtype, scale=0.3), torch.randint(0, V, (T,), generator=g).to(DEV)
        up = 2.0 ** (torch.arange(T, device=DEV) * 26.0 / (T - 1) - 17.0) * (1 - 2 * (torch.arange(T, device=DEV) % 2))
        up[5] = 0
        for tile in (0, 1, 2, 3):
            with Tune(vocab_tile=tile, vocab_piece_kb=kb):
                dh, dw, db = _backward(h, w, b, y, up, reduction="none")
                again = _backward(h, w, b, y, up, reduction="none")
                leaf = h.detach().requires_grad_()
                only, = torch.autograd.grad(training.linear_cross_entropy(leaf, w, y, b, reduction="none"), leaf, up)
            _own_rows(h, w, b, y, up, dh)
            _own_rows(h, w, b, y, up, only)
            rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
            _head_check(h, w, b, y, -100, up, rows, dh, dw, db)
            assert all(torch.equal(x, z) for x, z in zip((dh, dw, db), again))


# ---- roundings --------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES[1:], ids=str)
def test_probabilities_are_rounded_once(dtype):
    # one token: a weight's gradient is one product, p rounded to the type times h, rounded to the type
    for D, V in [(64, 8192), (40, 20000)]:
        g = _gen(D, V, 73)
        h, w, b, y = _head(1, D, V, dtype, False, g)
        p, off = _softmax(h, w, None)
        p = p.scatter_add(1, y[:, None], torch.full((1, 1), -1.0, dtype=torch.float64, device=DEV))
        want = p.t() @ h.double()
        bound = (off + p.abs() * U[dtype] + TINY[dtype] * 2.0 ** -14).t() @ h.double().abs()
        bound = bound + (U[dtype] + 4 * E) * (want.abs() + bound) + TINY[dtype]
        for dw in (training.linear_cross_entropy_grad(h, w, y, reduction="sum")[2], _backward(h, w, None, y, None, reduction="sum")[1]):
            _within(dw, want, bound, "dweight")


# ---- infinities -------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_tokens_that_do_not_count_leave_nothing_whatever_weights_hold(dtype):
    for T, D, V in [(4, 40, 200), (70, 48, 300), (20, 1024, 8200), (300, 64, 513)]:
        print(T, D, V, flush=True)
        g = _gen(T, D, V, 77)
        h, w, b, y = _head(T, D, V, dtype, True, g)
        h[:, 1] = h[:, 1].abs() + 0.25
        y = y % 100
        y[2::5] = -100
        h[2::5] = float("nan")
        other = torch.arange(D, device=DEV) != 1    # there it is 0 times infinity
        for words in ([150], [100, 150, V - 1]):
            w[words, 1] = -float("inf")
            for up in (None, _rand(g, T)):
                dh, dw, db = _backward(h, w, b, y, up, reduction="mean" if up is None else "none")
                assert (dh[y == -100][:, other] == 0).all()
            _, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b)
            assert (dh[y == -100][:, other] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_an_infinite_weight_takes_a_word_out(dtype):
    for T, D, V, kb in [(4, 40, 200, 0), (20, 40, 200, 0), (70, 48, 300, 0), (150, 33, 700, 1), (300, 256, 515, 0), (20, 1024, 8200, 0),
                        (20, 1023, 8300, 0), (100, 1024, 8200, 0),
                        (20, 1023, 14500, 0)]:
        g = _gen(T, D, V, 74)
        h, w, b, y = _head(T, D, V, dtype, True, g)
        h[:, 1] = h[:, 1].abs().clamp(min=0.25)
        h[::3, 1], h[1::3, 1] = 1.0, 0.3      # with and without bits behind bfloat16's
        out = torch.tensor([0, V // 2, V - 1], device=DEV)
        y = 1 + y % (V // 2 - 1)
        y[2::5] = -100
        masked, bias = w.clone(), b.clone()
        masked[out, 1], bias[out] = 0.0, -float("inf")
        w[out, 1] = -float("inf")
        w[out[1], 2], masked[out[1], 2] = 0.3, 0.3
        other = torch.arange(D, device=DEV) != 1
        share = torch.full((T,), 1.0 / int((y != -100).sum()), device=DEV)
        for tile in (-1, 0, 1, 2, 3):
            print(T, D, V, tile, flush=True)
            tune = dict(vocab_tile=tile) if tile >= 0 else {}
            if kb:
                tune["vocab_piece_kb"] = kb
            with Tune(**tune):
                rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
                _, *step = training.linear_cross_entropy_grad(h, w, y, b)
                auto = _backward(h, w, b, y, None)
            for dh, dw, db in (step, auto):
                # 0 times infinity where the weight is, nothing else
                assert dh[y != -100][:, 1].isnan().all()
                dh = torch.where(other, dh, _masked_column(h, masked, bias, y, share, dtype))
                _head_check(h, masked, bias, y, -100, share, rows, dh, dw, db)


def _masked_column(h, w, b, y, share, dtype):
    """The definition's ``dhidden``, in place of a column that is not looked at."""
    s = torch.where((y != -100)[:, None], h, torch.zeros_like(h)).double() @ w.double().t() + b.double()
    p = s.softmax(1).scatter_add(1, y.clamp(min=0)[:, None], torch.full((len(y), 1), -1.0, dtype=torch.float64, device=DEV))
    return ((p * (share * (y != -100)).double()[:, None]) @ w.double()).to(dtype)


def test_float32_infinities_do_what_they_do_in_64_bits():
    # every path of float32, and every kind of product that an infinity may be in
    for T, D, V in [(5, 8, 20), (17, 8, 20), (40, 2048, 4200), (40, 2047, 4200), (40, 2047, 7200), (200, 40, 300)]:
        print(T, D, V, flush=True)
        g = _gen(T, D, V, 75)
        h, w, b, y = _head(T, D, V, torch.float32, False, g)
        y = y % 7
        h[0, 2], w[:, 2] = -float("inf"), w[:, 2].abs() + 0.1   # every logit of a token -inf
        h[1, 3] = float("inf")                                  # signs of both kinds
        w[V - 1, 4], h[:, 4] = float("inf"), -h[:, 4].abs() - 0.1   # a word taken out
        w[V - 2, 5], h[2, 5] = float("inf"), 0.0                # 0 times infinity
        h[3:, 5] = -0.5
        rows = training.linear_cross_entropy(h, w, y, reduction="none")
        s = h.double() @ w.double().t()
        assert s[2, V - 2].isnan() and s[0].isneginf().sum() >= V - 2
        assert rows[:3].isnan().all()
        s = s[3:, :V - 2]
        want = s.logsumexp(1) - s.gather(1, y[3:, None])[:, 0]
        size = (h[3:].abs().double() @ w[:V - 2].abs().double().t()).amax(1)
        _within(rows[3:], want, 2 * (D + 8) * E * size + (6 * size + 20) * E, "loss")


# ---- weights as they are -----------------------------------------------------------------------------------------

@pytest.mark.parametrize("T", [17, 64, 100, 127])
def test_weights_as_they_are_from_where_rows_that_begin_anywhere_take_them(T):
    # 7 * 2^21 weights and more, that come one float at a time, and on both sides of where planes take over
    for D, V, before, behind in [(1021, 14500, 0, 0), (1024, 14400, 1, 2), (2050, 7200, 2, 0), (1023, 14349, 0, 1), (1023, 14351, 0, 0),
                                 (31, 520000, 0, 0)]:
        print(T, D, V, before, behind, flush=True)
        g = _gen(T, D, V, 80)
        h, w, b, y = _head(T, D, V, torch.float32, True, g)
        y[0], y[1], y[2] = V - 1, 0, 128
        y[3::5] = -100
        wide = torch.full((V, before + D + behind), float("nan"), device=DEV)
        wide[:, before:before + D] = w
        wide = wide[:, before:before + D]
        share = torch.full((T,), 1.0 / int((y != -100).sum()), device=DEV)
        rows = training.linear_cross_entropy(h, wide, y, b, reduction="none")
        loss, dh, dw, db = training.linear_cross_entropy_grad(h, wide, y, b)
        _head_check(h, w, b, y, -100, share, rows, dh, dw, db)
        again = training.linear_cross_entropy_grad(h, wide, y, b)
        assert all(torch.equal(x, z) for x, z in zip((loss, dh, dw, db), again))


# ---- losses -----------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_a_loss_may_be_changed_in_place(reduction):
    g = _gen(76)
    h, w, b, y = _head(9, 16, 30, torch.float32, True, g)
    want = _backward(h, w, b, y, torch.full((9,) if reduction == "none" else (), 0.5, device=DEV), reduction=reduction)
    leaves = [x.detach().requires_grad_() for x in (h, w, b)]
    loss = training.linear_cross_entropy(leaves[0], leaves[1], y, leaves[2], reduction=reduction)
    assert loss._base is None
    before = loss.detach().clone()
    loss /= 2
    loss += 3.0
    assert torch.equal(loss, before / 2 + 3.0)
    loss.sum().backward()
    assert all(torch.equal(x.grad, z) for x, z in zip(leaves, want))
    for loss in (training.linear_cross_entropy(h, w, y, b, reduction=reduction),
                 training.linear_cross_entropy_grad(h, w, y, b, reduction=reduction)[0]):
        assert loss._base is None and loss.shape == before.shape
        before = loss.clone()
        loss *= 2
        assert torch.equal(loss, before * 2)


# ---- what is recorded -------------------------------------------------------------------------------------------

def test_forward_mode_is_refused_on_the_gpu():
    import torch.autograd.forward_ad as forward_ad
    g = _gen(78)
    h, w, b, y = _head(9, 16, 30, torch.float32, True, g)
    leaf = w.clone().requires_grad_()
    with forward_ad.dual_level():
        dual = {k: forward_ad.make_dual(t, torch.ones_like(t)) for k, t in dict(h=h, w=w, b=b).items()}
        for call in (lambda: training.embedding(y, dual["w"]), lambda: training.embedding_grad(y, dual["h"], 30),
                     lambda: training.linear_cross_entropy(dual["h"], w, y, b), lambda: training.linear_cross_entropy(h, dual["w"], y, b),
                     lambda: training.linear_cross_entropy(h, leaf, y, dual["b"]), lambda: training.gradient_norm([h, dual["w"]]),
                     lambda: training.clip_gradients_([h.clone()], 1.0, out=[dual["h"]])):
            with pytest.raises(NotImplementedError, match="forward"):
                call()


# ---- tensors that overlap -----------------------------------------------------------------------------------------

def test_clipping_refuses_to_write_what_another_tensor_reads():
    a, b = torch.ones(1000, device=DEV), torch.ones(1000, device=DEV)
    flat, wide = torch.ones(3000, device=DEV), torch.ones(40, 30, device=DEV)
    half = flat.view(torch.bfloat16)
    for grads, out in (([a, b], [b, a]), ([a], [a.view(torch.bfloat16)[:1000]]), ([flat[:1000]], [flat[1:1001]]),
                       ([flat[1:1001]], [flat[:1000]]), ([flat[:1000], flat[500:600]], [a, flat[550:650]]),
                       ([flat[:1000], flat[2000:3000]], [flat[2999:3000].expand(1000), a]), ([a, a], [a, b]), ([a, b], [a, a]),
                       ([half[:1000]], [flat[:1000]]), ([a, b, flat[:1]], [flat[:1000], flat[1000:2000], b[:1]]),
                       # however they lie
                       ([wide[:, :20], wide[:, 19:]], None), ([wide[:, :20], wide[:, :20]], None),
                       ([wide[:, :7], wide.t()[3:9]], None), ([wide[:, :1].expand(40, 30)], None),
                       ([a[:40], a[40:80]], [wide[:, 3], wide[:, 3]])):
        before = [t.clone() for t in grads + (out or [])]
        with pytest.raises(ValueError, match="memory"):
            training.clip_gradients_(grads, 1.0, out=out)
        assert all(torch.equal(t, was) for t, was in zip(grads + (out or []), before))


def test_clipping_takes_tensors_that_lie_beside_each_other():
    g = _gen(81)
    for make in (lambda f, w: ([f[:1000], f[1000:1010]], [f[:1000], f[1010:1020]]),       # one in place, one to its neighbour
                 lambda f, w: ([f[:10], f[:10], f[5:15]], [f[20:30], f[30:40], f[40:50]]),  # sources may overlap
                 lambda f, w: ([w[:, :20], w[:, 20:]], None), lambda f, w: ([w[::2], w[1::2]], None),
                 lambda f, w: ([w[:, :20], f[:800]], [w[:, 10:], f[800:1600]])):           # copied before anything is written
        flat, wide = _rand(g, 3000), _rand(g, 40, 30)
        grads, out = make(flat, wide)
        before = [t.double().clone() for t in grads]
        norm = torch.stack([t.norm() for t in before]).norm()
        got = training.clip_gradients_(grads, 0.5, out=out)
        assert abs(got.double() - norm) <= E * norm
        for t, was in zip(grads if out is None else out, before):
            want = was * (0.5 / (norm + 1e-6))
            assert ((t.double() - want).abs() <= 4 * E * want.abs()).all()
