"""GPU: the distillation of a linear head (deepshift_amd.training.linear_distillation) against its definition in 64 bits.

Bounds are derived, not tuned.  With u the rounding of the operands' type (2^-24, 2^-8, 2^-11), e = 2^-23 and c the temperature:

* a student's logit over c is off by d = ((D + 8) e (sum |h w| + |b|)) / c + 2 e |s|: a product of D terms, a factor, a sum;
* its logarithm of the sum of exponentials by the largest d of the row and (6 m + 20) e, m the row's largest |s|;
* a teacher's probability q of a word x below its best by q (2 |x| + K + 16) e: an exponential of a rounded argument over a sum;
* a loss is a sum of K terms q (log q - log p) in 32 bits; the gradient p - q is off by what both are, and where it goes into a
  product by one more rounding to the operands' type; a product by the sum of these times the other operand and the additions'
  n e, and the output's rounding.
"""
import math

import pytest
import torch

from deepshift_amd import training
from tests.conftest import Tune

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def _gen(*key):
    return torch.Generator().manual_seed(hash(key) & 0x7fffffff)


def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g times the bound" % (
        what, int(bad.sum()), bad.numel(), float((off / bound.clamp(min=1e-300)).nan_to_num(float("inf")).max()))


def _case(T, D, V, K, dtype, bias, *key, spread=2.0):
    g = _gen(T, D, V, K, *key)
    h, w = _rand(g, T, D, dtype=dtype), _rand(g, V, D, dtype=dtype, scale=spread / math.sqrt(max(D, 1)))
    b = _rand(g, V, dtype=dtype, scale=0.3) if bias else None
    # words of all parts of the vocabulary, in any order, without repetitions where there are enough
    ids = torch.rand(T, max(V, K), generator=g).argsort(1)[:, :K] % V
    logits = torch.randn(T, K, generator=g) * 3
    if T > 3:
        ids[1::5, K // 2:] = -1     # some have fewer, some none
        ids[2::7] = -7
    return h, w, b, ids.to(DEV), logits.to(DEV)


def _teacher(ids, logits, V, c):
    """Probabilities [T, V] of each word, how far off they may be, and sum of q log q and its bound, in 64 bits."""
    T, K = ids.shape
    there = (ids >= 0) & (logits > -math.inf)
    x = torch.where(there, logits.double() / c, -math.inf)
    top = torch.where(there.any(1), x.amax(1), 0.0)
    e = (x - top[:, None]).exp()
    q = e / e.sum(1, keepdim=True).clamp(min=1e-300)
    below = torch.where(there, top[:, None] - x, 0.0)
    off = q * (2 * below + K + 16) * E
    at = ids.clamp(min=0)
    whole = torch.zeros(T, V, dtype=torch.float64, device=DEV)
    whole_off = torch.zeros_like(whole)
    whole.scatter_add_(1, at, q)
    whole_off.scatter_add_(1, at, off)
    logq = torch.where(q > 0, q.clamp(min=1e-300).log(), 0.0)
    return there.any(1), at, q, off, logq, whole, whole_off


def _check(h, w, b, ids, logits, c, share, losses, dh=None, dw=None, db=None):
    """``share`` [T]: the gradient of each row's loss."""
    dtype, (T, D), V, K = h.dtype, h.shape, w.shape[0], ids.shape[1]
    kept, at, q, q_off, logq, whole, whole_off = _teacher(ids, logits, V, c)
    H, W = h.double(), w.double()
    H[~kept] = 0    # tokens that do not count leave nothing
    s, size = H @ W.t().contiguous(), H.abs() @ W.abs().t().contiguous()
    if b is not None:
        s, size = s + b.double(), size + b.double().abs()
    s, size = s / c, size / c
    finite = s.isfinite()
    d = torch.where(finite, (D + 8) * E * size + 2 * E * s.abs(), 0.0)
    row_d = d.amax(1, keepdim=True)
    most = torch.where(finite, s.abs(), 0.0).amax(1, keepdim=True)
    lse = s.logsumexp(1, keepdim=True)
    logp = s.gather(1, at) - lse
    terms = torch.where(q > 0, q * (logq - logp), 0.0)
    want = torch.where(kept, terms.sum(1), 0.0) * c * c
    off = torch.where(q > 0, q_off * (logq.abs() + logp.abs() + 1) + q * (d.gather(1, at) + row_d + (6 * most + 20 + 4 * logq.abs()) * E), 0.0)
    bound = (off.sum(1) + (K + 8) * E * terms.abs().sum(1)) * c * c * kept
    _within(losses, want, bound + 1e-300, "loss")
    if dh is None:
        return want, bound
    p = (s - lse).exp()
    g = (share.double() * kept)[:, None] * c
    soft = p * (2 * row_d + (4 * most + 16) * E) + whole_off + E * (p + whole)
    P = (p - whole) * g
    G = (soft + (p - whole).abs() * 2 * U[dtype]) * g.abs() + TINY[dtype] * 2.0 ** -14 * g.abs().max()
    u, tiny = U[dtype], TINY[dtype]
    for name, got, left, right, n in (("dhidden", dh, P, W, V), ("dweight", dw, P.t().contiguous(), H, T)):
        size = left.abs() @ right.abs()
        off = (G if name == "dhidden" else G.t().contiguous()) @ right.abs()
        exact = left @ right
        _within(got, exact, off + (n + 16) * E * size + (u + 4 * E) * (exact.abs() + off) + tiny, name)
    if db is not None:
        exact = P.sum(0)
        _within(db, exact, (soft * g.abs()).sum(0) + (T + 8) * E * P.abs().sum(0) + u * exact.abs() * 1.01 + tiny, "dbias")
    return want, bound


SHAPES = [(1, 1, 1, 1), (1, 8, 2, 2), (3, 5, 7, 3), (64, 512, 10, 4), (2, 64, 1000, 10), (65, 64, 1000, 33), (130, 100, 257, 64),
          (16, 1000, 513, 65), (257, 136, 300, 5), (300, 256, 515, 100), (513, 96, 129, 16), (33, 2056, 777, 20), (20, 64, 2000, 1024)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tile", [None, 0, 1, 2, 3])
def test_losses_and_gradients(dtype, tile):
    for i, (T, D, V, K) in enumerate(SHAPES):
        print(T, D, V, K, flush=True)
        h, w, b, ids, logits = _case(T, D, V, K, dtype, i % 2 == 0)
        logits = logits.to(TYPES[i % 3])
        c = [1.0, 2.0, 0.7][i % 3]
        n = max(1, int((ids >= 0).any(1).sum()))
        with Tune(vocab_tile=tile):
            rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
            loss, dh, dw, db = training.linear_distillation_grad(h, w, ids, logits, b, c)
            again = training.linear_distillation_grad(h, w, ids.int(), logits, b, c)
        want, bound = _check(h, w, b, ids, logits, c, torch.full((T,), 1.0 / n, device=DEV), rows, dh, dw, db)
        assert abs(loss.double() - want.sum() / n) <= (bound.sum() + 4 * E * want.abs().sum()) / n + 1e-300
        assert torch.equal(loss, again[0]) and torch.equal(dh, again[1]) and torch.equal(dw, again[2])
        assert (db is None) == (b is None) and (db is None or torch.equal(db, again[3]))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_pieces_of_the_vocabulary_and_stretches(dtype):
    for T, D, V, K in [(100, 72, 1000, 40), (33, 100, 777, 7), (260, 64, 513, 20), (8, 24, 768, 100)]:
        h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 3)
        ids[0, 0], ids[-1, 0] = V - 1, 0
        ones = torch.ones(T, device=DEV)
        for tune in (dict(vocab_piece_kb=1), dict(vocab_piece_kb=1, vocab_split=3), dict(vocab_split=5), dict(vocab_split=1)):
            for tile in (0, 1, 2, 3):
                print(T, D, V, tune, tile, flush=True)
                with Tune(vocab_tile=tile, **tune):
                    rows = training.linear_distillation(h, w, ids, logits, b, 1.5, "none")
                    loss, dh, dw, db = training.linear_distillation_grad(h, w, ids, logits, b, 1.5, "sum")
                    got = _autograd(h, w, ids, logits, b, 1.5, "sum")
                _check(h, w, b, ids, logits, 1.5, ones, rows, dh, dw, db)
                _check(h, w, b, ids, logits, 1.5, ones, rows, *got[1:])


@pytest.mark.parametrize("T", [1, 8, 16, 17, 100])
def test_few_tokens_of_large_float32_weights(T):
    # weights as they are, four floats at a time and one, and in planes
    for D, V in ((1024, 8200), (1023, 16000), (64, 500)):
        h, w, b, ids, logits = _case(T, D, V, 12, torch.float32, True, 4)
        n = max(1, int((ids >= 0).any(1).sum()))
        rows = training.linear_distillation(h, w, ids, logits, b, 2.0, "none")
        loss, dh, dw, db = training.linear_distillation_grad(h, w, ids, logits, b, 2.0)
        _check(h, w, b, ids, logits, 2.0, torch.full((T,), 1.0 / n, device=DEV), rows, dh, dw, db)
        got = _autograd(h, w, ids, logits, b, 2.0, "mean")
        _check(h, w, b, ids, logits, 2.0, torch.full((T,), 1.0 / n, device=DEV), rows, *got[1:])


def _autograd(h, w, ids, logits, b, c, reduction, grad=None):
    leaves = [t.detach().requires_grad_() for t in (h, w, b) if t is not None]
    loss = training.linear_distillation(leaves[0], leaves[1], ids, logits, leaves[2] if b is not None else None, c, reduction)
    return [loss.detach()] + list(torch.autograd.grad(loss, leaves, grad))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_under_autograd(dtype, reduction):
    T, D, V, K = 90, 48, 300, 17
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 5)
    n = int((ids >= 0).any(1).sum())
    g = _gen(6)
    grad = _rand(g, T) if reduction == "none" else torch.tensor(0.37, device=DEV)
    share = grad if reduction == "none" else grad.expand(T) / (n if reduction == "mean" else 1)
    got = _autograd(h, w, ids, logits, b, 3.0, reduction, grad)
    rows = training.linear_distillation(h, w, ids, logits, b, 3.0, "none")
    want, bound = _check(h, w, b, ids, logits, 3.0, share, rows, *got[1:])
    # any number of leading axes, and one operand alone
    shaped = _autograd(h.view(9, 10, D), w, ids.view(9, 10, K), logits.view(9, 10, K), b, 3.0, reduction,
                       grad.view(9, 10) if reduction == "none" else grad)
    assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(shaped, got))
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == k) for k, t in enumerate((h, w, b))]
        loss = training.linear_distillation(leaves[0], leaves[1], ids, logits, leaves[2], 3.0, reduction)
        alone, = torch.autograd.grad(loss, leaves[i], grad)
        assert torch.equal(alone, got[1 + i])
    # the one call for all may take other tiles, so that its sums add up in another order
    for loss in (got[0], training.linear_distillation_grad(h, w, ids, logits, b, 3.0, reduction)[0]):
        if reduction == "none":
            _within(loss, want, bound + 1e-300, "loss")
        else:
            m = n if reduction == "mean" else 1
            assert abs(loss.double() - want.sum() / m) <= (bound.sum() + 4 * E * want.abs().sum()) / m


def test_words_in_two_places_and_in_any_order():
    T, D, V, K = 40, 32, 600, 24
    h, w, b, ids, logits = _case(T, D, V, K, torch.float32, True, 7)
    ids[0] = 5                       # all of it on one word
    ids[3, ::2] = ids[3, 1::2]
    ones = torch.ones(T, device=DEV)
    rows = training.linear_distillation(h, w, ids, logits, b, reduction="none")
    step = training.linear_distillation_grad(h, w, ids, logits, b, reduction="sum")
    _check(h, w, b, ids, logits, 1.0, ones, rows, *step[1:])
    order = torch.rand(T, K, generator=_gen(8)).argsort(1).to(DEV)
    mixed = training.linear_distillation(h, w, ids.gather(1, order), logits.gather(1, order), b, reduction="none")
    _, bound = _check(h, w, b, ids, logits, 1.0, ones, rows)
    assert ((mixed - rows).abs() <= 2 * bound).all()
    # a teacher with one word is a target
    one = ids[:, :1].clone()
    one[one < 0] = -100
    want = training.linear_cross_entropy(h, w, one[:, 0], b, reduction="none")
    got = training.linear_distillation(h, w, one, logits[:, :1], b, reduction="none")
    assert torch.allclose(got, want, rtol=1e-5, atol=1e-5)
    p, q = training.linear_distillation_grad(h, w, one, logits[:, :1], b)[1:], training.linear_cross_entropy_grad(h, w, one[:, 0], b)[1:]
    assert all(torch.allclose(a, c, rtol=1e-4, atol=1e-7) for a, c in zip(p, q))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_places_without_words_and_tokens_that_do_not_count(dtype):
    T, D, V, K = 50, 40, 400, 9
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 9)
    ids[2::7] = -1
    kept = (ids >= 0).any(1)
    n = int(kept.sum())
    want = training.linear_distillation_grad(h, w, ids, logits, b)
    # a place is empty by its number or by its logit, whatever the other is
    same = logits.clone()
    same[ids < 0] = float("nan")
    assert all(torch.equal(p, q) for p, q in zip(training.linear_distillation_grad(h, w, ids, same, b), want))
    by_logit, numbers = logits.clone(), ids.clone()
    by_logit[ids < 0] = -float("inf")
    numbers[ids < 0] = 3
    assert all(torch.equal(p, q) for p, q in zip(training.linear_distillation_grad(h, w, numbers, by_logit, b), want))
    numbers[ids < 0] = 2 ** 40
    assert all(torch.equal(p, q) for p, q in zip(training.linear_distillation_grad(h, w, numbers, by_logit, b), want))
    # tokens that do not count may hold anything
    for bad in (float("nan"), float("inf")):
        wild = h.clone()
        wild[~kept] = bad
        for reduction in ("mean", "sum", "none"):
            p = training.linear_distillation_grad(wild, w, ids, logits, b, reduction=reduction)
            q = training.linear_distillation_grad(h, w, ids, logits, b, reduction=reduction)
            assert all(torch.equal(x, y) for x, y in zip(p, q))
            p, q = _autograd(wild, w, ids, logits, b, 1.0, reduction, torch.ones(T, device=DEV) if reduction == "none" else None), \
                _autograd(h, w, ids, logits, b, 1.0, reduction, torch.ones(T, device=DEV) if reduction == "none" else None)
            assert all(torch.equal(x, y) for x, y in zip(p, q))
    assert n < T and (want[1][~kept] == 0).all()
    # none counts
    for reduction in ("mean", "sum", "none"):
        got = training.linear_distillation_grad(h, w, torch.full_like(ids, -1), logits, b, reduction=reduction)
        assert all((t == 0).all() for t in got)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_empty_places_in_front(dtype):
    for T, K in ((60, 9), (60, 300), (1100, 9)):
        h, w, b, ids, logits = _case(T, 40, 400, K, dtype, True, 24)
        ids = torch.randint(0, 400, (T, K), generator=_gen(25, K)).to(DEV)
        ids[::2, :K - 1], logits[1::4, :K - 2] = -1, -float("inf")
        ids[3::8] = -1
        n = int(((ids >= 0) & (logits > -float("inf"))).any(1).sum())
        rows = training.linear_distillation(h, w, ids, logits, b, 2.0, "none")
        step = training.linear_distillation_grad(h, w, ids, logits, b, 2.0)
        assert n < T
        _check(h, w, b, ids, logits, 2.0, torch.full((T,), 1.0 / n, device=DEV), rows, *step[1:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_what_is_no_number_or_no_word_stays_in_its_token(dtype):
    T, D, V, K = 30, 40, 300, 6
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 10)
    ids[:] = ids.abs() % V
    want = training.linear_distillation_grad(h, w, ids, logits, b, reduction="none")
    others = [i for i in range(T) if i != 4]
    wrong = []
    for value in (V, 2 ** 40):
        numbers = ids.clone()
        numbers[4, 2] = value
        wrong.append((h, numbers, logits))
    for value in (float("nan"), float("inf")):
        values = logits.clone()
        values[4, 2] = value
        wrong.append((h, ids, values))
    hidden = h.clone()
    hidden[4, 3] = float("nan")
    wrong.append((hidden, ids, logits))
    for hidden, numbers, values in wrong:
        got = training.linear_distillation_grad(hidden, w, numbers, values, b, reduction="none")
        assert torch.equal(got[0][others], want[0][others]) and got[0][4].isnan()
        assert torch.equal(got[1][others], want[1][others]) and got[1][4].isnan().all()
        assert training.linear_distillation(hidden, w, numbers, values, b).isnan()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_words_taken_out_and_large_logits(dtype):
    T, D, V, K = 40, 64, 500, 8
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 11)
    ids[:] = ids.abs() % (V // 2)
    b[V // 2:] = -float("inf")        # words nobody teaches
    ones = torch.ones(T, device=DEV)
    rows = training.linear_distillation(h, w, ids, logits, b, 2.0, "none")
    step = training.linear_distillation_grad(h, w, ids, logits, b, 2.0, "sum")
    kept = _check(h, w, b, ids, logits, 2.0, ones, rows, *step[1:])
    assert kept[0].isfinite().all()
    # a taught one: the loss is infinite, the gradient is not
    ids[7, 1] = V - 1
    rows = training.linear_distillation(h, w, ids, logits, b, 2.0, "none")
    assert rows[7] == float("inf") and rows[:7].isfinite().all() and rows[8:].isfinite().all()
    assert all(t.isfinite().all() for t in training.linear_distillation_grad(h, w, ids, logits, b, 2.0, "sum")[1:])
    # far apart, on both sides
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 12, spread=60.0)
    logits = logits * 30
    for c in (1.0, 8.0):
        rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
        step = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
        _check(h, w, b, ids, logits, c, ones, rows, *step[1:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(dtype):
    T, D, V, K = 60, 64, 300, 10
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 13)
    g = _gen(14)
    wide_h, wide_w = _rand(g, T, D + 5, dtype=dtype), _rand(g, V, 2 * D, dtype=dtype, scale=0.2)
    wide_ids, wide_logits = torch.stack([ids, ids], 2), torch.cat([logits, logits], 1)
    ones = torch.ones(T, device=DEV)
    for h2, w2, i2, l2 in ((wide_h[:, :D], wide_w[:, 3:D + 3], wide_ids[..., 1], wide_logits[:, K:]),
                           (h.t().contiguous().t(), w.t().contiguous().t(), ids.t().contiguous().t(), logits.t().contiguous().t()),
                           (h[:1].expand(T, D), w[:1].expand(V, D), ids[:1].expand(T, K), logits[:1].expand(T, K))):
        rows = training.linear_distillation(h2, w2, i2, l2, b, reduction="none")
        step = training.linear_distillation_grad(h2, w2, i2, l2, b, reduction="sum")
        _check(h2, w2, b, i2, l2, 1.0, ones, rows, *step[1:])
    one = training.linear_distillation(h[0], w, ids[0], logits[0], b, reduction="none")
    assert one.shape == () and torch.equal(one, training.linear_distillation(h[:1], w, ids[:1], logits[:1], b, reduction="none")[0])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_words_of_one_tile(dtype):
    # more of them than a tile keeps at hand, neighbours and the same ones again, and more than there are
    T, D, V = 40, 48, 700
    for K, low, high in ((40, 100, 160), (9, 250, 262), (64, 640, 700), (50, 0, 7)):
        h, w, b, _, logits = _case(T, D, V, K, dtype, True, 20)
        ids = torch.randint(low, high, (T, K), generator=_gen(21, K)).to(DEV)
        ids[5] = -1
        ones = torch.ones(T, device=DEV)
        for tune in (dict(), dict(vocab_piece_kb=1)):
            for tile in (None, 0, 1, 2, 3):
                with Tune(vocab_tile=tile, **tune):
                    rows = training.linear_distillation(h, w, ids, logits, b, 1.3, "none")
                    step = training.linear_distillation_grad(h, w, ids, logits, b, 1.3, "sum")
                    got = _autograd(h, w, ids, logits, b, 1.3, "sum")
                _check(h, w, b, ids, logits, 1.3, ones, rows, *step[1:])
                _check(h, w, b, ids, logits, 1.3, ones, rows, *got[1:])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_temperatures_at_both_ends(dtype):
    T, D, V, K = 30, 40, 300, 8
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 22)
    ones = torch.ones(T, device=DEV)
    for c in (2.0 ** 20, 1000.0, 0.03, 2.0 ** -20):
        rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
        step = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
        # float16 ends at 65504, and gradients are 2^20 (p - q) w there
        beyond = c > 1e6 and dtype == torch.float16
        assert not any(t.isnan().any() for t in step) and (beyond or all(t.isfinite().all() for t in step))
        _check(h, w, b, ids, logits, c, ones, rows, *(() if beyond else step[1:]))


@pytest.mark.parametrize("T", [3, 64, 65, 500, 1300])
def test_words_that_most_tokens_teach(T):
    # bfloat16: what P loses by its rounding is kept for them, 2^-16 of it is left
    dtype, D, V, K, c = torch.bfloat16, 72, 9001, 12, 1.4
    h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 26)
    ids = torch.randint(0, V, (T, K), generator=_gen(27)).to(DEV)
    often = torch.tensor([8999, 4321, 300], device=DEV)
    ids[:, :3], logits[:, :3] = often, logits[:, :3] + torch.tensor([6.0, 5.5, 5.0], device=DEV)
    ones = torch.ones(T, device=DEV)
    for tune in (dict(), dict(vocab_piece_kb=max(1, T * 4)), dict(vocab_split=3)):
        for tile in (None, 0, 1, 2, 3):
            with Tune(vocab_tile=tile, **tune):
                rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
                step = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
                got = _autograd(h, w, ids, logits, b, c, "sum")
            for dh, dw, db in (step[1:], got[1:]):
                _check(h, w, b, ids, logits, c, ones, rows, dh, dw, db)
                _, _, _, _, _, whole, whole_off = _teacher(ids, logits, V, c)
                H = h.double()
                s = (H @ w.double().t().contiguous() + b.double()) / c
                size = (H.abs() @ w.double().abs().t().contiguous() + b.double().abs()) / c
                d = ((D + 8) * E * size + 2 * E * s.abs()).amax(1, keepdim=True)
                p = s.softmax(1)
                P = ((p - whole) * c)[:, often].t().contiguous()
                soft = (p * (2 * d + (4 * s.abs().amax(1, keepdim=True) + 16) * E) + whole_off + E * (p + whole)) * c
                off = soft[:, often].t().contiguous() + P.abs() * 2.0 ** -15
                exact = P @ H
                bound = off @ H.abs() + (2 * T + 16) * E * (P.abs() @ H.abs()) + 1.01 * U[dtype] * exact.abs()
                _within(dw[often], exact, bound, "dweight of frequent words")
            again = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum") if not tune and tile is None else step
            assert all(torch.equal(x, y) for x, y in zip(again, step))


def test_many_tokens():
    # more of them than a launch's second axis has workgroups for, too
    for dtype, T in [(dtype, 70001) for dtype in TYPES] + [(torch.bfloat16, 530001), (torch.float32, 530001)]:
        D, V, K = 16, 50, 3
        h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 23)
        n = int((ids >= 0).any(1).sum())
        rows = training.linear_distillation(h, w, ids, logits, b, 2.0, "none")
        step = training.linear_distillation_grad(h, w, ids, logits, b, 2.0)
        want, bound = _check(h, w, b, ids, logits, 2.0, torch.full((T,), 1.0 / n, device=DEV), rows, *step[1:])
        assert abs(step[0].double() - want.sum() / n) <= (bound.sum() + 4 * E * want.abs().sum()) / n


def test_gradients_against_differences():
    T, D, V, K, c = 20, 16, 50, 6, 1.7
    h, w, b, ids, logits = _case(T, D, V, K, torch.float32, True, 15)
    got = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")[1:]
    kept, _, q, _, logq, whole, _ = _teacher(ids, logits, V, c)

    def value(h, w, b):
        logp = ((h @ w.t().contiguous() + b) / c).log_softmax(1)
        return c * c * ((q * logq).sum() - (whole * logp).sum())

    g = _gen(16)
    operands = [t.double() for t in (h, w, b)]
    for i in range(3):
        way = torch.randn(operands[i].shape, generator=g, dtype=torch.float64).to(DEV)
        step = 1e-3
        ends = [value(*[t + s * step * way if k == i else t for k, t in enumerate(operands)]) for s in (1, -1, 2, -2)]
        slope = (8 * (ends[0] - ends[1]) - (ends[2] - ends[3])) / (12 * step)
        along = (got[i].double() * way).sum()
        # float32: some hundred roundings of the terms' size; the differences: step^4 of the fifth derivative
        assert abs(along - slope) <= 300 * E * (got[i].double().abs() * way.abs()).sum() + 1e-7 * abs(slope) + 1e-7


def test_no_tokens_and_no_features():
    V, K = 7, 3
    for T, D in ((0, 8), (5, 0), (0, 0)):
        h, w, b = [torch.randn(*s, device=DEV, requires_grad=True) for s in ((T, D), (V, D), (V,))]
        ids, logits = torch.randint(0, V, (T, K), device=DEV), torch.randn(T, K, device=DEV)
        loss = training.linear_distillation(h, w, ids, logits, b)
        dh, dw, db = torch.autograd.grad(loss, (h, w, b))
        assert dh.shape == h.shape and (dw == 0).all() and dw.shape == w.shape and db.isfinite().all()
        if T:
            rows = training.linear_distillation(h, w, ids, logits, b, reduction="none").detach()
            want, bound = _check(h.detach(), w.detach(), b.detach(), ids, logits, 1.0, None, rows)
        else:
            assert loss == 0 and (db == 0).all()


def test_offsets_beyond_32_bits():
    # weights of 2.2 G elements; what is taught lies at their end
    T, D, V, K = 70, 4096, 540000, 3
    g = _gen(17)
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=DEV)
    w[-300:] = _rand(g, 300, D, dtype=torch.bfloat16, scale=1 / 64)
    h = _rand(g, T, D, dtype=torch.bfloat16)
    ids = torch.randint(V - 300, V, (T, K), generator=g).to(DEV)
    logits = _rand(g, T, K)
    loss, dh, dw, _ = training.linear_distillation_grad(h, w, ids, logits, reduction="sum")
    # all other words have a logit of 0: a bias of one word that has all their exponentials stands for them
    some = torch.cat([torch.zeros(1, D, dtype=torch.float64, device=DEV), w[-300:].double()])
    s = h.double() @ some.t().contiguous()
    s[:, 0] = math.log(V - 300)
    p, q = s.softmax(1), torch.zeros(T, 301, dtype=torch.float64, device=DEV)
    q.scatter_add_(1, ids - (V - 301), logits.double().softmax(1))
    P = (p - q)[:, 1:]
    exact = P.t().contiguous() @ h.double()
    bound = (P.abs() * 2.5 * U[torch.bfloat16] + 1e-7).t().contiguous() @ h.double().abs() + 2 * U[torch.bfloat16] * exact.abs()
    _within(dw[-300:], exact, bound, "dweight")
    exact = P @ some[1:]
    bound = (P.abs() * 2.5 * U[torch.bfloat16] + 1e-7) @ some[1:].abs() + 2 * U[torch.bfloat16] * exact.abs()
    _within(dh, exact, bound, "dhidden")


def test_another_stream_and_captured_replays():
    for dtype in (torch.float32, torch.bfloat16):
        T, D, V, K = 100, 64, 500, 12
        h, w, b, ids, logits = _case(T, D, V, K, dtype, True, 18)
        want = training.linear_distillation_grad(h, w, ids, logits, b, 2.0)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = training.linear_distillation_grad(h, w, ids, logits, b, 2.0)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = training.linear_distillation_grad(h, w, ids, logits, b, 2.0)
        with torch.cuda.graph(other, pool=graph.pool()):
            backward = _autograd(h, w, ids, logits, b, 3.0, "mean")
        for i in range(3):
            h.copy_(_rand(_gen(i), T, D, dtype=dtype))
            ids.copy_(torch.randint(-1, V, (T, K), generator=_gen(i)))
            for replay, results, call in ((graph, captured, lambda: training.linear_distillation_grad(h, w, ids, logits, b, 2.0)),
                                          (other, backward, lambda: _autograd(h, w, ids, logits, b, 3.0, "mean")),
                                          (graph, captured, lambda: training.linear_distillation_grad(h, w, ids, logits, b, 2.0))):
                replay.replay()
                torch.cuda.synchronize()
                assert all(torch.equal(p, q) for p, q in zip(results, call())), "replay %d" % i


def test_two_streams_at_once():
    for dtype in TYPES:
        cases = [_case(90, 64, 5000, 12, dtype, True, 28, i) for i in range(2)]
        want = [training.linear_distillation_grad(h, w, ids, logits, b, 2.0) for h, w, b, ids, logits in cases]
        streams = [torch.cuda.Stream() for _ in cases]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for _ in range(10):
            for (h, w, b, ids, logits), s, results in zip(cases, streams, got):
                with torch.cuda.stream(s):
                    results.append(training.linear_distillation_grad(h, w, ids, logits, b, 2.0))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for results, first in zip(got, want) for one in results for p, q in zip(one, first))


def test_the_heads_module():
    torch.manual_seed(0)
    head = training.LinearCrossEntropy(48, 200).to(DEV)
    h = torch.randn(30, 48, device=DEV, requires_grad=True)
    best = torch.randn(30, 200, device=DEV).topk(9, 1)
    loss = head.distill(h, best.indices, best.values, temperature=2.0)
    want = training.linear_distillation(h.detach(), head.weight.detach(), best.indices, best.values, head.bias.detach(), 2.0)
    assert torch.equal(loss, want)
    (0.5 * loss + 0.5 * head(h, best.indices[:, 0])).backward()
    assert h.grad.isfinite().all() and head.weight.grad.isfinite().all() and head.bias.grad.abs().max() > 0


def test_refusals_on_the_gpu():
    T, D, V, K = 4, 8, 20, 3
    h, w, b, ids, logits = _case(T, D, V, K, torch.float32, True, 19)
    f = training.linear_distillation
    for error, call in ((ValueError, lambda: f(h, w, ids[:, :0], logits[:, :0], b)), (ValueError, lambda: f(h, w, ids[:, 0], logits[:, 0], b)),
                        (ValueError, lambda: f(h, w, ids, logits[:, :2], b)), (TypeError, lambda: f(h, w, ids.float(), logits, b)),
                        (TypeError, lambda: f(h, w, ids, logits.double(), b)), (TypeError, lambda: f(h, w.half(), ids, logits, b)),
                        (ValueError, lambda: f(h, w, ids.cpu(), logits, b)), (ValueError, lambda: f(h, w, ids, logits.cpu(), b)),
                        (ValueError, lambda: f(h, w, ids, logits, b[:5])), (ValueError, lambda: f(h, w, ids, logits, b, 0.0)),
                        (ValueError, lambda: f(h, w, ids, logits, b, float("nan"))), (ValueError, lambda: f(h, w, ids, logits, b, 1.0, "max")),
                        (ValueError, lambda: f(h, w, ids.repeat(1, 500), logits.repeat(1, 500), b))):
        with pytest.raises(error):
            call()
    h.requires_grad_()
    dh, = torch.autograd.grad(f(h, w, ids, logits, b), h, create_graph=True)
    with pytest.raises(RuntimeError):
        dh.sum().backward()


def _check_frequent(h, w, b, ids, logits, c, often, dw):
    """``dw`` of a step with reduction 'sum', at words whose P keeps what it loses by its rounding to bfloat16: 2^-16 of it is left."""
    (T, D), V = h.shape, w.shape[0]
    kept, _, _, _, _, whole, whole_off = _teacher(ids, logits, V, c)
    H = torch.where(kept[:, None], h.double(), 0.0)
    s = H @ w.double().t().contiguous()
    size = H.abs() @ w.double().abs().t().contiguous()
    if b is not None:
        s, size = s + b.double(), size + b.double().abs()
    s, size = s / c, size / c
    d = ((D + 8) * E * size + 2 * E * s.abs()).amax(1, keepdim=True)
    p = s.softmax(1)
    P = ((p - whole) * c * kept[:, None])[:, often].t().contiguous()
    soft = (p * (2 * d + (4 * s.abs().amax(1, keepdim=True) + 16) * E) + whole_off + E * (p + whole)) * c * kept[:, None]
    off = soft[:, often].t().contiguous() + P.abs() * 2.0 ** -15
    exact = P @ H
    bound = off @ H.abs() + (2 * T + 16) * E * (P.abs() @ H.abs()) + 1.01 * U[h.dtype] * exact.abs()
    _within(dw[often], exact, bound, "dweight of frequent words")


def _frequent(T, D, V, K, often, strength, *key):
    """A case whose first words are the same for all tokens, the others anywhere."""
    h, w, b, _, logits = _case(T, D, V, K, torch.bfloat16, True, *key)
    ids = torch.randint(0, V, (T, K), generator=_gen(*key, 1)).to(DEV)
    ids[:, :len(often)] = torch.tensor(often, device=DEV)
    logits[:, :len(often)] = logits[:, :len(often)] * 0.3 + strength
    return h, w, b, ids, logits


def test_frequent_words_beside_rare_ones_of_more_weight():
    # words of other groups that one token teaches, with nearly all of its probability, and that lie in the frequent words' places of
    # a table of 4096, as a multiplication by the golden ratio finds them
    T, D, V, K, c, often = 500, 1000, 60001, 12, 1.3, [8999, 4321, 300, 55000]
    h, w, b, ids, logits = _frequent(T, D, V, K, often, 4.0, 41)
    places = (torch.arange(V) * 2654435761) % 2 ** 32 >> 20
    for i, word in enumerate(often):
        rare = [int(r) for r in (places == places[word]).nonzero() if int(r) // 256 != word // 256]
        assert len(rare) >= 3
        for j, r in enumerate(rare):
            ids[40 * i + j, 5], logits[40 * i + j, 5] = r, 16.0
    rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
    step = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
    got = _autograd(h, w, ids, logits, b, c, "sum")
    _check(h, w, b, ids, logits, c, torch.ones(T, device=DEV), rows, *step[1:])
    for dw in (step[2], got[2]):
        _check_frequent(h, w, b, ids, logits, c, often, dw)


@pytest.mark.parametrize("first", ["none", "others"])
def test_frequent_words_of_sequences(first):
    # tokens of equal sequences in a row, whose first ones (prompts, what begins a text) have no words, or words of their own
    T, D, V, K, c, often = 512, 1000, 5003, 256, 1.3, [4999, 2321, 300]
    h, w, b, ids, logits = _frequent(T, D, V, K, often, 4.0, 42)
    logits[:, 3:] = logits[:, 3:] / 3 - 2
    starts = torch.arange(T, device=DEV) % 8 < 2
    if first == "none":
        ids[starts] = -1
    else:
        ids[starts] = torch.randint(600, 1800, (int(starts.sum()), K), generator=_gen(43)).to(DEV)
        logits[starts] = 0.0
    rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
    step = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
    got = _autograd(h, w, ids, logits, b, c, "sum")
    _check(h, w, b, ids, logits, c, torch.ones(T, device=DEV), rows, *step[1:])
    for dw in (step[2], got[2]):
        _check_frequent(h, w, b, ids, logits, c, often, dw)


@pytest.mark.parametrize("K", [12, 256, 1024])
def test_frequent_words_of_a_few_tokens_among_many_that_do_not_count(K):
    D, V, c, often = 1000, 5003, 1.3, [4999, 2321, 300]
    for T in (513, 5000, 40000):
        h, w, b, ids, logits = _frequent(T, D, V, K, often, 4.0, 44)
        logits[:, 3:] = logits[:, 3:] / 3 - 2
        ids[torch.arange(T, device=DEV) % (T // 20) != T // 20 - 1] = -1
        step = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
        # (sums over the tokens that count: the others are zeros)
        kept = (ids[:, 0] >= 0)
        _check_frequent(h[kept], w, b, ids[kept], logits[kept], c, often, step[2])
    ids[:] = -1
    assert all((t == 0).all() for t in training.linear_distillation_grad(h, w, ids, logits, b, c, "sum"))


@pytest.mark.parametrize("T", [2, 64, 65, 128, 129, 1500])
def test_frequent_words_of_small_vocabularies(T):
    D, c = 264, 1.3
    for V, often in ((40, [7, 3]), (300, [299, 5]), (1000, [999, 300, 5]), (4096, [4095, 2000, 0]), (4097, [4096, 2000, 0])):
        h, w, b, ids, logits = _frequent(T, D, V, 8, often, 3.0, 45)
        rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
        step = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
        got = _autograd(h, w, ids, logits, b, c, "sum")
        again = training.linear_distillation_grad(h, w, ids, logits, b, c, "sum")
        assert all(torch.equal(p, q) for p, q in zip(step, again))
        for dh, dw, db in (step[1:], got[1:]):
            print(T, V, flush=True)
            _check(h, w, b, ids, logits, c, torch.ones(T, device=DEV), rows, dh, dw, db)
            _check_frequent(h, w, b, ids, logits, c, often, dw)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_that_lie_in_other_ways(dtype):
    # of single losses: what a sum, a mean, a part of them or a repeated one hands back
    h, w, b, ids, logits = _case(4 * 15, 40, 300, 6, dtype, True, 46)
    for make in (lambda loss: loss.sum(), lambda loss: loss.mean(), lambda loss: loss.t()[::2].sum(),
                 lambda loss: loss[:1].expand(5, 15).sum(), lambda loss: (loss.t() @ torch.ones(4, 2, device=DEV)).sum()):
        leaves = [t.detach().requires_grad_() for t in (h, w, b)]
        loss = training.linear_distillation(leaves[0].view(4, 15, 40), leaves[1], ids.view(4, 15, 6), logits.view(4, 15, 6), leaves[2],
                                            reduction="none")
        given, = torch.autograd.grad(make(loss), loss, retain_graph=True)
        got = torch.autograd.grad(make(loss), leaves)
        _check(h, w, b, ids, logits, 1.0, given.reshape(-1), loss.detach().reshape(-1), *got)
    # a single token without an axis of its own
    leaves = [t.detach().requires_grad_() for t in (h[3], w, b)]
    loss = training.linear_distillation(leaves[0], leaves[1], ids[3], logits[3], leaves[2], 2.0)
    assert loss.shape == ()
    got = torch.autograd.grad(loss, leaves)
    _check(h[3:4], w, b, ids[3:4], logits[3:4], 2.0, torch.ones(1, device=DEV), loss.detach()[None], got[0][None], got[1], got[2])


def test_frequent_words_of_tokens_whose_loss_is_used():
    # single losses times a mask of zeros and ones, as a program forms their mean over answers without their prompts
    T, D, V, K, c, often = 512, 1000, 5003, 256, 1.3, [4999, 2321, 300]
    h, w, b, ids, logits = _frequent(T, D, V, K, often, 4.0, 47)
    logits[:, 3:] = logits[:, 3:] / 3 - 2
    mask = (torch.arange(T, device=DEV) % 64 == 63).float()
    ids[mask == 0] = torch.randint(600, 1800, (int((mask == 0).sum()), K), generator=_gen(48)).to(DEV)
    rows = training.linear_distillation(h, w, ids, logits, b, c, "none")
    _, dh, dw, db = _autograd(h, w, ids, logits, b, c, "none", mask)
    _check(h, w, b, ids, logits, c, mask, rows, dh, dw, db)
    kept = mask == 1
    _check_frequent(h[kept], w, b, ids[kept], logits[kept], c, often, dw)
