"""GPU: the operators of a training step (deepshift_amd.training) against their definition in 64 bits.

Bounds are derived, not tuned.  With u the rounding of the output's type (2^-24, 2^-8, 2^-11) and e = 2^-23:

* a lookup is one multiplication in 32 bits and one rounding: equal bit for bit;
* a sum of n values in 32 bits, in any grouping, is off by at most n e sum |x|;
* a logit of D products is off by d = (D + 8) e (sum |h w| + |b|); its loss by twice the largest d of the row plus the
  rounding of a few operations on values up to the largest logit;
* a probability p is off by p (2 d + (4 |s| + 16) e) and, on its way into the second product, by one more rounding to the
  operands' type (none worth counting for float32, whose three planes hold 24 bits); a gradient by the sum of these times the
  other operand, the additions' n e, and the output's rounding.
"""
import math

import pytest
import torch

from deepshift_amd import _lib, modules, training
from tests.conftest import Tune

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
# half the smallest positive value of a type: what a result near zero may be off by
TINY = {torch.float32: 2.0 ** -126, torch.bfloat16: 2.0 ** -126, torch.float16: 2.0 ** -25}


def _gen(*key):
    return torch.Generator().manual_seed(hash(key) & 0x7fffffff)


def _rand(g, *shape, dtype=torch.float32, scale=1.0):
    return (torch.randn(shape, generator=g) * scale).to(dtype).to(DEV)


def _within(got, want, bound, what):
    got = got.double()
    off = (got - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g times the bound" % (
        what, int(bad.sum()), bad.numel(), float((off / bound.clamp(min=1e-300)).nan_to_num(float("inf")).max()))


# ---- embedding ------------------------------------------------------------------------------------------------

EMBED_SHAPES = [(1, 1, 1), (1, 1000, 512), (7, 3, 5), (64, 10, 8), (63, 1000, 36), (130, 7, 1000), (513, 4097, 260),
                (2065, 10007, 385), (300, 50, 4096)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("scale", [1.0, 22.627417])
def test_embedding_is_one_product_and_one_rounding(dtype, scale):
    for T, V, D in EMBED_SHAPES:
        print(T, V, D, flush=True)
        g = _gen(T, V, D)
        w = _rand(g, V, D, dtype=dtype)
        ids = torch.randint(0, V, (T,), generator=g).to(DEV)
        want = (w.float()[ids] * scale).to(dtype)
        for i in (ids, ids.int(), ids.view(T, 1), torch.stack([ids, ids], 1)[:, 0]):
            assert torch.equal(training.embedding(i, w, scale), want.view(i.shape + (D,)))
        # rows apart, and columns apart
        wide = _rand(g, V, D + 3, dtype=dtype)
        assert torch.equal(training.embedding(ids, wide[:, :D], scale), (wide[:, :D].float()[ids] * scale).to(dtype))
        assert torch.equal(training.embedding(ids, wide[:, 3:], scale), (wide[:, 3:].float()[ids] * scale).to(dtype))
        columns = w.t().contiguous().t()
        assert torch.equal(training.embedding(ids, columns, scale), want)


def test_embedding_of_no_tokens_and_of_numbers_that_are_no_words():
    w = _rand(_gen(1), 6, 4)
    assert training.embedding(torch.zeros(0, dtype=torch.int64, device=DEV), w).shape == (0, 4)
    assert training.embedding(torch.zeros(2, 0, 3, dtype=torch.int32, device=DEV), w).shape == (2, 0, 3, 4)
    out = training.embedding(torch.tensor([0, -1, 6, 5, 2 ** 40], device=DEV), w)
    assert torch.equal(out[[0, 3]], w[[0, 5]]) and out[[1, 2, 4]].isnan().all()


def _embed_grad_check(ids, grad, V, scale, padding, dtype, got):
    T, D = grad.shape
    kept = (ids >= 0) & (ids < V)
    if padding is not None:
        kept &= ids != padding
    want = torch.zeros(V, D, dtype=torch.float64, device=DEV)
    size = torch.zeros(V, D, dtype=torch.float64, device=DEV)
    want.index_add_(0, ids[kept], grad[kept].double())
    size.index_add_(0, ids[kept], grad[kept].double().abs())
    n = torch.bincount(ids[kept], minlength=V)[:, None]
    _within(got, want * scale, (n + 2) * E * size * scale + U[dtype] * want.abs() * scale + TINY[dtype], "dweight")
    assert (got[n[:, 0] == 0] == 0).all()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("radix", [0, 1], ids=["ranks", "radix"])
def test_embedding_gradient(dtype, radix):
    for T, V, D in EMBED_SHAPES + [(5000, 3, 40), (17000, 70000, 16), (20000, 300000, 8), (16384, 2, 8), (4096, 1, 12)]:
        print(T, V, D, flush=True)
        g = _gen(T, V, D, 1)
        # a few words have most of the tokens
        ids = (torch.rand(T, generator=g) ** 6 * V).long().clamp(max=V - 1).to(DEV)
        grad = _rand(g, T, D, dtype=dtype)
        with Tune(embed_radix=radix):
            got = training.embedding_grad(ids, grad, V, 0.5)
            _embed_grad_check(ids, grad, V, 0.5, None, dtype, got)
            assert torch.equal(got, training.embedding_grad(ids.int(), grad, V, 0.5)), "a second call differs"
            if T > 1:
                ids[T // 2] = -1
                ids[T // 3] = V
                # what belongs to padding, or to no word, is not looked at
                grad[(ids == 0) | (ids == -1) | (ids == V)] = float("nan")
                got = training.embedding_grad(ids, grad, V, 2.0, padding_idx=0)
                _embed_grad_check(ids, grad, V, 2.0, 0, dtype, got)


def test_embedding_gradient_layouts_and_empty_sizes():
    g = _gen(5)
    ids = torch.randint(0, 50, (4, 33), generator=g).to(DEV)
    grad = _rand(g, 4, 33, 24)
    want = training.embedding_grad(ids, grad, 50)
    wide = torch.zeros(4, 33, 31, device=DEV)
    wide[..., 5:29] = grad
    assert torch.equal(training.embedding_grad(ids, wide[..., 5:29], 50), want)
    assert torch.equal(training.embedding_grad(ids, grad.transpose(0, 2).contiguous().transpose(0, 2), 50), want)
    assert torch.equal(training.embedding_grad(ids, grad[:, :1, :1].expand(4, 33, 24), 50),
                       training.embedding_grad(ids, grad[:, :1, :1].expand(4, 33, 24).contiguous(), 50))
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert torch.equal(training.embedding_grad(none, torch.zeros(0, 7, device=DEV), 5), torch.zeros(5, 7, device=DEV))
    assert training.embedding_grad(ids, grad, 0).shape == (0, 24)
    assert training.embedding_grad(ids, grad[..., :0], 50).shape == (50, 0)
    assert (training.embedding_grad(torch.full_like(ids, 3), grad, 50, padding_idx=3) == 0).all()


def test_embedding_offsets_beyond_32_bits():
    V, D = 300000, 8200   # 4.9 GB of bfloat16
    w = torch.zeros(V, D, dtype=torch.bfloat16, device=DEV)
    last = _rand(_gen(2), D, dtype=torch.bfloat16)
    w[V - 1] = last
    ids = torch.tensor([V - 1, 0, V - 1], device=DEV)
    out = training.embedding(ids, w, 2.0)
    assert torch.equal(out[0], last * 2) and torch.equal(out[2], out[0]) and (out[1] == 0).all()
    got = training.embedding_grad(ids, out, V, 0.25)
    assert torch.equal(got[V - 1], last) and (got[V - 2] == 0).all() and (got[V // 2] == 0).all()


@pytest.mark.parametrize("T, V", [(6144, 400), (6145, 400), (8192, 510), (8192, 511), (12288, 1125), (12289, 1125), (12288, 262143)])
def test_embedding_gradient_where_the_sort_changes(T, V):
    g = _gen(T, V)
    ids = torch.randint(0, V, (T,), generator=g).to(DEV)
    ids[::5] = V // 2
    ids[1::7] = -1     # no word
    grad = _rand(g, T, 20)
    real = ids >= 0
    got = training.embedding_grad(ids, grad, V, 2.0, padding_idx=3)
    want, size = (torch.zeros(V, 20, dtype=torch.float64, device=DEV).index_add_(0, ids[real], x[real]) * 2 for x in
                  (grad.double(), grad.double().abs()))
    want[3], size[3] = 0, 0
    _within(got, want, (T + 2) * E * size + TINY[torch.float32], "gradient")
    assert (got[3] == 0).all() and torch.equal(got, training.embedding_grad(ids.int(), grad, V, 2.0, padding_idx=3))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_embedding_of_rows_that_begin_anywhere(dtype):
    for T, V, D, before in [(9000, 300, 257, 0), (20000, 3000, 131, 0), (17000, 65, 513, 0), (9000, 50, 384, 1), (100, 40, 385, 3),
                            (5, 3, 1, 1), (9, 7, 9, 0)]:
        print(T, V, D, before, flush=True)
        g = _gen(T, V, D)
        wide = torch.full((V, D + before), float("nan"), dtype=dtype, device=DEV)
        wide[:, before:] = _rand(g, V, D, dtype=dtype)
        ids = torch.randint(0, V, (T,), generator=g).to(DEV)
        ids[::3] = V - 1
        assert torch.equal(training.embedding(ids, wide[:, before:], 0.5), (wide[:, before:].float()[ids] * 0.5).to(dtype))
        flat = torch.full((T, D + before), float("nan"), dtype=dtype, device=DEV)
        flat[:, before:] = _rand(g, T, D, dtype=dtype)
        grad = flat[:, before:]
        got = training.embedding_grad(ids, grad, V, 0.5)
        want = torch.zeros(V, D, dtype=torch.float64, device=DEV).index_add_(0, ids, grad.double()) * 0.5
        size = torch.zeros(V, D, dtype=torch.float64, device=DEV).index_add_(0, ids, grad.double().abs()) * 0.5
        _within(got, want, (T + 2) * E * size + U[dtype] * want.abs() * 1.01 + TINY[dtype], "gradient")
        assert torch.equal(got, training.embedding_grad(ids, grad, V, 0.5))


def test_embedding_module_under_autograd():
    torch.manual_seed(0)
    m = training.ScaledEmbedding(40, 12, scale=3.0, padding_idx=-1).to(DEV)
    assert (m.weight[39] == 0).all()
    ids = torch.randint(0, 40, (3, 9), device=DEV)
    ids[0, 0] = 39
    grad = torch.randn(3, 9, 12, device=DEV)
    m(ids).backward(grad)
    want = torch.zeros(40, 12, dtype=torch.float64, device=DEV).index_add_(0, ids.view(-1), grad.double().view(-1, 12) * 3)
    want[39] = 0
    torch.testing.assert_close(m.weight.grad.double(), want, rtol=0, atol=27 * E * 3 * float(grad.abs().sum(1).max()) * 3)
    assert (m.weight.grad[39] == 0).all()


# ---- cross entropy ----------------------------------------------------------------------------------------------

def _head(T, D, V, dtype, bias, g, spread=2.0):
    h = _rand(g, T, D, dtype=dtype)
    w = _rand(g, V, D, dtype=dtype, scale=spread / math.sqrt(max(D, 1)))
    b = _rand(g, V, dtype=dtype, scale=0.3) if bias else None
    y = torch.randint(0, V, (T,), generator=g).to(DEV)
    return h, w, b, y


def _head_check(h, w, b, y, ignore, share, losses, dh=None, dw=None, db=None):
    """``share`` [T]: the gradient of each row's loss."""
    dtype, (T, D), V = h.dtype, h.shape, w.shape[0]
    kept = y != ignore
    H, W = h.double(), w.double()
    H[~kept] = 0    # tokens that do not count leave nothing
    s, size = H @ W.t(), H.abs() @ W.abs().t()
    if b is not None:
        s, size = s + b.double(), size + b.double().abs()
    finite = s.isfinite()
    delta = torch.where(finite, (D + 8) * E * size, 0.0)
    d = delta.amax(1, keepdim=True)
    most = torch.where(finite, s.abs(), 0.0).amax(1, keepdim=True)
    lse = s.logsumexp(1, keepdim=True)
    at = y.clamp(0, V - 1)[:, None]
    want = torch.where(kept, (lse - s.gather(1, at))[:, 0], 0.0)
    _within(losses, want, (2 * d + (6 * most + 20) * E)[:, 0] * kept + 1e-300, "loss")
    if dh is None:
        return
    p = (s - lse).exp()
    hot = torch.zeros_like(p).scatter_(1, at, 1.0)
    g = (share.double() * kept)[:, None]
    err = p * (2 * d + (4 * most + 16) * E) + (p - hot).abs() * 2 * U[dtype]
    # probabilities travel as shares of the largest gradient, float16 ones times 2^15
    P, G = (p - hot) * g, err * g.abs() + TINY[dtype] * 2.0 ** -14 * g.abs().max()
    u, tiny = U[dtype], TINY[dtype]
    for name, got, left, right, n in (("dhidden", dh, P, W, V), ("dweight", dw, P.t(), H, T)):
        terms = left.abs() @ right.abs()
        off = (G if name == "dhidden" else G.t()) @ right.abs()
        exact = left @ right
        _within(got, exact, off + (n + 16) * E * terms + (u + 4 * E) * (exact.abs() + off) + tiny, name)
    if db is not None:
        err = p * (2 * d + (4 * most + 16) * E) * g.abs()
        exact = P.sum(0)
        _within(db, exact, err.sum(0) + (T + 8) * E * P.abs().sum(0) + u * exact.abs() * 1.01 + tiny, "dbias")


HEAD_SHAPES = [(1, 1, 1), (1, 8, 2), (3, 5, 7), (64, 512, 10), (2, 64, 1000), (65, 64, 1000), (130, 100, 257), (16, 1000, 513),
               (257, 136, 300), (300, 256, 515), (513, 96, 129), (33, 2056, 777)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tile", [0, 1, 2, 3])
def test_cross_entropy_and_gradients(dtype, tile):
    for i, (T, D, V) in enumerate(HEAD_SHAPES):
        print(T, D, V, flush=True)
        g = _gen(T, D, V)
        h, w, b, y = _head(T, D, V, dtype, i % 2 == 0, g)
        if i % 3 == 1 and T > 2:
            y[::3] = -100
        n = max(1, int((y != -100).sum()))
        with Tune(vocab_tile=tile):
            rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
            loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b)
            again = training.linear_cross_entropy_grad(h, w, y.int(), b)
        _head_check(h, w, b, y, -100, torch.full((T,), 1.0 / n, device=DEV), rows, dh, dw, db)
        total = rows.double().sum() / n
        assert abs(loss.double() - total) <= 4 * E * rows.double().abs().sum() / n + 1e-300
        assert torch.equal(loss, again[0]) and torch.equal(dh, again[1]) and torch.equal(dw, again[2])
        assert (db is None) == (b is None) and (db is None or torch.equal(db, again[3]))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_in_pieces_and_stretches(dtype):
    # pieces of 256 words: each leaves its part of dhidden behind what the earlier ones left
    for T, D, V in [(100, 72, 1000), (33, 100, 777), (260, 64, 513)]:
        g = _gen(T, D, V, 3)
        h, w, b, y = _head(T, D, V, dtype, True, g)
        ones = torch.ones(T, device=DEV)
        for tune in (dict(vocab_piece_kb=1), dict(vocab_piece_kb=1, vocab_split=3), dict(vocab_split=5), dict(vocab_split=1)):
            for tile in (0, 1, 2, 3):
                print(T, D, V, tune, tile, flush=True)
                with Tune(vocab_tile=tile, **tune):
                    rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
                    loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b, reduction="sum")
                _head_check(h, w, b, y, -100, ones, rows, dh, dw, db)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("bias", [False, True])
def test_cross_entropy_keeps_the_last_piece(dtype, bias):
    # targets in every piece, the last piece shorter than the others, or of a single word, or of a whole tile
    for T, D, V in [(70, 40, 517), (129, 64, 1025), (8, 24, 768), (300, 33, 900)]:
        g = _gen(T, D, V, 7)
        h, w, b, y = _head(T, D, V, dtype, bias, g)
        y[0], y[1], y[T // 2] = V - 1, 0, 256
        y[2::7] = -100
        kept = int((y != -100).sum())
        for tile in (0, 1, 2, 3):
            print(T, D, V, tile, flush=True)
            with Tune(vocab_tile=tile, vocab_piece_kb=1):
                rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
                loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b)
                again = training.linear_cross_entropy_grad(h, w, y, b)
            _head_check(h, w, b, y, -100, torch.full((T,), 1.0 / kept, device=DEV), rows, dh, dw, db)
            assert all(x is z or torch.equal(x, z) for x, z in zip((loss, dh, dw, db), again))


@pytest.mark.parametrize("T", [1, 2, 3, 4, 5, 8, 9, 15, 16, 17])
def test_cross_entropy_of_a_few_tokens(T):
    # features around a wave's 256, words around a workgroup's 32, rows at every alignment
    for i, (D, V) in enumerate([(1, 1), (3, 2), (4, 31), (5, 33), (255, 64), (256, 65), (257, 1000), (700, 300), (1030, 2085),
                               (1030, 8201)]):
        print(T, D, V, flush=True)
        g = _gen(T, D, V, 5)
        h, w, b, y = _head(T, D, V, torch.float32, i % 2 == 0, g)
        y[0] = V - 1
        if T > 2:
            y[1::4] = -100
            h[1::4] = float("nan")
        kept = int((y != -100).sum())
        clean = torch.where((y != -100)[:, None], h, torch.zeros_like(h))
        wide_h, wide_w = torch.full((T, D + 3), float("nan"), device=DEV), torch.full((V, D + 1), float("inf"), device=DEV)
        wide_h[:, 2:D + 2], wide_w[:, 1:] = h, w
        share = torch.full((T,), 1.0 / kept, device=DEV)
        for hh, ww, tune in ((h, w, {}), (wide_h[:, 2:D + 2], wide_w[:, 1:], {}), (h, w, dict(vocab_piece_kb=1))):
            with Tune(**tune):
                rows = training.linear_cross_entropy(hh, ww, y, b, reduction="none")
                loss, dh, dw, db = training.linear_cross_entropy_grad(hh, ww, y, b)
                again = training.linear_cross_entropy_grad(hh, ww, y, b)
            _head_check(clean, w, b, y, -100, share, rows, dh, dw, db)
            assert (dh[y == -100] == 0).all()
            assert all(x is z or torch.equal(x, z) for x, z in zip((loss, dh, dw, db), again))
        # the gradients by themselves, of rows with gradients of their own
        grads = _rand(g, T)
        leaves = [x.detach().requires_grad_() for x in (h, w) + ((b,) if b is not None else ())]
        training.linear_cross_entropy(leaves[0], leaves[1], y, *leaves[2:], reduction="none").backward(grads)
        _head_check(clean, w, b, y, -100, grads, rows, leaves[0].grad, leaves[1].grad, leaves[2].grad if b is not None else None)


@pytest.mark.parametrize("T", [17, 40, 64, 65, 130])
def test_cross_entropy_of_weights_as_they_are(T):
    # many weights, few tokens: words around a tile's 128, features around a stage's 32
    for i, (D, V) in enumerate([(1024, 8193), (4, 2097153), (2052, 4224), (36, 233100), (1056, 7999)]):
        print(T, D, V, flush=True)
        g = _gen(T, D, V, 6)
        h, w, b, y = _head(T, D, V, torch.float32, i % 2 == 0, g)
        y[0], y[1], y[2] = V - 1, 0, 128
        y[3::5] = -100
        h[3::5] = float("nan")
        kept = int((y != -100).sum())
        clean = torch.where((y != -100)[:, None], h, torch.zeros_like(h))
        share = torch.full((T,), 1.0 / kept, device=DEV)
        for tune in ({}, dict(vocab_piece_kb=3 * 2 * T * (V // 3) // 1024)):
            with Tune(**tune):
                rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
                loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b)
                again = training.linear_cross_entropy_grad(h, w, y, b)
            _head_check(clean, w, b, y, -100, share, rows, dh, dw, db)
            assert all(x is z or torch.equal(x, z) for x, z in zip((loss, dh, dw, db), again))
        del again, dh, dw, db
        leaves = [x.detach().requires_grad_() for x in (h, w) + ((b,) if b is not None else ())]
        training.linear_cross_entropy(leaves[0], leaves[1], y, *leaves[2:], reduction="sum").backward()
        _head_check(clean, w, b, y, -100, torch.ones(T, device=DEV), rows, leaves[0].grad, leaves[1].grad,
                    leaves[2].grad if b is not None else None)


@pytest.mark.parametrize("T", [17, 64, 100])
def test_cross_entropy_of_weights_as_they_are_wherever_rows_begin(T):
    for D, V, before, behind in [(1021, 8300, 0, 0), (3, 2796203, 0, 0), (1024, 8200, 1, 2), (2050, 4097, 2, 0), (1023, 8201, 0, 1)]:
        print(T, D, V, before, behind, flush=True)
        g = _gen(T, D, V, 9)
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


def test_cross_entropy_of_extreme_weights_as_they_are():
    # the largest float32, and the smallest, split without loss
    g = _gen(1, 2, 3)
    T, D, V = 20, 1024, 8200
    h, w, b, y = _head(T, D, V, torch.float32, False, g)
    for small, large in ((2.0 ** -100, 2.0 ** 97), (2.0 ** 60, 2.0 ** -62)):
        rows = training.linear_cross_entropy(h * small, w * large, y, reduction="none")
        with Tune(vocab_tile=1):
            want = training.linear_cross_entropy(h * small, w * large, y, reduction="none")
        _head_check(h * small, w * large, None, y, -100, torch.ones(T, device=DEV), rows)
        _head_check(h * small, w * large, None, y, -100, torch.ones(T, device=DEV), want)
    w[:, 0] = torch.finfo(torch.float32).max
    h[:, 0] = 2.0 ** -125
    rows = training.linear_cross_entropy(h, w, y, reduction="none")
    _head_check(h, w, None, y, -100, torch.ones(T, device=DEV), rows)


def test_cross_entropy_of_a_few_tokens_with_words_taken_out():
    g = _gen(8, 8)
    h, w, b, y = _head(6, 20, 200, torch.float32, True, g)
    b[30:170] = float("-inf")
    y = y % 30
    rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
    loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b, reduction="sum")
    _head_check(h, w, b, y, -100, torch.ones(6, device=DEV), rows, dh, dw, db)
    assert (dw[30:170] == 0).all() and (db[30:170] == 0).all()
    assert training.linear_cross_entropy(h, w, torch.full_like(y, 100), b, reduction="none").isposinf().all()
    assert training.linear_cross_entropy(h, w, y, torch.full_like(b, float("-inf")), reduction="none").isnan().all()
    # logits far apart
    h, w = h * 2.0 ** 30, w * 2.0 ** 40
    rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
    s = h.double() @ w.double().t() + b.double()
    size = (h.abs().double() @ w.abs().double().t())[:, :30].amax(1) + (h.abs().double() @ w.abs().double().t())[:, 170:].amax(1)
    _within(rows, s.logsumexp(1) - s.gather(1, y[:, None])[:, 0], 2 * 28 * E * size + 8 * E * size, "loss")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_layouts(dtype):
    g = _gen(11)
    h, w, b, y = _head(60, 64, 301, dtype, True, g)
    want = training.linear_cross_entropy_grad(h, w, y, b)
    wide_h = torch.full((60, 80), float("nan"), dtype=dtype, device=DEV)
    wide_w = torch.full((301, 71), float("nan"), dtype=dtype, device=DEV)
    wide_h[:, 8:72], wide_w[:, 3:67] = h, w
    wide_b = torch.zeros(602, dtype=dtype, device=DEV)
    wide_b[::2] = b
    for hh, ww in ((wide_h[:, 8:72], w), (h, wide_w[:, 3:67]), (wide_h[:, 8:72], wide_w[:, 3:67]),
                   (h.t().contiguous().t(), w.t().contiguous().t())):
        got = training.linear_cross_entropy_grad(hh, ww, y, wide_b[::2])
        assert all(torch.equal(a, c) for a, c in zip(got, want))
    got = training.linear_cross_entropy_grad(h.view(3, 20, 64), w, y.view(3, 20), b)
    assert got[1].shape == (3, 20, 64) and torch.equal(got[1].view(60, 64), want[1]) and torch.equal(got[2], want[2])
    same = h[:1].expand(60, 64)
    assert torch.equal(training.linear_cross_entropy(same, w, y, b, reduction="none"),
                       training.linear_cross_entropy(same.contiguous(), w, y, b, reduction="none"))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_masks(dtype):
    g = _gen(12)
    T, D, V = 70, 48, 300
    h, w, b, y = _head(T, D, V, dtype, True, g)
    # words taken out by a bias of -inf, whole tiles of them
    b[40:290] = float("-inf")
    y = torch.where(y % 2 == 0, y % 40, 290 + y % 10)
    rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
    loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b, reduction="sum")
    _head_check(h, w, b, y, -100, torch.ones(T, device=DEV), rows, dh, dw, db)
    assert (dw[40:290] == 0).all() and (db[40:290] == 0).all()
    # the lowest value of the type does the same as far as the type's exponent goes
    low = b.clone()
    low[40:290] = torch.finfo(dtype).min
    rows2 = training.linear_cross_entropy(h, w, y, low, reduction="none")
    assert torch.equal(rows, rows2)
    # a target that was taken out costs infinitely much
    assert training.linear_cross_entropy(h, w, torch.full_like(y, 100), b, reduction="none").isposinf().all()
    # every word taken out: no distribution
    assert training.linear_cross_entropy(h, w, y, torch.full_like(b, float("-inf")), reduction="none").isnan().all()
    # tokens that do not count may hold anything
    y2 = y.clone()
    y2[::5] = 7777
    kept = y2 != 7777
    h2 = h.clone()
    h2[::5] = float("nan")
    h2[5] = float("inf")
    rows = training.linear_cross_entropy(h2, w, y2, b, ignore_index=7777, reduction="none")
    loss, dh, dw, db = training.linear_cross_entropy_grad(h2, w, y2, b, ignore_index=7777)
    _head_check(torch.where(kept[:, None], h2, torch.zeros_like(h2)), w, b, y2, 7777,
                torch.full((T,), 1.0 / int(kept.sum()), device=DEV), rows, dh, dw, db)
    assert (dh[::5] == 0).all() and torch.isfinite(loss)
    # nothing counts
    loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, torch.full_like(y, -100), b)
    assert loss == 0 and (dh == 0).all() and (dw == 0).all() and (db == 0).all()
    # an ignored number that is a word
    rows = training.linear_cross_entropy(h, w, y, b, ignore_index=int(y[0]), reduction="none")
    assert (rows[y == y[0]] == 0).all() and (rows[y != y[0]] != 0).all()


def test_cross_entropy_of_no_tokens_no_features_and_wrong_targets():
    w = _rand(_gen(3), 9, 16)
    b = _rand(_gen(4), 9)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    loss, dh, dw, db = training.linear_cross_entropy_grad(torch.zeros(0, 16, device=DEV), w, none, b)
    assert loss == 0 and dh.shape == (0, 16) and (dw == 0).all() and (db == 0).all()
    y = torch.tensor([1, 8], device=DEV)
    loss, dh, dw, db = training.linear_cross_entropy_grad(torch.zeros(2, 0, device=DEV), torch.zeros(9, 0, device=DEV), y, b)
    p = b.double().softmax(0)
    assert abs(loss.double() + p[y].log().mean()) < 1e-6 and dh.shape == (2, 0) and dw.shape == (9, 0)
    want = p.clone()
    want[1] -= 0.5
    want[8] -= 0.5
    assert (db.double() - want).abs().max() < 1e-6
    h = _rand(_gen(5), 3, 16)
    rows = training.linear_cross_entropy(h, w, torch.tensor([0, 9, -1], device=DEV), b, reduction="none")
    assert rows[0].isfinite() and rows[1:].isnan().all()
    assert training.linear_cross_entropy_grad(h, w, torch.tensor([0, 9, 2], device=DEV), b)[2].isnan().any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_cross_entropy_of_large_and_far_apart_logits(dtype):
    g = _gen(21)
    T, D, V = 40, 64, 500
    h, w, b, y = _head(T, D, V, dtype, False, g, spread=60.0)
    rows = training.linear_cross_entropy(h, w, y, reduction="none")
    loss, dh, dw, _ = training.linear_cross_entropy_grad(h, w, y, reduction="sum")
    _head_check(h, w, None, y, -100, torch.ones(T, device=DEV), rows, dh, dw)
    h[3, 2] = float("inf")
    rows = training.linear_cross_entropy(h, w, y, reduction="none")
    assert rows[3].isnan() and rows[:3].isfinite().all() and rows[4:].isfinite().all()


def test_float32_head_keeps_24_bits():
    # values next to the largest float32 and tiny ones, whose planes round up and underflow
    h = torch.tensor([[3.4e38, 1e-30, 1.0, 0.0]], device=DEV)
    w = torch.tensor([[1e-38, 1.0, 1 / 3, 5.0], [1e-39, 1e30, 1e-3, 0.0], [-1e-38, 0.0, 1.0, 1.0]], device=DEV)
    rows = training.linear_cross_entropy(h, w, torch.tensor([1], device=DEV), reduction="none")
    s = h.double() @ w.double().t()
    assert abs(rows.double() - (s.logsumexp(1) - s[:, 1])).item() < 20 * E


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("reduction", ["none", "sum", "mean"])
def test_cross_entropy_under_autograd(dtype, reduction):
    g = _gen(31)
    T, D, V = 50, 40, 200
    h, w, b, y = _head(T, D, V, dtype, True, g)
    y[::7] = -100
    kept = y != -100
    for t in (h, w, b):
        t.requires_grad_()
    loss = training.linear_cross_entropy(h, w, y, b, reduction=reduction)
    assert loss.dtype == torch.float32
    if reduction == "none":
        up = _rand(g, T, scale=1e-6)     # small: float16 must not lose it
        share = up
    else:
        up = torch.tensor(-0.5, device=DEV)
        share = torch.full((T,), -0.5 / (int(kept.sum()) if reduction == "mean" else 1), device=DEV)
    dh, dw, db = torch.autograd.grad(loss, (h, w, b), up)
    with torch.no_grad():
        rows = training.linear_cross_entropy(h, w, y, b, reduction="none")
        _head_check(h.detach(), w.detach(), b.detach(), y, -100, share, rows, dh, dw, db)
    # only what is asked for
    only = training.linear_cross_entropy(h.detach(), w, y, b.detach(), reduction="sum")
    dw2, = torch.autograd.grad(only, (w,))
    assert dw2.shape == w.shape


def test_cross_entropy_gradient_against_differences():
    # along a direction x of unit length per token, a loss f has f(e) - f(-e) = 2 e f' + e^3/3 f'''; |f'''| <= 6 m^3 with m the
    # largest change of a logit per e, and each f is off by the bound of its logits
    g = _gen(41)
    T, D, V = 20, 30, 90
    h, w, b, y = _head(T, D, V, torch.float32, True, g)
    _, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b, reduction="sum")
    e = 2.0 ** -6
    for which, grad in ((0, dh), (1, dw), (2, db)):
        x = _rand(g, *(h, w, b)[which].shape)
        x /= x.norm()
        ends = []
        for side in (e, -e):
            args = [h, w, b]
            args[which] = args[which] + side * x
            ends.append(training.linear_cross_entropy(args[0], args[1], y, args[2], reduction="none").double().sum())
        slope = (ends[0] - ends[1]) / (2 * e)
        change = (x @ w.t() if which == 0 else h @ x.t() if which == 1 else x.expand(T, V)).abs().amax(1).double()
        size = (h.abs() @ w.abs().t() + b.abs()).max().double()
        bound = float((change ** 3).sum() * e * e + T * (2 * (D + 8) * size + 6 * size + 20) * E / e)
        assert abs(slope - (grad.double() * x.double()).sum()) <= bound
        assert bound < 0.2 * float(grad.norm()), "the bound says nothing"


def test_cross_entropy_offsets_beyond_32_bits():
    V, D = 140000, 16392    # 4.6 GB of bfloat16
    g = torch.Generator(device=DEV).manual_seed(3)
    w = torch.empty(V, D, dtype=torch.bfloat16, device=DEV)
    for part in w.split(10000):
        part.copy_(torch.randn(part.shape, generator=g, device=DEV) / 64)
    h = torch.randn(2, D, generator=g, device=DEV).bfloat16()
    y = torch.tensor([V - 1, V - 70000], device=DEV)
    rows = training.linear_cross_entropy(h, w, y, reduction="none")
    loss, dh, dw, _ = training.linear_cross_entropy_grad(h, w, y, reduction="sum")
    H = h.double()
    s = torch.cat([H @ part.double().t() for part in w.split(10000)], 1)
    p = s.softmax(1)
    assert ((s.logsumexp(1) - s.gather(1, y[:, None])[:, 0]) - rows.double()).abs().max() < 1e-3
    p.scatter_add_(1, y[:, None], torch.full((2, 1), -1.0, dtype=torch.float64, device=DEV))
    want = sum(p[:, i * 10000:(i + 1) * 10000] @ part.double() for i, part in enumerate(w.split(10000)))
    size = sum(p[:, i * 10000:(i + 1) * 10000].abs() @ part.double().abs() for i, part in enumerate(w.split(10000)))
    assert ((dh.double() - want).abs() <= 2.0 ** -7 * size).all()
    for v in (0, V - 70000, V - 1, 65535, 65536):
        want = p[:, v] @ H
        assert ((dw[v].double() - want).abs() <= 2.0 ** -7 * (p[:, v].abs() @ H.abs()) + 1e-30).all()


# ---- clipping ---------------------------------------------------------------------------------------------------

def _sets(g):
    yield [(5,)]
    yield [(1,), (0,), (3, 0), (64, 3, 7, 7), (16384,), (16385,), (33, 1000)]
    yield [(512, 784), (512,), (512, 512), (512,), (10, 512), (10,)]
    yield [(int(n),) for n in torch.randint(1, 300, (300,), generator=g)]
    yield [(3000000,), (7,), ()]


@pytest.mark.parametrize("to", TYPES, ids=str)
@pytest.mark.parametrize("dtype", TYPES + ["mixed"], ids=str)
def test_clipping(dtype, to):
    g = _gen(51)
    for shapes in _sets(g):
        print(len(shapes), flush=True)
        grads = [_rand(g, *s, dtype=TYPES[i % 3] if dtype == "mixed" else dtype) for i, s in enumerate(shapes)]
        norm = math.sqrt(sum(float((t.double() ** 2).sum()) for t in grads))
        assert abs(training.gradient_norm(grads).item() - norm) <= 2.0 ** -23 * norm
        for most in (norm / 3, norm * 2):
            out = [torch.empty(t.shape, dtype=to, device=DEV) for t in grads]
            before = [t.clone() for t in grads]
            got = training.clip_gradients_(grads, most, out=out)
            assert got.shape == () and abs(got.item() - norm) <= 2.0 ** -23 * norm
            f = min(1.0, most / (norm + 1e-6))
            for t, o, was in zip(grads, out, before):
                assert torch.equal(t, was)
                want = was.double() * f
                _within(o, want, want.abs() * (U[to] + 3 * E) + TINY[to], "clipped")
            inplace = [t.clone() for t in grads]
            training.clip_gradients_(inplace, most)
            for t, was in zip(inplace, before):
                want = was.double() * f
                _within(t, want, want.abs() * (U[was.dtype] + 3 * E) + TINY[was.dtype], "clipped in place")
                assert f < 1 or torch.equal(t, was)


def test_clipping_extreme_values():
    big = [torch.full((1000,), 3e38, device=DEV), torch.full((7,), 1e-38, device=DEV)]
    norm = training.clip_gradients_(big, 1.0)
    assert norm.isinf()       # 3e38 * sqrt(1000) is more than float32 holds; the factor still comes from the 64-bit norm
    assert abs(big[0].double().norm().item() - 1.0) < 1e-6
    mid = [torch.full((4,), 1e38, device=DEV)]
    assert abs(training.gradient_norm(mid).item() / 2e38 - 1) < 1e-6
    small = [torch.full((4,), 1e-30, device=DEV)]
    assert abs(training.gradient_norm(small).item() / 2e-30 - 1) < 1e-6
    zero = [torch.zeros(3, device=DEV)]
    assert training.clip_gradients_(zero, 0.0).item() == 0 and (zero[0] == 0).all()
    inf = [torch.tensor([1.0, float("inf"), -2.0], device=DEV)]
    assert training.clip_gradients_(inf, 1.0).isinf()
    assert inf[0][0] == 0 and inf[0][1].isnan() and inf[0][2] == 0
    nan = [torch.tensor([1.0, float("nan")], device=DEV), torch.ones(3, device=DEV)]
    assert training.clip_gradients_(nan, 1.0).isnan() and nan[1].isnan().all()


def test_clipping_layouts():
    g = _gen(52)
    base = _rand(g, 40, 30)
    pieces = [base[:, 3:20], base.t()[20:25], base[:7, 27], _rand(g, 2, 3, 8, 8).to(memory_format=torch.channels_last)]
    plain = [t.clone(memory_format=torch.contiguous_format) for t in pieces]
    keep = base.clone()
    want = [t.clone() for t in plain]
    n1, n2 = training.clip_gradients_(pieces, 0.5), training.clip_gradients_(want, 0.5)
    # the same values in the same places, whatever lies between them
    torch.testing.assert_close(n1, n2, rtol=2.0 ** -22, atol=0)
    for a, b in zip(pieces, want):
        torch.testing.assert_close(a, b, rtol=2.0 ** -21, atol=0)
    assert torch.equal(base[:, :3], keep[:, :3]) and torch.equal(base[7:, 25:], keep[7:, 25:])
    out = [torch.empty_like(t.transpose(0, 1).contiguous()).transpose(0, 1) if t.dim() == 2 else torch.empty_like(t) for t in plain]
    training.clip_gradients_(plain, 0.5, out=out)
    for a, b in zip(out, want):
        torch.testing.assert_close(a, b, rtol=2.0 ** -21, atol=0)
    # unaligned starts
    flat = _rand(g, 5000)
    a, b = flat[1:4001], flat[1:4001].clone()
    training.clip_gradients_([a], 1.0)
    training.clip_gradients_([b], 1.0)
    torch.testing.assert_close(a, b, rtol=2.0 ** -21, atol=0)


def test_autograd_hears_of_clipped_tensors_and_refuses_second_derivatives():
    g = _gen(53)
    a, b = _rand(g, 30), _rand(g, 30)
    before = a._version, b._version
    training.clip_gradients_([a], 0.1)
    training.clip_gradients_([a], 0.1, out=[b])
    training.gradient_norm([a, b])
    assert a._version == before[0] + 1 and b._version == before[1] + 1
    with torch.inference_mode():
        c = torch.ones(4, device=DEV)
        assert training.clip_gradients_([c], 1.0).item() == 2.0 and c[0] < 0.6
    h, w = _rand(g, 5, 8).requires_grad_(), _rand(g, 6, 8).requires_grad_()
    y = torch.arange(5, device=DEV)
    for loss, of in ((training.linear_cross_entropy(h, w, y), h), (training.embedding(y, w).square().sum(), w)):
        first, = torch.autograd.grad(loss, of, create_graph=True)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(first.sum(), of)


def test_rows_far_apart():
    g = _gen(54)
    h, w, b, y = _head(3, 16, 20, torch.bfloat16, True, g)
    far = torch.zeros(3 * 2100000, dtype=torch.bfloat16, device=DEV).view(3, 2100000)
    far[:, 8:24] = h
    want = training.linear_cross_entropy_grad(h, w, y, b)
    got = training.linear_cross_entropy_grad(far[:, 8:24], w, y, b)
    assert all(torch.equal(x, z) for x, z in zip(got, want))
    assert torch.equal(training.embedding(torch.tensor([2, 0], device=DEV), far[:, 8:24]), h[[2, 0]])


def test_clip_grad_norm_of_parameters():
    torch.manual_seed(1)
    m = torch.nn.Sequential(modules.LinearShift(20, 30), torch.nn.ReLU(), modules.LinearShift(30, 5)).to(DEV)
    (m(torch.randn(8, 20, device=DEV)) ** 2).sum().backward()
    want = [p.grad.clone() for p in m.parameters()]
    norm = torch.nn.utils.get_total_norm(want)
    got = training.clip_grad_norm_(m.parameters(), 0.1)
    torch.testing.assert_close(got, norm, rtol=1e-5, atol=0)
    for p, was in zip(m.parameters(), want):
        torch.testing.assert_close(p.grad, was * (0.1 / (norm + 1e-6)), rtol=1e-5, atol=1e-12)
    m[0].bias.grad[0] = float("inf")
    before = [p.grad.clone() for p in m.parameters()]
    with pytest.raises(RuntimeError, match="norm"):
        training.clip_grad_norm_(m.parameters(), 0.1, error_if_nonfinite=True)
    assert all(torch.equal(p.grad, was) for p, was in zip(m.parameters(), before))
    for p in m.parameters():
        p.grad = None
    assert training.clip_grad_norm_(m.parameters(), 0.1).item() == 0


# ---- streams, graphs, refusals ------------------------------------------------------------------------------------

def _step(ids, table, w, b, y):
    h = training.embedding(ids, table, 2.0)
    loss, dh, dw, db = training.linear_cross_entropy_grad(h, w, y, b)
    dt = training.embedding_grad(ids, dh, table.shape[0], 2.0)
    grads = [dt, dw, db]
    norm = training.clip_gradients_(grads, 0.01)
    return [loss, norm] + grads


def test_another_stream_and_captured_replays():
    g = _gen(61)
    V, D, T = 500, 64, 200
    table, w, b = _rand(g, V, D), _rand(g, V, D, scale=0.2), _rand(g, V)
    ids, y = torch.randint(0, V, (T,), generator=g).to(DEV), torch.randint(0, V, (T,), generator=g).to(DEV)
    want = [t.clone() for t in _step(ids, table, w, b, y)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = _step(ids, table, w, b, y)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, c) for a, c in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = _step(ids, table, w, b, y)
    for i in range(3):
        ids2 = torch.randint(0, V, (T,), generator=g).to(DEV)
        ids.copy_(ids2)
        graph.replay()
        torch.cuda.synchronize()
        want = _step(ids, table, w, b, y)
        assert all(torch.equal(a, c) for a, c in zip(captured, want)), "replay %d" % i


def test_refusals():
    f = torch.zeros(4, 8, device=DEV)
    w = torch.zeros(5, 8, device=DEV)
    ids = torch.zeros(4, dtype=torch.int64, device=DEV)
    with pytest.raises(TypeError):
        training.embedding(ids.float(), w)
    with pytest.raises(TypeError):
        training.embedding(ids, w.double())
    with pytest.raises(ValueError):
        training.embedding(ids, w[0])
    with pytest.raises(ValueError):
        training.embedding(ids.cpu(), w)
    with pytest.raises(ValueError):
        training.embedding(ids, w, float("inf"))
    with pytest.raises(ValueError):
        training.embedding_grad(ids, f[:3], 5)
    with pytest.raises(ValueError):
        training.embedding_grad(ids, f, 5, padding_idx=5)
    with pytest.raises(ValueError):
        training.embedding_grad(ids, f, -1)
    with pytest.raises(TypeError):
        training.linear_cross_entropy(f, w.bfloat16(), ids)
    with pytest.raises(ValueError):
        training.linear_cross_entropy(f, w[:, :7], ids)
    with pytest.raises(ValueError):
        training.linear_cross_entropy(f, w, ids[:3])
    with pytest.raises(ValueError):
        training.linear_cross_entropy(f, w, ids, torch.zeros(4, device=DEV))
    with pytest.raises(ValueError):
        training.linear_cross_entropy(f, w, ids, reduction="average")
    with pytest.raises(ValueError):
        training.linear_cross_entropy(f, w[:0], ids)
    with pytest.raises(TypeError):
        training.linear_cross_entropy(f, w, ids.float())
    with pytest.raises(ValueError):
        training.clip_gradients_([], 1.0)
    with pytest.raises(ValueError):
        training.clip_gradients_([f], -1.0)
    with pytest.raises(ValueError):
        training.clip_gradients_([f], float("nan"))
    with pytest.raises(ValueError):
        training.clip_gradients_([f, f], 1.0)
    with pytest.raises(ValueError):
        training.clip_gradients_([f], 1.0, out=[w])
    with pytest.raises(ValueError):
        training.clip_gradients_([f, w], 1.0, out=[f])
    with pytest.raises(TypeError):
        training.clip_gradients_([f.double()], 1.0)
    with pytest.raises(ValueError):
        training.clip_gradients_([f.cpu()], 1.0)
    # what is written may not overlap, what is only read may
    run = torch.ones(10, device=DEV)
    for grads, out in (([run[:6], run[4:]], None), ([run[:4], run[4:8]], [run[:4], run[3:7]]), ([f, None], None)):
        with pytest.raises((ValueError, TypeError)):
            training.clip_gradients_(grads, 1.0, out=out)
    assert training.gradient_norm([run[:6], run[4:]]).item() == pytest.approx(12 ** 0.5, rel=2.0 ** -22)
    training.clip_gradients_([run[4:8], run[:0], run[:4], run[8:]], 1.0)
    L = _lib.lib()
    ws = torch.empty(1 << 20, dtype=torch.uint8, device=DEV)
    assert L.ds_embed(ids.data_ptr(), 3, w.data_ptr(), 8, f.data_ptr(), 4, 5, 8, 1.0, 0, None) == -1
    assert L.ds_embed(ids.data_ptr(), 8, w.data_ptr(), 7, f.data_ptr(), 4, 5, 8, 1.0, 0, None) == -1
    assert L.ds_embed_grad(ids.data_ptr(), 8, f.data_ptr(), 8, w.data_ptr(), 4, 5, 8, -1, 1.0, 0, ws.data_ptr(), 16, None) == -4
    assert L.ds_embed_grad(ids.data_ptr(), 8, f.data_ptr(), 8, w.data_ptr(), 4, 5, 8, -1, 1.0, 7, ws.data_ptr(), 1 << 20, None) == -1


# ---- together -----------------------------------------------------------------------------------------------------

def test_a_step_of_the_token_model_against_plain_torch():
    from deepshift_amd import train_tokens
    torch.manual_seed(5)
    with torch.device(DEV):
        model = train_tokens.TokenModel(300, 32, 2)
    generator = torch.Generator(device=DEV).manual_seed(1)
    pair, target = train_tokens.batch(200, 300, torch.device(DEV), generator, ignored=0.2)
    loss = model(pair, target)
    loss.backward()
    got = {n: p.grad.clone() for n, p in model.named_parameters()}
    model.zero_grad()
    x = torch.nn.functional.embedding(pair, model.embedding.weight).mul(model.embedding.scale).flatten(1)
    for norm, layer in zip(model.norms, model.layers):
        x = x + torch.relu(layer(norm(x)))
    want = torch.nn.functional.cross_entropy(model.head.logits(x), target)
    want.backward()
    torch.testing.assert_close(loss, want, rtol=1e-5, atol=0)
    for n, p in model.named_parameters():
        # the same float32 layers between: what differs is the order of sums
        assert (got[n] - p.grad).norm() <= 1e-4 * p.grad.norm(), n


@pytest.mark.parametrize("shift_type", ["PS", "Q"])
def test_the_token_model_learns(shift_type):
    from deepshift_amd import train_tokens
    first, last = train_tokens.main(["--steps", "60", "--tokens", "2048", "--vocabulary", "64", "--width", "128", "--depth", "1",
                                     "--shift-type", shift_type, "--lr", "0.01"])
    assert last < 0.8 * first
