"""GPU: the gated block (deepshift_amd.training.gated_linear) against its definition in 64 bits.

Bounds are derived, not tuned.  With u the rounding of the operands' type (2^-24, 2^-8, 2^-11) and e = 2^-23:

* a projection of D products is off by d = (D + 16) e (sum |x w| + |b|) (float32's planes leave out less than 2^-24 of a product);
* an activation or its slope at g is off by its own steepness times what g is off by, and by (g^2 + |g| + 16) e of itself: its
  argument is rounded once, and the error function's tail moves g^2 times as much;
* gradients use the projections in 32 bits, and dz is rounded to the operands' type once for its products
  (float16's dz is scaled: what is below 2^-39 of the largest is lost);
* a sum of n products in 32 bits, in any grouping, is off by n e sum |a b| and what its terms are off by; results are rounded once.
"""
import math

import pytest
import torch
import torch.nn.functional as F_

from deepshift_amd import training
from tests.conftest import Tune

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -100, torch.bfloat16: 2.0 ** -100, torch.float16: 2.0 ** -24}
KINDS = ["silu", "gelu", "relu", "sigmoid"]
STEEP = {"silu": 1.1, "gelu": 1.13, "relu": 1.0, "sigmoid": 0.25}    # largest slopes
BENT = {"silu": 0.5, "gelu": 0.8, "relu": 0.0, "sigmoid": 0.1}       # largest second derivatives
FUNCTIONS = {"silu": F_.silu, "gelu": F_.gelu, "relu": torch.relu, "sigmoid": torch.sigmoid}


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


def _slope(kind, g):
    with torch.enable_grad():
        g = g.clone().requires_grad_()
        return torch.autograd.grad(FUNCTIONS[kind](g).sum(), g)[0]


def _check(x, w, b, kind, grad, out, dx=None, dw=None, db=None):
    dtype = x.dtype
    u, tiny = U[dtype], TINY[dtype]
    T, D, F = x.shape[:-1].numel(), x.shape[-1], w.shape[0] // 2
    xd, wd = x.reshape(T, D).double(), w.double()
    bd = torch.zeros(2 * F, dtype=torch.float64, device=DEV) if b is None else b.double()
    z = xd @ wd.t().contiguous() + bd
    d = (D + 16) * E * (xd.abs() @ wd.abs().t().contiguous() + bd.abs())
    g, up, dg, dup = z[:, :F], z[:, F:], d[:, :F], d[:, F:]
    act = FUNCTIONS[kind](g)
    off_act = STEEP[kind] * dg + (g * g + g.abs() + 16) * E * act.abs()
    y = act * up
    _within(out.reshape(T, F), y, (off_act * (up.abs() + dup) + act.abs() * dup) * (1 + u) + (u + E) * y.abs() + tiny, "out")
    if dx is None and dw is None and db is None:
        return
    dy = grad.reshape(T, F).double()
    slope = _slope(kind, g)
    off_slope = BENT[kind] * dg + (g * g + g.abs() + 16) * E * (slope.abs() + (g * g).clamp(max=1))
    if kind == "relu":
        off_slope = torch.where(g.abs() <= dg, 1.0, 0.0).double()
    off_act = STEEP[kind] * dg + (g * g + g.abs() + 16) * E * act.abs()
    dz = torch.cat([dy * up * slope, dy * act], 1)
    off = torch.cat([dy.abs() * (off_slope * (up.abs() + dup) + slope.abs() * dup), dy.abs() * off_act], 1) + 4 * E * dz.abs()
    loose = off.clone()
    loose += u * (dz.abs() + off)
    if dtype == torch.float16:
        loose += dz.abs().max() * 2.0 ** -38 if dz.numel() else 0
    for name, got, a, b_, n in (("dx", dx, (dz, loose), (wd, None), 2 * F), ("dw", dw, (dz.t(), loose.t()), (xd, None), T)):
        if got is None:
            continue
        left, leftoff, right = a[0].contiguous(), a[1].contiguous(), b_[0]
        want = left @ right
        bound = leftoff @ right.abs() + (n + 16) * E * (left.abs() @ right.abs())
        _within(got.reshape(want.shape), want, bound * (1 + u) + u * want.abs() + tiny, name)
    if db is not None:
        want = dz.sum(0)
        _within(db, want, (off.sum(0) + (T + 16) * E * dz.abs().sum(0)) * (1 + u) + u * want.abs() + tiny, "db")


def _step(x, w, b, kind, grad):
    leaves = [t.detach().requires_grad_() for t in (x, w, b) if t is not None]
    out = training.gated_linear(leaves[0], leaves[1], leaves[2] if b is not None else None, kind)
    return [out.detach()] + list(torch.autograd.grad(out, leaves, grad))


def _case(T, D, F, dtype, bias, *key):
    g = _gen(T, D, F, *key)
    return (_rand(g, T, D, dtype=dtype), _rand(g, 2 * F, D, dtype=dtype, scale=1.5 / math.sqrt(D)),
            _rand(g, 2 * F, dtype=dtype, scale=0.5) if bias else None, _rand(g, T, F, dtype=dtype))


SHAPES = [(1, 1, 1), (1, 8, 8), (3, 5, 7), (2, 64, 32), (64, 64, 64), (65, 100, 33), (130, 64, 256), (300, 257, 129),
          (257, 128, 500), (1, 512, 1000), (17, 1024, 96)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("tile", [None, 0, 1, 2, 3])
def test_results_and_gradients(dtype, tile):
    for i, (T, D, F) in enumerate(SHAPES):
        print(T, D, F, flush=True)
        kind, bias = KINDS[i % 4], i % 3 != 0
        x, w, b, grad = _case(T, D, F, dtype, bias)
        with Tune(vocab_tile=tile):
            got = _step(x, w, b, kind, grad)
            plain = training.gated_linear(x, w, b, kind)
            again = _step(x, w, b, kind, grad)
        assert torch.equal(plain, got[0])
        assert all(torch.equal(p, q) for p, q in zip(got, again))
        _check(x, w, b, kind, grad, *got)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_activations(dtype, kind):
    x, w, b, grad = _case(200, 96, 160, dtype, True, kind)
    _check(x, w, b, kind, grad, *_step(x, w, b, kind, grad))
    # far out on both sides
    x, w, b, grad = _case(40, 64, 64, dtype, True, kind, 1)
    x = x * 12
    _check(x, w, b, kind, grad, *_step(x, w, b, kind, grad))


@pytest.mark.parametrize("T", [1, 16, 17, 130])
def test_few_tokens_of_large_float32_weights(T):
    # weights that are split into planes where they are needed; from some number of tokens on beforehand
    for D, F in ((1024, 4096), (1028, 4099)):
        x, w, b, _ = _case(T, D, F, torch.float32, True)
        _check(x, w, b, "silu", None, training.gated_linear(x, w, b, "silu"))
    big = w.clone()
    big[5, 3] = 3.4e38
    big[4099 + 7, 9] = -3.4e38
    out = training.gated_linear(x * 1e-3, big, b, "relu")
    want = torch.relu((x * 1e-3).double() @ big[:F].t().double() + b[:F].double()) * \
        ((x * 1e-3).double() @ big[F:].t().double() + b[F:].double())
    here = want.abs() < 3e38
    assert torch.allclose(out.double()[here], want[here], rtol=1e-3, atol=1e-3)    # what is compared is that nothing is lost


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_one_token_and_a_few(dtype):
    # weights as they lie, whole pieces of them and what is left, rows anywhere
    for i, (D, F) in enumerate(((4096, 24), (2048, 1), (1032, 70), (2049, 33), (1, 3), (777, 50), (8192 + 520, 9))):
        wide = _rand(_gen(D, F), 2 * F, D + 3, dtype=dtype, scale=1.5 / math.sqrt(D))
        for T in (1, 2, 3, 4, 5, 8, 9):
            x, w, b, grad = _case(T, D, F, dtype, T % 2 == 0, i)
            for weight in (w, wide[:, 1:D + 1]):
                print(T, D, F, flush=True)
                got = _step(x, weight, b, KINDS[(T + i) % 4], grad)
                assert torch.equal(got[0], training.gated_linear(x, weight, b, KINDS[(T + i) % 4]))
                _check(x, weight, b, KINDS[(T + i) % 4], grad, *got)
    x, w, b, _ = _case(1, 512, 64, dtype, True)
    graph = torch.cuda.CUDAGraph()
    training.gated_linear(x, w, b)
    with torch.cuda.graph(graph):
        out = training.gated_linear(x, w, b)
    for i in range(3):
        x.copy_(_rand(_gen(i), 1, 512, dtype=dtype))
        graph.replay()
        assert torch.equal(out, training.gated_linear(x, w, b))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(dtype):
    g = _gen(3)
    T, D, F = 70, 64, 72
    x, w, b, grad = _case(T, D, F, dtype, True)
    wide_x, wide_w = _rand(g, T, D + 9, dtype=dtype), _rand(g, 2 * F, 2 * D, dtype=dtype, scale=0.2)
    wide_grad = _rand(g, T, F + 5, dtype=dtype)
    for name, (x2, w2, b2, g2) in {
            "rows apart": (wide_x[:, :D], wide_w[:, :D], b, wide_grad[:, :F]),
            "odd starts": (wide_x[:, 9:], wide_w[:, 3:D + 3], b, wide_grad[:, 5:]),
            "columns apart": (x.t().contiguous().t(), w.t().contiguous().t(), b.repeat_interleave(2)[::2], grad.t().contiguous().t()),
            "one for all": (x[:1].expand(T, D), w[:1].expand(2 * F, D), b[:1].expand(2 * F), grad[:1, :1].expand(T, F))}.items():
        print(name, flush=True)
        _check(x2, w2, b2, "silu", g2, *_step(x2, w2, b2, "silu", g2))
    # any number of leading axes
    for shape in ((7, 10), (7, 2, 5)):
        got = _step(x.view(*shape, D), w, b, "gelu", grad.view(*shape, F))
        want = _step(x, w, b, "gelu", grad)
        assert got[0].shape == shape + (F,) and got[1].shape == shape + (D,)
        assert all(torch.equal(p.reshape(q.shape), q) for p, q in zip(got, want))
    one = _step(x[0], w, b, "silu", grad[0])
    assert one[0].shape == (F,) and one[1].shape == (D,)
    _check(x[:1], w, b, "silu", grad[:1], *one)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_of_one_operand_alone(dtype):
    x, w, b, grad = _case(50, 40, 24, dtype, True, 4)
    want = _step(x, w, b, "gelu", grad)
    for i in range(3):
        leaves = [t.detach().requires_grad_(i == k) for k, t in enumerate((x, w, b))]
        got, = torch.autograd.grad(training.gated_linear(*leaves, "gelu"), leaves[i], grad)
        assert torch.equal(got, want[1 + i])


def test_float16_gradients_keep_their_bits_whatever_their_size():
    for size in (1e-7, 1e-4, 1.0, 200.0):
        x, w, b, grad = _case(100, 64, 48, torch.float16, True, 5)
        grad = (grad.float() * size).half()
        _check(x, w, b, "silu", grad, *_step(x, w, b, "silu", grad))
    # nothing at all, and one value that is none
    zero = torch.zeros_like(grad)
    assert all((t == 0).all() for t in _step(x, w, b, "silu", zero)[1:])
    for bad in (float("inf"), float("nan")):
        grad = _rand(_gen(6), 100, 48, dtype=torch.float16)
        want = _step(x, w, b, "silu", grad)
        grad[3, 4] = bad
        got = _step(x, w, b, "silu", grad)
        rows = [i for i in range(100) if i != 3]
        words = [i for i in range(96) if i % 48 != 4]
        off = (got[1].float()[rows] - want[1].float()[rows]).abs().max() <= 2 * U[torch.float16] * want[1].float()[rows].abs().max()
        assert off and not got[1][3].isfinite().any()
        assert got[2][words].isfinite().all() and not got[2][4].isfinite().any() and not got[2][52].isfinite().any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_what_is_no_number_stays_where_it_belongs(dtype):
    x, w, b, grad = _case(80, 64, 40, dtype, True, 7)
    want = _step(x, w, b, "silu", grad)
    bad = x.clone()
    bad[9, 5] = float("nan")
    got = _step(bad, w, b, "silu", grad)
    others = [i for i in range(80) if i != 9]
    assert torch.equal(got[0][others], want[0][others]) and got[0][9].isnan().all()
    assert torch.equal(got[1][others], want[1][others]) and got[1][9].isnan().all()
    bad = w.clone()
    bad[6, 5] = float("nan")
    got = _step(x, bad, b, "silu", grad)
    others = [i for i in range(40) if i != 6]
    assert torch.equal(got[0][:, others], want[0][:, others]) and got[0][:, 6].isnan().all()
    words = others + [i + 40 for i in others]
    assert torch.equal(got[3][words], want[3][words])


def test_gradients_against_differences():
    x, w, b, grad = _case(30, 24, 20, torch.float32, True, 8)
    g = _gen(9)
    for kind in ("silu", "gelu", "sigmoid"):
        got = _step(x, w, b, kind, grad)

        def value(x, w, b):
            z = x @ w.t().contiguous() + b
            return (FUNCTIONS[kind](z[:, :20]) * z[:, 20:] * grad.double()).sum()

        operands = [t.double() for t in (x, w, b)]
        for i in range(3):
            way = torch.randn(operands[i].shape, generator=g, dtype=torch.float64).to(DEV)
            step = 1e-3
            ends = [value(*[t + s * step * way if k == i else t for k, t in enumerate(operands)]) for s in (1, -1, 2, -2)]
            slope = (8 * (ends[0] - ends[1]) - (ends[2] - ends[3])) / (12 * step)
            along = (got[1 + i].double() * way).sum()
            # float32: a thousand roundings of the terms' size at most; the differences: step^4 of the fifth derivative
            assert abs(along - slope) <= 1000 * E * (got[1 + i].double().abs() * way.abs()).sum() + 1e-6 * abs(slope) + 1e-6


def test_many_tokens():
    # more of them than a launch's second axis has workgroups of 64 for, too
    for dtype in TYPES:
        for T, D, F in ((70001, 16, 24), (4300001, 8, 8)):
            x, w, b, grad = _case(T, D, F, dtype, True, 12)
            _check(x, w, b, "silu", grad, *_step(x, w, b, "silu", grad))


def test_two_streams_at_once():
    for dtype in TYPES:
        cases = [_case(90, 64, 200, dtype, True, 14, i) for i in range(2)]
        want = [_step(x, w, b, "gelu", grad) for x, w, b, grad in cases]
        streams = [torch.cuda.Stream() for _ in cases]
        for s in streams:
            s.wait_stream(torch.cuda.current_stream())
        got = [[], []]
        for _ in range(10):
            for (x, w, b, grad), s, results in zip(cases, streams, got):
                with torch.cuda.stream(s):
                    results.append(_step(x, w, b, "gelu", grad))
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for results, first in zip(got, want) for one in results for p, q in zip(one, first))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_a_few_tokens_of_shared_memory(dtype):
    x, w, b, grad = _case(3, 64, 40, dtype, True, 13)
    for x2, w2 in ((x[:1].expand(3, 64), w), (x, w[:1].expand(80, 64)), (x.t().contiguous().t(), w.t().contiguous().t())):
        _check(x2, w2, b, "gelu", grad, *_step(x2, w2, b, "gelu", grad))


def test_empty_sizes():
    for T, D, F in ((0, 8, 4), (5, 0, 4), (5, 8, 0), (0, 0, 0)):
        x, w, b = [torch.randn(*s, device=DEV, requires_grad=True) for s in ((T, D), (2 * F, D), (2 * F,))]
        out = training.gated_linear(x, w, b)
        assert out.shape == (T, F)
        if D == 0 and F:
            _check(x.detach(), w.detach(), b.detach(), "silu", None, out.detach())
        dx, dw, db = torch.autograd.grad(out.sum(), (x, w, b))
        assert dx.shape == x.shape and dw.shape == w.shape and db.shape == b.shape
        assert (dx == 0).all() and (dw == 0).all()
        if T == 0:
            assert (db == 0).all()


def test_offsets_beyond_32_bits():
    # halves of the weights 2.2 GB apart, results of 2.1 G elements
    T, D, F = 2, 16, 70000000 // 2
    w = torch.zeros(2 * F, D, dtype=torch.bfloat16, device=DEV)
    g = _gen(10)
    w[-100:] = _rand(g, 100, D, dtype=torch.bfloat16)
    w[F - 100:F] = _rand(g, 100, D, dtype=torch.bfloat16)
    x = _rand(g, T, D, dtype=torch.bfloat16)
    out = training.gated_linear(x, w)
    ends = torch.cat([w[F - 100:F], w[-100:]])
    _check(x, ends, None, "silu", None, out[:, -100:])
    assert (out[:, :F - 100] == 0).all()
    del out, w
    T, D, F = 70000, 16, 32768
    w, x = _rand(g, 2 * F, D, dtype=torch.bfloat16), _rand(g, T, D, dtype=torch.bfloat16)
    out = training.gated_linear(x, w)
    _check(x[-50:], w, None, "silu", None, out[-50:])


def test_another_stream_and_captured_replays():
    for dtype in TYPES:
        x, w, b, grad = _case(100, 72, 60, dtype, True, 11)
        want = _step(x, w, b, "silu", grad)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _step(x, w, b, "silu", grad)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = _step(x, w, b, "silu", grad)
        with torch.cuda.graph(other, pool=graph.pool()):
            twice = _step(x, w, b, "gelu", grad)
        for i in range(3):
            x.copy_(_rand(_gen(i), 100, 72, dtype=dtype))
            grad.mul_(0.5)
            for replay, kind, results in ((graph, "silu", captured), (other, "gelu", twice), (graph, "silu", captured)):
                replay.replay()
                torch.cuda.synchronize()
                want = _step(x, w, b, kind, grad)
                assert all(torch.equal(p, q) for p, q in zip(results, want)), "replay %d" % i


def test_module():
    torch.manual_seed(0)
    block = training.GatedLinear(48, 40, activation="gelu").to(DEV)
    x = torch.randn(5, 7, 48, device=DEV)
    out = block(x)
    _check(x, block.weight.detach(), block.bias.detach(), "gelu", None, out.detach())
    out.sum().backward()
    assert block.weight.grad.shape == (80, 48) and block.bias.grad.shape == (80,)


@pytest.mark.parametrize("shift_type", ["PS", "Q"])
def test_weights_of_powers_of_two(shift_type):
    torch.manual_seed(1)
    block = training.GatedShift(48, 40, activation="silu", shift_type=shift_type, weight_bits=5).to(DEV)
    layer = block.layer
    x = torch.randn(9, 48, device=DEV)
    grad = torch.randn(9, 40, device=DEV)
    out = block(x)
    weight, inputs = layer.float_weight().detach(), layer.float_input(x).detach()
    _check(inputs, weight, layer.bias.detach(), "silu", None, out.detach())
    z = layer(x)
    assert torch.allclose(out, F_.silu(z[:, :40]) * z[:, 40:], rtol=1e-4, atol=1e-4 * float(z.detach().abs().max()) ** 2)
    parameters = list(layer.parameters())
    got = torch.autograd.grad(out, parameters, grad)
    leaf = weight.clone().requires_grad_()
    dw, = torch.autograd.grad(training.gated_linear(inputs, leaf, layer.bias, "silu"), leaf, grad)
    want = torch.autograd.grad(layer.float_weight(), [p for p in parameters if p is not layer.bias], dw)
    assert all(torch.equal(p, q) for p, q in zip([p for p, q in zip(got, parameters) if q is not layer.bias], want))
    # on the shift kernels
    layer.use_kernel = True
    with torch.no_grad():
        z = layer(x)
        assert torch.equal(block(x), F_.silu(z[:, :40]) * z[:, 40:])


def test_refusals_on_the_gpu():
    x, w, b = torch.zeros(4, 8, device=DEV), torch.zeros(12, 8, device=DEV), torch.zeros(12, device=DEV)
    for error, call in ((ValueError, lambda: training.gated_linear(x, w[:11], b)), (ValueError, lambda: training.gated_linear(x, w.t(), b)),
                        (TypeError, lambda: training.gated_linear(x, w.half(), b)), (ValueError, lambda: training.gated_linear(x, w, b[:6])),
                        (TypeError, lambda: training.gated_linear(x, w.cpu(), b)), (ValueError, lambda: training.gated_linear(x, w, b, "tanh")),
                        (TypeError, lambda: training.gated_linear(x.double(), w, b)), (ValueError, lambda: training.gated_linear(x[0, 0], w, b))):
        with pytest.raises(error):
            call()
    x.requires_grad_()
    dx, = torch.autograd.grad(training.gated_linear(x, w).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_activations_on_the_same_inputs_every_time(dtype, kind):
    # (strings hash to other numbers in every process: seeds are numbers)
    x, w, b, grad = _case(200, 96, 160, dtype, True, KINDS.index(kind), 61)
    _check(x, w, b, kind, grad, *_step(x, w, b, kind, grad))
    x, w, b, grad = _case(40, 64, 64, dtype, True, KINDS.index(kind), 62)
    x = x * 12
    _check(x, w, b, kind, grad, *_step(x, w, b, kind, grad))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("kind", KINDS)
def test_infinite_operands(dtype, kind):
    # infinities of x, of either half's weights, of both and of a bias: results as the formula has them, the others as ever
    for T, D, F, tiles in ((90, 72, 40, (None, 0, 1, 2, 3)), (3, 200, 50, (None,)), (40, 1024, 4096, (None,)), (300, 257, 129, (None,))):
        x, w, b, _ = _case(T, D, F, dtype, True, KINDS.index(kind), 63)
        inf = float("inf")
        x[T // 2, 5], x[1, D - 1] = inf, -inf
        w[6, 7], w[F + 9, 5], w[F - 1, D - 1], b[F + 11], b[3] = -inf, inf, inf, inf, -inf
        z = x.double() @ w.double().t().contiguous() + b.double()
        want = FUNCTIONS[kind](z[:, :F]) * z[:, F:]
        for tile in tiles:
            print(T, D, F, tile, flush=True)
            with Tune(vocab_tile=tile):
                out = training.gated_linear(x, w, b, kind)
            assert torch.equal(out.isnan(), want.isnan())
            assert torch.equal(out.isposinf(), want.isposinf()) and torch.equal(out.isneginf(), want.isneginf())
            rows = [t for t in range(T) if t not in (T // 2, 1)]
            units = [f for f in range(F) if f not in (6, 9, F - 1, 11, 3)]
            both = units + [F + f for f in units]
            _check(x[rows], w[both], b[both], kind, None, out[rows][:, units])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_that_lie_in_other_ways(dtype):
    # what a sum, a mean, a transposed or a repeated result hands back
    x, w, b, grad = _case(60, 40, 24, dtype, True, 64)
    for make in (lambda out: out.sum(), lambda out: (out.t() * grad.t()).sum(), lambda out: out[:, :1].sum(),
                 lambda out: (out.unsqueeze(0) * grad).sum() + out.mean()):
        leaves = [t.detach().requires_grad_() for t in (x, w, b)]
        out = training.gated_linear(*leaves)
        given, = torch.autograd.grad(make(out), out, retain_graph=True)
        got = torch.autograd.grad(make(out), leaves)
        _check(x, w, b, "silu", given, out.detach(), *got)
