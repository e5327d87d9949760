"""GPU: the gated recurrence (deepshift_amd.training.gated_recurrence) against its definition in 64 bits.

Bounds are derived, not tuned.  With u the rounding of the output's type (2^-24, 2^-8, 2^-11) and e = 2^-23: a gate's sides are
off by at most 4 e of themselves (an exponential, an addition, a reciprocal and a product of a unit in the last place each), and
a token adds at most four roundings to what reaches it, its share in the products over stretches included.  So a state is off by
E[t] = a[t] E[t - 1] + 8 e S[t], with S[t] = a[t] S[t - 1] + (1 - a[t]) |x[t]| the sum of its magnitudes, and the gradient of
one by the same along the way back; what is formed from them adds the products' own errors and one rounding.
"""
import pytest
import torch

from deepshift_amd import training
from tests.conftest import Tune

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
E = 2.0 ** -23
TYPES = [torch.float32, torch.bfloat16, torch.float16]
U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
TINY = {torch.float32: 2.0 ** -120, torch.bfloat16: 2.0 ** -120, torch.float16: 2.0 ** -24}


def _gen(*key):
    return torch.Generator().manual_seed(hash(key) & 0x7fffffff)


def _rand(g, *shape, dtype=torch.float32, scale=1.0, shift=0.0):
    return (torch.randn(shape, generator=g) * scale + shift).to(dtype).to(DEV)


def _within(got, want, bound, what):
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    assert not bad.any(), "%s: %d of %d values off, worst %.3g times the bound" % (
        what, int(bad.sum()), bad.numel(), float((off / bound.clamp(min=1e-300)).nan_to_num(float("inf")).max()))


class Exact:
    """Results and their bounds in 64 bits, token by token."""

    def __init__(self, x, gate, state, lengths, grad=None, grad_last=None):
        B, T, D = x.shape
        u, tiny = U[x.dtype], TINY[x.dtype]
        inside = torch.ones(B, T, 1, dtype=torch.bool, device=DEV)
        if lengths is not None:
            inside = (torch.arange(T, device=DEV) < lengths.clamp(0, T)[:, None])[..., None]
        v = torch.where(inside, x.double(), 0)
        a = torch.where(inside, torch.sigmoid(gate.double()), 1)
        away = torch.where(inside, torch.sigmoid(-gate.double()), 0)
        zero = torch.zeros(B, D, dtype=torch.float64, device=DEV)
        h = zero if state is None else state.double()
        s, off = h.abs(), zero
        hs, ss, offs = [h], [s], [off]
        for t in range(T):
            h = a[:, t] * h + away[:, t] * v[:, t]
            s = a[:, t] * s + away[:, t] * v[:, t].abs()
            off = a[:, t] * off + torch.where(inside[:, t], 8 * E * s, 0)
            hs.append(h), ss.append(s), offs.append(off)
        hs, ss, offs = torch.stack(hs, 1), torch.stack(ss, 1), torch.stack(offs, 1)
        self.out = torch.where(inside, hs[:, 1:], 0)
        self.out_bound = torch.where(inside, offs[:, 1:] * (1 + u) + u * hs[:, 1:].abs() + tiny, 0)
        self.last, self.last_bound = h, off + TINY[torch.float32]
        if grad is None and grad_last is None:
            return
        dh = torch.zeros_like(v) if grad is None else torch.where(inside, grad.double(), 0)
        m = zero if grad_last is None else grad_last.double()
        n, off = m.abs(), zero
        dx, dg, bx, bg = [], [], [], []
        for t in range(T - 1, -1, -1):
            l, big = dh[:, t] + m, dh[:, t].abs() + n
            here = inside[:, t]
            apart, apart_abs = hs[:, t] - v[:, t], ss[:, t] + v[:, t].abs()
            slope = a[:, t] * away[:, t]
            dx.append(torch.where(here, away[:, t] * l, 0))
            bx.append(torch.where(here, away[:, t] * (off + 6 * E * big), 0))
            dg.append(torch.where(here, slope * l * apart, 0))
            bg.append(torch.where(here, slope * (off * apart.abs() + big * (offs[:, t] + 16 * E * apart_abs)), 0))
            off = torch.where(here, a[:, t] * (off + 8 * E * big), off)
            m, n = a[:, t] * l, a[:, t] * big
        self.grads, self.grad_bounds = [], []
        for values, bounds in ((dx, bx), (dg, bg)):
            value = torch.stack(values[::-1], 1) if values else torch.zeros_like(v)
            bound = torch.stack(bounds[::-1], 1) if bounds else torch.zeros_like(v)
            self.grads.append(value)
            self.grad_bounds.append(torch.where(inside, bound * (1 + u) + u * value.abs() + tiny, 0))
        self.grads.append(m), self.grad_bounds.append(off + TINY[torch.float32])


def _check(x, gate, state, lengths, grad, grad_last, got):
    want = Exact(x, gate, state, lengths, grad, grad_last)
    _within(got[0], want.out, want.out_bound, "out")
    _within(got[1], want.last, want.last_bound, "last")
    for name, value, exact, bound in zip(("dx", "dgate", "dstate"), got[2:], getattr(want, "grads", ()),
                                         getattr(want, "grad_bounds", ())):
        if value is not None:
            _within(value, exact, bound, name)


def _step(x, gate, state, lengths, grad, grad_last):
    x, gate = x.detach().requires_grad_(), gate.detach().requires_grad_()
    state = None if state is None else state.detach().requires_grad_()
    leaves = [t for t in (x, gate, state) if t is not None]
    out, last = training.gated_recurrence(x, gate, state, lengths)
    pairs = [(o, g) for o, g in ((out, grad), (last, grad_last)) if g is not None]
    grads = list(torch.autograd.grad([o for o, _ in pairs], leaves, [g for _, g in pairs]))
    return [out.detach(), last.detach()] + grads


SHAPES = [(1, 1, 1), (3, 1, 64), (64, 1, 512), (2, 8, 5), (2, 9, 130), (1, 63, 66), (2, 64, 258), (2, 65, 128), (5, 129, 385),
          (3, 1000, 257), (1, 2500, 64)]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("segments", [None, 1, 3])
def test_states_and_gradients(dtype, segments):
    for B, T, D in SHAPES:
        for ragged in (False, True):
            print(B, T, D, ragged, flush=True)
            g = _gen(B, T, D, ragged)
            x, gate = _rand(g, B, T, D, dtype=dtype), _rand(g, B, T, D, dtype=dtype, scale=1.5, shift=1.5)
            state = _rand(g, B, D) if ragged or T % 2 else None
            lengths = None
            if ragged:
                lengths = torch.randint(0, T + 1, (B,), generator=g).to(DEV)
                lengths[0] = 0
                lengths[-1] = T
            grad, grad_last = _rand(g, B, T, D, dtype=dtype), _rand(g, B, D)
            with Tune(recur_segments=segments):
                got = _step(x, gate, state, lengths, grad, grad_last)
                again = _step(x, gate, state, lengths, grad, grad_last)
                plain = training.gated_recurrence(x, gate, state, lengths)
            assert all(torch.equal(p, q) for p, q in zip(got, again))
            assert torch.equal(plain[0], got[0]) and torch.equal(plain[1], got[1])
            _check(x, gate, state, lengths, grad, grad_last, got)


def test_what_lies_behind_a_sequences_end_is_not_looked_at():
    for dtype in TYPES:
        for T, D in ((20, 70), (300, 130)):
            g = _gen(T, D)
            B = 5
            lengths = torch.tensor([0, 1, T - 1, T, 7], device=DEV)
            x, gate, grad = [_rand(g, B, T, D, dtype=dtype) for _ in range(3)]
            state, grad_last = _rand(g, B, D), _rand(g, B, D)
            want = _step(x, gate, state, lengths, grad, grad_last)
            behind = torch.arange(T, device=DEV) >= lengths[:, None]
            for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
                for t in (x, gate, grad):
                    t[behind] = bad
                got = _step(x, gate, state, lengths, grad, grad_last)
                assert all(torch.equal(p, q) for p, q in zip(got, want))
            assert all((t[behind] == 0).all() for t in (got[0], got[2], got[3]))
            assert torch.equal(got[1][0], state[0]) and torch.equal(got[4][0], grad_last[0])
            # lengths in 32 bits, and such as are held to [0, T]
            wild = torch.tensor([-3, 1, T - 1, T + 9, 7], device=DEV, dtype=torch.int32)
            assert all(torch.equal(p, q) for p, q in zip(_step(x, gate, state, wild, grad, grad_last), want))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_sequences_in_pieces_go_on_from_the_last_state(dtype):
    g = _gen(5)
    B, T, D = 3, 150, 100
    x, gate, state = _rand(g, B, T, D, dtype=dtype), _rand(g, B, T, D, dtype=dtype, shift=2.0), _rand(g, B, D)
    want = Exact(x, gate, state, None)
    for cuts in ([0, 1, 2, 40, 149, 150], list(range(T + 1))):
        h, outs = state, []
        for s, t in zip(cuts, cuts[1:]):
            out, h = training.gated_recurrence(x[:, s:t], gate[:, s:t], h)
            outs.append(out)
        _within(torch.cat(outs, 1), want.out, want.out_bound, "out")
        _within(h, want.last, want.last_bound, "last")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_layouts(dtype):
    g = _gen(6)
    for B, T, D in ((2, 70, 64), (3, 33, 65), (2, 1, 130)):
        wide = _rand(g, B, T, 2 * D + 1, dtype=dtype)
        state, grad_last = _rand(g, B, D), _rand(g, B, D)
        grad = _rand(g, B, T, D, dtype=dtype)
        forms = {
            "halves": (wide[..., :D], wide[..., D:2 * D], grad),
            "odd starts": (wide[..., 1:D + 1], wide[..., D + 1:], grad),
            "tokens first": (wide[..., :D].transpose(0, 1).contiguous().transpose(0, 1), wide[..., D:2 * D],
                             grad.transpose(0, 1).contiguous().transpose(0, 1)),
            "channels apart": (wide[..., :2 * D:2], wide[..., 1:2 * D:2], grad.mT.contiguous().mT),
            "every other token": (wide.repeat_interleave(2, 1)[:, ::2, :D], wide[..., D:2 * D], grad),
            "one for all": (wide[:1, :, :D].expand(B, T, D), wide[:, :1, D:2 * D].expand(B, T, D), grad[:1, :1, :1].expand(B, T, D)),
        }
        for name, (x, gate, gr) in forms.items():
            print(name, flush=True)
            got = _step(x, gate, state, None, gr, grad_last)
            _check(x, gate, state, None, gr, grad_last, got)


def test_gradients_of_one_result_alone():
    g = _gen(7)
    for T in (1, 5, 200):
        x, gate, state = _rand(g, 2, T, 70), _rand(g, 2, T, 70), _rand(g, 2, 70)
        grad, grad_last = _rand(g, 2, T, 70), _rand(g, 2, 70)
        _check(x, gate, state, None, grad, None, _step(x, gate, state, None, grad, None))
        _check(x, gate, state, None, None, grad_last, _step(x, gate, state, None, None, grad_last))
        # of one operand alone
        want = _step(x, gate, state, None, grad, grad_last)
        for i in range(3):
            leaves = [t.detach().requires_grad_(i == k) for k, t in enumerate((x, gate, state))]
            out, last = training.gated_recurrence(*leaves)
            got, = torch.autograd.grad((out, last), leaves[i], (grad, grad_last))
            assert torch.equal(got, want[2 + i])


def test_gradients_of_a_shared_state():
    g = _gen(8)
    B, T, D = 4, 30, 66
    x, gate, first = _rand(g, B, T, D), _rand(g, B, T, D), _rand(g, D)
    grad, grad_last = _rand(g, B, T, D), _rand(g, B, D)
    leaf = first.clone().requires_grad_()
    out, last = training.gated_recurrence(x, gate, leaf.expand(B, D))
    got, = torch.autograd.grad((out, last), leaf, (grad, grad_last))
    want = Exact(x, gate, first.expand(B, D), None, grad, grad_last)
    _within(got, want.grads[2].sum(0), (want.grad_bounds[2] + B * E * want.grads[2].abs()).sum(0), "dstate")


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_extreme_gates(dtype):
    g = _gen(9)
    B, T, D = 2, 40, 64
    x, state = _rand(g, B, T, D, dtype=dtype), _rand(g, B, D)
    grad, grad_last = _rand(g, B, T, D, dtype=dtype), _rand(g, B, D)
    top = torch.finfo(dtype).max
    # kept for good, replaced at once, and a little of each
    for values in ([float("inf")], [-float("inf")], [top], [-top], [float("inf"), -float("inf")], [80.0, -80.0, 100.0, -100.0],
                   [15.0, -15.0, 0.0]):
        gate = torch.tensor(values, dtype=dtype, device=DEV)[torch.randint(0, len(values), (B, T, D), generator=g).to(DEV)]
        _check(x, gate, state, None, grad, grad_last, _step(x, gate, state, None, grad, grad_last))


def test_what_is_no_number_stays_in_its_channel():
    g = _gen(10)
    for T in (5, 200):
        x, gate, state, grad, last = (_rand(g, 2, T, 64), _rand(g, 2, T, 64), _rand(g, 2, 64), _rand(g, 2, T, 64),
                                      _rand(g, 2, 64))
        want = _step(x, gate, state, None, grad, last)
        for bad in (float("nan"), float("inf")):
            for which in range(5):
                args = [t.clone() for t in (x, gate, state, grad, last)]
                t = args[which]
                (t[1, T // 2] if t.dim() == 3 else t[1])[7] = bad
                got = _step(args[0], args[1], args[2], None, args[3], args[4])
                for p, q in zip(got, want):
                    p, q = p.clone(), q.clone()
                    p[1, ..., 7] = q[1, ..., 7] = 0
                    assert torch.equal(p, q)
                if which in (0, 1) and bad != bad:
                    assert got[0][1, T // 2:, 7].isnan().all() and not got[0][1, :T // 2, 7].isnan().any()


def test_gradients_against_differences():
    g = _gen(11)
    B, T, D = 2, 90, 33
    x, gate, state = _rand(g, B, T, D), _rand(g, B, T, D, shift=1.0), _rand(g, B, D)
    grad, grad_last = _rand(g, B, T, D), _rand(g, B, D)
    got = _step(x, gate, state, None, grad, grad_last)
    bounds = Exact(x, gate, state, None, grad, grad_last).grad_bounds

    def value(x, gate, state):
        h, total = state, 0.0
        for t in range(T):
            a = torch.sigmoid(gate[:, t])
            h = a * h + (1 - a) * x[:, t]
            total = total + (h * grad[:, t].double()).sum()
        return total + (h * grad_last.double()).sum()

    operands = [t.double() for t in (x, gate, state)]
    for i in range(3):
        way = torch.randn(operands[i].shape, generator=g, dtype=torch.float64).to(DEV)
        step = 1e-4
        ends = [value(*[t + s * step * way if k == i else t for k, t in enumerate(operands)]) for s in (1, -1, 2, -2)]
        slope = (8 * (ends[0] - ends[1]) - (ends[2] - ends[3])) / (12 * step)     # off by step^4 of the fifth derivative
        along = (got[2 + i].double() * way).sum()
        assert abs(along - slope) <= (bounds[i] * way.abs()).sum() + 1e-9 * abs(slope) + 1e-7, i


def test_empty_sizes():
    for B, T, D in ((0, 5, 4), (2, 5, 0), (2, 0, 4), (0, 0, 0)):
        x, gate = [torch.randn(B, T, D, device=DEV, requires_grad=True) for _ in range(2)]
        state = torch.randn(B, D, device=DEV, requires_grad=True)
        out, last = training.gated_recurrence(x, gate, state)
        assert out.shape == (B, T, D) and last.shape == (B, D) and (T > 0 or torch.equal(last, state))
        grads = torch.autograd.grad((out.sum() + last.sum(),), (x, gate, state))
        assert [t.shape for t in grads] == [x.shape, gate.shape, state.shape]
        if T == 0:
            assert torch.equal(grads[2], torch.ones(B, D, device=DEV))
    assert (training.gated_recurrence(torch.zeros(2, 0, 4, device=DEV), torch.zeros(2, 0, 4, device=DEV))[1] == 0).all()


def test_offsets_beyond_32_bits():
    # 2.1 G elements of one operand, of which the last sequence is checked
    B, T, D = 3, 11000, 65536
    x = torch.zeros(B, T, D, dtype=torch.bfloat16, device=DEV)
    gate = torch.zeros(1, 1, D, dtype=torch.bfloat16, device=DEV).expand(B, T, D)
    g = _gen(12)
    x[-1, -300:] = _rand(g, 300, D, dtype=torch.bfloat16)
    out, last = training.gated_recurrence(x, gate)
    want = Exact(x[-1:, -300:, -200:], gate[-1:, -300:, -200:], None, None)
    _within(out[-1:, -300:, -200:], want.out, want.out_bound, "out")
    _within(last[-1:, -200:], want.last, want.last_bound, "last")
    assert (out[0, :, -1] == 0).all() and (out[-1, :-300, -1] == 0).all()


def test_another_stream_and_captured_replays():
    g = _gen(13)
    for B, T, D in ((4, 1, 64), (2, 2000, 64)):
        x, gate, state = _rand(g, B, T, D), _rand(g, B, T, D), _rand(g, B, D)
        grad, grad_last = _rand(g, B, T, D), _rand(g, B, D)
        want = _step(x, gate, state, None, grad, grad_last)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = _step(x, gate, state, None, grad, grad_last)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(p, q) for p, q in zip(got, want))
        graph, other = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            captured = _step(x, gate, state, None, grad, grad_last)
        with torch.cuda.graph(other, pool=graph.pool()):
            twice = _step(gate, x, state, None, grad, grad_last)
        for i in range(3):
            x.copy_(_rand(g, B, T, D))
            graph.replay()
            other.replay()
            torch.cuda.synchronize()
            want = _step(gate, x, state, None, grad, grad_last)
            assert all(torch.equal(p, q) for p, q in zip(twice, want)), "replay %d" % i
            graph.replay()
            torch.cuda.synchronize()
            want = _step(x, gate, state, None, grad, grad_last)
            assert all(torch.equal(p, q) for p, q in zip(captured, want)), "replay %d" % i


def test_second_derivatives_are_refused():
    x, gate = [torch.randn(2, 3, 4, device=DEV, requires_grad=True) for _ in range(2)]
    dx, = torch.autograd.grad(training.gated_recurrence(x, gate)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        dx.sum().backward()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_gradients_that_lie_in_other_ways(dtype):
    # what a sum, a mean, a transposed or a repeated result hands back, of even and odd channels
    for B, T, D in ((3, 70, 66), (2, 9, 5), (1, 300, 1), (4, 1, 130)):
        g = _gen(B, T, D, 71)
        x, gate, state = _rand(g, B, T, D, dtype=dtype), _rand(g, B, T, D, dtype=dtype, shift=1.0), _rand(g, B, D)
        weight = _rand(g, B, T, D, dtype=dtype)
        for make in (lambda out, last: out.sum() + last.sum(), lambda out, last: (out.transpose(0, 1) * weight.transpose(0, 1)).sum(),
                     lambda out, last: out.mean(1).sum() + last[:, :1].sum(), lambda out, last: out[:, -1:].expand(B, 3, D).sum(),
                     lambda out, last: (out.transpose(1, 2) @ weight.float().to(dtype)).sum() if dtype == torch.float32 else last.t().sum()):
            leaves = [t.detach().requires_grad_() for t in (x, gate, state)]
            out, last = training.gated_recurrence(*leaves)
            given = torch.autograd.grad(make(out, last), (out, last), retain_graph=True, allow_unused=True)
            got = torch.autograd.grad(make(out, last), leaves)
            _check(x, gate, state, None, given[0], given[1], [out.detach(), last.detach()] + list(got))
