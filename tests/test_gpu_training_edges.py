"""GPU: what deepshift_amd.training does at the edges of its definition.

Bounds are those of test_gpu_training.py, but for what each test says.
"""
import pytest
import torch

from deepshift_amd import training
from tests.test_gpu_training import DEV, E, _gen, _rand

pytestmark = pytest.mark.gpu


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
