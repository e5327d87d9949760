"""CPU: what deepshift_amd.training refuses rather than answer wrongly."""
import itertools

import pytest
import torch

from deepshift_amd import training


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
