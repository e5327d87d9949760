"""CPU: the float path of the shift layers leaves its parameters where they are."""
import pytest
import torch

from deepshift_amd import modules, modules_q

LAYERS = [lambda **o: modules.LinearShift(6, 4, **o), lambda **o: modules_q.LinearShiftQ(6, 4, **o),
          lambda **o: modules.Conv2dShift(3, 4, 3, **o), lambda **o: modules_q.Conv2dShiftQ(3, 4, 3, **o)]


def _parameter(layer):
    return layer.shift if hasattr(layer, "shift") else layer.weight


def _input(layer):
    return torch.randn(2, 6) if hasattr(layer, "in_features") else torch.randn(2, 3, 8, 8)


@pytest.mark.parametrize("make", LAYERS)
def test_a_forward_pass_clamps_in_the_parameters_own_memory(make):
    layer = make()
    p = _parameter(layer)
    p.data.mul_(300.0)
    at, version, alias = p.data_ptr(), p._version, p.detach()
    before = alias.clone()
    lowest, highest = layer.shift_range if hasattr(layer, "shift") else (-2.0 ** layer.shift_range[1], 2.0 ** layer.shift_range[1])
    for _ in range(2):
        layer(_input(layer)).sum().backward()
        assert p.data_ptr() == at and p._version - version <= 1 and p.is_leaf and p.requires_grad and not p.is_inference()
        # what is written later through the same memory is what the next pass reads
        assert torch.equal(alias, p) and p.min() >= lowest and p.max() <= highest
    assert (before.abs() > max(abs(lowest), abs(highest))).any() and p.grad is not None


@pytest.mark.parametrize("make", LAYERS)
def test_parameters_made_without_gradients_and_passes_without_them(make):
    with torch.inference_mode():
        made = make()
    made(_input(made))
    layer = make()
    with torch.inference_mode():
        layer(_input(layer))
    with torch.no_grad():
        layer(_input(layer))
    layer(_input(layer)).sum().backward()
    assert _parameter(layer).grad is not None


def test_an_expanded_parameter_is_taken_as_it_was():
    layer = modules.LinearShift(6, 4)
    layer.shift = torch.nn.Parameter(torch.full((1, 6), -90.0).expand(4, 6))
    same = modules.LinearShift(6, 4)
    same.load_state_dict(layer.state_dict())
    x = torch.randn(3, 6)
    assert torch.equal(layer(x), same(x)) and (layer.shift == layer.shift_range[0]).all()
    # rows of another order have memory of their own
    layer.shift = torch.nn.Parameter(torch.full((6, 4), -90.0).t())
    at = layer.shift.data_ptr()
    assert torch.equal(layer(x), same(x)) and layer.shift.data_ptr() == at
