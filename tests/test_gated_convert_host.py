"""CPU: models with gated blocks are converted to shift layers with them."""
import copy

import pytest
import torch
import torch.nn as nn
import torch.nn.functional as F

from deepshift_amd import convert, modules, modules_q, training


def _model(bias):
    torch.manual_seed(0)
    return nn.Sequential(nn.Linear(6, 8), nn.Sequential(training.GatedLinear(8, 5, bias=bias, activation="gelu")), nn.Linear(5, 3))


@pytest.mark.parametrize("shift_type", ["PS", "Q"])
@pytest.mark.parametrize("bias", [True, False])
def test_gated_blocks_become_gated_shift(shift_type, bias):
    model = _model(bias)
    weight = model[1][0].weight.detach().clone()
    model, _ = convert.convert_to_shift(model, 100, shift_type, convert_weights=True)
    block = model[1][0]
    kind = modules.LinearShift if shift_type == "PS" else modules_q.LinearShiftQ
    assert isinstance(block, training.GatedShift) and type(block.layer) is kind and type(model[0]) is kind and type(model[2]) is kind
    assert (block.in_features, block.out_features, block.activation) == (8, 5, "gelu")
    assert tuple(block.layer.float_weight().shape) == (10, 8) and (block.layer.bias is not None) == bias
    # its weights are the block's, to the nearest power of two
    sizes = block.layer.float_weight().detach()
    assert torch.equal(sizes.sign(), weight.sign()) and ((sizes / weight).log2().abs() <= 0.5 + 1e-5)[weight.abs() > 2.0 ** -14].all()
    assert convert.count_layer_type(model, kind) == 3 and convert.count_layer_type(model, training.GatedLinear) == 0
    rounded = convert.round_shift_weights(model, clone=True)
    assert torch.equal(rounded[1][0].layer.float_weight(), sizes)


def test_a_part_of_the_layers():
    model, count = convert.convert_to_shift(_model(True), 2, "PS", convert_all_linear=False, convert_weights=True)
    assert count == 2 and type(model[0]) is nn.Linear and type(model[2]) is modules.LinearShift
    assert isinstance(model[1][0], training.GatedShift)
    model, count = convert.convert_to_shift(_model(True), 1, "PS", convert_all_linear=False, convert_weights=True)
    assert count == 1 and type(model[1][0]) is training.GatedLinear


@pytest.mark.parametrize("shift_type", ["PS", "Q"])
def test_converted_blocks_run_on_the_shift_kernels(shift_type):
    model = copy.deepcopy(_model(True))
    model, _ = convert.convert_to_shift(model, 100, shift_type, convert_weights=True, use_kernel=True, use_cuda=False)
    x = torch.randn(4, 7, 6)
    with torch.no_grad():
        got = model(x)
        block = model[1][0]
        inner = model[0](x)
        gate, up = F.linear(inner, block.layer.float_weight(), block.layer.bias).chunk(2, -1)
        want = model[2](F.gelu(gate) * up)
    # inputs and biases are off by 2^-16, times at most 8 weights of up to 1, a slope of 1.13, factors below 8 and 5 weights more
    assert got.shape == (4, 7, 3) and (got - want).abs().max() <= 2.0 ** -8


def test_a_layer_of_another_size_is_refused():
    with pytest.raises(ValueError, match="layer must have"):
        training.GatedShift(8, 5, layer=modules.LinearShift(8, 5))
    layer = modules.LinearShift(8, 10)
    assert training.GatedShift(8, 5, layer=layer).layer is layer
