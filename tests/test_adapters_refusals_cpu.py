"""What the adapters' layers refuse or warn of, without a GPU."""
import warnings

import pytest
import torch

from rocm_qlora import LoRALinear, QuantLinear
from rocm_qlora.lora import AdapterRows, MultiLoRALinear, attach_adapters, multi_lora


def merged(q):
    """As LoRALinear.merge_lora leaves the quantized layer: its forward reads the merged weight."""
    q.merged_fp16_weight = torch.zeros(q.out_features, q.in_features, dtype=torch.float16)
    q.merged_mode = True
    return q


def test_merged_quantized_layers_are_refused():
    with pytest.raises(RuntimeError, match="merged"):
        MultiLoRALinear(merged(QuantLinear(64, 32, bits=4)), 2)
    layer = MultiLoRALinear(QuantLinear(64, 32, bits=4), 1)
    merged(layer.base_layer)
    with pytest.raises(RuntimeError, match="merged"):
        layer(torch.zeros(2, 64), AdapterRows.single(2))


def test_attach_adapters_refuses_a_merged_weight_before_it_changes_the_model():
    first = LoRALinear(QuantLinear(64, 64, bits=4), r=4)
    shared = QuantLinear(64, 64, bits=4)
    second = LoRALinear(shared, r=4)  # not merged itself; its quantized layer is, by another
    merged(shared)
    model = torch.nn.Sequential(first, second)
    with pytest.raises(RuntimeError, match="merged"):
        attach_adapters(model, 2)
    assert model[0] is first and model[1] is second


def test_scaling_that_asks_for_a_gradient_is_refused():
    x, a, b = torch.zeros(4, 32), torch.zeros(1, 4, 32), torch.zeros(1, 8, 4)
    s = torch.ones(1, requires_grad=True)
    with pytest.raises(RuntimeError, match="scaling"):
        multi_lora(x, a, b, s, AdapterRows.single(4))
    with torch.no_grad(), pytest.raises(RuntimeError, match="GPU"):  # nothing is recorded: as any other
        multi_lora(x, a, b, s, AdapterRows.single(4))


def test_attach_adapters_warns_of_the_dropout_it_leaves_out():
    model = torch.nn.Sequential(LoRALinear(QuantLinear(64, 64, bits=4), r=4, lora_dropout=0.1))
    with pytest.warns(UserWarning, match="dropout"):
        attach_adapters(model, 2)
    assert isinstance(model[0], MultiLoRALinear)
    with warnings.catch_warnings():
        warnings.simplefilter("error")
        attach_adapters(torch.nn.Sequential(LoRALinear(QuantLinear(64, 64, bits=4), r=4)), 2)
