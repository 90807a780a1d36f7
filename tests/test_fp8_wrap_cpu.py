"""wrap_model_for_fp8 on models that it wraps in part or not at all (no GPU: layers are replaced, none is run)."""
import pytest
import torch.nn as nn

from rocm_qlora import LoRALinear, MXFP4Linear, QuantLinear
from rocm_qlora.fp8 import FP8Config, FP8LinearWrapper, fp8_linear, wrap_model_for_fp8

SUPPORTED = {"fp8_supported": True, "fp8_dtypes_available": True, "reason": "Supported"}


@pytest.fixture
def supported(monkeypatch):
    monkeypatch.setattr(fp8_linear, "detect_fp8_support", lambda: dict(SUPPORTED))


def mixed():
    return nn.ModuleDict({"a": LoRALinear(QuantLinear(64, 32, bits=4), r=4),
                          "b": nn.Sequential(LoRALinear(MXFP4Linear(64, 32), r=4)),
                          "c": LoRALinear(QuantLinear(64, 32, bits=8), r=4)})


def test_a_mixed_model_is_refused_as_it_stands(supported):
    model = mixed()
    before = dict(model.named_modules())
    with pytest.raises(TypeError, match="b.0: an MXFP4Linear"):
        wrap_model_for_fp8(model)
    after = dict(model.named_modules())
    assert list(before) == list(after) and all(before[n] is after[n] for n in before)
    # without the layer that is not wrapped, the others are
    del model["b"]
    model, status = wrap_model_for_fp8(model)
    assert status["layers_wrapped"] == 2 and status["backend"] == "native"


def test_a_mixed_model_that_is_not_run_in_fp8(supported, monkeypatch):
    """Without FP8 the wrappers run their layers unchanged, an MXFP4Linear's among them."""
    model, status = wrap_model_for_fp8(mixed(), FP8Config(enabled=False))
    assert status["layers_wrapped"] == 3 and status["backend"] == "bf16" and not status["enabled"]
    monkeypatch.setattr(fp8_linear, "detect_fp8_support", lambda: dict(SUPPORTED, fp8_supported=False))
    model = mixed()
    assert wrap_model_for_fp8(model)[1]["layers_wrapped"] == 0 and isinstance(model["a"], LoRALinear)


def test_what_is_wrapped_stays_wrapped_once(supported):
    model = nn.Sequential(LoRALinear(QuantLinear(64, 32, bits=4), r=4), LoRALinear(QuantLinear(64, 32, bits=4), r=4))
    lora = list(model)
    wrap_model_for_fp8(model)
    model.append(LoRALinear(QuantLinear(64, 32, bits=4), r=4))
    model, status = wrap_model_for_fp8(model)
    assert status["layers_wrapped"] == 1
    assert [m.base for m in model][:2] == lora and all(isinstance(m, FP8LinearWrapper) and m.backend == "native" for m in model)
    # a wrapper that runs its layer unchanged may be followed by one that does not
    model = wrap_model_for_fp8(nn.Sequential(lora[0]), FP8Config(enabled=False))[0]
    model, status = wrap_model_for_fp8(model)
    assert status["layers_wrapped"] == 1 and model[0].backend == "bf16" and model[0].base.backend == "native"
