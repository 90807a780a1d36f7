"""merge_and_export_fp16 of models with MXFP4 layers: their weights are buffers of codes, which the export would leave out."""
import os

import pytest
import torch
import torch.nn as nn

from rocm_qlora import LoRALinear, MXFP4Experts, MXFP4Linear
from rocm_qlora.export.gguf_export import merge_and_export_fp16


@pytest.mark.parametrize("layer", [lambda: MXFP4Linear(64, 32), lambda: MXFP4Experts(2, 64, 32), lambda: LoRALinear(MXFP4Linear(64, 32), r=4),
                                   lambda: nn.Sequential(MXFP4Linear(64, 32, bias=False))])
def test_a_model_with_mxfp4_weights_is_refused(tmp_path, layer):
    path = str(tmp_path / "w.pt")
    for model in (nn.Sequential(nn.Linear(8, 64), layer()), layer()):
        with pytest.raises(TypeError, match="MXFP4"):
            merge_and_export_fp16(model, path)
    assert not os.path.exists(path)


def test_a_model_without_them_is_written(tmp_path):
    path = str(tmp_path / "w.pt")
    merge_and_export_fp16(nn.Sequential(nn.Linear(8, 4)), path)
    assert set(torch.load(path, weights_only=True)) == {"0.weight", "0.bias"}
