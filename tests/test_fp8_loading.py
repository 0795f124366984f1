"""e4m3 modules against what a pack's quantization config says of them."""
from __future__ import annotations

import pytest
import torch
from safetensors.torch import save_file

from dsv4_carve_b200 import loader
from tests import fp8_reference as R


@pytest.mark.parametrize("non_routed", [{"bits": 6, "modules": ["attn.wo"]}, {"layers": {"layers.0.attn.wo": {"bits": 6}}}])
def test_a_module_that_the_config_lists_as_exl3_has_to_be_exl3(tmp_path, non_routed, monkeypatch):
    """Listed modules that are stored in e4m3 are refused; others load as e4m3."""
    tensors = {}
    for name in ("wo", "wq"):
        q, s = R.e4m3_weight((256, 128), 1, "cpu")
        tensors[f"layers.0.attn.{name}.weight"], tensors[f"layers.0.attn.{name}.scale"] = q, s
    save_file(tensors, str(tmp_path / "model.safetensors"))
    ck = loader.Checkpoint(tmp_path)
    config = loader.Exl3QuantConfig.from_dict({"quant_method": "exl3", "bits": 2, "non_routed_exl3": non_routed})
    assert config.matches_non_routed("layers.0.attn.wo") and not config.matches_non_routed("layers.0.attn.wq")
    monkeypatch.setattr(loader, "LinearFP8", lambda w, s, **kw: kw["key"])
    with pytest.raises(KeyError, match="layers.0.attn.wo.trellis"):
        loader.load_linear(ck, "layers.0.attn.wo", "cpu", config)
    assert loader.load_linear(ck, "layers.0.attn.wq", "cpu", config) == "layers.0.attn.wq"
    assert loader.load_linear(ck, "layers.0.attn.wo", "cpu") == "layers.0.attn.wo"
