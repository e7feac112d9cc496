"""Models with adapters, on the host: what is wrapped and what is refused."""
import pytest
import torch
from torch import nn

from diffuser_b200 import artifact, modules
from oracle import torch_ref as T


def _model(quantized=True):
    make = (lambda: modules.Ltx23Nf4Linear(64, 128, bias=False)) if quantized else (lambda: nn.Linear(128, 64, bias=False))
    return nn.ModuleDict({"a": make(), "b": make()})


def test_weights_are_not_loaded_over_adapters(tmp_path):
    state = _model(quantized=False).state_dict()
    tensors, n = artifact.quantize_state(state, lambda key: True, "nf4", quantize_nf4=T.ltx23_nf4_quantize,
                                         quantize_fp8=T.fp8_quantize)
    artifact.write_artifact(str(tmp_path), tensors, "nf4", n)
    art = artifact.open_artifact(str(tmp_path))
    model = _model()
    artifact.load_quantized(model, art)
    modules.attach_adapters(model, 2, 8, lambda key: key.startswith("a"))
    kept = model["a"]
    with pytest.raises(RuntimeError, match="before attach_adapters"):
        artifact.load_quantized(model, art)
    assert model["a"] is kept and isinstance(kept, modules.AdapterLinear)


def test_a_linear_in_two_places_is_wrapped_in_both():
    model = _model()
    model["again"] = model["a"]
    model["block"] = nn.ModuleDict({"c": model["b"], "list": nn.ModuleList([model["a"]])})
    model["twin"] = model["block"]
    names = modules.attach_adapters(model, 2, 8)
    banks = [m for m in model.modules() if isinstance(m, modules.AdapterLinear)]
    assert len(banks) == 2 and names[:2] == ["a", "b"]
    assert model["again"] is model["a"] is model["block"]["list"][0] and model["block"]["c"] is model["b"]
    assert not any(isinstance(m, modules.Ltx23Nf4Linear) and not n.endswith("base") for n, m in model.named_modules())
    assert modules.attach_adapters(model, 2, 8) == []
    assert [m for m in model.modules() if isinstance(m, modules.AdapterLinear)] == banks
