"""diffuser_b200 -- a B200-native (sm_100a) quantized weight-only linear engine
for diffuseR's NF4 and fp8-e4m3 DiT linears.

Public surface (mirrors the reference's R API names):
  ops.ltx23_nf4_quantize / ops.ltx23_nf4_dequantize / ops.fp8_quantize /
  ops.fp8_dequantize / ops.nf4_linear / ops.fp8_linear
  modules.ltx23_nf4_linear / modules.ltx23_fp8_linear / modules.swap_quant_linears
  ops.adapter_plan / adapter_add / adapter_backward, ops.checkpoint_pack /
  checkpoint_unpack, ops.nf4_linear_dgrad / fp8_linear_dgrad (no counterpart in
  the reference, as are the next two lines)
  modules.AdapterLinear / attach_adapters / select_adapters
  flux.gated_norm / gated_norm_backward
  tp.ColumnParallelQuantLinear (column-parallel over NCCL)
The compute path is the C-ABI library built from ``csrc/`` (see build.py);
there is no CPU fallback.
"""
from . import build  # noqa: F401

__all__ = ["build", "ops", "modules"]


def __getattr__(name):
    if name in ("ops", "modules", "tp", "flux"):
        import importlib
        return importlib.import_module(f".{name}", __name__)
    raise AttributeError(name)
