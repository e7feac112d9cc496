"""Linears made after attach_adapters pass gradients on as those before it do."""
import pytest
import torch
from torch import nn

from diffuser_b200 import modules, tp


def _nf4(n, k):
    return modules.Ltx23Nf4Linear(n, k, bias=False)


def test_concatenated_linears_keep_the_mark():
    mods = [_nf4(64, 128) for _ in range(3)]
    assert not modules.concat_nf4_linears(mods).differentiable
    mods[1].differentiable = True
    assert modules.concat_nf4_linears(mods).differentiable
    assert modules.fuse_gated_pair(*mods[1:], act="swiglu").differentiable


@pytest.mark.parametrize("call", ["forward", "forward_nccl"])
def test_a_marked_column_parallel_linear_drops_no_gradient(call):
    lin = tp.ColumnParallelNf4Linear.__new__(tp.ColumnParallelNf4Linear)
    nn.Module.__init__(lin)
    lin.in_features = 64
    x = torch.zeros(2, 64, dtype=torch.bfloat16, requires_grad=True)
    with pytest.raises(RuntimeError, match="CPU path"):
        getattr(lin, call)(x)
    lin.differentiable = True
    with pytest.raises(RuntimeError, match="gradients"):
        getattr(lin, call)(x)
    with torch.no_grad(), pytest.raises(RuntimeError, match="CPU path"):
        getattr(lin, call)(x)
