"""Scales and codes of 8-bit activations for every maximum that bf16 can hold."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_every_maximum():
    from diffuser_b200 import ops
    bits = torch.arange(0x7F80, dtype=torch.int32)  # zero, subnormals, normals
    top = bits.to(torch.int16).view(torch.bfloat16)
    part = torch.tensor([1, -1, .5, -.5, .25, .75, .3, -.3, .01, .004, .0039, 0, .99, -.66, .125, 1 / 127.])
    x = (top.float()[:, None] * part).to(torch.bfloat16)
    scales = top.float().clamp_min(1e-12) / 127  # IEEE division, on the host
    codes = (x.float() / scales[:, None]).round().to(torch.int8)
    p = ops.checkpoint_pack(x.cuda())
    assert torch.equal(p.scales.cpu()[:, 0], scales)
    assert torch.equal(p.codes.cpu(), codes)
    assert torch.equal(ops.checkpoint_unpack(p).cpu(), (codes.float() * scales[:, None]).to(torch.bfloat16))
