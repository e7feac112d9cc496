"""Adapter outputs in column ranges of buffers that hold other operands."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_outputs_in_shared_buffers():
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    m, k, n = 20, 64, 64
    ids, off = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0], [0, m]))
    plan = ops.adapter_plan(ids, off, m, 1)
    bank = (rn(1, 8, k), rn(1, 8, n), torch.ones(1, device="cuda"))
    buf = rn(m, 256)
    x, y = buf[:, :64], buf[:, 64:128]
    want, hidden = ops.adapter_add(y, x, *bank, plan, return_hidden=True)
    for at in (72, 56, 8):  # columns that are y's in part, x's and y's, x's in part
        with pytest.raises(ValueError, match="overlap"):
            ops.adapter_add(y, x, *bank, plan, out=buf[:, at:at + 64])
    with pytest.raises(ValueError, match="overlap"):
        ops.adapter_backward(y, x, hidden, *bank, plan, out=buf[:, 120:184])
    packed = ops.checkpoint_pack(x)
    spare = packed.codes.view(torch.bfloat16)  # [m, 32]
    with pytest.raises(ValueError, match="overlap x"):
        ops.adapter_backward(y[:10], ops.PackedActivation(packed.codes[:10], packed.scales[:10]), hidden[:10], *bank,
                             ops.adapter_plan(ids, torch.tensor([0, 10], dtype=torch.int32, device="cuda"), 10, 1),
                             out=spare.view(-1)[:640].view(10, 64))
    assert torch.equal(ops.adapter_add(y, x, *bank, plan, out=buf[:, 128:192]), want)
    assert torch.equal(ops.adapter_add(y, x, *bank, plan, out=y), want)
    dx = ops.adapter_backward(buf[:, 128:192], x, hidden, *bank, plan)[0]
    assert torch.equal(ops.adapter_backward(buf[:, 128:192], x, hidden, *bank, plan, out=buf[:, 192:256])[0], dx)
    with pytest.raises(ValueError, match="overlap down"):
        wide = rn(40, 64)
        ops.adapter_add(rn(m, n), rn(m, k), wide[:8].view(1, 8, 64), *bank[1:], plan, out=wide[4:24])
