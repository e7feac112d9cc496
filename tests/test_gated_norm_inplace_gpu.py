"""In-place forms of the gated norm give the bits of the others."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 2304])
def test_results_in_the_place_of_operands(d):
    from diffuser_b200 import _lib, flux
    b, n, ld = 2, 75, d + 8
    g = torch.Generator(device="cuda").manual_seed(d)
    buf = torch.randn(4, b * n, ld, generator=g, device="cuda").to(torch.bfloat16)
    x, y, dh, ds = (t[:, :d].contiguous().view(b, n, d) for t in buf)
    s, h = flux.gated_norm(x, y, post="rms", pre="layer")
    grads = flux.gated_norm_backward(ds, dh, s, y, post="rms", pre="layer")
    stream = torch.cuda.current_stream().cuda_stream
    for into in (0, 1):  # s where x or y was
        rows, out = buf.clone(), torch.empty(b * n, ld, dtype=torch.bfloat16, device="cuda")
        at = [t.data_ptr() for t in rows]
        _lib.call("dq_gated_norm", at[0], ld, at[1], ld, b * n, n, d, 0, 0, 0, 0, 0, 0, 0, 1, 2, 1.0, 1e-6, 0,
                  at[into], ld, out.data_ptr(), ld, stream)
        assert torch.equal(rows[into, :, :d].reshape(b, n, d), s) and torch.equal(out[:, :d].reshape(b, n, d), h)
        assert torch.equal(rows[:, :, d:], buf[:, :, d:])
    # dx where ds was, dy where y was
    rows = buf.clone()
    at = [t.data_ptr() for t in rows]
    ws = torch.empty(_lib.lib().dq_gated_norm_backward_workspace(b * n, n, d), dtype=torch.uint8, device="cuda")
    _lib.call("dq_gated_norm_backward", at[3], ld, at[2], ld, s.data_ptr(), d, at[1], ld, b * n, n, d, 0, 0, 0, 0, 0, 0, 1, 2,
              1.0, 1e-6, at[3], ld, at[1], ld, 0, 0, 0, 0, 0, ws.data_ptr(), ws.numel(), stream)
    assert torch.equal(rows[3, :, :d].reshape(b, n, d), grads["dx"])
    assert torch.equal(rows[1, :, :d].reshape(b, n, d), grads["dy"])
    assert torch.equal(rows[:, :, d:], buf[:, :, d:])
