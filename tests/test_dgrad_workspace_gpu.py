"""Input gradients ask for the decoded weight only where they decode it first."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("fmt", ["nf4", "fp8"])
def test_workspace_of_an_input_gradient(fmt):
    from diffuser_b200 import _lib, ops
    n, k = 2048, 1024
    w = torch.randn(n, k, device="cuda") * 0.1
    if fmt == "nf4":
        packed, absmax = ops.ltx23_nf4_quantize(w)
        call = lambda dy: ops.nf4_linear_dgrad(dy, packed, absmax, k)  # noqa: E731
        raw = lambda dy, dx, p, b: _lib.call(  # noqa: E731
            "dq_linear_nf4_dgrad", dy.data_ptr(), dy.shape[0], n, packed.data_ptr(), absmax.data_ptr(), 0, k,
            dx.data_ptr(), p, b, torch.cuda.current_stream().cuda_stream)
    else:
        w8, s = ops.fp8_quantize(w)
        s = float(s)
        call = lambda dy: ops.fp8_linear_dgrad(dy, w8, s)  # noqa: E731
        raw = lambda dy, dx, p, b: _lib.call(  # noqa: E731
            "dq_linear_fp8_dgrad", dy.data_ptr(), dy.shape[0], n, w8.data_ptr(), s, k, dx.data_ptr(), p, b,
            torch.cuda.current_stream().cuda_stream)
    for m, decoded in ((1, False), (300, False), (600, True)):
        dy = torch.randn(m, n, device="cuda").to(torch.bfloat16)
        want = call(dy)
        dx = torch.empty_like(want)
        if decoded:
            ws = torch.empty(_lib.lib().dq_linear_dgrad_workspace_for(m, n, k), dtype=torch.uint8, device="cuda")
            raw(dy, dx, ws.data_ptr(), ws.numel())
            for p, b in ((0, 0), (ws.data_ptr(), ws.numel() - 1), (ws.data_ptr() + 8, ws.numel())):
                with pytest.raises(_lib.DqError, match="workspace"):
                    raw(dy, dx, p, b)
        else:
            raw(dy, dx, 0, 0)
        assert torch.equal(dx, want), m
        # what the Python call holds beside its result
        torch.cuda.synchronize()
        held = torch.cuda.memory_allocated()
        torch.cuda.reset_peak_memory_stats()
        out = call(dy)
        beside = torch.cuda.max_memory_allocated() - held - out.numel() * 2
        assert (beside >= 2 * n * k) == decoded and (decoded or beside < 4096), (m, beside)
    with pytest.raises(ValueError):
        ops.nf4_linear_dgrad(dy, w[:0].byte(), w[:0], 0)
