"""The factors' gradients without the input's, as a first layer wants them."""
import pytest
import torch

pytestmark = pytest.mark.gpu


# 16-row tiles, 128-row tiles with one split of the rows and with several
@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("lengths,ids,k,n,r", [([1, 3, 2], [1, -1, 0], 256, 136, 24), ([], [], 64, 64, 8),
                                               ([90, 70], [0, 2], 128, 320, 16), ([700, 5, 800], [2, -1, 0], 272, 136, 40)])
def test_factor_gradients_alone_have_the_same_bits(lengths, ids, k, n, r, packed):
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(k)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    m, a = sum(lengths) + 4, 3
    offsets = torch.tensor([1] + lengths).cumsum(0).to(torch.int32).cuda()
    plan = ops.adapter_plan(torch.tensor(ids, dtype=torch.int32, device="cuda"), offsets, m, a)
    down, up, scale = rn(a, r, k), rn(a, r, n), torch.rand(a, generator=g, device="cuda") + 0.5
    x, dy = rn(m, k), rn(m, n)
    _, hidden = ops.adapter_add(rn(m, n), x, down, up, scale, plan, return_hidden=True)
    x = ops.checkpoint_pack(x) if packed else x
    _, wd, wu = ops.adapter_backward(dy, x, hidden, down, up, scale, plan)
    dx, ddown, dup = ops.adapter_backward(dy, x, hidden, down, up, scale, plan, inputs=False)
    assert dx is None and torch.equal(ddown, wd) and torch.equal(dup, wu)
    for kw in (dict(dx=rn(m, k)), dict(out=rn(m, k)), dict(factors=False)):
        with pytest.raises(ValueError, match="inputs"):
            ops.adapter_backward(dy, x, hidden, down, up, scale, plan, inputs=False, **kw)
    assert ops.device_error() == 0


def test_a_first_layer_allocates_no_input_gradient():
    from diffuser_b200 import modules, ops
    n, k, m = 64, 1024, 2048
    lin = modules.Ltx23Nf4Linear(n, k, bias=False).cuda()
    lin.set_nf4_weight(*ops.ltx23_nf4_quantize(torch.randn(n, k, device="cuda")))
    mod = modules.AdapterLinear(lin, 1, 8)
    mod.selection = modules.AdapterSelection(torch.zeros(1, dtype=torch.int32, device="cuda"), 1)
    x, dy = (torch.randn(m, c, device="cuda").to(torch.bfloat16) for c in (k, n))
    mod(x).backward(dy)
    mod.down.grad = mod.up.grad = None
    y = mod(x)
    torch.cuda.synchronize()
    held = torch.cuda.memory_allocated()
    torch.cuda.reset_peak_memory_stats()
    y.backward(dy)
    # the gradients, g [m, 8] and the partial sums of up to 8 splits; a gradient of x would be 4 MB more
    assert torch.cuda.max_memory_allocated() - held < m * k * 2
