"""Adapter calls at their edges, against 64-bit formulas."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H = torch.finfo(torch.bfloat16).eps / 2
U = 2.0 ** -23


def _rn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _one_adapter(m):
    from diffuser_b200 import ops
    off = torch.tensor([0, m], dtype=torch.int32, device="cuda")
    return ops.adapter_plan(torch.zeros(1, dtype=torch.int32, device="cuda"), off, m, 1)


# 16-row tiles (3 tokens) and 128-row ones (200), ranks that fill their class and not
@pytest.mark.parametrize("m", [3, 200])
@pytest.mark.parametrize("r", [8, 16, 24, 40, 64, 96, 128])
def test_an_infinite_input_gives_an_infinity(m, r):
    """One infinity in x, positive weights where it is multiplied: every v of
    its row is infinite and so is every out, and none is NaN, whatever the rank
    is padded to."""
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(r)
    k, n, at = 256, 264, m // 2
    x, y = _rn(g, m, k), _rn(g, m, n)
    down, up = _rn(g, 1, r, k, std=k ** -0.5), _rn(g, 1, r, n).abs() + 0.125
    down[0, :, 5] = 0.5
    x[at, 5] = float("inf")
    one, plan = torch.ones(1, device="cuda"), _one_adapter(m)
    out, hidden = ops.adapter_add(y, x, down, up, one, plan, return_hidden=True)
    keep = torch.arange(m, device="cuda") != at
    assert (hidden[at] == float("inf")).all() and (out[at] == float("inf")).all()
    assert out[keep].isfinite().all() and hidden[keep].isfinite().all()
    # and back: the same products with the factors' parts exchanged
    dy = _rn(g, m, n)
    dy[at, 7] = float("inf")
    dx, _, _ = ops.adapter_backward(dy, x, hidden, down.abs() + 0.125, up, one, plan)
    assert (dx[at] == float("inf")).all() and dx[keep].isfinite().all()


def _linear(fmt, seed):
    from diffuser_b200 import modules
    lin = (modules.Ltx23Nf4Linear if fmt == "nf4" else modules.Ltx23Fp8Linear)(64, 128, bias=True).cuda()
    _set(lin, fmt, seed)
    return lin


def _set(lin, fmt, seed):
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(64, 128, generator=g, device="cuda") * 0.1
    if fmt == "nf4":
        lin.set_nf4_weight(*ops.ltx23_nf4_quantize(w))
    else:
        w8, s = ops.fp8_quantize(w)
        lin.set_fp8_weight(w8, s.cpu())


@pytest.mark.parametrize("adapted", [False, True])
@pytest.mark.parametrize("act", [None, "gelu_tanh"])
@pytest.mark.parametrize("fmt", ["nf4", "fp8"])
def test_a_weight_replaced_before_the_backward_pass(fmt, act, adapted):
    """The gradient is that of the weight the forward pass used, or none."""
    from diffuser_b200 import modules
    lin = _linear(fmt, 1)
    mod = modules.AdapterLinear(lin, 1, 8) if adapted else lin
    lin.differentiable = True
    if adapted:
        mod.selection = modules.AdapterSelection(torch.zeros(1, dtype=torch.int32, device="cuda"), 1)
    x = torch.randn(9, 128, device="cuda").to(torch.bfloat16).requires_grad_()
    dy = torch.randn(9, 64, device="cuda").to(torch.bfloat16)
    want, = torch.autograd.grad(mod(x, act=act), x, dy)
    y = mod(x, act=act)
    _set(lin, fmt, 2)
    if fmt == "nf4":  # in place: the old weight is gone
        with pytest.raises(RuntimeError, match="changed"):
            y.backward(dy)
    else:  # another tensor: the old one is still held
        assert torch.equal(torch.autograd.grad(y, x, dy)[0], want)
    assert not torch.equal(torch.autograd.grad(mod(x, act=act), x, dy)[0], want)


def test_a_bias_replaced_before_the_backward_pass():
    lin = _linear("nf4", 3)
    lin.differentiable = True
    x = torch.randn(9, 128, device="cuda").to(torch.bfloat16).requires_grad_()
    y = lin(x, act="gelu_tanh")
    with torch.no_grad():
        lin.bias.add_(1)
    with pytest.raises(RuntimeError, match="changed"):
        y.sum().backward()
    lin(x).sum().backward()  # without an activation the bias is not read again


# one to eight clusters of CTAs per 16-row tile, by the tiles, the columns and
# what a rank leaves resident
@pytest.mark.parametrize("r", [16, 32, 64, 128])
@pytest.mark.parametrize("tiles,n", [(1, 16392), (2, 12288), (4, 8200), (5, 16384), (8, 4096), (17, 6152)])
def test_small_batches_of_wide_outputs(tiles, n, r):
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(tiles)
    k, m = 264, tiles
    x, y, dy = _rn(g, m, k), _rn(g, m, n), _rn(g, m, n)
    down, up, scale = _rn(g, m, r, k, std=k ** -0.5), _rn(g, m, r, n, std=r ** -0.5), torch.rand(m, generator=g, device="cuda") + 0.5
    ids = torch.arange(m, dtype=torch.int32, device="cuda")
    plan = ops.adapter_plan(ids, torch.arange(m + 1, dtype=torch.int32, device="cuda"), m, m)
    out, hidden = ops.adapter_add(y, x, down, up, scale, plan, return_hidden=True)
    v = scale.double()[:, None] * torch.einsum("mk,mrk->mr", x.double(), down.double())
    v_err = (k + 8) * U * scale.double()[:, None] * torch.einsum("mk,mrk->mr", x.double().abs(), down.double().abs())
    assert ((hidden.double() - v).abs() <= 1.01 * (v_err + H * v.abs())).all()
    ref = y.double() + torch.einsum("mr,mrn->mn", v, up.double())
    size = torch.einsum("mr,mrn->mn", H * v.abs() + v_err, up.double().abs()) + (r + 4) * U * (
        torch.einsum("mr,mrn->mn", v.abs(), up.double().abs()) + y.double().abs())
    assert ((out.double() - ref).abs() <= 1.01 * (size + H * ref.abs())).all()
    assert ops.device_error() == 0


def test_linears_quantized_or_joined_after_the_adapters_pass_gradients_on():
    from diffuser_b200 import modules
    model = torch.nn.Sequential(_linear("nf4", 1), torch.nn.Linear(64, 64, bias=False).cuda().to(torch.bfloat16))
    modules.attach_adapters(model, 1, 8, lambda key: key.startswith("0"))
    modules.swap_quant_linears(model, lambda key: key.startswith("1"))
    joined = modules.concat_nf4_linears([model[1], model[1]])
    x = torch.randn(5, 128, device="cuda").to(torch.bfloat16).requires_grad_()
    dy = torch.randn(5, 64, device="cuda").to(torch.bfloat16)
    one, = torch.autograd.grad(model[1](model[0](x)), x, dy)
    two, = torch.autograd.grad(joined(model[0](x))[:, 64:], x, dy)
    # the same products, summed next to zeros: a rounding each of two results
    assert one.any() and ((one - two).double().norm() / one.double().norm()).item() <= 2 * H
