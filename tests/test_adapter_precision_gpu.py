"""How many roundings a result carries, with bounds that one more, or one term
less, breaks.

H = 2^-8 is half a bf16 step, the most one rounding is off; spread evenly its
mean square is H^2 / 3.  U = 2^-23 covers a float32 operation."""
import pytest
import torch
from torch import nn

from test_adapter_modules_gpu import _adapted64, _far, _fill, _linear

pytestmark = pytest.mark.gpu

H = torch.finfo(torch.bfloat16).eps / 2
U = 2.0 ** -23


def _activated(z, act):
    gelu = lambda t: nn.functional.gelu(t, approximate="tanh")  # noqa: E731
    if act == "gelu_tanh":
        return gelu(z)
    gate, up = z.unflatten(-1, (-1, 2, 16)).unbind(-2)
    return ((nn.functional.silu if act == "swiglu" else gelu)(gate) * up).flatten(-2)


# 16-row tiles (37 tokens of 5 adapters) and 128-row ones (180 of 1)
@pytest.mark.parametrize("m,a", [(37, 5), (180, 1)])
@pytest.mark.parametrize("act", [None, "gelu_tanh", "swiglu", "geglu_tanh"])
def test_an_activated_sum_is_rounded_once(act, m, a):
    """From the bf16 intermediate that the call returns, y + hidden . up and its
    activation stay in float32 up to the result: H of the result and the float32
    operations' error.  The activation's arguments are up to 1 + r + 1 sums; its
    exponential and reciprocal are within 2^-21, the product with its argument
    of some tens within 2^-17 of it, slopes are below 1.13."""
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(m)
    k, n, r = 256, 544, 24
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    x, y, down, up = rn(m, k), rn(m, n), rn(a, r, k) / 16, rn(a, r, n) / 4
    off = torch.tensor([i * m // a for i in range(a)] + [m], dtype=torch.int32, device="cuda")
    plan = ops.adapter_plan(torch.arange(a, dtype=torch.int32, device="cuda"), off, m, a)
    out, hidden = ops.adapter_add(y, x, down, up, torch.ones(a, device="cuda"), plan, act=act, return_hidden=True)
    mine = torch.repeat_interleave(torch.arange(a, device="cuda"), off.diff().long())
    z, size = y.double(), y.double().abs()
    for i in range(a):
        rows = mine == i
        z[rows] += hidden[rows].double() @ up[i].double()
        size[rows] += hidden[rows].double().abs() @ up[i].double().abs()
    err = (r + 2) * U * size
    if act is None:
        ref, tol = z, err
    elif act == "gelu_tanh":
        ref = _activated(z, act)
        tol = 1.13 * err + 2.0 ** -17 * (z.abs() + ref.abs())
    else:
        ref = _activated(z, act)
        (zg, zu), (eg, eu) = (t.unflatten(-1, (-1, 2, 16)).unbind(-2) for t in (z, err))
        tol = (zu.abs() * (1.13 * eg + 2.0 ** -17 * 2 * zg.abs()) + zg.abs() * 1.13 * eu).flatten(-2)
    tol = 1.01 * (tol + H * ref.abs()) + 1e-30
    assert ((out.double() - ref).abs() <= tol).all()
    # the sum rounded before its activation, or the activation before its product, would not pass
    if act is not None:
        twice = _activated(z.to(torch.bfloat16).double(), act).to(torch.bfloat16).double()
        assert ((twice - ref).abs() > tol).any()


def _norm(t, kind, weight=None):
    """The norm, "rms" or "layer", or one with a term of its derivative left out."""
    mean = t.mean(-1, keepdim=True) if kind.startswith("layer") else torch.zeros_like(t[..., :1])
    if kind == "layer, no mean":
        mean = mean.detach()
    scale = ((t - mean).square().mean(-1, keepdim=True) + 1e-6).rsqrt()
    return (t - mean) * (scale.detach() if kind.endswith("no projection") else scale) * (1 if weight is None else weight)


@pytest.mark.parametrize("pack", [False, True])
@pytest.mark.parametrize("seq", [5, 150])
def test_a_block_is_within_the_sum_of_its_roundings(pack, seq):
    """gated norm, NF4 projection with adapters, GELU, fp8 projection with
    adapters, gated norm.  Nine results are rounded on the way to h (s, h, base,
    sum, GELU, base, sum, s, h) and as many on the way back; independent ones
    add up in squares, sqrt(9 / 3) H = 1.7 H forward and 2.4 H backward, taken
    twice for the factors between them.  An 8-bit activation is off by a code's
    1 / sqrt(12) in the mean square, a code max / 127 of its run, max up to four
    times its rms."""
    from diffuser_b200 import flux, modules
    ids, dim, inner = [1, -1, 0, 1], 256, 384
    lin1, w1, b1 = _linear("nf4", inner, dim, 1)
    lin2, w2, b2 = _linear("fp8", dim, inner, 2)
    up1, up2 = (modules.AdapterLinear(m, 2, 12, pack_activations=pack) for m in (lin1, lin2))
    for i, m in enumerate((up1, up2)):
        _fill(m, 3 + i)
        m.selection = modules.AdapterSelection(torch.tensor(ids, dtype=torch.int32, device="cuda"), 2)
    g = torch.Generator(device="cuda").manual_seed(6)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()  # noqa: E731
    v = dict(x=rn(4, seq, dim), y0=rn(4, seq, dim), gate0=rn(4, dim), gate1=rn(4, dim), scale=rn(4, dim), shift=rn(4, dim),
             weight=rn(dim), down1=up1.down, up1=up1.up, down2=up2.down, up2=up2.up)
    s1, h1 = flux.gated_norm(v["x"], v["y0"], v["gate0"], pre="rms", scale=v["scale"], shift=v["shift"])
    y1 = up2(up1(h1, act="gelu_tanh"))
    s2, h2 = flux.gated_norm(s1, y1, v["gate1"], post="rms", post_weight=v["weight"], pre="layer", residual_scale=0.5)
    d = [torch.randn(t.shape, generator=g, device="cuda").to(torch.bfloat16) for t in (s2, h2)]
    grads = dict(zip(v, torch.autograd.grad([s2, h2], list(v.values()), d)))

    def reference(post="rms", last="layer", share=True):
        q = {k: t.detach().double().requires_grad_() for k, t in v.items()}
        col = lambda t: t.unsqueeze(1)  # noqa: E731
        r1 = q["x"] + col(q["gate0"]) * q["y0"]
        rh = _norm(r1, "rms") * (1 + col(q["scale"])) + col(q["shift"])
        z = _adapted64(rh, w1, b1, q["down1"], q["up1"], up1.scale, ids)
        z = nn.functional.gelu(z, approximate="tanh")
        if not share:  # adapter 1's part of the second projection's dx
            low = lambda t: _adapted64(t, w2 * 0, b2 * 0, q["down2"], q["up2"], up2.scale, [1, -1, -1, 1])  # noqa: E731
            z = _adapted64(z, w2, b2, q["down2"], q["up2"], up2.scale, [-1, -1, 0, -1]) + low(z.detach())
        else:
            z = _adapted64(z, w2, b2, q["down2"], q["up2"], up2.scale, ids)
        r2 = r1 + 0.5 * col(q["gate1"]) * _norm(z, post, q["weight"])
        r3 = _norm(r2, last)
        return r2, r3, dict(zip(q, torch.autograd.grad([r2, r3], list(q.values()), [t.double() for t in d])))

    r2, r3, ref = reference()
    forward, backward = 2 * 3 ** 0.5 * H, 2 * 6 ** 0.5 * H + (4 / (127 * 12 ** 0.5) if pack else 0)
    assert _far(s2, r2.detach()) <= forward and _far(h2, r3.detach()) <= forward
    for k, t in ref.items():
        assert _far(grads[k], t) <= backward, k
    # a derivative with one term left out is farther off than that (the first
    # norm's projection, 1 / sqrt(256) of a path that brings x a seventh of its
    # gradient, is below it: the norm's own test has it element by element)
    for k, kw in (("x", dict(last="layer, no mean")), ("x", dict(last="layer, no projection")),
                  ("down2", dict(post="rms, no projection")), ("down1", dict(share=False)), ("x", dict(share=False))):
        assert _far(grads[k], reference(**kw)[2][k]) > backward, (k, kw)
