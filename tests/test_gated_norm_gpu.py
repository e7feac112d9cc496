"""gated_norm (norm behind a block, gate, residual, norm before the next) and
its gradients against 64-bit formulas and against the unfused glue.

Tolerances: H = 2^-8 is half a bf16 step, one per rounded result; float32
arithmetic on D features is within (log2 D + 16) 2^-23 of the sum of magnitudes
(block sums are trees; rsqrt is within 2 ulp)."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H = torch.finfo(torch.bfloat16).eps / 2
F32 = 30 * 2.0 ** -23


def _rn(g, *shape, std=1.0, mean=0.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std + mean).to(torch.bfloat16)


def _operands(seed, b, s, d, post, weights, gate, mod):
    g = torch.Generator(device="cuda").manual_seed(seed)
    t = dict(x=_rn(g, b, s, d, std=1.5, mean=0.3), y=_rn(g, b, s, d, std=2.0, mean=-0.2),
             ds=_rn(g, b, s, d, std=0.1), dh=_rn(g, b, s, d, std=0.1))
    kw = dict(gate=_rn(g, b, d, std=0.7) if gate else None,
              scale=_rn(g, b, d, std=0.3) if mod else None, shift=_rn(g, b, d, std=0.3) if mod else None,
              post_weight=_rn(g, d, std=0.2, mean=1) if weights and post else None,
              pre_weight=_rn(g, d, std=0.2, mean=1) if weights else None)
    return t, kw


def _norm64(v, kind, w, eps):
    if kind == "layer":
        v = torch.nn.functional.layer_norm(v, (v.shape[-1],), eps=eps)
    elif kind == "rms":
        v = v * torch.rsqrt(v.square().mean(-1, keepdim=True) + eps)
    return v if w is None else v * w


def _added64(y, kw, post, rs, eps):
    p = _norm64(y, post, kw["post_weight"], eps)
    return rs * (p if kw["gate"] is None else p * kw["gate"].unsqueeze(1))


def _pre64(s, kw, pre, eps):
    h = _norm64(s, pre, kw["pre_weight"], eps)
    if kw["scale"] is not None:
        h = h * (1 + kw["scale"].unsqueeze(1))
    return h if kw["shift"] is None else h + kw["shift"].unsqueeze(1)


CASES = [
    # b, s, d, post, pre, weights, gate, mod, residual_scale
    (1, 1, 4, None, "rms", False, False, False, 1.0),
    (1, 1, 64, "rms", "rms", True, True, True, 1.0),
    (2, 77, 2304, "rms", "rms", True, True, True, 0.5),
    (3, 5, 1028, "layer", "layer", True, True, True, 0.2236),
    (2, 300, 516, None, "layer", False, True, True, 1.0),
    (1, 700, 3076, "rms", "layer", False, True, False, 1.0),
    (4, 33, 4096, "layer", "rms", True, False, True, 2.0),
    (2, 19, 8192, "rms", "rms", False, True, True, 1.0),
    (37, 1, 260, "rms", "layer", True, True, True, 1.0),
    (1, 2, 6148, None, "layer", True, True, True, 1.0),
]


@pytest.mark.parametrize("case", CASES)
def test_forward_matches_the_formula(case):
    from diffuser_b200 import flux
    b, s, d, post, pre, weights, gate, mod, rs = case
    t, kw = _operands(1, b, s, d, post, weights, gate, mod)
    k64 = {k: None if v is None else v.double() for k, v in kw.items()}
    for rounding in ("once", "ops"):
        out, h = flux.gated_norm(t["x"], t["y"], post=post, pre=pre, residual_scale=rs, eps=1e-5,
                                 rounding=rounding, **kw)
        added = _added64(t["y"].double(), k64, post, rs, 1e-5)
        ref = t["x"].double() + added
        # rounding after each op: up to four roundings before the sum's
        steps = 4 if rounding == "ops" else 0
        tol = H * ref.abs() + (F32 + steps * H) * added.abs() * 1.02 + F32 * t["x"].double().abs()
        assert ((out.double() - ref).abs() <= 1.01 * tol + 1e-30).all()
        # the next norm reads the stored s
        o64 = out.double()
        ref = _pre64(o64, k64, pre, 1e-5)
        shift = torch.zeros_like(ref) if kw["shift"] is None else k64["shift"].unsqueeze(1).expand_as(ref)
        part = (ref - shift).abs()
        # the deviation from the mean is off by the mean's own float32 error
        spread = (o64.abs().mean(-1, keepdim=True) + o64.abs()) * (part.sum(-1, keepdim=True) > 0) / \
            (o64.var(-1, unbiased=False, keepdim=True) if pre == "layer" else o64.square().mean(-1, keepdim=True)).add(1e-5).sqrt()
        amp = 1.0
        for w, plus in ((k64["pre_weight"], 0), (k64["scale"], 1)):
            if w is not None:
                amp = amp * (w.unsqueeze(-2) + plus if w.dim() == 2 else w).abs()
        tol = H * ref.abs() + (F32 + (4 * H if rounding == "ops" else 0)) * part * 1.02 + F32 * (spread * amp + shift.abs())
        assert ((h.double() - ref).abs() <= 1.01 * tol + 1e-30).all()


@pytest.mark.parametrize("d", [260, 1024, 3076, 4096, 8192])
def test_ops_rounding_gives_the_bits_of_the_unfused_glue(d):
    from diffuser_b200 import flux
    t, kw = _operands(2, 2, 45, d, None, False, True, True)
    s, h = flux.gated_norm(t["x"], t["y"], kw["gate"], pre="layer", scale=kw["scale"], shift=kw["shift"],
                           rounding="ops")
    want = flux.gated_residual(t["x"], kw["gate"], t["y"])
    assert torch.equal(s, want)
    assert torch.equal(h, flux.adaln_modulate(want, kw["scale"], kw["shift"]))


def _exact_grads(t, s, kw, post, pre, rs, eps, use_ds):
    leaf = {k: v.double().requires_grad_() for k, v in dict(y=t["y"], **kw).items() if v is not None}
    full = {k: leaf.get(k) for k in kw}
    added = _added64(leaf["y"], full, post, rs, eps)
    x = (s.double() - added.detach()).requires_grad_()
    total = x + added
    h = _pre64(total, full, pre, eps)
    loss = (h * t["dh"].double()).sum()
    if use_ds:
        loss = loss + (total * t["ds"].double()).sum()
    names = ["x", *leaf]
    return dict(zip(names, torch.autograd.grad(loss, [x, *leaf.values()])))


@pytest.mark.parametrize("use_ds", [True, False])
@pytest.mark.parametrize("case", CASES)
def test_backward_matches_the_formula(case, use_ds):
    from diffuser_b200 import flux
    b, s, d, post, pre, weights, gate, mod, rs = case
    t, kw = _operands(3, b, s, d, post, weights, gate, mod)
    stored, _ = flux.gated_norm(t["x"], t["y"], post=post, pre=pre, residual_scale=rs, eps=1e-5, **kw)
    run = lambda: flux.gated_norm_backward(t["ds"] if use_ds else None, t["dh"], stored, t["y"], post=post, pre=pre,  # noqa: E731
                                           residual_scale=rs, eps=1e-5, **kw)
    got = run()
    ref = _exact_grads(t, stored, kw, post, pre, rs, 1e-5, use_ds)
    assert {k for k, v in got.items() if v is not None} == {"d" + k for k in ref}
    for k, v in ref.items():
        g = got["d" + k].double()
        if k in ("x", "y"):
            # float32 terms of the row's size: each element's error is within
            # F32 of the row's largest term, times the (up to) 4 sums it passes
            big = v.abs().amax(-1, keepdim=True)
            if k == "y":
                # dq before the projection that removes its mean and its part along y
                big = torch.maximum(big, 4 * ref["x"].abs().amax(-1, keepdim=True) * rs * _largest(kw, post, t["y"]))
            else:
                big = torch.maximum(big, 4 * _largest_dt(t["dh"], stored, kw, pre))
            tol = H * v.abs() + 4 * F32 * big
        else:
            # the terms of a sum over tokens are within F32 of their size; the
            # sizes are bounded by those of its factors
            terms = _sum_terms(k, t, stored, ref["x"], kw, post, pre, rs)
            tol = 4 * F32 * terms + 4 * F32 * terms.amax()
        assert ((g - v).abs() <= 1.01 * tol + 1e-30).all(), (k, ((g - v).abs() / (tol + 1e-30)).max().item())
    for k, v in run().items():
        assert v is None or torch.equal(v, got[k])


def _rstd(v, kind):
    v = v.double()
    if kind is None:
        return torch.ones_like(v[..., :1])
    m = v.var(-1, unbiased=False, keepdim=True) if kind == "layer" else v.square().mean(-1, keepdim=True)
    return (m + 1e-5).rsqrt()


def _largest(kw, post, y):
    f = 1.0
    for w in (kw["gate"], kw["post_weight"]):
        if w is not None:
            f = f * w.double().abs().amax()
    return f * _rstd(y, post)


def _largest_dt(dh, s, kw, pre):
    f = dh.double().abs().amax(-1, keepdim=True)
    if kw["scale"] is not None:
        f = f * (1 + kw["scale"].double()).abs().amax()
    if kw["pre_weight"] is not None:
        f = f * kw["pre_weight"].double().abs().amax()
    return f * _rstd(s, pre)


def _sum_terms(k, t, s, dx, kw, post, pre, rs):
    one = lambda w, plus=0.0: 1.0 if w is None else (w.double() + plus).abs().unsqueeze(1) if w.dim() == 2 else w.double().abs()  # noqa: E731
    dh = t["dh"].double().abs()
    that = (s.double().abs() + s.double().abs().mean(-1, keepdim=True)) * _rstd(s, pre)
    yhat = (t["y"].double().abs() + t["y"].double().abs().mean(-1, keepdim=True)) * _rstd(t["y"], post)
    dxa = dx.abs() + 4 * _largest_dt(t["dh"], s, kw, pre)
    term = {"shift": dh, "scale": dh * that * one(kw["pre_weight"]), "pre_weight": dh * that * one(kw["scale"], 1.0),
            "gate": rs * dxa * yhat * one(kw["post_weight"]), "post_weight": rs * dxa * yhat * one(kw["gate"])}[k]
    return term.sum((0, 1)) if k.endswith("weight") else term.sum(1)


def test_operands_may_be_strided_views():
    from diffuser_b200 import flux
    t, kw = _operands(4, 2, 9, 128, "rms", True, True, True)
    args = dict(post="rms", pre="layer")
    want = flux.gated_norm(t["x"], t["y"], **args, **kw)
    grads = flux.gated_norm_backward(t["ds"], t["dh"], want[0], t["y"], **args, **kw)
    wide = torch.zeros(2, 9, 300, dtype=torch.bfloat16, device="cuda")
    wide[..., 4:132], wide[..., 140:268] = t["x"], t["y"]
    mods = torch.stack([kw["gate"], kw["shift"], kw["scale"]], 1).flatten(1)  # chunks of one projection
    g, sh, sc = mods.chunk(3, dim=1)
    kw2 = dict(kw, gate=g, scale=sc, shift=sh)
    for x, y in ((wide[..., 4:132], wide[..., 140:268]),
                 (t["x"].transpose(0, 1).contiguous().transpose(0, 1), t["y"].transpose(1, 2).contiguous().transpose(1, 2)),
                 (torch.nn.functional.pad(t["x"], (1, 2))[..., 1:129], t["y"])):
        got = flux.gated_norm(x, y, **args, **kw2)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    got = flux.gated_norm_backward(t["ds"].transpose(0, 1).contiguous().transpose(0, 1), t["dh"], want[0],
                                   wide[..., 140:268], **args, **kw2)
    for k, v in grads.items():
        assert torch.equal(got[k], v), k


def test_rows_that_are_not_finite_stay_in_their_rows():
    from diffuser_b200 import flux
    t, kw = _operands(5, 2, 400, 256, "rms", True, True, True)
    args = dict(post="rms", pre="rms")
    s, h = flux.gated_norm(t["x"], t["y"], **args, **kw)
    grads = flux.gated_norm_backward(t["ds"], t["dh"], s, t["y"], **args, **kw)
    x, y = t["x"].clone(), t["y"].clone()
    x[0, 7, 3], y[1, 399, 9] = float("nan"), float("inf")
    s2, h2 = flux.gated_norm(x, y, **args, **kw)
    bad = torch.zeros(2, 400, dtype=torch.bool, device="cuda")
    bad[0, 7] = bad[1, 399] = True
    assert torch.equal(s2[~bad], s[~bad]) and torch.equal(h2[~bad], h[~bad]) and not h2[bad].isfinite().any()
    g2 = flux.gated_norm_backward(t["ds"], t["dh"], s2, y, **args, **kw)
    assert torch.equal(g2["dx"][~bad], grads["dx"][~bad]) and torch.equal(g2["dy"][~bad], grads["dy"][~bad])
    assert torch.equal(g2["dshift"], grads["dshift"]) and not g2["dscale"].isfinite().any()


def test_empty_batches_and_refusals():
    from diffuser_b200 import flux
    t, kw = _operands(6, 2, 3, 64, "rms", True, True, True)
    z = t["x"][:, :0]
    s, h = flux.gated_norm(z, z, post="rms", **kw)
    assert s.shape == z.shape and h.shape == z.shape
    g = flux.gated_norm_backward(None, z, z, z, post="rms", **kw)
    assert not g["dgate"].any() and not g["dpost_weight"].any()
    for bad, err in ((dict(post="batch"), ValueError), (dict(pre=None), ValueError), (dict(rounding="none"), ValueError),
                     (dict(post_weight=kw["post_weight"]), ValueError), (dict(gate=kw["gate"][:1]), TypeError),
                     (dict(pre_weight=kw["pre_weight"].float()), TypeError)):
        with pytest.raises(err):
            flux.gated_norm(t["x"], t["y"], **bad)
    with pytest.raises(ValueError):
        flux.gated_norm(t["x"], t["y"][:, :2])
    with pytest.raises(ValueError):
        flux.gated_norm(t["x"][..., :62], t["y"][..., :62])
    with pytest.raises(TypeError):
        flux.gated_norm(t["x"], t["y"].float())
    with pytest.raises(ValueError):
        flux.gated_norm(t["x"][0], t["y"][0])


def test_captured_and_replayed():
    from diffuser_b200 import flux
    t, kw = _operands(7, 2, 130, 512, "rms", True, True, True)

    def step():
        s, h = flux.gated_norm(t["x"], t["y"], post="rms", **kw)
        return (s, h, *flux.gated_norm_backward(t["ds"], t["dh"], s, t["y"], post="rms", **kw).values())

    want = [v.clone() for v in step()]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for v in got:
        v.zero_()
    graph.replay()
    for p, q in zip(got, want):
        assert torch.equal(p, q)
