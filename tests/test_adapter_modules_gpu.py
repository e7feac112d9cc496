"""Adapters, gated norms, 8-bit activations and input gradients as modules use
them: a block forward and backward, a FLUX transformer with adapters, and the
unchanged bits of the FLUX block boundary.

H = 2^-8 is half a bf16 step.  A chain of n rounded results is within n H of
the 64-bit chain in the 2-norm, times two for the condition of its products; an
8-bit activation adds half a code, max / 254 of its run."""
import pytest
import torch
from torch import nn

pytestmark = pytest.mark.gpu

H = torch.finfo(torch.bfloat16).eps / 2


def _far(got, ref):
    return ((got.double() - ref).norm() / ref.norm()).item()


def _linear(fmt, n, k, seed, bias=True):
    """A quantized module and the 64-bit weight and bias it stands for."""
    from diffuser_b200 import modules, ops
    g = torch.Generator(device="cuda").manual_seed(seed)
    w = torch.randn(n, k, generator=g, device="cuda") * k ** -0.5
    if fmt == "nf4":
        lin = modules.Ltx23Nf4Linear(n, k, bias=bias).cuda()
        p, a = ops.ltx23_nf4_quantize(w)
        lin.set_nf4_weight(p, a)
        wd = ops.ltx23_nf4_dequantize(p, a, (n, k)).double()
    else:
        lin = modules.Ltx23Fp8Linear(n, k, bias=bias).cuda()
        w8, s = ops.fp8_quantize(w)
        lin.set_fp8_weight(w8, s.cpu())
        wd = ops.fp8_dequantize(w8, float(s)).double()
    if bias:
        with torch.no_grad():
            lin.bias.copy_(torch.randn(n, generator=g, device="cuda") * 0.1)
        lin.bias = nn.Parameter(lin.bias.to(torch.bfloat16), requires_grad=False)
    return lin, wd, lin.bias.double() if bias else 0.0


def _fill(mod, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    a, r, k = mod.down.shape
    with torch.no_grad():
        mod.down.copy_(torch.randn(a, r, k, generator=g, device="cuda") * k ** -0.5)
        mod.up.copy_(torch.randn(a, r, mod.out_features, generator=g, device="cuda") * r ** -0.5)
        mod.scale.copy_(torch.rand(a, generator=g, device="cuda") + 0.5)


def _adapted64(x, wd, bias, down, up, scale, ids):
    """x [B, S, K] through the weight and each element's adapter, in 64 bits."""
    rows = [x[i] @ wd.T + bias + (scale[a].double() * (x[i] @ down[a].T) @ up[a] if a >= 0 else 0.0)
            for i, a in enumerate(ids)]
    return torch.stack(rows)


@pytest.mark.parametrize("pack", [False, True])
@pytest.mark.parametrize("seq", [5, 150])
def test_a_block_forward_and_backward(pack, seq):
    # gated norm -> NF4 projection with adapters -> GELU -> fp8 projection with adapters -> gated norm
    from diffuser_b200 import flux, modules
    ids, dim, inner = [1, -1, 0, 1], 256, 384
    lin1, w1, b1 = _linear("nf4", inner, dim, 1)
    lin2, w2, b2 = _linear("fp8", dim, inner, 2)
    up1, up2 = (modules.AdapterLinear(m, 2, 12, pack_activations=pack) for m in (lin1, lin2))
    assert up1.down.shape == (2, 16, dim)
    for i, m in enumerate((up1, up2)):
        _fill(m, 3 + i)
        m.selection = modules.AdapterSelection(torch.tensor(ids, dtype=torch.int32, device="cuda"), 2)
    g = torch.Generator(device="cuda").manual_seed(5)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16).requires_grad_()  # noqa: E731
    x, y0 = rn(4, seq, dim), rn(4, seq, dim)
    gates = [rn(4, dim) for _ in range(2)]
    scale, shift, weight = rn(4, dim), rn(4, dim), rn(dim)
    s1, h1 = flux.gated_norm(x, y0, gates[0], pre="rms", scale=scale, shift=shift)
    y1 = up2(up1(h1, act="gelu_tanh"))
    s2, h2 = flux.gated_norm(s1, y1, gates[1], post="rms", post_weight=weight, pre="layer", residual_scale=0.5)
    d1, d2 = torch.randn(s2.shape, generator=g, device="cuda"), torch.randn(h2.shape, generator=g, device="cuda")
    d1, d2 = d1.to(torch.bfloat16), d2.to(torch.bfloat16)
    leaves = dict(x=x, y0=y0, gate0=gates[0], gate1=gates[1], scale=scale, shift=shift, weight=weight, down1=up1.down,
                  up1=up1.up, down2=up2.down, up2=up2.up)
    grads = dict(zip(leaves, torch.autograd.grad([s2, h2], list(leaves.values()), [d1, d2])))

    v = {k: t.detach().double().requires_grad_() for k, t in leaves.items()}
    rms = lambda t: t * (t.square().mean(-1, keepdim=True) + 1e-6).rsqrt()  # noqa: E731
    m = lambda t: t.unsqueeze(1)  # noqa: E731
    r1 = v["x"] + m(v["gate0"]) * v["y0"]
    rh = rms(r1) * (1 + m(v["scale"])) + m(v["shift"])
    z = _adapted64(rh, w1, b1, v["down1"], v["up1"], up1.scale, ids)
    z = _adapted64(nn.functional.gelu(z, approximate="tanh"), w2, b2, v["down2"], v["up2"], up2.scale, ids)
    r2 = r1 + 0.5 * m(v["gate1"]) * (rms(z) * v["weight"])
    r3 = nn.functional.layer_norm(r2, (dim,), eps=1e-6)
    ref = dict(zip(v, torch.autograd.grad([r2, r3], list(v.values()), [d1.double(), d2.double()])))
    # forward: s1, h1, y (2 linears x (base, hidden, sum)), gelu, s2, h2: 11 results
    assert _far(s2, r2.detach()) <= 22 * H and _far(h2, r3.detach()) <= 22 * H
    # backward: as many again; an 8-bit activation's half code against its rms is at most 4 / 254
    for k, t in ref.items():
        assert grads[k].dtype == torch.bfloat16
        assert _far(grads[k], t) <= 44 * H + (4 / 254 if pack else 0), k
    # the inactive adapter slots and the frozen base
    assert grads["up1"].shape == up1.up.shape and lin1.bias.grad is None
    with torch.no_grad():
        again = up2(up1(h1, act="gelu_tanh"))
    assert _far(again, y1.detach().double()) <= 4 * H


def test_adapters_of_checkpoints_and_gated_bases():
    from diffuser_b200 import modules
    lin, wd, _ = _linear("nf4", 128, 64, 7, bias=False)
    lin.to_gated("swiglu")
    mod = modules.AdapterLinear(lin, 3, 4)
    g = torch.Generator(device="cuda").manual_seed(8)
    a, b = torch.randn(4, 64, generator=g, device="cuda"), torch.randn(128, 4, generator=g, device="cuda")
    mod.set_adapter(2, a, b, 0.25)
    mod.selection = modules.AdapterSelection(torch.tensor([2, -1], dtype=torch.int32, device="cuda"), 3)
    x = torch.randn(2, 9, 64, generator=g, device="cuda").to(torch.bfloat16)
    with torch.no_grad():
        out = mod(x)
    ad, bd = a.to(torch.bfloat16).double(), b.to(torch.bfloat16).double()
    z = x.double() @ wd.T
    z[0] += 0.25 * (x[0].double() @ ad.T) @ bd.T
    ref = nn.functional.silu(z[..., :64]) * z[..., 64:]
    assert out.shape == (2, 9, 64) and _far(out, ref) <= 8 * H
    with pytest.raises(RuntimeError, match="gated"):
        mod(x)
    with pytest.raises(ValueError):
        mod.set_adapter(0, a, b[:64], 1.0)
    with pytest.raises(IndexError):
        mod.set_adapter(3, a, b)
    with pytest.raises(ValueError, match="whole number"):
        with torch.no_grad():
            mod(x[:, :1].reshape(2, 64)[:1])
    with pytest.raises(TypeError):
        modules.AdapterLinear(nn.Linear(64, 64), 1, 8)
    with pytest.raises(ValueError):
        modules.AdapterLinear(lin, 1, 200)


def _tiny_flux():
    from diffuser_b200 import flux
    return flux.build_flux_nf4("cuda", seed=1, in_channels=16, num_layers=1, num_single_layers=2,
                               attention_head_dim=64, num_attention_heads=4, joint_attention_dim=128,
                               pooled_projection_dim=64, axes_dims_rope=(16, 24, 24))


def _flux_inputs(batch, s_img=35, s_txt=9):
    from diffuser_b200 import flux
    g = torch.Generator(device="cuda").manual_seed(2)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    ids = torch.cat([torch.zeros(s_txt, 3), flux.prepare_latent_image_ids(5, 7)]).cuda()
    return (rn(batch, s_img, 16), rn(batch, s_txt, 128), rn(batch, 64),
            torch.full((batch,), 0.5, device="cuda"), flux.pos_embed(ids, (16, 24, 24)))


def test_flux_block_boundary_keeps_its_bits():
    from diffuser_b200 import flux
    model, inputs = _tiny_flux(), _flux_inputs(2)
    with torch.no_grad():
        fused = model(*inputs)
        flux.FUSED_BOUNDARY = False
        try:
            apart = model(*inputs)
        finally:
            flux.FUSED_BOUNDARY = True
    assert torch.equal(fused, apart)


def test_flux_with_adapters_serves_every_element_its_own():
    from diffuser_b200 import modules
    model, inputs = _tiny_flux(), _flux_inputs(3)
    with torch.no_grad():
        bare = model(*inputs)
        wrapped = modules.attach_adapters(model, 2, 8)
        assert len(wrapped) == 14 + 2 * 6 and not any("qkv" in w for w in wrapped)
        for i, m in enumerate(m for m in model.modules() if isinstance(m, modules.AdapterLinear)):
            _fill(m, 20 + i)
            m.up.mul_(0.3)
        none = model(*inputs)
        # (q, k and v now run apart: the same sums in another kernel's tiles)
        assert _far(none, bare.double()) <= 8 * H
        ids = torch.tensor([1, -1, 0], dtype=torch.int32, device="cuda")
        modules.select_adapters(model, ids)
        mixed = model(*inputs)
        for i, a in enumerate(ids.tolist()):
            one = tuple(t[i:i + 1] for t in inputs[:4]) + inputs[4:]
            modules.select_adapters(model, torch.tensor([a], dtype=torch.int32, device="cuda"))
            alone = model(*one)
            assert _far(mixed[i:i + 1], alone.double()) <= 16 * H, i
        assert _far(mixed[1:2], none[1:2].double()) <= 16 * H
        # Against the same model with plain adapters (float32, the base's own
        # output): per adapted linear the two differ by the rounding of hidden,
        # H of the added term, and by results that then round apart.  A block
        # reaches the output only through its gate, rms 0.02 sqrt(256) rms(silu)
        # < 0.2 for weights of N(0, 0.02^2), so the added terms, about as large as
        # the projections, move the output by a few times 0.01 and their
        # roundings by H times that; bf16 results one step apart add up to 4 H.
        modules.select_adapters(model, ids)

        def plain(m):
            def forward(x, act=None, out=None):
                y = m.project(x).float()
                rows = y.view(3, -1, m.out_features) if y.dim() == 2 else y
                for i, a in enumerate(ids.tolist()):
                    if a >= 0:
                        xi = x.reshape(3, -1, m.in_features)[i].float()
                        rows[i] += m.scale[a] * (xi @ m.down[a].float().T) @ m.up[a].float()
                y = rows.view(*x.shape[:-1], m.out_features)
                y = (nn.functional.gelu(y, approximate="tanh") if act else y).to(torch.bfloat16)
                return y if out is None else out.copy_(y)
            return forward

        layers = [m for m in model.modules() if isinstance(m, modules.AdapterLinear)]
        kept = [m.forward for m in layers]
        for m in layers:
            m.forward = plain(m)
        want = model(*inputs)
        for m, f in zip(layers, kept):
            m.forward = f
        for i in (0, 2):
            assert _far(mixed[i], want[i].double()) <= 4 * H < _far(mixed[i], none[i].double())
        # a captured step follows the selection
        sel = modules.select_adapters(model, ids.clone())
        model(*inputs)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = model(*inputs)
        sel.update_(torch.tensor([-1, 0, 1], dtype=torch.int32, device="cuda"))
        graph.replay()
        want = model(*inputs)
        assert torch.equal(out, want)
        modules.select_adapters(model, None)
        assert torch.equal(model(*inputs), none)
        with pytest.raises(ValueError):
            modules.select_adapters(nn.Linear(2, 2), ids)


def _reference64(model, ids):
    """The model in 64 bits: dequantized weights, plain adapters, tensor ops."""
    import copy
    from diffuser_b200 import modules, ops

    class Plain(nn.Module):
        def __init__(self, m):
            super().__init__()
            base = m.base if isinstance(m, modules.AdapterLinear) else m
            self.out_features = base.out_features
            w = ops.ltx23_nf4_dequantize(base.weight_nf4, base.weight_absmax.float(),
                                         (base.out_features, base.in_features))
            self.weight = nn.Parameter(w.double(), requires_grad=False)
            self.bias = None if base.bias is None else nn.Parameter(base.bias.detach().double(), requires_grad=False)
            self.bank = None
            if base is not m:
                self.down, self.up = (nn.Parameter(t.detach().double()) for t in (m.down, m.up))
                self.bank = m.scale.double()

        def forward(self, x):
            y = nn.functional.linear(x, self.weight, self.bias)
            if self.bank is None:
                return y
            rows = x.view(len(ids), -1, x.shape[-1])
            add = [self.bank[a] * (r @ self.down[a].T) @ self.up[a] if a >= 0 else r.new_zeros(r.shape[0], y.shape[-1])
                   for r, a in zip(rows, ids)]
            return y + torch.stack(add).view(y.shape)

    ref = copy.deepcopy(model)
    for name, mod in list(ref.named_modules()):
        inner = isinstance(mod, (modules.Ltx23Nf4Linear, modules.AdapterLinear))
        if inner and not name.endswith(".base") and not name.endswith("_qkv"):
            parent = modules._walk(ref, name.split(".")[:-1])
            leaf = name.split(".")[-1]
            if leaf.isdigit():
                parent[int(leaf)] = Plain(mod)
            else:
                setattr(parent, leaf, Plain(mod))
    return ref.double()


# all linears, those of the attentions (the rest pass gradients on), and those
# of the feed-forwards alone (next to the concatenated q, k, v)
@pytest.mark.parametrize("which", ["all", "attn", "ff"])
def test_flux_trains_its_adapters(which):
    from diffuser_b200 import modules
    model, inputs = _tiny_flux(), _flux_inputs(3)
    bare = model(*inputs).detach()
    accept = {"all": None, "attn": lambda key: ".attn." in key,
              "ff": lambda key: ".ff" in key or "proj_mlp" in key}[which]
    assert modules.attach_adapters(model, 3, 8, accept, pack_activations=False)
    for i, m in enumerate(m for m in model.modules() if isinstance(m, modules.AdapterLinear)):
        _fill(m, 40 + i)
    assert modules.attach_adapters(model, 3, 8, accept if accept else lambda key: False) == []  # they keep theirs
    ids = [2, -1, 0]
    x = inputs[0].clone().requires_grad_()
    if which == "ff":  # (the concatenated q, k, v stay) the bits of the bare model, differentiable now
        assert torch.equal(model(*inputs).detach(), bare)
    modules.select_adapters(model, torch.tensor(ids, dtype=torch.int32, device="cuda"))
    out = model(x, *inputs[1:])
    with torch.no_grad():
        assert _far(out, model(*inputs).double()) <= 8 * H  # the recorded call's values
    g = torch.Generator(device="cuda").manual_seed(5)
    dout = torch.randn(out.shape, generator=g, device="cuda").to(torch.bfloat16)
    out.backward(dout)
    ref = _reference64(model, ids)
    x64 = inputs[0].double().requires_grad_()
    want = ref(x64, *(t.double() for t in inputs[1:4]), inputs[4])
    want.backward(dout.double())
    # About 40 roundings lie on a path through the blocks and as many on the way
    # back, each of at most H and H / sqrt(3) in the mean square: independent
    # ones add up to sqrt(80 / 3) H = 0.02, and sums of paths that partly cancel
    # (the residual adds, the norms' means) to a few times that.  A path that is
    # cut loses a share of the gradient, not a few per cent of it.
    assert _far(out, want.detach()) <= 0.1
    assert _far(x.grad, x64.grad) <= 0.1
    plain = dict(ref.named_modules())
    banks = [(n, m) for n, m in model.named_modules() if isinstance(m, modules.AdapterLinear)]
    assert len(banks) == {"all": 26, "attn": 8 + 2 * 3, "ff": 4 + 2}[which]
    for name, m in banks:
        for mine, theirs in ((m.down.grad, plain[name].down.grad), (m.up.grad, plain[name].up.grad)):
            assert _far(mine, theirs) <= 0.1, name
            assert not mine[1].any() and mine[0].any() and mine[2].any(), name


def test_selections_and_plans_are_guarded():
    from diffuser_b200 import modules, ops
    lin, _, _ = _linear("nf4", 64, 64, 3)
    mod = modules.AdapterLinear(lin, 2, 8)
    _fill(mod, 1)
    ids = torch.tensor([1, 0], dtype=torch.int32, device="cuda")
    sel = mod.selection = modules.AdapterSelection(ids, 2)
    x = torch.randn(2, 6, 64, device="cuda").to(torch.bfloat16).requires_grad_()
    before = mod(x).detach()
    ids.zero_()  # the caller's own tensor
    assert torch.equal(mod(x), before) and sel.ids.tolist() == [1, 0]
    # a plan rebuilt between a call and its backward pass
    y = mod(x)
    sel.update_(torch.tensor([0, 0], dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="rebuilt"):
        y.sum().backward()
    mod(x).sum().backward()
    for bad in (torch.zeros(1, dtype=torch.int32, device="cuda"), torch.zeros(2, dtype=torch.int64, device="cuda"), [0, 1]):
        with pytest.raises(ValueError):
            sel.update_(bad)
    # a plan made inside a capture would hold nothing until its replay
    stream = torch.cuda.Stream()
    with torch.no_grad(), torch.cuda.stream(stream):
        stream.wait_stream(torch.cuda.default_stream())
        graph = torch.cuda.CUDAGraph()
        graph.capture_begin()
        try:
            with pytest.raises(RuntimeError, match="before a capture"):
                sel.plan(2)
        finally:
            graph.capture_end()
        want = mod(x)  # its plan from another stream
    torch.cuda.default_stream().wait_stream(stream)
    assert torch.equal(want, mod(x).detach())
    # one factor frozen, both frozen, the input frozen
    d = torch.randn(2, 6, 64, device="cuda").to(torch.bfloat16)
    grads = {}
    for frozen in ((), ("down",), ("down", "up"), ("x",)):
        for n, t in (("down", mod.down), ("up", mod.up), ("x", x)):
            t.requires_grad_(n not in frozen)
            t.grad = None
        mod(x).backward(d)
        for n, t in (("down", mod.down), ("up", mod.up), ("x", x)):
            assert (t.grad is None) == (n in frozen), (frozen, n)
            if t.grad is not None:
                assert torch.equal(t.grad, grads.setdefault(n, t.grad.clone())), (frozen, n)
    # a copy of the module has its own plans
    import copy
    twin = copy.deepcopy(mod)
    assert twin.selection is not sel and not twin.selection._plans and torch.equal(twin(x).detach(), mod(x).detach())
    plan = copy.deepcopy(sel.plan(12))
    assert plan.address == plan.words.data_ptr() != sel.plan(12).address
    # no tokens
    with torch.no_grad():
        assert mod(x[:, :0]).shape == (2, 0, 64)
    assert ops.device_error() == 0


@pytest.mark.parametrize("act", [None, "gelu_tanh", "swiglu"])
@pytest.mark.parametrize("fmt", ["nf4", "fp8"])
def test_a_frozen_linear_passes_gradients_on(fmt, act):
    from diffuser_b200 import modules
    lin, wd, bias = _linear(fmt, 128, 192, 6)
    if act == "swiglu":
        lin.to_gated("swiglu")
    x = torch.randn(3, 7, 192, device="cuda").to(torch.bfloat16).requires_grad_()
    call = lambda: lin(x, act=act if act == "gelu_tanh" else None)  # noqa: E731
    assert not call().requires_grad  # outside autograd, as ever
    lin.differentiable = True
    y = call()
    with torch.no_grad():
        assert torch.equal(y, call())
    dy = torch.randn(y.shape, device="cuda").to(torch.bfloat16)
    y.backward(dy)
    x64 = x.detach().double().requires_grad_()
    z = x64 @ wd.T + bias
    if act == "gelu_tanh":
        z = nn.functional.gelu(z, approximate="tanh")
    elif act == "swiglu":
        z = nn.functional.silu(z[..., :64]) * z[..., 64:]
    z.backward(dy.double())
    # roundings: the projection, two of the activation, its gradient's three and dx
    assert _far(y, z.detach()) <= 8 * H and _far(x.grad, x64.grad) <= 2 * 8 * H
    with pytest.raises(RuntimeError, match="out"):
        lin(x, out=torch.empty(21, 128 if act != "swiglu" else 64, device="cuda", dtype=torch.bfloat16))


@pytest.mark.parametrize("pack", [False, True])
@pytest.mark.parametrize("seq", [5, 150])
def test_a_training_step_captured_and_replayed(seq, pack):
    """Two linears with an activation between them, forward and backward in one
    graph (no eager graph over the same factors alive), on other inputs and for
    another selection."""
    from diffuser_b200 import modules, ops
    mods = [modules.AdapterLinear(_linear("nf4", n, k, 5 + i)[0], 3, 8, pack) for i, (n, k) in enumerate([(256, 128), (64, 256)])]
    for i, m in enumerate(mods):
        _fill(m, 11 + i)
    sel = modules.AdapterSelection(torch.tensor([2, -1, 0], dtype=torch.int32, device="cuda"), 3)
    for m in mods:
        m.selection = sel
    g = torch.Generator(device="cuda").manual_seed(3)
    rn = lambda *s: torch.randn(*s, generator=g, device="cuda").to(torch.bfloat16)  # noqa: E731
    leaves = [p for m in mods for p in (m.down, m.up)]
    x, dy = rn(3, seq, 128).requires_grad_(), rn(3, seq, 64)

    def step():
        for t in (*leaves, x):
            t.grad = None
        y = mods[1](mods[0](x, act="gelu_tanh"))
        y.backward(dy)
        return y.detach()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    held = [t.grad for t in (*leaves, x)]
    for ids in ([0, 1, -1], [1, 1, 1]):
        with torch.no_grad():
            x.copy_(rn(3, seq, 128))
        dy.copy_(rn(3, seq, 64))
        sel.update_(torch.tensor(ids, dtype=torch.int32, device="cuda"))
        graph.replay()
        replayed = [out.clone(), *(t.clone() for t in held)]
        eager = [step(), *(t.grad for t in (*leaves, x))]
        for i, (a, b) in enumerate(zip(replayed, eager)):
            assert torch.equal(a, b), (ids, i)
    assert ops.device_error() == 0
    with pytest.raises(TypeError):
        modules.attach_adapters(_linear("nf4", 64, 64, 1)[0], 1, 8)
