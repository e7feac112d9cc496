"""Adapters beside the quantized linears, their backward pass, 8-bit activation
checkpoints and the linears' input gradients, against 64-bit formulas.

Tolerances are element by element.  H = 2^-8 is half a bf16 step; the device
rounds the [tokens, rank] intermediate once to bf16 and each result once, and
accumulates in float32 (an error of at most n 2^-23 of the sum of magnitudes
for n terms, counting the reordering); second-order terms are covered by the
factor 1.01."""
import pytest
import torch

pytestmark = pytest.mark.gpu

H = torch.finfo(torch.bfloat16).eps / 2
U = 2.0 ** -23


def _rn(g, *shape, std=1.0):
    return (torch.randn(*shape, generator=g, device="cuda") * std).to(torch.bfloat16)


def _batch(seed, lengths, ids, pad, k, n, r, a, lead=0):
    """Operands of a batch: `lead` tokens before the first request, `pad` behind the last."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    offsets = torch.tensor([lead] + list(lengths)).cumsum(0).to(torch.int32).cuda()
    m = lead + sum(lengths) + pad
    token = torch.full((m,), -1, dtype=torch.int64)
    at = lead
    for length, i in zip(lengths, ids):
        token[at:at + length] = i
        at += length
    return dict(m=m, ids=torch.tensor(ids, dtype=torch.int32).cuda(), offsets=offsets, token=token.cuda(),
                x=_rn(g, m, k), y=_rn(g, m, n), dy=_rn(g, m, n, std=0.3), dx0=_rn(g, m, k, std=0.3),
                down=_rn(g, a, r, k, std=k ** -0.5), up=_rn(g, a, r, n, std=r ** -0.5),
                scale=torch.rand(a, generator=g, device="cuda") + 0.5)


def _plan(b):
    from diffuser_b200 import ops
    return ops.adapter_plan(b["ids"], b["offsets"], b["m"], b["down"].shape[0])


def _low_rank(b, x, first, second, base):
    """(base + scale x first^T second, v = scale x first^T, tolerance without the final rounding)."""
    out, err = base.double().clone(), torch.zeros(base.shape, dtype=torch.float64, device="cuda")
    v = torch.zeros(b["m"], first.shape[1], dtype=torch.float64, device="cuda")
    v_err = torch.zeros_like(v)
    for a in range(first.shape[0]):
        rows = (b["token"] == a).nonzero().flatten()
        p, q, s = first[a].double(), second[a].double(), float(b["scale"][a])
        xr = x[rows].double()
        v[rows] = s * xr @ p.T
        v_err[rows] = (x.shape[1] + 8) * U * s * (xr.abs() @ p.abs().T)
        out[rows] += v[rows] @ q
        err[rows] = (H * v[rows].abs() + v_err[rows]) @ q.abs() + (q.shape[0] + 2) * U * (v[rows].abs() @ q.abs())
    return out, v, err + 4 * U * base.double().abs(), v_err


def _close(got, ref, tol, what):
    off = (got.double() - ref).abs() - 1.01 * tol
    assert got.isfinite().all(), what
    assert off.max().item() <= 0, (what, off.max().item(), int(off.argmax()))


CASES = {
    # lengths, ids, pad, k, n, r, a, lead
    "one_token": ([1], [0], 0, 64, 64, 8, 1, 0),
    "no_requests": ([], [], 5, 64, 64, 8, 2, 0),
    "single_tokens": ([1] * 37, [i % 6 - 1 for i in range(37)], 0, 264, 520, 16, 5, 0),
    "empty_requests": ([0, 3, 0, 0, 18, 0], [1, 2, 0, 2, 1, 1], 3, 72, 40, 24, 3, 2),
    "all_without": ([7, 9], [-1, -1], 1, 64, 64, 16, 2, 0),
    "same_adapter_twice": ([5, 6, 7], [1, 0, 1], 0, 128, 96, 32, 2, 0),
    "odd_large": ([300, 1, 129, 257], [2, 0, 2, 1], 33, 520, 328, 40, 3, 1),
    "rank_64": ([200, 90], [1, 0], 0, 512, 264, 64, 2, 0),
    "rank_128": ([150, 260], [0, 1], 6, 320, 584, 128, 2, 0),
    "rank_128_tokens": ([1] * 9, [3, 3, 0, 1, 3, -1, 2, 0, 3], 0, 256, 512, 128, 4, 0),
    "rank_96_tokens": ([2] * 9, [3, 3, 0, 1, 3, -1, 2, 0, 3], 0, 256, 776, 96, 4, 0),
    "one_long": ([1537], [0], 0, 2056, 264, 16, 1, 0),
    "many_adapters": ([3, 1, 4, 1, 5, 9, 2, 6, 5, 3, 5, 8], [50, 3, 11, 50, 69, 0, 3, 12, 13, 14, 69, 1], 0, 136, 72, 8, 70, 0),
}


@pytest.mark.parametrize("name", CASES)
def test_adapter_add_matches_the_formula(name):
    from diffuser_b200 import ops
    b = _batch(1, *CASES[name])
    ref, v, err, v_err = _low_rank(b, b["x"], b["down"], b["up"], b["y"])
    plan = _plan(b)
    out, hidden = ops.adapter_add(b["y"], b["x"], b["down"], b["up"], b["scale"], plan, return_hidden=True)
    _close(out, ref, err + H * ref.abs(), "out")
    _close(hidden, v, v_err + H * v.abs(), "hidden")
    none = b["token"] < 0
    assert torch.equal(out[none], b["y"][none]) and not hidden[none].any()
    # in place: the same bits, tokens without an adapter untouched
    y = b["y"].clone()
    assert ops.adapter_add(y, b["x"], b["down"], b["up"], b["scale"], plan, out=y) is y
    assert torch.equal(y, out)
    assert ops.device_error() == 0


@pytest.mark.parametrize("name", ["single_tokens", "odd_large"])
@pytest.mark.parametrize("act", ["gelu_tanh", "swiglu", "geglu_tanh"])
def test_adapter_add_applies_the_activation(name, act):
    from diffuser_b200 import ops
    lengths, ids, pad, k, _, r, a, lead = CASES[name]
    b = _batch(2, lengths, ids, pad, k, 544, r, a, lead)
    ref, _, err, _ = _low_rank(b, b["x"], b["down"], b["up"], b["y"])
    err = err + H * ref.abs()  # the sum is rounded before the activation
    gelu = lambda t: torch.nn.functional.gelu(t, approximate="tanh")  # noqa: E731
    if act == "gelu_tanh":
        # |gelu'| <= 1.13; the device's tanh is within 1e-6
        ref, tol = gelu(ref), 1.13 * err + 1e-6 * (1 + ref.abs())
    else:
        blocks = ref.view(b["m"], -1, 2, 16)
        ge, ue = err.view(b["m"], -1, 2, 16).unbind(2)
        gate, up = blocks.unbind(2)
        f, df = (torch.nn.functional.silu, 1.1) if act == "swiglu" else (gelu, 1.13)
        act_err = df * ge + 1e-6 * (1 + gate.abs()) + H * f(gate).abs()  # the activation is rounded too
        tol = (act_err * (up.abs() + ue) + f(gate).abs() * ue).reshape(b["m"], -1)
        ref = (f(gate) * up).reshape(b["m"], -1)
    out = ops.adapter_add(b["y"], b["x"], b["down"], b["up"], b["scale"], _plan(b), act=act)
    _close(out, ref, tol + H * ref.abs(), act)


def _packed(x):
    from diffuser_b200 import ops
    p = ops.checkpoint_pack(x)
    return p, p.codes.double() * p.scales.double().repeat_interleave(128, 1)[:, :x.shape[1]]


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("name", CASES)
def test_adapter_backward_matches_the_formula(name, packed):
    from diffuser_b200 import ops
    lengths, ids, pad, k, n, r, a, lead = CASES[name]
    k = (k + 15) // 16 * 16
    b = _batch(3, lengths, ids, pad, k, n, r, a, lead)
    plan = _plan(b)
    _, hidden = ops.adapter_add(b["y"], b["x"], b["down"], b["up"], b["scale"], plan, return_hidden=True)
    x, xd = _packed(b["x"]) if packed else (b["x"], b["x"].double())
    dx, ddown, dup = ops.adapter_backward(b["dy"], x, hidden, b["down"], b["up"], b["scale"], plan, dx=b["dx0"])
    ref, g, err, g_err = _low_rank(b, b["dy"], b["up"], b["down"], b["dx0"])
    _close(dx, ref, err + H * ref.abs(), "dx")
    dyd, hd = b["dy"].double(), hidden.double()
    # g is rounded once to bf16, and once more with the scale of an 8-bit x
    g_err = g_err + (2 if packed else 1) * H * g.abs()
    for ad in range(a):
        rows = (b["token"] == ad).nonzero().flatten()
        c = (rows.numel() + 8) * U
        ref = g[rows].T @ xd[rows]
        tol = (g_err[rows].T + c * g[rows].abs().T) @ xd[rows].abs() + H * ref.abs()
        _close(ddown[ad], ref, tol, ("ddown", ad))
        ref = hd[rows].T @ dyd[rows]
        _close(dup[ad], ref, c * (hd[rows].abs().T @ dyd[rows].abs()) + H * ref.abs(), ("dup", ad))
    # the same bits again, and in place
    acc = b["dx0"].clone()
    again = ops.adapter_backward(b["dy"], x, hidden, b["down"], b["up"], b["scale"], plan, dx=acc, out=acc)
    assert again[0] is acc
    for p, q in zip((dx, ddown, dup), again):
        assert torch.equal(p, q)


def test_gradients_agree_with_differences_of_the_forward_pass():
    # loss = <dy, out> is linear in x and in either factor: a step along the
    # gradient changes it by the gradient's product with the step, up to the
    # roundings of the two forward results and of the gradient itself
    from diffuser_b200 import ops
    b = _batch(4, [70, 130, 61], [1, 0, 1], 5, 256, 192, 16, 2)
    plan = _plan(b)
    y0 = torch.zeros_like(b["y"])
    _, hidden = ops.adapter_add(y0, b["x"], b["down"], b["up"], b["scale"], plan, return_hidden=True)
    grads = ops.adapter_backward(b["dy"], b["x"], hidden, b["down"], b["up"], b["scale"], plan)
    for what, grad in zip(("x", "down", "up"), grads):
        grad = grad.double()
        step = grad * (b[what].double().std() / grad.std())
        moved = dict(b, **{what: (b[what].double() + step).to(torch.bfloat16)})
        step = moved[what].double() - b[what].double()
        loss, size = [], 0.0
        for v in (b, moved):
            ref, _, err, _ = _low_rank(v, v["x"], v["down"], v["up"], y0)
            out = ops.adapter_add(y0, v["x"], v["down"], v["up"], v["scale"], plan)
            loss.append((out.double() * b["dy"].double()).sum())
            size += ((err + H * ref.abs()) * b["dy"].double().abs()).sum()
        size += (2 * H * grad.abs() * step.abs()).sum()
        pred = (grad * step).sum()
        assert (loss[1] - loss[0] - pred).abs() <= size < pred, (what, loss, pred, size)


def test_neighbours_that_are_not_finite_do_not_travel():
    # rows of another adapter, of none and behind the last request hold NaN and infinities
    from diffuser_b200 import ops
    b = _batch(6, [9, 20, 150, 3, 40], [0, 1, 0, -1, 2], 7, 128, 96, 16, 3, 2)
    plan = _plan(b)
    clean = b["token"] == 0
    args = (b["down"], b["up"], b["scale"], plan)
    want, hidden = ops.adapter_add(b["y"], b["x"], *args, return_hidden=True)
    wx, wd, wu = ops.adapter_backward(b["dy"], b["x"], hidden, *args, dx=b["dx0"])
    bad = torch.where(torch.arange(b["m"], device="cuda") % 2 == 0, float("nan"), float("inf"))[:, None]
    dirty = {k: torch.where(clean[:, None], b[k], bad.to(torch.bfloat16)) for k in ("x", "y", "dy", "dx0")}
    out, hidden = ops.adapter_add(dirty["y"], dirty["x"], *args, return_hidden=True)
    assert torch.equal(out[clean], want[clean]) and out[~clean].isfinite().sum() == 0
    for x in (dirty["x"], ops.checkpoint_pack(dirty["x"])):
        dx, ddown, dup = ops.adapter_backward(dirty["dy"], x, hidden, *args, dx=dirty["dx0"])
        assert torch.equal(dx[clean], wx[clean]) and torch.equal(dup[0], wu[0])
        assert ddown[0].isfinite().all() and (not isinstance(x, torch.Tensor) or torch.equal(ddown[0], wd[0]))


def test_adapter_operands_may_be_strided_views_and_batches():
    from diffuser_b200 import ops
    b = _batch(7, [40, 61], [1, 0], 0, 96, 64, 24, 2)
    plan = _plan(b)
    args = (b["down"], b["up"], b["scale"], plan)
    want = ops.adapter_add(b["y"], b["x"], *args)
    wide = torch.zeros(b["m"], 200, dtype=torch.bfloat16, device="cuda")
    wide[:, 8:104], wide[:, 104:168] = b["x"], b["y"]
    buf = torch.full((b["m"], 96), 7.0, dtype=torch.bfloat16, device="cuda")
    ops.adapter_add(wide[:, 104:168], wide[:, 8:104], *args, out=buf[:, 16:80])
    assert torch.equal(buf[:, 16:80], want) and (buf[:, :16] == 7).all() and (buf[:, 80:] == 7).all()
    odd = torch.zeros(b["m"], 101, dtype=torch.bfloat16, device="cuda")  # rows that are not 16-byte aligned
    odd[:, 3:99] = b["x"]
    assert torch.equal(ops.adapter_add(b["y"], odd[:, 3:99], *args), want)
    with pytest.raises(ValueError, match="out"):
        ops.adapter_add(b["y"], b["x"], *args, out=odd[:, 3:67])
    # [batch, tokens, features], transposed storage
    xt = b["x"].t().contiguous().t()
    assert torch.equal(ops.adapter_add(b["y"].view(1, -1, 64), xt.view(1, -1, 96), *args), want.view(1, -1, 64))


def test_plan_rebuilds_in_place_inside_a_captured_graph():
    from diffuser_b200 import ops
    b = _batch(8, [1] * 24, [i % 4 for i in range(24)], 0, 256, 320, 16, 4)
    ids, offsets = b["ids"].clone(), b["offsets"].clone()
    plan = ops.adapter_plan(ids, offsets, b["m"], 4)
    args = (b["down"], b["up"], b["scale"], plan)

    def step():
        plan.update_(ids, offsets)
        out, hidden = ops.adapter_add(b["y"], b["x"], *args, return_hidden=True)
        return (out, *ops.adapter_backward(b["dy"], b["x"], hidden, *args, dx=b["dx0"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):  # two graphs hold workspaces of their own
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, step()))
    for lengths, use in (([1] * 24, [3, -1] * 12), ([0] * 20 + [24, 0, 0, 0], [2] * 24)):
        ids.copy_(torch.tensor(use, dtype=torch.int32))
        offsets.copy_(torch.tensor([0] + lengths).cumsum(0).to(torch.int32))
        want = None
        for graph, got in graphs:
            graph.replay()
            if want is None:
                torch.cuda.synchronize()
                fresh = ops.adapter_plan(ids.clone(), offsets.clone(), b["m"], 4)
                out, hidden = ops.adapter_add(b["y"], b["x"], *args[:3], fresh, return_hidden=True)
                want = (out, *ops.adapter_backward(b["dy"], b["x"], hidden, *args[:3], fresh, dx=b["dx0"]))
            for p, q in zip(got, want):
                assert torch.equal(p, q)
    assert ops.device_error() == 0


def test_calls_on_two_streams_do_not_share_workspaces():
    from diffuser_b200 import ops
    cases = [_batch(s, [700, 900], [1, 0], 0, 1024, 1024, 32, 2) for s in (9, 10)]
    plans = [_plan(b) for b in cases]
    want = [ops.adapter_add(b["y"], b["x"], b["down"], b["up"], b["scale"], p) for b, p in zip(cases, plans)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cases]
    got = [[], []]
    for _ in range(20):
        for i, (b, p, st) in enumerate(zip(cases, plans, streams)):
            with torch.cuda.stream(st):
                got[i].append(ops.adapter_add(b["y"], b["x"], b["down"], b["up"], b["scale"], p))
    torch.cuda.synchronize()
    for i in range(2):
        for o in got[i]:
            assert torch.equal(o, want[i])


@pytest.mark.parametrize("ids,offsets,kept", [
    ([0, 5, 1, -2], [0, 3, 6, 9, 12], [0, 0, 0, -1, -1, -1, 1, 1, 1, -1, -1, -1]),  # ids out of range: none
    ([0, 1, 1, 0], [0, 6, 3, 9, 12], [-1] * 12),      # offsets that decrease
    ([0, 1, 1, 0], [0, 3, 6, 9, 13], [-1] * 12),      # offsets past the batch
    ([0, 1, 1, 0], [-1, 3, 6, 9, 12], [-1] * 12),     # offsets before it
])
def test_bad_indices_are_reported_and_stay_in_range(ids, offsets, kept):
    from diffuser_b200 import _lib, ops
    b = _batch(11, [3] * 4, [0, 1, 1, 0], 0, 64, 64, 8, 2)
    assert ops.device_error() == 0
    plan = ops.adapter_plan(torch.tensor(ids, dtype=torch.int32, device="cuda"),
                            torch.tensor(offsets, dtype=torch.int32, device="cuda"), 12, 2)
    out = ops.adapter_add(b["y"], b["x"], b["down"], b["up"], b["scale"], plan)
    assert ops.device_error() == _lib.DQ_ERR_INDEX and ops.device_error() == 0
    b["token"] = torch.tensor(kept).cuda()
    ref, _, err, _ = _low_rank(b, b["x"], b["down"], b["up"], b["y"])
    _close(out, ref, err + H * ref.abs(), "out")


def test_offsets_past_32_bits():
    from diffuser_b200 import ops
    m, n, k = (1 << 31) // 16384 + 300, 16384, 64  # the last rows start past 2^31 elements
    g = torch.Generator(device="cuda").manual_seed(12)
    y = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
    x, down, up = _rn(g, m, k), _rn(g, 2, 8, k, std=0.1), _rn(g, 2, 8, n, std=0.3)
    scale = torch.ones(2, device="cuda")
    ids = torch.tensor([0, 1], dtype=torch.int32, device="cuda")
    offsets = torch.tensor([0, 5, m], dtype=torch.int32, device="cuda")
    plan = ops.adapter_plan(ids, offsets, m, 2)
    _, hidden = ops.adapter_add(y, x, down, up, scale, plan, out=y, return_hidden=True)
    rows = slice(m - 200, m)
    ref = hidden[rows].double() @ up[1].double()
    tol = (10 * U * (hidden[rows].double().abs() @ up[1].double().abs())) + H * ref.abs()
    _close(y[rows], ref, tol, "last rows")
    # y as the gradient: dup = hidden^T dy needs every row
    _, _, dup = ops.adapter_backward(y, x, hidden, down, up, scale, plan)
    ref = torch.zeros(8, n, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(ref)
    for lo in range(5, m, 8192):
        hd, dy = hidden[lo:lo + 8192].double().T, y[lo:lo + 8192].double()
        ref += hd[:, :dy.shape[0]] @ dy
        size += hd.abs()[:, :dy.shape[0]] @ dy.abs()
    # 16 tokens per MMA: at most m / 16 additions one after another, and 16 within one
    _close(dup[1], ref, (m // 16 + 40) * U * size + H * ref.abs(), "dup")


def test_adapter_refusals():
    from diffuser_b200 import ops
    b = _batch(13, [4, 4], [0, 1], 0, 64, 64, 8, 2)
    plan = _plan(b)
    down, up, scale = b["down"], b["up"], b["scale"]
    add = lambda y=b["y"], x=b["x"], d=down, u=up, s=scale, p=plan, **kw: ops.adapter_add(y, x, d, u, s, p, **kw)  # noqa: E731
    for kw in (dict(x=b["x"][:5]), dict(x=b["x"][:, :56]), dict(u=up[:1]), dict(y=b["y"][:3], x=b["x"][:3]),
               dict(act="relu"), dict(out=torch.empty(3, 64, dtype=torch.bfloat16, device="cuda"))):
        with pytest.raises(ValueError):
            add(**kw)
    for kw in (dict(x=b["x"].float()), dict(s=scale.double()), dict(d=down.float()), dict(p=None),
               dict(d=down.transpose(1, 2))):
        with pytest.raises(TypeError):
            add(**kw)
    with pytest.raises(ValueError, match="multiples of 8"):
        add(d=down[:, :4].contiguous(), u=up[:, :4].contiguous())
    with pytest.raises(ops._lib.DqError):  # a gated act changes the rows' width: not in place
        add(out=b["y"][:, :32], act="swiglu")
    with pytest.raises(ValueError):
        ops.adapter_plan(b["ids"], b["offsets"][:-1], 8, 2)
    with pytest.raises(TypeError):
        ops.adapter_plan(b["ids"].long(), b["offsets"], 8, 2)
    with pytest.raises(ValueError):
        ops.adapter_plan(b["ids"], b["offsets"], 8, 0)
    with pytest.raises(RuntimeError, match="CUDA"):
        add(x=b["x"].cpu())
    hidden = torch.zeros(8, 8, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(TypeError):
        ops.adapter_backward(b["dy"], b["x"], hidden[:, :4], down, up, scale, plan)
    with pytest.raises(ValueError):
        ops.adapter_backward(b["dy"], ops.checkpoint_pack(b["x"][:4]), hidden, down, up, scale, plan)


# ---------------------------------------------------------------- checkpoints
def _pack_reference(x):
    m, k = x.shape
    nb = -(-k // 128)
    xb = torch.nn.functional.pad(x.float(), (0, nb * 128 - k)).view(m, nb, 128)
    amax = xb.abs().amax(2).clamp_min(1e-12)
    scales = amax / torch.full_like(amax, 127)
    codes = (xb / scales[:, :, None]).round().to(torch.int8).view(m, -1)[:, :k]
    return codes, scales


@pytest.mark.parametrize("m,k", [(1, 16), (3, 128), (5, 144), (77, 1040), (300, 4096), (1, 16384)])
def test_checkpoint_matches_its_definition_bit_for_bit(m, k):
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(k)
    x = _rn(g, m, k)
    x[:, ::37] *= 30
    if m > 2:
        x[1] = 0                                  # a row of zeros
        x[2] = (torch.arange(k, device="cuda") % 255 - 127).to(torch.bfloat16) / 2  # many ties
    p = ops.checkpoint_pack(x)
    codes, scales = _pack_reference(x)
    assert torch.equal(p.scales, scales) and torch.equal(p.codes, codes)
    want = (codes.float() * scales.repeat_interleave(128, 1)[:, :k]).to(torch.bfloat16)
    assert torch.equal(ops.checkpoint_unpack(p), want)
    # half a code of the run's scale, and the bf16 rounding
    tol = 0.5 * scales.double().repeat_interleave(128, 1)[:, :k] * (1 + 2 ** -10) + H * x.double().abs()
    _close(want, x.double(), tol, "restored")


def test_checkpoint_of_views_tiny_values_and_rows_that_are_not_finite():
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(3)
    wide = _rn(g, 6, 400)
    p = ops.checkpoint_pack(wide[:, 8:264])
    q = ops.checkpoint_pack(wide[:, 8:264].contiguous())
    assert torch.equal(p.codes, q.codes) and torch.equal(p.scales, q.scales)
    out = torch.full((6, 320), 3.0, dtype=torch.bfloat16, device="cuda")
    ops.checkpoint_unpack(p, out=out[:, 32:288])
    assert torch.equal(out[:, 32:288], ops.checkpoint_unpack(q)) and (out[:, :32] == 3).all()
    b3 = _rn(g, 2, 5, 160)
    assert ops.checkpoint_unpack(ops.checkpoint_pack(b3)).shape == (2, 5, 160)
    x = _rn(g, 4, 256)
    x[0, 5], x[1, 200], x[2, 3] = float("nan"), float("inf"), -float("inf")
    x[3] *= 1e-30
    r = ops.checkpoint_unpack(ops.checkpoint_pack(x))
    assert r[0, :128].isnan().all() and r[1, 128:].isnan().all() and r[2, :128].isnan().all()
    assert r[0, 128:].isfinite().all() and r[1, :128].isfinite().all() and not r[3].any()
    assert ops.checkpoint_pack(x[:0]).codes.shape == (0, 256)
    with pytest.raises(ValueError):
        ops.checkpoint_pack(x[:, :40])
    with pytest.raises(TypeError):
        ops.checkpoint_pack(x.float())
    with pytest.raises(ValueError):
        ops.PackedActivation(p.codes, p.scales[:, :1])
    with pytest.raises(ValueError):
        ops.checkpoint_unpack(p, out=out[:, 1:257])


# ------------------------------------------------------------ input gradients
@pytest.mark.parametrize("m,n,k", [(1, 64, 64), (3, 72, 128), (130, 520, 320), (257, 1032, 192), (1030, 264, 576)])
@pytest.mark.parametrize("fmt", ["nf4", "nf4_bf16", "fp8"])
def test_input_gradient_matches_the_dequantized_weight(m, n, k, fmt):
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(n)
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    dy = _rn(g, m, n)
    if fmt == "fp8":
        k -= 48  # rows of 16-multiples
        w8, s = ops.fp8_quantize(w[:, :k].contiguous())
        got, wd = ops.fp8_linear_dgrad(dy, w8, float(s)), ops.fp8_dequantize(w8, float(s))
    else:
        packed, absmax = ops.ltx23_nf4_quantize(w)
        am = absmax.to(torch.bfloat16) if fmt == "nf4_bf16" else absmax
        got, wd = ops.nf4_linear_dgrad(dy, packed, am, k), ops.ltx23_nf4_dequantize(packed, absmax, (n, k))
    ref = dy.double() @ wd.double()
    tol = (n + 8) * U * (dy.double().abs() @ wd.double().abs()) + H * ref.abs()
    _close(got, ref, tol, fmt)
    assert ops.device_error() == 0


def test_input_gradient_refusals_and_batches():
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(1)
    w = torch.randn(64, 128, generator=g, device="cuda") * 0.02
    packed, absmax = ops.ltx23_nf4_quantize(w)
    dy = _rn(g, 2, 3, 64)
    assert ops.nf4_linear_dgrad(dy, packed, absmax, 128).shape == (2, 3, 128)
    assert ops.nf4_linear_dgrad(dy[:, :0], packed, absmax, 128).shape == (2, 0, 128)
    with pytest.raises(ValueError):
        ops.nf4_linear_dgrad(dy, packed, absmax, 96)
    with pytest.raises(ValueError):
        ops.nf4_linear_dgrad(dy[..., :32], packed, absmax, 128)
    with pytest.raises(TypeError):
        ops.nf4_linear_dgrad(dy.float(), packed, absmax, 128)
    with pytest.raises(ValueError, match="% 8"):
        ops.fp8_linear_dgrad(dy[..., :60], torch.zeros(60, 64, dtype=torch.float8_e4m3fn, device="cuda"), 1.0)


# few tokens: the weight is decoded next to the product (one launch); one token
# tile and two, ragged token counts, sums split 1, 2, 4 and 8 ways, ends inside a
# 64-row step and inside a 128-feature slab
@pytest.mark.parametrize("m,n,k", [(512, 2048, 192), (333, 2056, 1024), (300, 4168, 4160), (256, 136, 64),
                                   (48, 200, 4096), (17, 72, 9024), (16, 64, 128), (400, 1000, 256)])
@pytest.mark.parametrize("fmt", ["nf4", "fp8"])
def test_input_gradient_of_few_tokens(m, n, k, fmt):
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(m)
    w = torch.randn(n, k, generator=g, device="cuda") * 0.02
    dy = _rn(g, m, n)
    if fmt == "fp8":
        k -= 16
        w8, s = ops.fp8_quantize(w[:, :k].contiguous())
        s = float(s)  # on the host before the capture
        call, wd = (lambda d: ops.fp8_linear_dgrad(d, w8, s)), ops.fp8_dequantize(w8, s)
    else:
        packed, absmax = ops.ltx23_nf4_quantize(w)
        call, wd = (lambda d: ops.nf4_linear_dgrad(d, packed, absmax, k)), ops.ltx23_nf4_dequantize(packed, absmax, (n, k))
    got = call(dy)
    ref = dy.double() @ wd.double()
    tol = (n + 8) * U * (dy.double().abs() @ wd.double().abs()) + H * ref.abs()
    _close(got, ref, tol, fmt)
    # the same sums in the same order on another stream, replayed from a graph
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        call(dy)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            again = call(dy)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(again, got)
    # a row that is not finite stays its own row's affair
    bad = dy.clone()
    bad[m // 2, 3], bad[m - 1] = float("nan"), float("inf")
    out = call(bad)
    keep = [i for i in range(m) if i not in (m // 2, m - 1)]
    assert torch.equal(out[keep], got[keep]) and out[m // 2].isnan().all() and not out[m - 1].isfinite().any()
    assert ops.device_error() == 0


def test_outputs_may_not_overlap_what_is_still_read():
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(2)
    ids, off = (torch.tensor(v, dtype=torch.int32, device="cuda") for v in ([0], [0, 20]))
    plan = ops.adapter_plan(ids, off, 20, 1)
    down, up, scale = _rn(g, 1, 8, 64), _rn(g, 1, 8, 64), torch.ones(1, device="cuda")
    x, y = _rn(g, 20, 64), _rn(g, 20, 64)
    want, hidden = ops.adapter_add(y, x, down, up, scale, plan, return_hidden=True)
    with pytest.raises(ValueError, match="overlap"):
        ops.adapter_add(y, x, down, up, scale, plan, out=x)
    both = torch.empty(40, 64, dtype=torch.bfloat16, device="cuda")
    both[1:21].copy_(y)
    with pytest.raises(ValueError, match="overlap"):
        ops.adapter_add(both[1:21], x, down, up, scale, plan, out=both[:20])
    assert torch.equal(ops.adapter_add(both[1:21], x, down, up, scale, plan, out=both[1:21]), want)
    dx = ops.adapter_backward(y, x, hidden, down, up, scale, plan)[0]
    for out in (y, x):
        with pytest.raises(ValueError, match="overlap"):
            ops.adapter_backward(y, x, hidden, down, up, scale, plan, out=out)
    only, none, none2 = ops.adapter_backward(y, x, hidden, down, up, scale, plan, factors=False)
    assert torch.equal(only, dx) and none is none2 is None
    # weights whose elements do not follow one another
    w8 = torch.zeros(64, 128, device="cuda").to(torch.float8_e4m3fn)
    with pytest.raises(TypeError):
        ops.fp8_linear_dgrad(_rn(g, 2, 128), w8.t(), 1.0)
    packed, absmax = ops.ltx23_nf4_quantize(torch.randn(64, 128, generator=g, device="cuda"))
    with pytest.raises(TypeError):
        ops.nf4_linear_dgrad(y, torch.stack([packed, packed], 1)[:, 0], absmax, 128)
    with pytest.raises(TypeError):
        ops.nf4_linear_dgrad(y, packed.to(torch.int8), absmax, 128)
    twice = torch.stack([absmax, absmax], 1)
    assert torch.equal(ops.nf4_linear_dgrad(y, packed, twice[:, 0], 128), ops.nf4_linear_dgrad(y, packed, absmax, 128))


# rows that start 16 but not 32 bytes aligned, by address and by stride
@pytest.mark.parametrize("offset,stride", [(8, 336), (0, 328), (16, 344)])
def test_checkpoint_rows_of_either_alignment(offset, stride):
    from diffuser_b200 import ops
    g = torch.Generator(device="cuda").manual_seed(9)
    x = _rn(g, 37, 304)
    want = ops.checkpoint_pack(x)
    wide = torch.zeros(37 * stride + 64, dtype=torch.bfloat16, device="cuda")
    view = wide[offset:].as_strided((37, 304), (stride, 1))
    view.copy_(x)
    got = ops.checkpoint_pack(view)
    assert torch.equal(got.codes, want.codes) and torch.equal(got.scales, want.scales)
    back = torch.full_like(wide, 7.0)
    out = back[offset:].as_strided((37, 304), (stride, 1))
    ops.checkpoint_unpack(want, out=out)
    assert torch.equal(out, ops.checkpoint_unpack(want))
    gaps = torch.ones_like(back, dtype=torch.bool)
    gaps[offset:].as_strided((37, 304), (stride, 1)).fill_(False)
    assert (back[gaps] == 7.0).all()


@pytest.mark.parametrize("m,n,k", [(7, 8, 64), (300, 24, 128), (600, 16, 64)])
@pytest.mark.parametrize("fmt", ["nf4", "fp8"])
def test_input_gradient_of_few_outputs(m, n, k, fmt):
    """Sums shorter than a step of 64 (the rest of dy's boxes and of the weight's
    tile is past their end), every dx written, nothing behind it."""
    from diffuser_b200 import _lib, ops
    g = torch.Generator(device="cuda").manual_seed(n)
    w, dy = torch.randn(n, k, generator=g, device="cuda") * 0.02, _rn(g, m, n)
    ws = torch.empty(2 * n * k + 256, dtype=torch.uint8, device="cuda")
    dx = torch.full((m + 3, k), 5.0, dtype=torch.bfloat16, device="cuda")
    stream = torch.cuda.current_stream().cuda_stream
    if fmt == "nf4":
        packed, absmax = ops.ltx23_nf4_quantize(w)
        wd = ops.ltx23_nf4_dequantize(packed, absmax, (n, k))
        _lib.call("dq_linear_nf4_dgrad", dy.data_ptr(), m, n, packed.data_ptr(), absmax.data_ptr(), 0, k, dx.data_ptr(),
                  ws.data_ptr(), ws.numel(), stream)
    else:
        w8, s = ops.fp8_quantize(w)
        wd = ops.fp8_dequantize(w8, float(s))
        _lib.call("dq_linear_fp8_dgrad", dy.data_ptr(), m, n, w8.data_ptr(), float(s), k, dx.data_ptr(), ws.data_ptr(),
                  ws.numel(), stream)
    ref = dy.double() @ wd.double()
    tol = (n + 8) * U * (dy.double().abs() @ wd.double().abs()) + H * ref.abs()
    _close(dx[:m], ref, tol, fmt)
    assert (dx[m:] == 5.0).all() and ops.device_error() == 0
