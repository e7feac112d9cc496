"""The operators around the quantized linears that serve and train adapters, as measurable cases.

Operators (``op`` of a case):
  adapter     y + scale_a * (x . down_a^T) . up_a for the tokens of many requests, each with an
              adapter of its own or none, beside a shared projection's output y
  adapter_bwd its gradients: d x (added to the projection's own), d down, d up; x in bf16 or as an
              8-bit activation checkpoint
  checkpoint  a bf16 activation packed to 8 bits and restored
  norm        s = x + residual_scale * gate * N_post(y);  h = N_pre(s) * w * (1 + scale) + shift
  norm_bwd    its gradients
  dgrad       a quantized linear's input gradient, dy . dequant(W)
"""
import math

import torch

own = False

NF4_LEVELS = (-1.0, -0.6961928009986877, -0.5250730514526367, -0.39491748809814453,
              -0.28444138169288635, -0.18477343022823334, -0.09105003625154495, 0.0,
              0.07958029955625534, 0.16093020141124725, 0.24611230194568634, 0.33791524171829224,
              0.44070982933044434, 0.5626170039176941, 0.7229568362236023, 1.0)
BLOCK8 = 128  # features per scale of an 8-bit activation checkpoint


def listed():
    return [
        # one request's modulation vector (one token) through one of eight resident adapters
        dict(name="adapter_one_token", op="adapter", tokens=1, requests=1, k=4096, n=4096, rank=16,
             adapters=8, pad=0, act="none"),
        # a serving batch of single tokens, most with an adapter of their own, some with none
        dict(name="adapter_48_single_tokens", op="adapter", tokens=48, requests=48, k=4096, n=12288,
             rank=16, adapters=24, pad=0, act="none"),
        # four ragged prompts in one padded batch, a feed-forward up projection with its GELU
        dict(name="adapter_ragged_prompts_gelu", op="adapter", tokens=4613, requests=4, k=4096,
             n=16384, rank=32, adapters=6, pad=123, act="gelu_tanh"),
        # fine-tuning step: adapters of three tenants on a square projection, bf16 activations
        dict(name="adapter_bwd_three_tenants", op="adapter_bwd", tokens=1531, requests=7, k=4096,
             n=4096, rank=24, adapters=3, pad=27, packed=False),
        # fine-tuning one adapter over an image + text sequence, activations kept in 8 bits
        dict(name="adapter_bwd_packed_image", op="adapter_bwd", tokens=4608, requests=1, k=4096,
             n=12288, rank=64, adapters=1, pad=0, packed=True),
        # a text stream's activation, and a video step's
        dict(name="checkpoint_text", op="checkpoint", tokens=512, k=4096),
        dict(name="checkpoint_video", op="checkpoint", tokens=6144, k=16384),
        # a short text stream with RMS norms on both sides of the block
        dict(name="norm_text_sandwich", op="norm", batch=2, seq=77, dim=2304, post="rms", pre="rms",
             weights=True, modulated=True, residual_scale=0.5),
        # an image stream with the AdaLN-Zero boundary (no norm after the block)
        dict(name="norm_image_adaln", op="norm", batch=1, seq=4608, dim=4096, post="none", pre="layer",
             weights=False, modulated=True, residual_scale=1.0),
        # the same stream's backward pass with norms on both sides
        dict(name="norm_bwd_image_sandwich", op="norm_bwd", batch=2, seq=2304, dim=4096, post="rms",
             pre="rms", weights=True, modulated=True, residual_scale=1.0),
        # input gradients: a text stream through an NF4 projection, a video step through an fp8 one
        dict(name="dgrad_nf4_text", op="dgrad", tokens=333, n=4096, k=4096, fmt="nf4"),
        dict(name="dgrad_fp8_video", op="dgrad", tokens=6144, n=12288, k=4096, fmt="fp8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(v, q):
    return max(q, int(round(v / q)) * q)


def draw(rng):
    op = rng.choice(["adapter", "adapter", "adapter_bwd", "checkpoint", "norm", "norm_bwd", "dgrad"])
    if op in ("adapter", "adapter_bwd"):
        tokens = _log(rng, 1, 4608)
        k, n = _mult(_log(rng, 512, 4096), 64), _mult(_log(rng, 512, 12288), 8)
        pad = rng.choice([0, 0, rng.randint(0, max(0, tokens // 8))])
        requests = rng.choice([1, min(tokens - pad, rng.randint(1, 12)), min(tokens - pad, _log(rng, 1, 256))])
        case = dict(op=op, tokens=tokens, requests=max(1, requests), k=k, n=n,
                    rank=8 * rng.choice([1, 2, 2, 3, 4, 8, 16]),
                    adapters=_log(rng, 1, 32 if op == "adapter" else 8), pad=pad)
        if op == "adapter":
            case["act"] = rng.choice(["none", "none", "gelu_tanh"])
        else:
            case["packed"] = rng.random() < 0.5
        return case
    if op == "checkpoint":
        return dict(op=op, tokens=_log(rng, 1, 6144), k=_mult(_log(rng, 64, 16384), 16))
    if op in ("norm", "norm_bwd"):
        return dict(op=op, batch=rng.randint(1, 4), seq=_log(rng, 1, 1152), dim=_mult(_log(rng, 64, 8192), 8),
                    post=rng.choice(["none", "rms", "layer"]), pre=rng.choice(["rms", "layer"]),
                    weights=rng.random() < 0.5, modulated=rng.random() < 0.7,
                    residual_scale=rng.choice([1.0, 0.5, 0.2236]))
    return dict(op=op, tokens=_log(rng, 1, 4608), n=_mult(_log(rng, 256, 12288), 64),
                k=_mult(_log(rng, 256, 4096), 64), fmt=rng.choice(["nf4", "fp8"]))


def _split(case, g):
    """Lengths of the requests (each at least one token) and their adapters (-1: none)."""
    live, r = case["tokens"] - case["pad"], case["requests"]
    cuts = (torch.randperm(live - 1, generator=g)[:r - 1] + 1).sort().values
    offsets = torch.cat([torch.zeros(1, dtype=torch.int64), cuts, torch.tensor([live])])
    ids = torch.randint(0, case["adapters"], (r,), generator=g)
    if r > 2:  # a few requests carry none
        ids[torch.rand(r, generator=g) < 0.125] = -1
    return ids.to(torch.int32), offsets.to(torch.int32)


def _token_adapter(ids, offsets, tokens):
    """The adapter of each token, -1 where it has none (padding rows too)."""
    lengths = (offsets[1:] - offsets[:-1]).long()
    of_token = torch.repeat_interleave(ids.long(), lengths)
    return torch.cat([of_token, of_token.new_full((tokens - of_token.numel(),), -1)])


def _pack_plain(x):
    """8-bit codes and float32 scales of a float32 activation, by rows and runs of BLOCK8 features."""
    m, k = x.shape
    nb = -(-k // BLOCK8)
    xb = torch.nn.functional.pad(x, (0, nb * BLOCK8 - k)).view(m, nb, BLOCK8)
    amax = xb.abs().amax(dim=2).clamp_min(1e-12)
    scales = amax / torch.full_like(amax, 127)  # a division: by a number it is a product with 1 / 127
    codes = (xb / scales[:, :, None]).round().view(m, -1)[:, :k].to(torch.int8)
    return codes.contiguous(), scales


def _unpack_plain(codes, scales):
    m, k = codes.shape
    return codes.to(scales.dtype) * scales.repeat_interleave(BLOCK8, dim=1)[:, :k]


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    h = torch.Generator().manual_seed(seed)

    def rn(*shape, std=1.0, dtype=torch.bfloat16):
        return (torch.randn(*shape, generator=g, device="cuda") * std).to(dtype)

    op, st = case["op"], dict(case=case)
    if op in ("adapter", "adapter_bwd"):
        m, k, n, r, a = case["tokens"], case["k"], case["n"], case["rank"], case["adapters"]
        ids, offsets = _split(case, h)
        st.update(x=rn(m, k), down=rn(a, r, k, std=k ** -0.5), up=rn(a, r, n, std=0.5 * r ** -0.5),
                  scale=torch.rand(a, generator=g, device="cuda") + 0.5,
                  ids=ids.cuda(), offsets=offsets.cuda(),
                  token_adapter=_token_adapter(ids, offsets, m).cuda())
        if op == "adapter":
            st["y"] = rn(m, n)
        else:
            st.update(dy=rn(m, n, std=0.1), dx0=rn(m, k, std=0.1))
            st["hidden"] = _down(st, st["x"].float(), st["down"])[0].to(torch.bfloat16)
            if case["packed"]:
                st["codes"], st["scales"] = _pack_plain(st.pop("x").float())
        if own:  # the tokens sorted by adapter: built once for a batch, used by every layer it passes
            from diffuser_b200 import ops
            st["plan"] = ops.adapter_plan(st["ids"], st["offsets"], m, a)
    elif op == "checkpoint":
        # activations with a few features that stand out, as normalized and gated inputs have
        x = rn(case["tokens"], case["k"], dtype=torch.float32)
        x *= 1 + 15 * (torch.rand(case["k"], generator=g, device="cuda") < 0.01)
        st["x"] = x.to(torch.bfloat16)
    elif op in ("norm", "norm_bwd"):
        b, s, d = case["batch"], case["seq"], case["dim"]
        st["y"] = rn(b, s, d, std=2.0)
        st["gate"] = rn(b, d, std=0.7) if case["modulated"] else None
        st["scale"], st["shift"] = (rn(b, d, std=0.3), rn(b, d, std=0.3)) if case["modulated"] else (None, None)
        st["pre_weight"] = rn(d, std=0.2) + 1 if case["weights"] else None
        st["post_weight"] = rn(d, std=0.2) + 1 if case["weights"] and case["post"] != "none" else None
        if op == "norm":
            st["x"] = rn(b, s, d, std=1.5)
        else:
            st.update(s=rn(b, s, d, std=1.5) + 0.1, ds=rn(b, s, d, std=0.1), dh=rn(b, s, d, std=0.1))
    else:
        m, n, k = case["tokens"], case["n"], case["k"]
        st["dy"] = rn(m, n, std=0.1)
        w = rn(n, k, std=0.02, dtype=torch.float32)
        if case["fmt"] == "nf4":
            blocks = w.view(-1, 64)
            st["absmax"] = blocks.abs().amax(dim=1)
            levels = torch.tensor(NF4_LEVELS, device="cuda")
            codes = torch.bucketize(blocks / st["absmax"][:, None], (levels[1:] + levels[:-1]) / 2).view(-1, 2)
            st["packed"] = (codes[:, 0] * 16 + codes[:, 1]).to(torch.uint8)
        else:
            st["w_scale"] = float(w.abs().max()) / 448
            st["w8"] = (w / st["w_scale"]).to(torch.float8_e4m3fn)
    return st


# ------------------------------------------------------------------ plain forms
def _down(st, x, bank):
    """scale_a * x . bank_a^T of each token's own adapter (zeros without one), and the same spread
    over the adapters' columns [tokens, adapters * rank], zero in all but the token's own."""
    a, r, _ = bank.shape
    own_columns = torch.nn.functional.one_hot(st["token_adapter"] + 1, a + 1)[:, 1:].to(x.dtype)
    v = (x @ bank.reshape(a * r, -1).to(x.dtype).T).view(-1, a, r)
    v = v * (own_columns * st["scale"].to(x.dtype))[:, :, None]
    return v.sum(dim=1), v.reshape(-1, a * r)


def _gelu_tanh(v):
    return 0.5 * v * (1 + torch.tanh(0.7978845608028654 * (v + 0.044715 * v * v * v)))


def _norm_plain(v, kind, eps):
    """(normalized v, reciprocal deviation) over the last axis."""
    if kind == "none":
        return v, torch.ones_like(v[..., :1])
    if kind == "layer":
        v = v - v.mean(dim=-1, keepdim=True)
    rstd = torch.rsqrt((v * v).mean(dim=-1, keepdim=True) + eps)
    return v * rstd, rstd


def _norm_grad_plain(d, t, rstd, kind):
    if kind == "none":
        return d
    out = d - t * (d * t).mean(dim=-1, keepdim=True)
    if kind == "layer":
        out = out - d.mean(dim=-1, keepdim=True)
    return out * rstd


def _norm_forward(st, f):
    case = st["case"]
    post = _norm_plain(f(st["y"]), case["post"], 1e-6)[0]
    if st["post_weight"] is not None:
        post = post * f(st["post_weight"])
    if st["gate"] is not None:
        post = post * f(st["gate"])[:, None]
    s = f(st["x"]) + case["residual_scale"] * post
    h = _norm_plain(s, case["pre"], 1e-6)[0]
    if st["pre_weight"] is not None:
        h = h * f(st["pre_weight"])
    if st["scale"] is not None:
        h = h * (1 + f(st["scale"]))[:, None] + f(st["shift"])[:, None]
    return s, h


def _norm_backward(st, f):
    case = st["case"]
    rs, dh = case["residual_scale"], f(st["dh"])
    t, rstd = _norm_plain(f(st["s"]), case["pre"], 1e-6)
    w = f(st["pre_weight"]) if st["pre_weight"] is not None else 1.0
    one = (1 + f(st["scale"]))[:, None] if st["scale"] is not None else 1.0
    out = dict(dshift=dh.sum(dim=1), dscale=(dh * t * w).sum(dim=1)) if st["scale"] is not None else {}
    if st["pre_weight"] is not None:
        out["dpre_weight"] = (dh * one * t).sum(dim=(0, 1))
    dx = f(st["ds"]) + _norm_grad_plain(dh * w * one, t, rstd, case["pre"])
    yhat, rstd = _norm_plain(f(st["y"]), case["post"], 1e-6)
    w = f(st["post_weight"]) if st["post_weight"] is not None else 1.0
    gate = f(st["gate"])[:, None] if st["gate"] is not None else 1.0
    if st["gate"] is not None:
        out["dgate"] = rs * (dx * yhat * w).sum(dim=1)
    if st["post_weight"] is not None:
        out["dpost_weight"] = rs * (dx * gate * yhat).sum(dim=(0, 1))
    dy = _norm_grad_plain(rs * dx * gate * w, yhat, rstd, case["post"])
    return dict(out, dx=dx, dy=dy)


def _weight(st, n, k):
    """The bf16 weight that the quantized one stands for, in float32."""
    if "packed" in st:
        levels = torch.tensor(NF4_LEVELS, device="cuda").to(torch.bfloat16).float()
        codes = torch.stack([st["packed"] >> 4, st["packed"] & 15], dim=1).long()
        w = levels[codes].view(-1, 64) * st["absmax"].to(torch.bfloat16).float()[:, None]
    else:
        w = st["w8"].float() * float(torch.tensor(st["w_scale"]).to(torch.bfloat16))
    return w.to(torch.bfloat16).float().view(n, k)


def _run_plain(st):
    case, op = st["case"], st["case"]["op"]
    if op == "adapter":
        spread = _down(st, st["x"].float(), st["down"])[1]
        out = st["y"].float() + spread @ st["up"].reshape(spread.shape[1], -1).float()
        return (_gelu_tanh(out) if case["act"] == "gelu_tanh" else out).to(torch.bfloat16)
    if op == "adapter_bwd":
        a, r = case["adapters"], case["rank"]
        x = _unpack_plain(st["codes"], st["scales"]) if case["packed"] else st["x"].float()
        dy = st["dy"].float()
        spread = _down(st, dy, st["up"])[1]
        own_columns = torch.nn.functional.one_hot(st["token_adapter"] + 1, a + 1)[:, 1:].float()
        hidden = (st["hidden"].float()[:, None] * own_columns[:, :, None]).reshape(-1, a * r)
        return dict(dx=(st["dx0"].float() + spread @ st["down"].reshape(a * r, -1).float()).to(torch.bfloat16),
                    ddown=(spread.T @ x).view(a, r, -1).to(torch.bfloat16),
                    dup=(hidden.T @ dy).view(a, r, -1).to(torch.bfloat16))
    if op == "checkpoint":
        codes, scales = _pack_plain(st["x"].float())
        return dict(restored=_unpack_plain(codes, scales).to(torch.bfloat16), scales=scales)
    if op == "norm":
        s, h = _norm_forward(st, lambda t: t.float())
        return dict(s=s.to(torch.bfloat16), h=h.to(torch.bfloat16))
    if op == "norm_bwd":
        out = _norm_backward(st, lambda t: t.float())
        return dict(out, dx=out["dx"].to(torch.bfloat16), dy=out["dy"].to(torch.bfloat16))
    return (st["dy"].float() @ _weight(st, case["n"], case["k"])).to(torch.bfloat16)


# -------------------------------------------------------- the framework's calls
def _norm_args(st):
    case = st["case"]
    return dict(gate=st["gate"], post=None if case["post"] == "none" else case["post"], pre=case["pre"],
                post_weight=st["post_weight"], pre_weight=st["pre_weight"], scale=st["scale"],
                shift=st["shift"], residual_scale=case["residual_scale"], eps=1e-6)


def _run_own(st):
    from diffuser_b200 import flux, ops
    case, op = st["case"], st["case"]["op"]
    if op == "adapter":
        return ops.adapter_add(st["y"], st["x"], st["down"], st["up"], st["scale"], st["plan"],
                               act=None if case["act"] == "none" else case["act"])
    if op == "adapter_bwd":
        x = ops.PackedActivation(st["codes"], st["scales"]) if case["packed"] else st["x"]
        dx, ddown, dup = ops.adapter_backward(st["dy"], x, st["hidden"], st["down"], st["up"], st["scale"],
                                              st["plan"], dx=st["dx0"])
        return dict(dx=dx, ddown=ddown, dup=dup)
    if op == "checkpoint":
        packed = ops.checkpoint_pack(st["x"])
        return dict(restored=ops.checkpoint_unpack(packed), scales=packed.scales)
    if op == "norm":
        s, h = flux.gated_norm(st["x"], st["y"], **_norm_args(st))
        return dict(s=s, h=h)
    if op == "norm_bwd":
        grads = flux.gated_norm_backward(st["ds"], st["dh"], st["s"], st["y"], **_norm_args(st))
        return {k: v for k, v in grads.items() if v is not None}
    if case["fmt"] == "nf4":
        return ops.nf4_linear_dgrad(st["dy"], st["packed"], st["absmax"], case["k"])
    return ops.fp8_linear_dgrad(st["dy"], st["w8"], st["w_scale"])


def run(state):
    return _run_own(state) if own else _run_plain(state)


def work(case):
    op = case["op"]
    if op in ("adapter", "adapter_bwd"):
        m, k, n, r = case["tokens"], case["k"], case["n"], case["rank"]
        used = min(case["adapters"], case["requests"])
        banks = 2 * used * r * (k + n)
        if op == "adapter":
            return dict(bytes=2 * (m * k + 2 * m * n) + banks, flops=2 * m * r * (k + n))
        x = m * k * (1 + 4 / BLOCK8) if case["packed"] else 2 * m * k
        return dict(bytes=x + 2 * (m * n + m * r + 2 * m * k) + banks + 2 * case["adapters"] * r * (k + n),
                    flops=4 * m * r * (k + n))
    if op == "checkpoint":
        e = case["tokens"] * case["k"]
        return dict(bytes=e * (2 + 2 * (1 + 4 / BLOCK8) + 2), flops=4 * e)
    if op in ("norm", "norm_bwd"):
        e = case["batch"] * case["seq"] * case["dim"]
        return dict(bytes=(8 if op == "norm" else 12) * e, flops=(16 if op == "norm" else 40) * e)
    m, n, k = case["tokens"], case["n"], case["k"]
    weight = n * k * (0.5 + 4 / 64) if case["fmt"] == "nf4" else n * k
    return dict(bytes=2 * m * (n + k) + weight, flops=2 * m * n * k)


# ------------------------------------------------------------- 64-bit definition
def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "adapter":
        out = st["y"].double()
        for i, a in enumerate(st["ids"].tolist()):
            if a >= 0:
                rows = slice(int(st["offsets"][i]), int(st["offsets"][i + 1]))
                v = st["x"][rows].double() @ st["down"][a].double().T
                out[rows] += v @ (st["up"][a].double() * float(st["scale"][a]))
        return torch.nn.functional.gelu(out, approximate="tanh") if case["act"] == "gelu_tanh" else out
    if op == "adapter_bwd":
        dx = st["dx0"].double()
        ddown = torch.zeros(st["down"].shape, dtype=torch.float64, device="cuda")
        dup = torch.zeros(st["up"].shape, dtype=torch.float64, device="cuda")
        for i, a in enumerate(st["ids"].tolist()):
            if a >= 0:
                rows = slice(int(st["offsets"][i]), int(st["offsets"][i + 1]))
                dy = st["dy"][rows].double()
                if case["packed"]:
                    x = torch.cat([c * s for c, s in zip(
                        st["codes"][rows].double().split(BLOCK8, dim=1),
                        st["scales"][rows].double().split(1, dim=1))], dim=1)
                else:
                    x = st["x"][rows].double()
                gr = dy @ st["up"][a].double().T * float(st["scale"][a])
                dx[rows] += gr @ st["down"][a].double()
                ddown[a] += gr.T @ x
                dup[a] += st["hidden"][rows].double().T @ dy
        return dict(dx=dx, ddown=ddown, dup=dup)
    if op == "checkpoint":
        restored, scales = [], []
        for xb in st["x"].double().split(BLOCK8, dim=1):
            s = xb.abs().amax(dim=1, keepdim=True).clamp_min(1e-12) / 127
            restored.append(torch.round(xb / s) * s)
            scales.append(s)
        return dict(restored=torch.cat(restored, dim=1), scales=torch.cat(scales, dim=1))
    if op in ("norm", "norm_bwd"):
        leaf = {k: v.double().requires_grad_() for k, v in st.items() if isinstance(v, torch.Tensor)}
        d = case["dim"]

        def norm(v, kind, w):
            if kind == "layer":
                v = torch.nn.functional.layer_norm(v, (d,), eps=1e-6)
            elif kind == "rms":
                v = v / torch.sqrt(v.square().mean(-1, keepdim=True) + 1e-6)
            return v if w is None else v * w

        post = norm(leaf["y"], case["post"], leaf.get("post_weight"))
        if "gate" in leaf:
            post = post * leaf["gate"].unsqueeze(1)
        add = case["residual_scale"] * post

        def pre(s):
            h = norm(s, case["pre"], leaf.get("pre_weight"))
            if "scale" in leaf:
                h = h * (1 + leaf["scale"].unsqueeze(1)) + leaf["shift"].unsqueeze(1)
            return h

        if op == "norm":
            s = leaf["x"] + add
            return dict(s=s.detach(), h=pre(s).detach())
        # the same s as given, reached from an x that makes up the difference
        s = (leaf["s"].detach() - add.detach()).requires_grad_()
        x, total = s, s + add
        h = pre(total)
        wanted = {"dx": x, "dy": leaf["y"]}
        for k in ("gate", "scale", "shift", "pre_weight", "post_weight"):
            if k in leaf:
                wanted["d" + k] = leaf[k]
        loss = (total * leaf["ds"].detach()).sum() + (h * leaf["dh"].detach()).sum()
        return dict(zip(wanted, torch.autograd.grad(loss, list(wanted.values()))))
    n, k = case["n"], case["k"]
    if case["fmt"] == "nf4":
        table = torch.tensor(NF4_LEVELS, dtype=torch.bfloat16, device="cuda").double()
        both = torch.stack([table[(st["packed"] // 16).long()], table[(st["packed"] % 16).long()]], dim=1)
        w = both.view(-1, 64) * st["absmax"].to(torch.bfloat16).double()[:, None]
    else:
        w = st["w8"].double() * float(torch.tensor(st["w_scale"]).to(torch.bfloat16))
    return st["dy"].double() @ w.to(torch.bfloat16).double().view(n, k)
