"""Drop-in module mirrors of diffuseR's quantized linears.

``ltx23_nf4_linear`` / ``ltx23_fp8_linear`` keep the reference's constructor,
setters, buffers and forward contract (R/nf4_ltx23.R:211-247,
R/fp8_ltx23.R:49-84), with forward() running the fused sm_100a kernel instead
of dequantize-into-a-buffer + cuBLAS.  ``swap_quant_linears`` mirrors the
loader swap ``do.call(`$<-`, list(parent, leaf, quant_mod))``
(R/quantize_flux.R:541-576).
"""
from __future__ import annotations

import re
import weakref

import torch
from torch import nn

from . import ops

NF4_BLOCK = ops.NF4_BLOCK


def _activate(y: torch.Tensor, act: str) -> torch.Tensor:
    """The activation of a projection's output, in tensor ops."""
    if act == "gelu_tanh":
        return nn.functional.gelu(y, approximate="tanh")
    gate, up = y.unflatten(-1, (-1, 2, 16)).unbind(-2)  # the gated row order
    gate = nn.functional.silu(gate) if act == "swiglu" else nn.functional.gelu(gate, approximate="tanh")
    return (gate * up).flatten(-2)


class _Frozen:
    """The tensors of a frozen linear that a call used and its backward pass
    reads again: held until then, and not to be written in between."""

    def __init__(self, tensors):
        self.tensors = tensors
        self.versions = self._versions()

    def _versions(self):  # (inference tensors count none)
        return [None if t is None or t.is_inference() else t._version for t in self.tensors]

    def again(self):
        if self._versions() != self.versions:
            raise RuntimeError("a frozen linear's weight was changed after the call whose backward pass needs it")
        return self.tensors


class _FrozenProjection(torch.autograd.Function):
    """A quantized linear whose input takes a gradient: the forward pass is the
    engine's, the backward pass its input gradient (behind an activation, whose
    argument is computed again)."""

    @staticmethod
    def forward(ctx, x, linear, act):
        weight, bias, factor = linear._operands(x.device)
        ctx.linear, ctx.act, ctx.factor = linear, act, factor
        ctx.frozen = _Frozen((*weight, *(() if act is None else (bias,))))
        if act is not None:
            ctx.save_for_backward(x)
        return linear._run(x, act, None, (weight, bias, factor))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        weight = ctx.frozen.again()
        if ctx.act is not None:
            *weight, bias = weight
            with torch.enable_grad():
                y = ctx.linear._run(ctx.saved_tensors[0], None, None, (weight, bias, ctx.factor)).requires_grad_()
                dy, = torch.autograd.grad(_activate(y, ctx.act), y, dy)
        return ctx.linear._input_grad(dy, weight, ctx.factor), None, None


def _run_linear(linear, x, act, out):
    if getattr(linear, "differentiable", False) and torch.is_grad_enabled() and x.requires_grad:
        if out is not None:
            raise RuntimeError("a differentiable call takes no out")
        return _FrozenProjection.apply(x, linear, act)
    return linear._run(x, act, out)


class Ltx23Nf4Linear(nn.Module):
    """NF4 linear (R/nf4_ltx23.R:211-247).

    Buffers ``weight_nf4`` (uint8 [N*K/2]) and ``weight_absmax`` (float32
    [N*K/64]) move with the module; uint8 survives dtype casts and absmax is
    kept float32 (the forward uses bf16(absmax), which a cast would not change).
    """

    def __init__(self, out_features: int, in_features: int, bias: bool = True):
        super().__init__()
        self.out_features = int(out_features)
        self.in_features = int(in_features)
        n = self.out_features * self.in_features
        self.register_buffer("weight_nf4", torch.zeros(n // 2, dtype=torch.uint8))
        self.register_buffer("weight_absmax", torch.ones(n // NF4_BLOCK, dtype=torch.float32))
        self.scales_bf16 = False
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features))
        else:
            self.register_parameter("bias", None)
        self.gated_act = None
        self.differentiable = False  # in its input (attach_adapters sets it)

    def set_nf4_weight(self, packed: torch.Tensor, absmax: torch.Tensor):
        """Copy packed codes and block scales into the buffers (R/nf4_ltx23.R:228-234)."""
        with torch.no_grad():
            self.weight_nf4.copy_(packed.reshape(-1))
            self.weight_absmax.copy_(absmax.reshape(-1))
        return self

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        want = torch.bfloat16 if getattr(self, "scales_bf16", False) else torch.float32
        if self.weight_absmax.dtype != want:
            self.weight_absmax = self.weight_absmax.to(want)
        return self

    def repack_scales_bf16(self):
        """Load-time repack of the block scales to bf16 (half the scale
        bytes).  The forward casts absmax to bf16 before scaling
        (R/nf4_ltx23.R:97), so the dequantized weights are unchanged."""
        self.weight_absmax = self.weight_absmax.to(torch.bfloat16)
        self.scales_bf16 = True
        return self

    def to_gated(self, act: str = "swiglu"):
        """Reorder the rows of a [gate; up] projection into the gated row
        order and fuse `act` ("swiglu": silu(gate) * up, "geglu_tanh") into
        every forward, which then returns out_features / 2 columns."""
        if act not in ops.GATED_ACTS:
            raise ValueError(f"act must be one of {ops.GATED_ACTS}")
        with torch.no_grad():
            p, a = ops.to_gated_rows_nf4(self.weight_nf4, self.weight_absmax, self.out_features,
                                         self.in_features)
            self.weight_nf4.copy_(p)
            self.weight_absmax.copy_(a)
            if self.bias is not None:
                self.bias.copy_(ops.to_gated_rows(self.bias.detach(), self.out_features))
        self.gated_act = act
        return self

    def forward(self, x: torch.Tensor, act: str | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
        return _run_linear(self, x, act or self.gated_act, out)

    def _operands(self, device):
        """(weight tensors, bias, per-tensor factor) of a call."""
        return (self.weight_nf4, self.weight_absmax), self.bias, None

    def _run(self, x, act, out, operands=None):
        (packed, absmax), bias, _ = operands or self._operands(x.device)
        return ops.nf4_linear(x, packed, absmax, self.out_features, bias, act=act, out=out)

    def _input_grad(self, dy, weight, factor):
        return ops.nf4_linear_dgrad(dy, *weight, self.in_features)

    def input_grad(self, dy: torch.Tensor) -> torch.Tensor:
        """dy . W for a gradient dy of the projection's output."""
        weight, _, factor = self._operands(dy.device)
        return self._input_grad(dy, weight, factor)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, format=nf4"


class Ltx23Fp8Linear(nn.Module):
    """fp8-e4m3 linear with a per-tensor scale (R/fp8_ltx23.R:49-84).

    As in the reference, the fp8 weight and its scale are plain attributes, not
    buffers, so ``.to()`` moves only the bias.  The reference streams them to
    the device on every forward; here the first forward on a device copies them
    once and keeps that copy resident (B200 holds every weight in HBM).
    """

    def __init__(self, out_features: int, in_features: int, bias: bool = True):
        super().__init__()
        self.out_features = int(out_features)
        self.in_features = int(in_features)
        self.weight_fp8 = None
        self.weight_scale = None
        self._resident = None
        self._scale_f = None
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features))
        else:
            self.register_parameter("bias", None)
        self.gated_act = None
        self.differentiable = False  # in its input (attach_adapters sets it)

    def set_fp8_weight(self, weight: torch.Tensor, scale, pin: bool = False):
        """Store the e4m3 weight and float32 scale (R/fp8_ltx23.R:60-68)."""
        if weight.dtype != torch.float8_e4m3fn:
            raise TypeError("weight must be float8_e4m3fn")
        if pin and not weight.is_cuda and torch.cuda.is_available():
            weight = weight.pin_memory()
        self.weight_fp8 = weight
        scale_t = torch.as_tensor(scale).detach().to(device="cpu", dtype=torch.float32)
        self.weight_scale = scale_t
        self._scale_f = float(scale_t)
        self._resident = weight if weight.is_cuda else None
        return self

    def to_gated(self, act: str = "swiglu"):
        """As Ltx23Nf4Linear.to_gated: rows into the gated row order, `act`
        fused into every forward (out_features / 2 output columns)."""
        if act not in ops.GATED_ACTS:
            raise ValueError(f"act must be one of {ops.GATED_ACTS}")
        if self.weight_fp8 is None:
            raise RuntimeError("set_fp8_weight() has not been called")
        self.weight_fp8 = ops.to_gated_rows(self.weight_fp8, self.out_features)
        self._resident = self.weight_fp8 if self.weight_fp8.is_cuda else None
        if self.bias is not None:
            with torch.no_grad():
                self.bias.copy_(ops.to_gated_rows(self.bias.detach(), self.out_features))
        self.gated_act = act
        return self

    def forward(self, x: torch.Tensor, act: str | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
        return _run_linear(self, x, act or self.gated_act, out)

    def _operands(self, device):
        """(weight tensors, bias, per-tensor factor) of a call."""
        return (self._weight_on(device),), self.bias, self._scale_f

    def _run(self, x, act, out, operands=None):
        (w8,), bias, factor = operands or self._operands(x.device)
        return ops.fp8_linear(x, w8, factor, bias, act=act, out=out)

    def _input_grad(self, dy, weight, factor):
        return ops.fp8_linear_dgrad(dy, *weight, factor)

    def input_grad(self, dy: torch.Tensor) -> torch.Tensor:
        """dy . W for a gradient dy of the projection's output."""
        weight, _, factor = self._operands(dy.device)
        return self._input_grad(dy, weight, factor)

    def _weight_on(self, device: torch.device) -> torch.Tensor:
        if self.weight_fp8 is None:
            raise RuntimeError("set_fp8_weight() has not been called")
        w8 = self._resident
        if w8 is None or w8.device != device:
            w8 = self.weight_fp8.to(device=device, non_blocking=True)
            self._resident = w8
        return w8

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, format=fp8"


def concat_nf4_linears(mods):
    """One NF4 linear whose output features are those of `mods`, in order.
    NF4 blocks of 64 never straddle a weight row, so a row range's packed codes
    and block scales are contiguous: concatenating the buffers concatenates
    the rows, with no repacking.  None unless every module is NF4 with the same
    in_features and scale dtype."""
    if not mods or any(not isinstance(m, Ltx23Nf4Linear) for m in mods):
        return None
    k = mods[0].in_features
    if any(m.in_features != k or m.weight_absmax.dtype != mods[0].weight_absmax.dtype for m in mods):
        return None
    dev = mods[0].weight_nf4.device
    fused = Ltx23Nf4Linear(sum(m.out_features for m in mods), k, bias=False).to(dev)
    fused.differentiable = any(m.differentiable for m in mods)
    if mods[0].scales_bf16:
        fused.repack_scales_bf16()
    fused.set_nf4_weight(torch.cat([m.weight_nf4 for m in mods]),
                         torch.cat([m.weight_absmax for m in mods]))
    if any(m.bias is not None for m in mods):
        dt = next(m.bias.dtype for m in mods if m.bias is not None)
        fused.bias = nn.Parameter(torch.cat([
            m.bias.detach().to(dt) if m.bias is not None
            else torch.zeros(m.out_features, dtype=dt, device=dev) for m in mods]), requires_grad=False)
    return fused


def fuse_gated_pair(gate: nn.Module, up: nn.Module, act: str = "geglu_tanh"):
    """One NF4 linear computing act(gate(x)) * up(x) with the gate fused into
    its epilogue (the gated MLP of a Gemma-style text encoder, whose gate_proj
    and up_proj are separate checkpoint weights, R/quantize_gemma3.R:126-130):
    the two weights' rows concatenated as [gate; up] and put in the gated row
    order.  NF4 only (fp8's per-tensor scales differ between the two)."""
    fused = concat_nf4_linears([gate, up])
    if fused is None or gate.out_features != up.out_features:
        raise ValueError("fuse_gated_pair needs two NF4 linears of the same shape")
    return fused.to_gated(act)


class Flux2FeedForward(nn.Module):
    """flux2_feed_forward (R/dit_flux2_modules.R:73-87) on quantized linears:
    ``linear_in`` (dim -> 2 * inner, [gate; up]) runs in the gated row order
    with SiLU(gate) * up fused into its epilogue, then ``linear_out``
    (inner -> dim_out).  Build it from the reference module's two linears with
    ``from_linears``; forward(x) returns the same values as
    linear_out(silu(h[..., :inner]) * h[..., inner:]) with h = linear_in(x)."""

    def __init__(self, linear_in: nn.Module, linear_out: nn.Module):
        super().__init__()
        self.linear_in = linear_in
        self.linear_out = linear_out

    @classmethod
    def from_linears(cls, linear_in: nn.Linear, linear_out: nn.Linear, fmt: str = "nf4"):
        holder = nn.Module()
        holder.linear_in, holder.linear_out = linear_in, linear_out
        swap_quant_linears(holder, lambda key: True, fmt)
        holder.linear_in.to_gated("swiglu")
        return cls(holder.linear_in, holder.linear_out)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return self.linear_out(self.linear_in(x))


# ------------------------------------------------------------------ adapters
class AdapterSelection:
    """Which adapter each batch element uses: ids, int32 on the GPU, one per
    element (-1: none).  Every adapted linear of a model shares it; the plan for
    a token count is built at its first use (an element's tokens follow one
    another, equally many for each).  Streams wait for one another here: a plan's
    build for the stream that set the ids, a use for the stream of the build.  A
    graph capture takes a selection and plans that were made before it (by a
    call, or by plan(tokens)); the graph reads their memory at every replay, so
    keep the selection for as long as the graph.  Of the plans that no capture
    took, the sixteen used last are kept, and those that are in use elsewhere."""

    KEPT = 16

    def __init__(self, ids: torch.Tensor, n_adapters: int):
        if not isinstance(ids, torch.Tensor) or not ids.is_cuda or ids.dtype != torch.int32 or ids.dim() != 1 or \
                ids.numel() == 0:
            raise ValueError("ids must be a 1-d int32 CUDA tensor, one entry per batch element")
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a selection made inside a capture would hold nothing until its replay")
        self.n_adapters = int(n_adapters)
        with torch.cuda.device(ids.device):
            self.ids = ids.clone()
            self._set = self._now()  # stream and event behind the last write of ids
        self._no_plans()

    def _no_plans(self):
        self._plans = weakref.WeakValueDictionary()  # tokens -> plan, every one alive
        self._built = weakref.WeakKeyDictionary()    # plan -> stream and event behind its last build
        self._recent: dict = {}                      # tokens -> plan, the KEPT used last, oldest first
        self._captured: dict = {}                    # tokens -> plan

    def __getstate__(self):  # a copy has ids and plans of its own
        with torch.cuda.device(self.ids.device):
            self._after(self._set, self.ids)
            return {"ids": self.ids.clone(), "n_adapters": self.n_adapters}

    def __setstate__(self, state):
        self.__dict__.update(state)
        self._no_plans()
        with torch.cuda.device(self.ids.device):
            self._set = self._now()

    def _offsets(self, tokens: int) -> torch.Tensor:
        batch = self.ids.numel()
        return torch.arange(batch + 1, dtype=torch.int32, device=self.ids.device) * (tokens // batch)

    def _now(self):
        stream = torch.cuda.current_stream(self.ids.device)
        return stream.cuda_stream, stream.record_event()

    def _after(self, mark, *written: torch.Tensor) -> None:
        """The current stream goes on behind `mark`, whose stream wrote these."""
        handle, event = mark
        if handle != ops._raw_stream(self.ids) and not torch.cuda.is_current_stream_capturing():
            stream = torch.cuda.current_stream(self.ids.device)
            stream.wait_event(event)
            for t in written:
                t.record_stream(stream)

    def plan(self, tokens: int) -> ops.AdapterPlan:
        plan = self._plans.get(tokens)
        if plan is None:
            batch = self.ids.numel()
            if tokens % batch != 0:
                raise ValueError(f"{tokens} tokens are not a whole number per element of a batch of {batch}")
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(f"the plan for {tokens} tokens must be built before a capture: run the call once, "
                                   "or selection.plan(tokens)")
            with torch.cuda.device(self.ids.device):
                self._after(self._set, self.ids)
                plan = ops.adapter_plan(self.ids, self._offsets(tokens), tokens, self.n_adapters)
                self._built[plan] = self._now()
            self._plans[tokens] = plan
        else:
            self._after(self._built[plan], plan.words)
        if torch.cuda.is_current_stream_capturing():
            self._captured[tokens] = plan
        self._recent.pop(tokens, None)
        self._recent[tokens] = plan
        if len(self._recent) > self.KEPT:
            del self._recent[next(iter(self._recent))]
        return plan

    def update_(self, ids: torch.Tensor) -> "AdapterSelection":
        """Other adapters for the same batch size: the plans built so far are
        rebuilt in place (captured graphs that read them see the new ones).  Not
        between a call and its backward pass, which then raises; calls on other
        streams must have finished."""
        if not isinstance(ids, torch.Tensor) or ids.shape != self.ids.shape or ids.dtype != torch.int32:
            raise ValueError(f"ids must hold {self.ids.numel()} int32 entries, as before")
        with torch.cuda.device(self.ids.device):
            capturing = torch.cuda.is_current_stream_capturing()
            self._after(self._set, self.ids)
            self.ids.copy_(ids)
            if not capturing:
                self._set = self._now()
            for tokens, plan in list(self._plans.items()):
                self._after(self._built[plan], plan.words)
                plan.update_(self.ids, self._offsets(tokens))
                if not capturing:
                    self._built[plan] = self._now()
        return self


class _AdaptedProjection(torch.autograd.Function):
    """base(x) + adapters, with the base frozen: gradients of x, down and up."""

    @staticmethod
    def forward(ctx, x, down, up, scale, plan, base, pack):
        operands = base.base._operands(x.device)
        y = base.base._run(x, None, None, operands)
        y, hidden = ops.adapter_add(y, x, down, up, scale, plan, out=y, return_hidden=True)
        if pack:
            packed = ops.checkpoint_pack(x)
            ctx.save_for_backward(hidden, down, up, scale, packed.codes, packed.scales)
        else:
            ctx.save_for_backward(hidden, down, up, scale, x)
        ctx.plan, ctx.version, ctx.base, ctx.pack = plan, plan.version, base.base, pack
        ctx.frozen, ctx.factor = _Frozen(operands[0]), operands[2]
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, dy):
        if ctx.plan.version != ctx.version:
            raise RuntimeError("the adapter plan was rebuilt for another batch after this call")
        hidden, down, up, scale, *x = ctx.saved_tensors
        x = ops.PackedActivation(*x) if ctx.pack else x[0]
        dx = ctx.base._input_grad(dy, ctx.frozen.again(), ctx.factor) if ctx.needs_input_grad[0] else None
        dx, ddown, dup = ops.adapter_backward(dy, x, hidden, down, up, scale, ctx.plan, dx=dx, out=dx,
                                              factors=ctx.needs_input_grad[1] or ctx.needs_input_grad[2],
                                              inputs=ctx.needs_input_grad[0])
        return dx, ddown, dup, None, None, None, None


class AdapterLinear(nn.Module):
    """A quantized linear with a bank of low-rank adapters beside it: every
    batch element's tokens pass the shared weight and its own adapter,
    y + scale_a * (x . down_a^T) . up_a.

    The bank's factors are parameters (bf16, ``down`` [A, r, K], ``up``
    [A, r, N]); the base is frozen.  Set ``selection`` (AdapterSelection), or
    pass a plan, before calling; without either the base runs alone.  With
    gradients enabled the call is differentiable in x and the factors, and
    keeps its input for the backward pass as it is or, with
    ``pack_activations``, in 8 bits.  (As for any leaf of PyTorch's autograd: do
    not capture a backward pass into a CUDA graph while an eager graph over the
    same factors is alive; delete its results first.)"""

    def __init__(self, base: nn.Module, n_adapters: int, rank: int, pack_activations: bool = False):
        super().__init__()
        if not isinstance(base, (Ltx23Nf4Linear, Ltx23Fp8Linear)):
            raise TypeError("AdapterLinear wraps a quantized linear")
        rank = -(-int(rank) // 8) * 8  # the kernels take multiples of 8; the rest stays zero
        if not 8 <= rank <= 128 or base.out_features % 8 != 0 or base.in_features % 8 != 0:
            raise ValueError("adapters need a rank of 1..128 and features that are multiples of 8")
        if pack_activations and base.in_features % 16 != 0:
            raise ValueError("8-bit activations need in_features % 16 == 0")
        self.base = base
        base.differentiable = True
        self.in_features, self.out_features = base.in_features, base.out_features
        self.pack_activations = bool(pack_activations)
        dev = base.weight_nf4.device if isinstance(base, Ltx23Nf4Linear) else \
            (base.weight_fp8.device if base.weight_fp8 is not None else None)
        zeros = lambda *shape: torch.zeros(*shape, dtype=torch.bfloat16, device=dev)  # noqa: E731
        self.down = nn.Parameter(zeros(n_adapters, rank, base.in_features))
        self.up = nn.Parameter(zeros(n_adapters, rank, base.out_features))
        self.register_buffer("scale", torch.ones(n_adapters, dtype=torch.float32, device=dev))
        self.selection: AdapterSelection | None = None

    def _apply(self, fn, recurse=True):
        super()._apply(fn, recurse)
        if self.scale.dtype != torch.float32:
            self.scale = self.scale.float()
        return self

    def set_adapter(self, index: int, a: torch.Tensor, b: torch.Tensor, scale: float = 1.0):
        """Install adapter `index` from its two factors as checkpoints store
        them, a [r, in_features] and b [out_features, r] (r up to the bank's
        rank), with the factor scale (alpha / r).  For a gated base b is in the
        [gate; up] row order."""
        r = a.shape[0]
        if a.shape != (r, self.in_features) or b.shape != (self.out_features, r) or r > self.down.shape[1]:
            raise ValueError(f"expected [r, {self.in_features}] and [{self.out_features}, r] with r <= "
                             f"{self.down.shape[1]}, got {tuple(a.shape)} and {tuple(b.shape)}")
        if not 0 <= index < self.down.shape[0]:
            raise IndexError(f"adapter {index} of {self.down.shape[0]}")
        with torch.no_grad():
            u = b.t()
            if self.base.gated_act is not None:
                u = u.index_select(1, ops.gated_row_order(self.out_features, b.device))
            self.down[index].zero_()[:r].copy_(a)
            self.up[index].zero_()[:r].copy_(u)
            self.scale[index] = float(scale)
        return self

    @property
    def bias(self):
        return self.base.bias

    def project(self, x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
        """The base's projection alone, without an activation."""
        return self.base._run(x, None, out)

    def input_grad(self, dy: torch.Tensor) -> torch.Tensor:
        return self.base.input_grad(dy)

    def forward(self, x: torch.Tensor, act: str | None = None, out: torch.Tensor | None = None,
                plan: ops.AdapterPlan | None = None) -> torch.Tensor:
        if plan is None:
            if self.selection is None:
                return self.base(x, act=act, out=out)
            plan = self.selection.plan(x.numel() // self.in_features)
        act = act or self.base.gated_act
        if torch.is_grad_enabled() and (x.requires_grad or self.down.requires_grad or self.up.requires_grad):
            if out is not None or act in ops.GATED_ACTS:
                raise RuntimeError("a differentiable call takes neither out nor a gated activation")
            y = _AdaptedProjection.apply(x, self.down, self.up, self.scale, plan, self, self.pack_activations)
            return y if act is None else _activate(y, act)
        down, up = self.down.detach(), self.up.detach()
        if act is None:
            y = self.project(x, out=out)
            return ops.adapter_add(y, x, down, up, self.scale, plan, out=y)
        return ops.adapter_add(self.project(x), x, down, up, self.scale, plan, act=act, out=out)

    def extra_repr(self) -> str:
        return f"adapters={self.down.shape[0]}, rank={self.down.shape[1]}"


def attach_adapters(model: nn.Module, n_adapters: int, rank: int, is_adapted_key=None,
                    pack_activations: bool = False) -> list[str]:
    """Wrap the model's quantized linears (those whose ``<name>.weight`` key
    is_adapted_key accepts; all of them without it) in AdapterLinear.  Linears
    that flux.fuse_qkv_projections concatenated are dropped where one of their
    parts is wrapped; linears that have a bank already keep it; one in several
    places gets one.  The model's
    modules are marked differentiable: with gradients enabled, the quantized
    linears that were not wrapped and the FLUX blocks' fused kernels then pass
    gradients on too.  Returns the wrapped names."""
    if isinstance(model, (Ltx23Nf4Linear, Ltx23Fp8Linear)):
        raise TypeError("a linear by itself is wrapped by AdapterLinear(linear, ...)")
    wrapped, made = [], {}
    for mod in model.modules():
        mod.differentiable = True
    for name, mod in list(model.named_modules(remove_duplicate=False)):
        if not isinstance(mod, (Ltx23Nf4Linear, Ltx23Fp8Linear)):
            continue
        segs = name.split(".")
        if isinstance(_walk(model, segs), AdapterLinear) or \
                (len(segs) > 1 and isinstance(_walk(model, segs[:-1]), AdapterLinear)):
            continue
        if segs[-1] in ("to_qkv", "add_qkv") or (is_adapted_key is not None and not is_adapted_key(name + ".weight")):
            continue
        parent = _walk(model, segs[:-1]) if len(segs) > 1 else model
        wrap = made.get(mod)  # (a linear in two places has one bank)
        if wrap is None:
            wrap = made[mod] = AdapterLinear(mod, n_adapters, rank, pack_activations)
        if segs[-1].isdigit():
            parent[int(segs[-1])] = wrap
        else:
            setattr(parent, segs[-1], wrap)
        for fused, parts in (("to_qkv", ("to_q", "to_k", "to_v")),
                             ("add_qkv", ("add_q_proj", "add_k_proj", "add_v_proj"))):
            if segs[-1] in parts and getattr(parent, fused, None) is not None:
                delattr(parent, fused)
        wrapped.append(name)
    return wrapped


def select_adapters(model: nn.Module, ids: torch.Tensor | None) -> AdapterSelection | None:
    """Give every adapted linear of `model` the adapters of the next batch: ids
    int32 on the GPU, one per batch element (-1: none); None takes them off."""
    layers = [m for m in model.modules() if isinstance(m, AdapterLinear)]
    if not layers:
        raise ValueError("the model has no adapted linears")
    counts = {m.down.shape[0] for m in layers}
    if len(counts) != 1:
        raise ValueError(f"the model's banks hold different numbers of adapters: {sorted(counts)}")
    selection = None if ids is None else AdapterSelection(ids, counts.pop())
    for m in layers:
        m.selection = selection
    return selection


# Reference-spelled aliases, so callers read like the R API.
ltx23_nf4_linear = Ltx23Nf4Linear
ltx23_fp8_linear = Ltx23Fp8Linear


def _walk(module: nn.Module, segments):
    cur = module
    for seg in segments:
        cur = cur[int(seg)] if seg.isdigit() else getattr(cur, seg, None)
        if cur is None:
            return None
    return cur


def swap_quant_linears(model: nn.Module, is_quant_key, fmt: str = "nf4",
                       device=None) -> list[str]:
    """Replace every ``nn.Linear`` whose ``<name>.weight`` key matches
    ``is_quant_key`` by an NF4 / fp8 module holding its quantized weight,
    adopting the original bias parameter (R/quantize_flux.R:541-576).

    Quantization runs on the GPU kernels of this package.  Returns the swapped
    keys.
    """
    if fmt not in ("nf4", "fp8"):
        raise ValueError("fmt must be 'nf4' or 'fp8'")
    swapped = []
    for name, mod in list(model.named_modules()):
        if not isinstance(mod, nn.Linear) or not is_quant_key(name + ".weight"):
            continue
        segs = name.split(".")
        parent = _walk(model, segs[:-1]) if len(segs) > 1 else model
        leaf = segs[-1]
        w = mod.weight.detach()
        dev = torch.device(device) if device is not None else w.device
        w = w.to(dev)
        n_out, n_in = w.shape
        has_bias = mod.bias is not None
        if fmt == "nf4":
            q = Ltx23Nf4Linear(n_out, n_in, bias=has_bias).to(dev)
            packed, absmax = ops.ltx23_nf4_quantize(w)
            q.set_nf4_weight(packed, absmax)
        else:
            q = Ltx23Fp8Linear(n_out, n_in, bias=has_bias).to(dev)
            w8, scale = ops.fp8_quantize(w)
            q.set_fp8_weight(w8, scale.cpu())
        if has_bias:
            q.bias = mod.bias
        q.differentiable = getattr(mod, "differentiable", False)
        if leaf.isdigit():
            parent[int(leaf)] = q
        else:
            setattr(parent, leaf, q)
        swapped.append(name + ".weight")
    return swapped


# R/checkpoint_flux.R:21-32 -- the FLUX.1 cast set (494 weights at full size).
FLUX_QUANT_CAST_PATTERN = re.compile(
    r"^("
    r"transformer_blocks\.[0-9]+\.("
    r"attn\.(to_q|to_k|to_v|add_q_proj|add_k_proj|add_v_proj|to_out\.0|to_add_out)"
    r"|ff\.net\.(0\.proj|2)|ff_context\.net\.(0\.proj|2)"
    r"|norm1\.linear|norm1_context\.linear"
    r")"
    r"|single_transformer_blocks\.[0-9]+\.("
    r"attn\.(to_q|to_k|to_v)|proj_mlp|proj_out|norm\.linear"
    r")"
    r")\.weight$")

# R/fp8_ltx23.R:15-18 -- the official LTX fp8 cast set.
LTX23_FP8_CAST_PATTERN = re.compile(
    r"^transformer_blocks\.[0-9]+\..*"
    r"(to_q|to_k|to_v|to_out\.0|ff\.net\.0\.proj|ff\.net\.2)\.weight$")


def flux_is_quant_key(key: str) -> bool:
    """R/checkpoint_flux.R:41-42."""
    return FLUX_QUANT_CAST_PATTERN.search(key) is not None


def ltx23_is_fp8_cast_key(key: str) -> bool:
    """R/fp8_ltx23.R:28-30."""
    return LTX23_FP8_CAST_PATTERN.search(key) is not None
