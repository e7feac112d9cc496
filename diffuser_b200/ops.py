"""Torch-facing wrappers over the C ABI: every op runs the sm_100a kernels.

These mirror the functional half of diffuseR's quantized-linear API
(R/nf4_ltx23.R, R/fp8_ltx23.R).  Tensors are passed to the library as raw
device pointers with torch's current CUDA stream.  There is no CPU path: a
CPU tensor, a non-bf16 activation or a missing library raises.
"""
from __future__ import annotations

import contextlib
import ctypes

import torch

from . import _lib

NF4_BLOCK = 64  # R/nf4_ltx23.R:23


def _require_cuda(t: torch.Tensor, name: str) -> None:
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor: the engine has no CPU path")


def _ptr(t):
    return None if t is None else ctypes.c_void_p(t.data_ptr())


def _stream(device: torch.device):
    return ctypes.c_void_p(torch.cuda.current_stream(device).cuda_stream)


def _dtype_code(t: torch.Tensor) -> int:
    if t.dtype == torch.float32:
        return _lib.DQ_DTYPE_F32
    if t.dtype == torch.bfloat16:
        return _lib.DQ_DTYPE_BF16
    raise TypeError(f"unsupported weight dtype {t.dtype}; expected float32 or bfloat16")


# ------------------------------------------------------------- workspaces
def workspace(device: torch.device, nbytes: int) -> torch.Tensor | None:
    """Scratch of one call (split-K partial sums, or a weight decoded to bf16 and
    its ready counters), from torch's allocator.  The allocator keeps it for the
    next call on the same stream, as the reference's per-shape dequant buffers
    are kept (R/nf4_ltx23.R:160-175), but calls on several streams never meet in
    it, and a captured graph owns what it replays into: one buffer per device,
    grown on demand, was written by two streams at once and freed under the
    graphs that held its address."""
    if nbytes == 0:
        return None
    return torch.empty(nbytes, dtype=torch.uint8, device=device)


def release_workspaces() -> None:
    """Give unused scratch back to the device
    (ltx23_release_dequant_buffers, R/nf4_ltx23.R:185-194)."""
    torch.cuda.empty_cache()


def workspace_size(M: int, N: int, K: int, fmt: int = _lib.DQ_FMT_NF4) -> int:
    return int(_lib.lib().dq_workspace_size(M, N, K, fmt))


# ----------------------------------------------------------------- quantize
def ltx23_nf4_quantize(x: torch.Tensor):
    """NF4-quantize a CUDA tensor (R/nf4_ltx23.R:35-61).

    Returns ``(packed uint8 [n/2], absmax float32 [n/64])``; ``n`` must be a
    multiple of 64 (the reference's error otherwise).
    """
    _require_cuda(x, "x")
    n = x.numel()
    if n % NF4_BLOCK != 0:
        raise ValueError(f"Tensor length must be a multiple of {NF4_BLOCK}")
    src = x.detach()
    if src.dtype not in (torch.float32, torch.bfloat16):
        src = src.to(torch.float32)
    src = src.contiguous()
    packed = torch.empty(n // 2, dtype=torch.uint8, device=x.device)
    absmax = torch.empty(n // NF4_BLOCK, dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check("dq_quantize_nf4", _lib.lib().dq_quantize_nf4(
            _ptr(src), _dtype_code(src), n, _ptr(packed), _ptr(absmax), _stream(x.device)))
    return packed, absmax


def fp8_quantize(x: torch.Tensor):
    """Per-tensor e4m3 quantization (R/quantize_flux.R:406-409).

    Returns ``(w8 float8_e4m3fn, scale float32 0-d tensor)``, both on x's device.
    """
    _require_cuda(x, "x")
    src = x.detach()
    if src.dtype not in (torch.float32, torch.bfloat16):
        src = src.to(torch.float32)
    src = src.contiguous()
    w8 = torch.empty(src.shape, dtype=torch.uint8, device=x.device)
    scale = torch.empty((), dtype=torch.float32, device=x.device)
    with torch.cuda.device(x.device):
        _lib.check("dq_quantize_fp8", _lib.lib().dq_quantize_fp8(
            _ptr(src), _dtype_code(src), src.numel(), _ptr(w8), _ptr(scale), _stream(x.device)))
    return w8.view(torch.float8_e4m3fn), scale


# --------------------------------------------------------------- dequantize
def ltx23_nf4_dequantize(packed: torch.Tensor, absmax: torch.Tensor, shape,
                         dtype=torch.bfloat16, out: torch.Tensor | None = None) -> torch.Tensor:
    """NF4 -> bf16 (R/nf4_ltx23.R:77-115), bit-exact with the byte-LUT path."""
    _require_cuda(packed, "packed")
    if dtype != torch.bfloat16:
        raise TypeError("the engine dequantizes to bfloat16 only")
    n = 1
    for s in shape:
        n *= int(s)
    if packed.numel() * 2 != n or absmax.numel() * NF4_BLOCK != n:
        raise ValueError("packed / absmax sizes do not match shape")
    if out is None:
        out = torch.empty(tuple(shape), dtype=torch.bfloat16, device=packed.device)
    if absmax.dtype == torch.bfloat16:
        with torch.cuda.device(packed.device):
            _lib.check("dq_dequant_nf4_scaled", _lib.lib().dq_dequant_nf4_scaled(
                _ptr(packed.contiguous()), _ptr(absmax.contiguous()), _lib.DQ_DTYPE_BF16, n,
                _ptr(out), _stream(packed.device)))
        return out
    am = absmax if absmax.dtype == torch.float32 else absmax.float()
    with torch.cuda.device(packed.device):
        _lib.check("dq_dequant_nf4", _lib.lib().dq_dequant_nf4(
            _ptr(packed.contiguous()), _ptr(am.contiguous()), n, _ptr(out), _stream(packed.device)))
    return out


def fp8_dequantize(w8: torch.Tensor, scale, dtype=torch.bfloat16,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """e4m3 -> bf16 times bf16(scale) (R/fp8_ltx23.R:79-80), bit-exact."""
    _require_cuda(w8, "w8")
    if dtype != torch.bfloat16:
        raise TypeError("the engine dequantizes to bfloat16 only")
    s = float(scale)
    if out is None:
        out = torch.empty(w8.shape, dtype=torch.bfloat16, device=w8.device)
    raw = w8.contiguous().view(torch.uint8)
    with torch.cuda.device(w8.device):
        _lib.check("dq_dequant_fp8", _lib.lib().dq_dequant_fp8(
            _ptr(raw), ctypes.c_float(s), raw.numel(), _ptr(out), _stream(w8.device)))
    return out


# ------------------------------------------------------------------- linear
def _prep_x(x: torch.Tensor, k: int) -> torch.Tensor:
    _require_cuda(x, "x")
    if x.dtype != torch.bfloat16:
        raise TypeError(f"activations must be bfloat16 on the GPU path, got {x.dtype}")
    if x.shape[-1] != k:
        raise ValueError(f"last dim of x is {x.shape[-1]}, expected in_features={k}")
    x2 = x.reshape(-1, k)
    if not x2.is_contiguous() or x2.data_ptr() % 16 != 0:
        x2 = x2.contiguous()
    return x2


def _prep_bias(bias, n: int, device):
    if bias is None:
        return None
    b = bias.detach()
    if b.dtype != torch.bfloat16:
        b = b.to(torch.bfloat16)
    if b.device != device:
        b = b.to(device)
    if b.numel() != n:
        raise ValueError("bias size does not match out_features")
    return b.contiguous()


_ACTS = {None: _lib.DQ_ACT_NONE, "gelu_tanh": _lib.DQ_ACT_GELU_TANH, "swiglu": _lib.DQ_ACT_SWIGLU,
         "geglu_tanh": _lib.DQ_ACT_GEGLU_TANH}
GATED_ACTS = ("swiglu", "geglu_tanh")


def _act_code(act, n: int) -> tuple[int, int]:
    """(C-ABI activation code, output width) of a linear with n weight rows."""
    if act not in _ACTS:
        raise ValueError(f"unknown activation {act!r}; expected one of {list(_ACTS)}")
    if act in GATED_ACTS:
        if n % 32 != 0:
            raise ValueError("a gated activation needs out_features % 32 == 0 (gated row order)")
        return _ACTS[act], n // 2
    return _ACTS[act], n


# ------------------------------------------------------------ gated rows
def gated_row_order(n: int, device=None) -> torch.Tensor:
    """Row permutation from the reference's [gate; up] halves of an n-row
    weight (R/dit_flux2_modules.R:77-84: silu(first half) * second half) to
    the gated row order of the epilogue: for each block b of 16 output
    features, rows 32b .. 32b+15 are gate rows 16b .. 16b+15 and rows
    32b+16 .. 32b+31 the up rows n/2 + 16b .. n/2 + 16b+15."""
    if n % 32 != 0:
        raise ValueError("the gated row order needs n % 32 == 0")
    h = n // 2
    b = torch.arange(n // 32).view(-1, 1) * 16
    i = torch.arange(16).view(1, -1)
    order = torch.stack([b + i, h + b + i], dim=1).reshape(-1)
    return order if device is None else order.to(device)


def to_gated_rows_nf4(packed: torch.Tensor, absmax: torch.Tensor, n: int, k: int):
    """NF4 buffers of a [gate; up] weight reordered into the gated row order:
    rows are whole byte ranges of the packed codes and of the block scales
    (K % 64 == 0), so the reorder is a row gather."""
    order = gated_row_order(n, packed.device)
    p = packed.reshape(n, k // 2).index_select(0, order).reshape(-1)
    a = absmax.reshape(n, k // NF4_BLOCK).index_select(0, order.to(absmax.device)).reshape(-1)
    return p, a


def to_gated_rows(t: torch.Tensor, n: int) -> torch.Tensor:
    """Rows of an fp8 weight [n, K] (or a bias [n]) in the gated row order."""
    order = gated_row_order(n, t.device)
    raw = t.view(torch.uint8) if t.dtype == torch.float8_e4m3fn else t
    out = raw.index_select(0, order)
    return out.view(torch.float8_e4m3fn) if t.dtype == torch.float8_e4m3fn else out


def _out_rows(out: torch.Tensor, m: int, n: int) -> int:
    """Row stride (elements) of a caller-given output viewed as [m, n] rows,
    which must be evenly spaced with unit stride along the features."""
    if out.dtype != torch.bfloat16 or not out.is_cuda:
        raise TypeError("out must be a bfloat16 CUDA tensor")
    if out.shape[-1] != n or out.numel() != m * n or out.stride(-1) != 1:
        raise ValueError(f"out must hold [{m}, {n}] with unit stride along the last dimension")
    ld = out.stride(-2) if out.dim() >= 2 else n
    for d in range(out.dim() - 2):
        if out.stride(d) != out.shape[d + 1] * out.stride(d + 1):
            raise ValueError("out's rows must be evenly spaced")
    return ld


def nf4_linear(x: torch.Tensor, packed: torch.Tensor, absmax: torch.Tensor,
               out_features: int, bias: torch.Tensor | None = None, act: str | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x . dequant_nf4(W)^T + bias (R/nf4_ltx23.R:235-246); act="gelu_tanh"
    applies GELU-tanh in the epilogue, as gelu_proj does after the projection;
    act="swiglu" / "geglu_tanh" gate a weight in the gated row order
    (to_gated_rows_nf4) and return out_features / 2 columns.  With `out`
    (e.g. a column range of a wider buffer) y is written there."""
    n = int(out_features)
    k = packed.numel() * 2 // n
    code, n_out = _act_code(act, n)
    x2 = _prep_x(x, k)
    m = x2.shape[0]
    b = _prep_bias(bias, n, x.device)
    if absmax.dtype == torch.bfloat16:
        # block scales repacked to bf16 at load time (bf16(absmax), the value
        # the forward uses): the dtype-tagged entry point
        y = out if out is not None else torch.empty((m, n_out), dtype=torch.bfloat16, device=x.device)
        ldy = _out_rows(y, m, n_out)
        with torch.cuda.device(x.device):
            ws_bytes = workspace_size(m, n, k, _lib.DQ_FMT_NF4)
            ws = workspace(x.device, ws_bytes)
            _lib.check("dq_linear_nf4_scaled", _lib.lib().dq_linear_nf4_scaled(
                _ptr(x2), m, k, _ptr(packed), _ptr(absmax), _lib.DQ_DTYPE_BF16, _ptr(b), n, code,
                _ptr(y), ldy, _ptr(ws), ws_bytes, _stream(x.device)))
        return y if out is not None else y.reshape(*x.shape[:-1], n_out)
    am = absmax if absmax.dtype == torch.float32 else absmax.float()
    if out is not None:
        ldy = _out_rows(out, m, n_out)
        with torch.cuda.device(x.device):
            ws_bytes = workspace_size(m, n, k, _lib.DQ_FMT_NF4)
            ws = workspace(x.device, ws_bytes)
            _lib.check("dq_linear_nf4_ld", _lib.lib().dq_linear_nf4_ld(
                _ptr(x2), m, k, _ptr(packed), _ptr(am), _ptr(b), n, code, _ptr(out), ldy,
                _ptr(ws), ws_bytes, _stream(x.device)))
        return out
    y = torch.empty((m, n_out), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        ws_bytes = workspace_size(m, n, k, _lib.DQ_FMT_NF4)
        ws = workspace(x.device, ws_bytes)
        if act is None:
            _lib.check("dq_linear_nf4", _lib.lib().dq_linear_nf4(
                _ptr(x2), m, k, _ptr(packed), _ptr(am), _ptr(b), n, _ptr(y),
                _ptr(ws), ws_bytes, _stream(x.device)))
        else:
            _lib.check("dq_linear_nf4_ex", _lib.lib().dq_linear_nf4_ex(
                _ptr(x2), m, k, _ptr(packed), _ptr(am), _ptr(b), n, code, _ptr(y),
                _ptr(ws), ws_bytes, _stream(x.device)))
    return y.reshape(*x.shape[:-1], n_out)


def fp8_linear(x: torch.Tensor, w8: torch.Tensor, scale: float,
               bias: torch.Tensor | None = None, act: str | None = None,
               out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x . (e4m3(W) * bf16(scale))^T + bias fused (R/fp8_ltx23.R:70-83);
    act="gelu_tanh" applies GELU-tanh in the epilogue, act="swiglu" /
    "geglu_tanh" gate a weight in the gated row order (to_gated_rows) and
    return half as many columns; with `out` y is written there (its rows may
    be spaced wider than the output width)."""
    n, k = int(w8.shape[0]), int(w8.shape[1])
    code, n_out = _act_code(act, n)
    x2 = _prep_x(x, k)
    m = x2.shape[0]
    b = _prep_bias(bias, n, x.device)
    raw = w8.view(torch.uint8)
    if out is not None:
        ldy = _out_rows(out, m, n_out)
        with torch.cuda.device(x.device):
            ws_bytes = workspace_size(m, n, k, _lib.DQ_FMT_FP8)
            ws = workspace(x.device, ws_bytes)
            _lib.check("dq_linear_fp8_ld", _lib.lib().dq_linear_fp8_ld(
                _ptr(x2), m, k, _ptr(raw), ctypes.c_float(float(scale)), _ptr(b), n, code,
                _ptr(out), ldy, _ptr(ws), ws_bytes, _stream(x.device)))
        return out
    y = torch.empty((m, n_out), dtype=torch.bfloat16, device=x.device)
    with torch.cuda.device(x.device):
        ws_bytes = workspace_size(m, n, k, _lib.DQ_FMT_FP8)
        ws = workspace(x.device, ws_bytes)
        if act is None:
            _lib.check("dq_linear_fp8", _lib.lib().dq_linear_fp8(
                _ptr(x2), m, k, _ptr(raw), ctypes.c_float(float(scale)), _ptr(b), n, _ptr(y),
                _ptr(ws), ws_bytes, _stream(x.device)))
        else:
            _lib.check("dq_linear_fp8_ex", _lib.lib().dq_linear_fp8_ex(
                _ptr(x2), m, k, _ptr(raw), ctypes.c_float(float(scale)), _ptr(b), n, code,
                _ptr(y), _ptr(ws), ws_bytes, _stream(x.device)))
    return y.reshape(*x.shape[:-1], n_out)


# ----------------------------------------------------------------- adapters
# The calls below are small next to a Python call, so their checks come in two
# parts: a short one that accepts the usual operands (contiguous, aligned), and
# the full one that names what is wrong or copies what is only laid out badly.
_NO_SWITCH = contextlib.nullcontext()
_BF16, _F32 = torch.bfloat16, torch.float32


def _on(t: torch.Tensor):
    """Makes t's device the current one for the duration of a call."""
    return _NO_SWITCH if t.get_device() == torch._C._cuda_getDevice() else torch.cuda.device(t.device)


def _raw_stream(t: torch.Tensor) -> int:
    """Handle of the current stream on t's device."""
    return torch._C._cuda_getCurrentRawStream(t.get_device())


def _scratch(nbytes: int, like: torch.Tensor) -> torch.Tensor:
    """Workspace of one call, from torch's allocator: calls on several streams
    and captured graphs each hold their own."""
    return torch.empty(max(int(nbytes), 16), dtype=torch.uint8, device=like.device)


def _same_device(t: torch.Tensor, name: str, like: torch.Tensor) -> None:
    _require_cuda(t, name)
    if t.device != like.device:
        raise ValueError(f"{name} is on {t.device}, expected {like.device}")


def _rows16(t: torch.Tensor, name: str, width: int, like: torch.Tensor) -> torch.Tensor:
    """t as bf16 rows [-1, width] with unit stride along the features, 16-byte
    aligned row starts and evenly spaced rows (copied when it is not)."""
    _same_device(t, name, like)
    if t.dtype != _BF16:
        raise TypeError(f"{name} must be bfloat16, got {t.dtype}")
    if t.dim() < 1 or t.shape[-1] != width:
        raise ValueError(f"{name} must have {width} features, got shape {tuple(t.shape)}")
    t2 = t if t.dim() == 2 else t.reshape(-1, width)
    if t2.stride(1) != 1 or t2.stride(0) % 8 != 0 or t2.stride(0) < width or t2.data_ptr() % 16 != 0:
        t2 = t2.new_empty(t2.shape).copy_(t2)
    return t2


def _row_operand(t: torch.Tensor, name: str, width: int, like: torch.Tensor, must_alias: bool = False):
    """(tensor that holds the rows, address, row stride, rows) of a bf16
    [..., width] operand; with must_alias it may not be a copy of t."""
    if isinstance(t, torch.Tensor) and t.dtype is _BF16 and t.is_contiguous() and \
            t.get_device() == like.get_device() and t.is_cuda and t.dim() and t.shape[-1] == width:
        p = t.data_ptr()
        if p % 16 == 0 and width % 8 == 0:
            return t, p, width, t.numel() // width
    t2 = _rows16(t, name, width, like)
    if must_alias and t2.data_ptr() != t.data_ptr():
        raise ValueError(f"{name} must have evenly spaced, 16-byte aligned rows with unit feature stride")
    m = t2.shape[0]
    return t2, t2.data_ptr(), (t2.stride(0) if m > 1 else max(t2.stride(0), width)), m


def _bank(down: torch.Tensor, up: torch.Tensor, scale: torch.Tensor, like: torch.Tensor):
    """(adapters, rank, in_features, out_features) of a checked adapter bank."""
    try:
        a, r, k = down.shape
        a2, r2, n = up.shape
        d = like.get_device()
        if down.dtype is up.dtype is _BF16 and scale.dtype is _F32 and a == a2 == scale.numel() and r == r2 and \
                scale.dim() == 1 and r % 8 == 0 and 0 < r <= 128 and k % 8 == 0 and n % 8 == 0 and \
                down.is_contiguous() and up.is_contiguous() and scale.is_contiguous() and \
                down.get_device() == up.get_device() == scale.get_device() == d:
            return a, r, k, n
    except (AttributeError, ValueError):
        pass
    for t, name in ((down, "down"), (up, "up")):
        _same_device(t, name, like)
        if t.dtype != _BF16 or t.dim() != 3 or not t.is_contiguous():
            raise TypeError(f"{name} must be a contiguous bfloat16 [adapters, rank, features] tensor")
    a, r, k = down.shape
    if up.shape[:2] != (a, r):
        raise ValueError("down and up must hold the same adapters and rank")
    _same_device(scale, "scale", like)
    if scale.dtype != _F32 or scale.shape != (a,) or not scale.is_contiguous():
        raise TypeError("scale must be a contiguous float32 [adapters] tensor")
    if r % 8 != 0 or r > 128 or k % 8 != 0 or up.shape[2] % 8 != 0:
        raise ValueError("rank (at most 128) and features must be multiples of 8")
    return a, r, k, up.shape[2]


class AdapterPlan:
    """The tokens of a batch sorted by adapter (adapter_plan builds it)."""

    def __init__(self, ids, offsets, n_adapters: int, tokens: int):
        self.tokens, self.requests, self.n_adapters = int(tokens), ids.numel(), int(n_adapters)
        lib = _lib.lib()
        nbytes = int(lib.dq_adapter_plan_bytes(self.tokens, self.requests, self.n_adapters))
        if nbytes == 0:
            raise ValueError("adapter_plan: tokens must be 0..2^30, requests at most 2^20 and n_adapters 1..65535")
        # bytes of adapter_add's workspace per unit of rank
        self.add_workspace = int(lib.dq_adapter_add_workspace(self.tokens, self.requests, 1, self.n_adapters))
        self.words = torch.empty(nbytes // 4, dtype=torch.int32, device=ids.device)
        self.address = self.words.data_ptr()
        self.version = 0  # how often it has been built
        self.update_(ids, offsets)

    def __setstate__(self, state):  # a copy holds its own words
        self.__dict__.update(state)
        self.address = self.words.data_ptr()

    def update_(self, ids: torch.Tensor, offsets: torch.Tensor) -> "AdapterPlan":
        """Rebuild in place for new ids / offsets of the same counts (also
        inside a graph capture: the plan's address does not change)."""
        for t, name in ((ids, "ids"), (offsets, "offsets")):
            _same_device(t, name, self.words)
            if t.dtype != torch.int32 or t.dim() != 1 or not t.is_contiguous():
                raise TypeError(f"{name} must be a contiguous 1-d int32 tensor")
        if ids.numel() != self.requests or offsets.numel() != self.requests + 1:
            raise ValueError("offsets must hold one more entry than ids, and both as many as before")
        with _on(self.words):
            _lib.check("dq_adapter_plan", _lib.lib().dq_adapter_plan(
                _ptr(ids), _ptr(offsets), self.requests, self.tokens, self.n_adapters, self.address,
                self.words.numel() * 4, _raw_stream(self.words)))
        self.version += 1
        return self


def adapter_plan(ids: torch.Tensor, offsets: torch.Tensor, tokens: int, n_adapters: int) -> AdapterPlan:
    """Sort a batch's tokens by adapter, on the device, once for every layer
    the batch passes.  ids int32 [R]: each request's adapter (-1: none);
    offsets int32 [R + 1]: request i holds tokens offsets[i] .. offsets[i+1]-1
    of the batch's `tokens`; tokens outside every request (padding) have no
    adapter.  Neither is read by the host: ids out of range count as none,
    offsets out of order leave every token without an adapter, and
    device_error() then returns DQ_ERR_INDEX."""
    _require_cuda(ids, "ids")
    return AdapterPlan(ids, offsets, n_adapters, tokens)


def _check_plan(plan: AdapterPlan, m: int, a: int, like: torch.Tensor) -> None:
    if not isinstance(plan, AdapterPlan):
        raise TypeError("plan must come from adapter_plan")
    if plan.tokens != m or plan.n_adapters != a:
        raise ValueError(f"the plan is for {plan.tokens} tokens and {plan.n_adapters} adapters, "
                         f"the operands hold {m} and {a}")
    if plan.words.get_device() != like.get_device():
        _same_device(plan.words, "plan", like)


def _whole(t: torch.Tensor, name: str):
    """A contiguous operand as one row of bytes."""
    n = t.numel() * t.element_size()
    return t.data_ptr(), n, n, 1, name


def _refuse_alias(out, others) -> None:
    """out's rows are written while other tokens of `others` are still read.
    Each is (address, row stride, row width, rows, name), in bytes; rows of one
    stride that keep to different columns do not meet."""
    p, ld, w, m, _ = out
    for q, ldq, wq, mq, name in others:
        if m == 0 or mq == 0 or p + (m - 1) * ld + w <= q or q + (mq - 1) * ldq + wq <= p:
            continue
        if ld == ldq and w <= (q - p) % ld <= ld - wq:
            continue
        raise ValueError(f"out must not overlap {name}")


def adapter_add(y: torch.Tensor, x: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                scale: torch.Tensor, plan: AdapterPlan, act: str | None = None,
                out: torch.Tensor | None = None, return_hidden: bool = False):
    """act(y + scale_a * (x . down_a^T) . up_a) for every token with its own
    adapter a (act(y) where it has none): the low-rank adapters of many
    requests beside a shared projection's output y [..., N], x [..., K] its
    input.  down bf16 [A, r, K], up bf16 [A, r, N] (the transposed second
    factor), scale float32 [A].  act as nf4_linear's; the gated ones take y and
    up in the gated row order and return N / 2 columns.  out may be y itself
    (in place, not with a gated act) but overlaps no other operand.  With
    return_hidden also the bf16 [tokens, r] scale_a * x . down_a^T that
    adapter_backward takes."""
    _require_cuda(y, "y")
    a, r, k, n = _bank(down, up, scale, y)
    code, n_out = (_lib.DQ_ACT_NONE, n) if act is None else _act_code(act, n)
    x2, xp, ldx, mx = _row_operand(x, "x", k, y)
    y2, yp, ldy, m = _row_operand(y, "y", n, y)
    if mx != m:
        raise ValueError(f"x holds {mx} tokens, y {m}")
    _check_plan(plan, m, a, y)
    if out is None:
        res = torch.empty_like(y) if n_out == n and y2 is y else \
            torch.empty((*y.shape[:-1], n_out), dtype=_BF16, device=y.device)
        op, ldo = res.data_ptr(), n_out
    else:
        res = out
        _, op, ldo, mo = _row_operand(out, "out", n_out, y, must_alias=True)
        if mo != m:
            raise ValueError(f"out holds {mo} tokens, y {m}")
        _refuse_alias((op, 2 * ldo, 2 * n_out, m, "out"), (
            (xp, 2 * ldx, 2 * k, m, "x"), *(() if op == yp else ((yp, 2 * ldy, 2 * n, m, "y unless it is y"),)),
            _whole(down, "down"), _whole(up, "up"), _whole(scale, "scale"), _whole(plan.words, "plan")))
    hidden = torch.empty((m, r), dtype=_BF16, device=y.device) if return_hidden else None
    nbytes = 0 if return_hidden else plan.add_workspace * r
    ws = _scratch(nbytes, y) if nbytes else None
    with _on(y):
        _lib.call("dq_adapter_add", yp, ldy, xp, ldx, m, plan.requests, k, n, down.data_ptr(), up.data_ptr(),
                  scale.data_ptr(), r, a, plan.address, code, op, ldo, 0 if hidden is None else hidden.data_ptr(),
                  0 if ws is None else ws.data_ptr(), nbytes, _raw_stream(y))
    return (res, hidden) if return_hidden else res


def adapter_backward(dy: torch.Tensor, x, hidden: torch.Tensor, down: torch.Tensor, up: torch.Tensor,
                     scale: torch.Tensor, plan: AdapterPlan, dx: torch.Tensor | None = None,
                     out: torch.Tensor | None = None, factors: bool = True, inputs: bool = True):
    """Gradients of adapter_add (without act): returns (dx, ddown, dup).

    dy [..., N] is the output's gradient; x the forward's input, as bf16
    [..., K] or as checkpoint_pack packed it; hidden what adapter_add returned.
    dx [..., K], if given, is the shared projection's input gradient
    (nf4_linear_dgrad / fp8_linear_dgrad): the adapters' part is added to it, in
    `out` (which may be dx, and overlaps no other operand) or a new tensor.
    ddown / dup have the layouts of down / up, zeros for adapters without
    tokens; with factors=False they are None, and neither is computed, nor with
    inputs=False (a first layer's) the gradient of x.  The same inputs give the
    same bits."""
    if not inputs and (dx is not None or out is not None or not factors):
        raise ValueError("inputs=False takes neither dx nor out, nor factors=False")
    _require_cuda(dy, "dy")
    a, r, k, n = _bank(down, up, scale, dy)
    dy2, dyp, lddy, m = _row_operand(dy, "dy", n, dy)
    _check_plan(plan, m, a, dy)
    if isinstance(x, PackedActivation):
        if x.codes.shape[-1] != k or x.codes.numel() != m * k:
            raise ValueError(f"the packed activation holds {tuple(x.codes.shape)}, expected [{m}, {k}]")
        _same_device(x.codes, "x", dy)
        x2, xp, ldx, scales = x.codes, x.codes.data_ptr(), k, x.scales.data_ptr()
    else:
        x2, xp, ldx, mx = _row_operand(x, "x", k, dy)
        scales = 0
        if mx != m:
            raise ValueError(f"x holds {mx} tokens, dy {m}")
    _same_device(hidden, "hidden", dy)
    if hidden.dtype != _BF16 or hidden.shape != (m, r) or not hidden.is_contiguous() or hidden.data_ptr() % 16 != 0:
        raise TypeError(f"hidden must be a contiguous bfloat16 [{m}, {r}] tensor")
    shape = (*dy.shape[:-1], k)
    res, dxp, lddx, op, ldo = None, 0, k, 0, k
    if inputs:
        base = torch.zeros(shape, dtype=_BF16, device=dy.device) if dx is None else dx
        dx2, dxp, lddx, md = _row_operand(base, "dx", k, dy)
        if md != m:
            raise ValueError(f"dx holds {md} tokens, dy {m}")
        if out is None:
            res = base if dx is None else torch.empty_like(dx) if dx2 is dx and dx.shape == shape else \
                torch.empty(shape, dtype=_BF16, device=dy.device)
            op = res.data_ptr()
        else:
            res = out
            _, op, ldo, mo = _row_operand(out, "out", k, dy, must_alias=True)
            if mo != m:
                raise ValueError(f"out holds {mo} tokens, dy {m}")
            size = x2.element_size()
            _refuse_alias((op, 2 * ldo, 2 * k, m, "out"), (
                (dyp, 2 * lddy, 2 * n, m, "dy"), (xp, size * ldx, size * k, m, "x"), _whole(hidden, "hidden"),
                *(() if op == dxp else ((dxp, 2 * lddx, 2 * k, m, "dx unless it is dx"),)),
                _whole(down, "down"), _whole(up, "up"), _whole(scale, "scale"), _whole(plan.words, "plan")))
    ddown, dup = (torch.empty_like(down), torch.empty_like(up)) if factors else (None, None)
    with _on(dy):
        nbytes = _lib.lib().dq_adapter_backward_workspace(m, plan.requests, k, n, r, a)
        ws = _scratch(nbytes, dy)
        _lib.call("dq_adapter_backward", dyp, lddy, xp, ldx, scales, hidden.data_ptr(), m, plan.requests, k, n,
                  down.data_ptr(), up.data_ptr(), scale.data_ptr(), r, a, plan.address, dxp, lddx, op, ldo,
                  0 if ddown is None else ddown.data_ptr(), 0 if dup is None else dup.data_ptr(), ws.data_ptr(),
                  nbytes, _raw_stream(dy))
    return res, ddown, dup


# ---------------------------------------------------- activation checkpoints
CHECKPOINT_RUN = 128


class PackedActivation:
    """An activation in 8 bits: int8 codes [..., K] and float32 scales
    [rows, ceil(K / 128)], one per row and run of 128 features."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor):
        _require_cuda(codes, "codes")
        _same_device(scales, "scales", codes)
        if codes.dtype != torch.int8 or scales.dtype != _F32 or codes.dim() < 1:
            raise TypeError("codes must be int8 and scales float32")
        k = codes.shape[-1]
        if k == 0 or k % 16 != 0:
            raise ValueError("an 8-bit activation needs a feature count that is a multiple of 16")
        if scales.shape != (codes.numel() // k, -(-k // CHECKPOINT_RUN)):
            raise ValueError("scales must hold one value per row and run of 128 features")
        self.codes = codes if codes.is_contiguous() and codes.data_ptr() % 16 == 0 else codes.contiguous().clone()
        self.scales = scales.contiguous()


def checkpoint_pack(x: torch.Tensor) -> PackedActivation:
    """Pack a bf16 activation [..., K] (K % 16 == 0) to 8 bits for the backward
    pass: per row and run of 128 features scale = max(max|x|, 1e-12) / 127,
    codes = x / scale rounded to the nearest (ties to even).  A run that is not
    finite comes back as NaN."""
    _require_cuda(x, "x")
    k = x.shape[-1] if x.dim() else 0
    if k == 0 or k % 16 != 0:
        raise ValueError("an 8-bit activation needs a feature count that is a multiple of 16")
    x2, xp, ldx, m = _row_operand(x, "x", k, x)
    packed = object.__new__(PackedActivation)
    packed.codes = codes = torch.empty_like(x, dtype=torch.int8, memory_format=torch.contiguous_format)
    packed.scales = scales = x.new_empty((m, -(-k // CHECKPOINT_RUN)), dtype=_F32)
    with _on(x):
        _lib.call("dq_checkpoint_pack", xp, ldx, m, k, codes.data_ptr(), scales.data_ptr(), _raw_stream(x))
    return packed


def checkpoint_unpack(packed: PackedActivation, out: torch.Tensor | None = None) -> torch.Tensor:
    """The bf16 activation that a packed one stands for."""
    if not isinstance(packed, PackedActivation):
        raise TypeError("packed must come from checkpoint_pack")
    codes = packed.codes
    k = codes.shape[-1]
    if out is None:
        res = torch.empty_like(codes, dtype=_BF16)
        op, ldo, m = res.data_ptr(), k, codes.numel() // k
    else:
        res = out
        _, op, ldo, m = _row_operand(out, "out", k, codes, must_alias=True)
        if m != codes.numel() // k:
            raise ValueError("out must hold the packed rows")
    with _on(codes):
        _lib.call("dq_checkpoint_unpack", codes.data_ptr(), packed.scales.data_ptr(), m, k, op, ldo,
                  _raw_stream(codes))
    return res


# -------------------------------------------------------- input gradients
def _prep_dgrad(dy: torch.Tensor, n: int, k: int, weight: torch.Tensor, dtypes):
    _same_device(weight, "weight", dy)
    if weight.dtype not in dtypes or not weight.is_contiguous():
        raise TypeError(f"the weight must be contiguous {' or '.join(str(t) for t in dtypes)}, got {weight.dtype}")
    if n == 0 or n % 8 != 0:
        raise ValueError("the input gradient needs out_features % 8 == 0")
    if dy.dtype != _BF16:
        raise TypeError(f"gradients must be bfloat16 on the GPU path, got {dy.dtype}")
    if dy.dim() < 1 or dy.shape[-1] != n:
        raise ValueError(f"last dim of dy is {tuple(dy.shape)[-1:]}, expected out_features={n}")
    dy2 = dy if dy.is_contiguous() and dy.data_ptr() % 16 == 0 else dy.new_empty(dy.shape).copy_(dy)
    dx = torch.empty((*dy.shape[:-1], k), dtype=_BF16, device=dy.device)
    m = dy2.numel() // n
    nbytes = _lib.lib().dq_linear_dgrad_workspace_for(m, n, k)
    ws = _scratch(nbytes, dy) if nbytes else None
    return dy2, dx, m, ws, 0 if ws is None else ws.data_ptr(), nbytes


def nf4_linear_dgrad(dy: torch.Tensor, packed: torch.Tensor, absmax: torch.Tensor,
                     in_features: int) -> torch.Tensor:
    """dx = dy . dequant_nf4(W), the input gradient of nf4_linear: dy bf16
    [..., N] -> [..., K].  absmax float32 or bf16 as for the forward."""
    _require_cuda(dy, "dy")
    k = int(in_features)
    n = packed.numel() * 2 // max(k, 1)
    if n * k != packed.numel() * 2 or absmax.numel() * NF4_BLOCK != n * k:
        raise ValueError("packed / absmax sizes do not match in_features")
    dy2, dx, m, ws, wsp, nbytes = _prep_dgrad(dy, n, k, packed, (torch.uint8,))
    _same_device(absmax, "absmax", dy)
    am = (absmax if absmax.dtype in (_F32, _BF16) else absmax.float()).contiguous()
    with _on(dy):
        _lib.call("dq_linear_nf4_dgrad", dy2.data_ptr(), m, n, packed.data_ptr(), am.data_ptr(),
                  _dtype_code(am), k, dx.data_ptr(), wsp, nbytes, _raw_stream(dy))
    return dx


def fp8_linear_dgrad(dy: torch.Tensor, w8: torch.Tensor, scale: float) -> torch.Tensor:
    """dx = dy . (e4m3(W) * bf16(scale)), the input gradient of fp8_linear."""
    _require_cuda(dy, "dy")
    if w8.dim() != 2:
        raise ValueError(f"w8 must be [out_features, in_features], got {tuple(w8.shape)}")
    n, k = int(w8.shape[0]), int(w8.shape[1])
    dy2, dx, m, ws, wsp, nbytes = _prep_dgrad(dy, n, k, w8, (torch.float8_e4m3fn, torch.uint8))
    with _on(dy):
        _lib.call("dq_linear_fp8_dgrad", dy2.data_ptr(), m, n, w8.data_ptr(), float(scale), k,
                  dx.data_ptr(), wsp, nbytes, _raw_stream(dy))
    return dx


def device_error(device=None) -> int:
    """Read and clear the device's kernel error word (DQ_OK, DQ_ERR_TIMEOUT or
    DQ_ERR_INDEX)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    code = ctypes.c_int(0)
    with torch.cuda.device(dev):
        _lib.check("dq_device_error", _lib.lib().dq_device_error(ctypes.byref(code), _stream(dev)))
    return code.value


def set_pair_mode(mode: int = 0) -> None:
    """0 = automatic, 1 = fused one-CTA tiles, 2 = fused CTA-pair tiles,
    3 = two-phase (the bf16 pair GEMM launch dequantizes the weight into bf16
    scratch one group of weight tiles ahead of its MMAs), 4 = two-phase with
    the dequantization as a separate launch before the GEMM, 5 = the small-M
    kernels (M <= 16, K % 128 == 0; the TMA-ring one where it applies),
    6 = the small-M kernel that loads the weight into registers."""
    _lib.check("dq_set_pair_mode", _lib.lib().dq_set_pair_mode(int(mode)))


def set_tile_override(bm: int = 0, splits: int = 0) -> None:
    """Force the x-tile height / split-K count (0 = automatic); for sweeps."""
    _lib.check("dq_set_tile_override", _lib.lib().dq_set_tile_override(int(bm), int(splits)))


def plan_info(M: int, N: int, K: int, fmt: int = _lib.DQ_FMT_NF4) -> dict:
    """The launch plan the linear uses for this shape on the current device."""
    vals = [ctypes.c_int(0) for _ in range(4)]
    _lib.check("dq_plan_info", _lib.lib().dq_plan_info(int(M), int(N), int(K), int(fmt),
                                                       *[ctypes.byref(v) for v in vals]))
    pair, bm, splits, grid = (v.value for v in vals)
    kernel = {0: "dq_gemm_kernel (one CTA)", 1: "dq_gemm2_kernel (CTA pair)",
              2: "bf16_gemm2_kernel (CTA pair, decoding its weight in-launch)",
              3: "smallm_kernel (weights loaded into registers, decoded into warp-MMA operands)",
              4: "smallm2_kernel (weights streamed through a TMA ring, decoded into warp-MMA "
                 "operands)"}[pair]
    return {"kernel": kernel, "pair": pair in (1, 2), "twophase": pair == 2, "smallm": pair in (3, 4),
            "ring": pair == 4,
            "bm": bm, "splits": splits, "grid": grid}
