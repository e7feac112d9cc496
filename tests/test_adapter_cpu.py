"""Host-side refusals of the adapter, activation-checkpoint, input-gradient and
gated-norm entry points: every check that needs no device."""
import ctypes

import pytest
import torch

from diffuser_b200 import _lib, flux, ops
from diffuser_b200 import build as B

SHAPE, ALIGN, ARG = 1, 2, 7


@pytest.fixture(scope="module")
def lib():
    B.build()
    return _lib.lib()


P = 0x1000
F = ctypes.c_float


def _add(lib, *, M=4, R=1, K=64, N=64, r=16, A=2, act=0, y=P, ldy=None, x=P, ldx=None, down=P, up=P, scale=P,
         plan=P, out=2 * P, ldo=None, hidden=None):
    n_out = N // 2 if act >= 2 else N
    return lib.dq_adapter_add(y, N if ldy is None else ldy, x, K if ldx is None else ldx, M, R, K, N, down, up,
                              scale, r, A, plan, act, out, n_out if ldo is None else ldo, hidden, P, 1 << 30, None)


@pytest.mark.parametrize("kw,status", [
    (dict(K=60), SHAPE), (dict(N=60), SHAPE), (dict(r=12), SHAPE), (dict(r=136), SHAPE), (dict(r=0), SHAPE),
    (dict(A=0), SHAPE), (dict(A=65536), SHAPE), (dict(M=-1), SHAPE), (dict(M=(1 << 30) + 1), SHAPE),
    (dict(R=-1), SHAPE), (dict(ldy=56), SHAPE), (dict(ldy=68), SHAPE), (dict(ldx=60), SHAPE), (dict(ldo=8), SHAPE),
    (dict(act=2, N=48), SHAPE), (dict(act=4), ARG), (dict(act=-1), ARG), (dict(y=None), ARG), (dict(x=None), ARG),
    (dict(down=None), ARG), (dict(up=None), ARG), (dict(scale=None), ARG), (dict(plan=None), ARG),
    (dict(out=None), ARG), (dict(act=2, out=P), ARG), (dict(out=P, ldo=72), SHAPE), (dict(y=P + 8), ALIGN),
    (dict(x=P + 2), ALIGN), (dict(up=P + 8), ALIGN), (dict(hidden=P + 4), ALIGN), (dict(out=P + 8), ALIGN),
    (dict(M=0), 0),
])
def test_adapter_add_checks_its_arguments(lib, kw, status):
    assert _add(lib, **kw) == status


def _bwd(lib, *, M=4, K=64, N=64, r=16, A=2, dy=P, x=P, ldx=None, x_scales=None, hidden=P, dx=P, lddx=None,
         dx_out=2 * P, ddown=P, dup=P, plan=P):
    return lib.dq_adapter_backward(dy, N, x, K if ldx is None else ldx, x_scales, hidden, M, 1, K, N, P, P, P, r, A,
                                   plan, dx, K if lddx is None else lddx, dx_out, K, ddown, dup, P, 1 << 30, None)


@pytest.mark.parametrize("kw,status", [
    (dict(K=60), SHAPE), (dict(r=20), SHAPE), (dict(K=72, x_scales=P), SHAPE), (dict(ldx=72, x_scales=P), SHAPE),
    (dict(ldx=60), SHAPE), (dict(lddx=60), SHAPE), (dict(dup=None), ARG), (dict(dy=None), ARG), (dict(dx=None), ARG),
    (dict(dx_out=None), ARG), (dict(x=None), ARG), (dict(hidden=None), ARG), (dict(plan=None), ARG),
    (dict(dx=P, dx_out=P, lddx=72), SHAPE), (dict(x_scales=P + 2), ALIGN), (dict(ddown=P + 2), ALIGN),
])
def test_adapter_backward_checks_its_arguments(lib, kw, status):
    assert _bwd(lib, **kw) == status


def test_plan_checks_its_arguments(lib):
    assert lib.dq_adapter_plan_bytes(-1, 1, 1) == 0 and lib.dq_adapter_plan_bytes(1, 1, 0) == 0
    n = lib.dq_adapter_plan_bytes(100, 3, 2)
    assert n > 400
    assert lib.dq_adapter_plan(P, P, 3, 100, 0, P, n, None) == SHAPE
    assert lib.dq_adapter_plan(None, P, 3, 100, 2, P, n, None) == ARG
    assert lib.dq_adapter_plan(P, None, 3, 100, 2, P, n, None) == ARG
    assert lib.dq_adapter_plan(P, P, 3, 100, 2, P + 4, n, None) == ALIGN
    assert lib.dq_adapter_plan(P, P, 3, 100, 2, P, n - 1, None) == 6
    assert "offset" in _lib.status_string(_lib.DQ_ERR_INDEX)


def test_plan_capacity_holds_every_split_into_groups(lib):
    # each nonempty bucket is padded by at most 15 rows and opens at most one more large tile
    for m, r, a in ((1, 1, 1), (17, 5, 3), (300, 300, 7), (4608, 4, 64), (0, 0, 1)):
        words = lib.dq_adapter_plan_bytes(m, r, a) // 4
        groups = min(a, r) + 1
        need = m + 15 * groups
        assert words >= 16 + (a + 2) + (a + 1) + need + need // 16 + 4 * (m // 128 + groups)


@pytest.mark.parametrize("args,status", [
    ((P, 64, 4, 60, P, P), SHAPE), ((P, 60, 4, 64, P, P), SHAPE), ((P, 68, 4, 64, P, P), SHAPE),
    ((P, 64, -1, 64, P, P), SHAPE), ((None, 64, 4, 64, P, P), ARG), ((P, 64, 4, 64, None, P), ARG),
    ((P + 8, 64, 4, 64, P, P), ALIGN), ((P, 64, 4, 64, P + 8, P), ALIGN), ((P, 64, 0, 64, P, P), 0)])
def test_checkpoint_pack_checks_its_arguments(lib, args, status):
    assert lib.dq_checkpoint_pack(*args, None) == status


def test_checkpoint_unpack_checks_its_arguments(lib):
    assert lib.dq_checkpoint_unpack(P, P, 4, 72, P, 72, None) == SHAPE
    assert lib.dq_checkpoint_unpack(P, P, 4, 64, P, 60, None) == SHAPE
    assert lib.dq_checkpoint_unpack(P, None, 4, 64, P, 64, None) == ARG
    assert lib.dq_checkpoint_unpack(P, P, 4, 64, P + 8, 64, None) == ALIGN


def test_dgrad_checks_its_arguments(lib):
    nf4 = lambda M=4, N=64, K=64, dy=P, w=P, am=P, sd=0, dx=P: lib.dq_linear_nf4_dgrad(  # noqa: E731
        dy, M, N, w, am, sd, K, dx, P, 1 << 30, None)
    assert nf4(N=60) == SHAPE and nf4(K=96) == SHAPE and nf4(M=-1) == SHAPE
    assert nf4(dy=None) == ARG and nf4(am=None) == ARG and nf4(dx=None) == ARG and nf4(sd=3) == ARG
    assert nf4(dy=P + 8) == ALIGN and nf4(w=P + 8) == ALIGN
    assert nf4(M=0) == 0
    assert lib.dq_linear_fp8_dgrad(P, 4, 64, P, F(1.0), 24, P, P, 1 << 30, None) == SHAPE
    assert lib.dq_linear_fp8_dgrad(P, 4, 64, None, F(1.0), 32, P, P, 1 << 30, None) == ARG
    assert lib.dq_linear_dgrad_workspace(64, 128) == 64 * 128 * 2


def _norm(lib, *, T=4, S=2, D=64, x=P, ldx=None, y=P, gate=P, ldg=None, scale=P, shift=P, ldm=None, pw=None, qw=None,
          post=0, pre=1, rounding=0, s=P, h=P):
    return lib.dq_gated_norm(x, D if ldx is None else ldx, y, D, T, S, D, gate, D if ldg is None else ldg, scale,
                             shift, D if ldm is None else ldm, pw, qw, post, pre, F(1.0), F(1e-6), rounding, s, D, h,
                             D, None)


@pytest.mark.parametrize("kw,status", [
    (dict(D=66), SHAPE), (dict(D=8196), SHAPE), (dict(T=5), SHAPE), (dict(S=0), SHAPE), (dict(T=-2), SHAPE),
    (dict(ldx=60), SHAPE), (dict(ldx=66), SHAPE), (dict(ldg=60), SHAPE), (dict(ldm=62), SHAPE), (dict(post=3), ARG),
    (dict(pre=0), ARG), (dict(pre=3), ARG), (dict(pw=P), ARG), (dict(rounding=2), ARG), (dict(x=None), ARG),
    (dict(h=None), ARG), (dict(y=P + 4), ALIGN), (dict(gate=P + 2), ALIGN), (dict(qw=P + 4), ALIGN), (dict(T=0), 0)])
def test_gated_norm_checks_its_arguments(lib, kw, status):
    assert _norm(lib, **kw) == status


def test_gated_norm_backward_checks_its_arguments(lib):
    def call(T=4, S=2, D=64, dh=P, s=P, post=0, pw=None, lddx=64, dx=P, dgate=P):
        return lib.dq_gated_norm_backward(None, 0, dh, 64, s, 64, P, 64, T, S, D, P, 64, P, 64, pw, None, post, 1,
                                          F(1.0), F(1e-6), dx, lddx, P, 64, dgate, P, P, None, None, P, 1 << 30, None)
    assert call(D=66) == SHAPE and call(T=3) == SHAPE and call(T=1 << 31, S=1) == SHAPE and call(lddx=60) == SHAPE
    assert call(dh=None) == ARG and call(s=None) == ARG and call(dx=None) == ARG and call(pw=P) == ARG
    assert call(dx=P + 4) == ALIGN and call(dgate=P + 2) == ALIGN
    assert lib.dq_gated_norm_backward_workspace(5, 2, 64) == 0


def test_python_entry_points_refuse_cpu_tensors():
    b = lambda *s: torch.zeros(*s, dtype=torch.bfloat16)  # noqa: E731
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adapter_plan(torch.zeros(1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 4, 1)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adapter_add(b(2, 64), b(2, 64), b(1, 8, 64), b(1, 8, 64), torch.ones(1), None)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.adapter_backward(b(2, 64), b(2, 64), b(2, 8), b(1, 8, 64), b(1, 8, 64), torch.ones(1), None)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.checkpoint_pack(b(2, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.PackedActivation(torch.zeros(2, 64, dtype=torch.int8), torch.ones(2, 1))
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.nf4_linear_dgrad(b(2, 64), torch.zeros(64 * 32, dtype=torch.uint8), torch.ones(64), 64)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.fp8_linear_dgrad(b(2, 64), torch.zeros(64, 64, dtype=torch.float8_e4m3fn), 1.0)
    with pytest.raises(RuntimeError, match="CUDA"):
        flux.gated_norm(b(1, 2, 64), b(1, 2, 64))
    with pytest.raises(RuntimeError, match="CUDA"):
        flux.gated_norm_backward(None, b(1, 2, 64), b(1, 2, 64), b(1, 2, 64))


def test_packed_calls_carry_every_argument(lib):
    """The packed form of an entry refuses what the entry itself refuses, so a
    word out of place shows: each argument is spoilt in turn."""
    from diffuser_b200 import _lib as L
    assert all(getattr(lib, name + "_packed")(None) == ARG for name in L.PACKED)
    # dq_checkpoint_pack: x, ldx, M, K, codes, scales, stream
    good = [1 << 20, 64, 0, 64, 1 << 20, 1 << 20, 0]
    L.call("dq_checkpoint_pack", *good)
    for at, bad in ((1, 60), (2, -1), (3, 40), (3, -16)):
        words = list(good)
        words[at] = bad
        with pytest.raises(L.DqError, match="dq_checkpoint_pack.*shape"):
            L.call("dq_checkpoint_pack", *words)
    # dq_gated_norm: a float past the integers, then an alignment
    norm = [16, 64, 16, 64, 4, 2, 64, 0, 0, 0, 0, 0, 0, 0, 0, 1, 1.0, 1e-6, 0, 16, 64, 16, 64, 0]
    for at, bad, status in ((4, 3, "shape"), (6, 62, "shape"), (14, 7, ""), (18, 5, ""), (20, 63, "shape"),
                            (21, 17, "align"), (0, 20, "align")):
        words = list(norm)
        words[at] = bad
        with pytest.raises(L.DqError, match=f"dq_gated_norm.*{status}"):
            L.call("dq_gated_norm", *words)
