"""Linear layers with activation and residual, what needs no GPU: their formulas in 64 bits with bounds on what a kernel may be off,
the gradients against differences, and the refusals of the entry points."""
import ctypes

import pytest
import scipy.sparse as sp
import numpy as np
import torch

import void_b200 as void
from void_b200 import _lib

BAD_ARG, ALIGN, SHAPE, WORKSPACE, TOO_LARGE = -1, -2, -3, -6, -8
ACTS = ("none", "relu", "gelu", "silu")
C1, C3 = 1.5957691216, 0.044715      # the framework's GELU: z * sigmoid(C1 (z + C3 z^3))
U = 2.0 ** -24
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 1e-44, torch.float16: 2.0 ** -25, torch.bfloat16: 1e-40}
# sigmoid and its products from the hardware's exponential and reciprocal: 2 ulp and 1 ulp, and as many for the polynomial in front
# (whose error is multiplied by |w| sigma(1 - sigma) |z| < |z|): 16 U |z| covers them
SIG = 16 * U


def act64(z, act):
    if act == "relu":
        return z.clamp_min(0)
    if act == "gelu":
        return z * torch.sigmoid(C1 * (z + C3 * z ** 3))
    return z * torch.sigmoid(z) if act == "silu" else z


def slope64(z, act):
    if act == "relu":
        return (z > 0).to(z.dtype)
    if act == "none":
        return torch.ones_like(z)
    s = torch.sigmoid(C1 * (z + C3 * z ** 3)) if act == "gelu" else torch.sigmoid(z)
    return s + z * s * (1 - s) * (C1 * (1 + 3 * C3 * z * z) if act == "gelu" else 1.0)


def product_error(a, b, dtype, terms, dense=False):
    """|a| . |b|^T times what a tensor-core sum of ``terms`` products may be off: fp32 sums that may truncate (2^-23 per addition, at
    most one per eight products, and sixteen for pieces that meet), for fp32 operands also their reduction to TF32 (A's tiles to the
    nearest, 2^-11; the other operand truncated: TF32 has ten bits behind the leading one, so what is cut off is below 2^-10 of the
    value).  dense: neither operand is a packed weight (the tiles' gradient), so both are truncated: (1 + 2^-10)^2 - 1 = 2^-9 + 2^-20."""
    tf32 = 2.0 ** -9 + 2.0 ** -20 if dense else 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -20
    unit = (terms / 8.0 + 16) * 2.0 ** -23 + (tf32 if dtype == torch.float32 else 0.0)
    return unit * (a.abs() @ b.abs().t())


def layer64(x, a, bias, residual, act, dtype, x_error=None):
    """z, y = act(z) + residual in 64 bits and a bound on a kernel's y; x_error: how far its x may already be off."""
    z = x @ a.t() + (0 if bias is None else bias)
    ez = product_error(x, a, dtype, x.shape[1]) + 4 * U * z.abs() + (0 if bias is None else 2 * U * bias.abs())
    if x_error is not None:
        ez = ez + x_error @ a.abs().t()
    y = act64(z, act)
    ey = 1.2 * ez + SIG * z.abs() * (act in ("gelu", "silu"))         # (slopes of gelu and silu stay below 1.13)
    if residual is not None:
        y = y + residual
        ey = ey + 2 * U * (y.abs() + residual.abs())
    return z, y, ez, ey


def rounded(e, y, dtype):
    return e + HALF[dtype] * (y.abs() + e) + TINY[dtype]


def layer_grads64(g, z, ez, x, a, act, dtype, bias_dtype):
    """(dx, dA, dbias) in 64 bits with their bounds.  z is kept in ``dtype``; second derivatives of gelu and silu stay below 0.8, and a
    relu whose z is within its error of zero may take the other side."""
    dz = g * slope64(z, act)
    kept = ez if act == "none" else rounded(ez, z, dtype)
    if act == "relu":
        e = g.abs() * (z.abs() <= kept)
    elif act == "none":
        e = torch.zeros_like(g)
    else:
        e = g.abs() * (0.85 * kept + SIG * (1 + z.abs()))
    e = e + 2 * U * dz.abs()
    er = e if act == "none" else rounded(e, dz, dtype)
    dx, da, db = dz @ a, dz.t() @ x, dz.sum(0)
    edx = er @ a.abs() + product_error(dz, a.t(), dtype, a.shape[0])
    eda = er.t() @ x.abs() + product_error(dz.t(), x.t(), dtype, x.shape[0], dense=True)
    edb = e.sum(0) + (g.shape[0] + 16) * U * dz.abs().sum(0)
    return [(dx, rounded(edx, dx, dtype)), (da, rounded(eda, da, dtype)), (db, rounded(edb, db, bias_dtype))]


def within(got, ref, bound):
    off = (got.double() - ref).abs() - bound
    assert bool((off <= 0).all()), (float(off.max()), float(bound.max()), float(ref.abs().max()))


@pytest.mark.parametrize("act", ACTS)
def test_gradient_formulas_are_the_derivatives(act):
    gen = torch.Generator().manual_seed(11)
    x, a, bias, g = (torch.randn(*s, generator=gen, dtype=torch.float64) for s in ((5, 7), (6, 7), (6,), (5, 6)))
    z, _, ez, _ = layer64(x, a, bias, None, act, torch.float32)
    dx, da, db = (t[0] for t in layer_grads64(g, z, ez, x, a, act, torch.float32, torch.float32))
    h = 1e-6
    for i, grad in enumerate((dx, da, db)):
        step = torch.randn(grad.shape, generator=gen, dtype=torch.float64)
        ends = [[t + (s * h * step if j == i else 0.0) for j, t in enumerate((x, a, bias))] for s in (1.0, -1.0)]
        diff = float(((layer64(*ends[0], None, act, torch.float32)[1] - layer64(*ends[1], None, act, torch.float32)[1]) * g).sum() / (2 * h))
        # (no z of this draw is within h of zero, so relu's kink is not crossed; the rest is of order h^2)
        assert abs(float((grad * step).sum()) - diff) < 1e-6 * (1 + abs(diff))


def _args(**kw):
    a = _lib.SpmmArgs()
    a.row_ptr, a.out, a.b, a.tiles, a.tile_cols = 1024, 1024, 1024, 1024, 1024
    a.nbr, a.nbc, a.nnz, a.M, a.K, a.N, a.ldb, a.ldc, a.transposed = 1, 1, 1, 32, 32, 4, 64, 32, 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("args, tail, kind, status", [
    (dict(transposed=0), {}, _lib.KIND_F16, BAD_ARG), (dict(transposed=3), {}, _lib.KIND_F16, BAD_ARG), ({}, {}, _lib.KIND_F8E4M3, BAD_ARG),
    ({}, {}, 9, BAD_ARG), ({}, dict(residual=1024, ldr=31), _lib.KIND_F16, SHAPE), ({}, dict(pre=1024, ldp=31), _lib.KIND_F16, SHAPE),
    (dict(out_dtype=1), dict(residual=1024, ldr=32, residual_dtype=2), _lib.KIND_F16, BAD_ARG),
    (dict(out_dtype=0), dict(residual=1024, ldr=32, residual_dtype=1), _lib.KIND_F16, BAD_ARG),
    (dict(M=-1), {}, _lib.KIND_F16, BAD_ARG), (dict(out=None), {}, _lib.KIND_F16, BAD_ARG), (dict(ldc=31), {}, _lib.KIND_F16, SHAPE),
    (dict(act=7), {}, _lib.KIND_F16, BAD_ARG), (dict(ldb=60), {}, _lib.KIND_F16, ALIGN), (dict(segs=1024), {}, _lib.KIND_F16, BAD_ARG),
    (dict(acc_out=1024), {}, _lib.KIND_F16, BAD_ARG), (dict(scale_mode=1), {}, _lib.KIND_I8, BAD_ARG),
])
def test_linear_entry_point_refuses(args, tail, kind, status):
    e = _lib.Epilogue()
    for k, v in tail.items():
        setattr(e, k, v)
    assert _lib.load().void_spmm_linear(ctypes.byref(_args(**args)), ctypes.byref(e), kind, None) == status


def test_linear_entry_points_refuse_null_structures_and_groups_of_other_layouts():
    lib, e, s = _lib.load(), _lib.Epilogue(), _lib.GroupStore()
    assert lib.void_spmm_linear(None, ctypes.byref(e), _lib.KIND_F16, None) == BAD_ARG
    assert lib.void_spmm_linear(ctypes.byref(_args()), None, _lib.KIND_F16, None) == BAD_ARG
    assert lib.void_spmm_grouped_linear(ctypes.byref(_args()), ctypes.byref(e), ctypes.byref(s), _lib.KIND_F16, None) == BAD_ARG
    assert lib.void_spmm_grouped_linear(ctypes.byref(_args(transposed=2)), ctypes.byref(e), ctypes.byref(s), _lib.KIND_F16, None) == BAD_ARG
    assert lib.void_spmm_grouped_linear(ctypes.byref(_args(transposed=2)), ctypes.byref(e), None, _lib.KIND_F16, None) == BAD_ARG
    assert lib.void_spmm_linear(ctypes.byref(_args(N=0, out=None)), ctypes.byref(e), _lib.KIND_F16, None) == 0


@pytest.mark.parametrize("bad, status", [
    (dict(elem=3), BAD_ARG), (dict(rows=-1), BAD_ARG), (dict(cols=-1), BAD_ARG), (dict(act=4), BAD_ARG), (dict(act=-1), BAD_ARG), (dict(ldg=7), BAD_ARG),
    (dict(ldz=7), BAD_ARG), (dict(lddz=7), BAD_ARG), (dict(be=2), BAD_ARG), (dict(g=None), BAD_ARG), (dict(z=None), BAD_ARG), (dict(dz=None), BAD_ARG),
    (dict(ws=None), WORKSPACE), (dict(ws_bytes=31), WORKSPACE), (dict(rows=2 ** 31 - 1), TOO_LARGE),
])
def test_activation_gradient_refuses(bad, status):
    v = dict(g=16, ldg=8, z=16, ldz=8, elem=1, rows=4, cols=8, act=2, dz=16, lddz=8, db=16, be=1, ws=16, ws_bytes=1 << 30)
    v.update(bad)
    ptr = lambda p: None if p is None else ctypes.c_void_p(p)   # noqa: E731
    assert _lib.load().void_activation_grad(ptr(v["g"]), v["ldg"], ptr(v["z"]), v["ldz"], v["elem"], v["rows"], v["cols"], v["act"], ptr(v["dz"]),
                                            v["lddz"], ptr(v["db"]), v["be"], ptr(v["ws"]), v["ws_bytes"], None) == status


def test_epilogue_mirror_matches_the_c_struct_layout():
    assert ctypes.sizeof(_lib.Epilogue) == 40
    assert [getattr(_lib.Epilogue, f).offset for f, _ in _lib.Epilogue._fields_] == [0, 8, 16, 20, 24, 32]


def _cpu_weight(m, k):
    return void.csr_to_void(sp.random(m, k, density=0.2, format="csr", dtype=np.float32, random_state=4))


def test_python_operators_refuse_what_they_cannot_do():
    a, back = _cpu_weight(64, 96), _cpu_weight(96, 64)
    x = torch.randn(4, 96)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.void_linear(a, x, residual=torch.randn(4, 64))
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.fused_sparse_mlp(x, a, back, residual=x)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.fused_sparse_mlp(x, a, back, norm=(None, None))
    with pytest.raises(AssertionError, match="residual"):
        void.fused_sparse_mlp(x, a, back, residual=torch.randn(4, 95))
    with pytest.raises(ValueError, match="unknown activation"):
        void.SparseLinear(96, 64, a, activation="gleu")
    with pytest.raises(NotImplementedError, match="not fused"):
        void.SparseLinear(96, 64, a, activation="tanh")
    with pytest.raises(AssertionError, match="w2 must have shape"):
        void.SparseFeedForward(a, a)


@pytest.mark.parametrize("bad, status", [
    (dict(kind=_lib.KIND_TF32), BAD_ARG), (dict(kind=_lib.KIND_I8), BAD_ARG), (dict(M=-1), BAD_ARG), (dict(K=-1), BAD_ARG), (dict(N=-1), BAD_ARG),
    (dict(ldx=63), BAD_ARG), (dict(ldz=31), BAD_ARG), (dict(bd=5), BAD_ARG), (dict(x=None), BAD_ARG), (dict(values=None), BAD_ARG), (dict(rows=None), BAD_ARG),
    (dict(at=None), BAD_ARG), (dict(cols=None), BAD_ARG), (dict(z=None), BAD_ARG), (dict(z=8), ALIGN), (dict(ldz=36), ALIGN),
    (dict(plan=None), BAD_ARG), (dict(plan=1024, offset_bytes=4), BAD_ARG), (dict(plan=1024, n_experts=0), BAD_ARG), (dict(M=0), 0), (dict(N=0), 0),
])
def test_relu_border_refuses(bad, status):
    v = dict(x=16, ldx=64, values=16, rows=16, at=16, cols=16, M=32, K=64, N=4, kind=_lib.KIND_F16, bias=None, bd=0, z=16, ldz=32, offset_bytes=0, n_experts=2)
    v.update(bad)
    ptr = lambda p: None if p is None else ctypes.c_void_p(p)   # noqa: E731
    x = None
    if "plan" in v:
        x = ctypes.byref(_lib.Experts(plan=v["plan"], n_experts=v["n_experts"], chunk=8, offset_bytes=v["offset_bytes"]))
    assert _lib.load().void_relu_border(ptr(v["x"]), v["ldx"], ptr(v["values"]), ptr(v["rows"]), ptr(v["at"]), ptr(v["cols"]), v["M"], v["K"], v["N"], v["kind"],
                                        ptr(v["bias"]), v["bd"], ptr(v["z"]), v["ldz"], x, None) == status
