"""Layers of experts, what needs no GPU: the refusals of the entry points and of the Python operators."""
import ctypes

import numpy as np
import pytest
import scipy.sparse as sp
import torch

import void_b200 as void
from void_b200 import _lib
from void_b200.experts import rows_by_length

BAD_ARG, ALIGN, SHAPE, WORKSPACE, TOO_LARGE = -1, -2, -3, -6, -8


def _cpu_weight(m, k, seed=4):
    return void.csr_to_void(sp.random(m, k, density=0.2, format="csr", dtype=np.float32, random_state=seed))


def test_mirror_matches_the_c_struct_layout():
    assert ctypes.sizeof(_lib.Experts) == 32
    assert [getattr(_lib.Experts, f).offset for f, _ in _lib.Experts._fields_] == [0, 8, 12, 16, 24, 28]


def test_plan_words():
    words = _lib.load().void_expert_plan_words
    assert words(0, 10, 8) == 0 and words(4, -1, 8) == 0 and words(4, 10, 0) == 0
    # head 4, bounds and chunk offsets of five words each (on 16 bytes: 16 in all), at most 100 // 8 + 4 chunks of four words
    assert words(4, 100, 8) == 16 + 4 * 16
    assert words(4, 3, 8) == 16 + 4 * 3          # (a chunk holds a token)
    assert words(4, 0, 8) == 16


@pytest.mark.parametrize("bad, status", [
    (dict(offsets=None), BAD_ARG), (dict(plan=None), BAD_ARG), (dict(n_experts=0), BAD_ARG), (dict(rows=-1), BAD_ARG), (dict(chunk=0), BAD_ARG),
    (dict(offset_bytes=2), BAD_ARG), (dict(plan=1032), ALIGN), (dict(offset_bytes=8, offsets=1028), ALIGN), (dict(rows=2 ** 31 - 1), TOO_LARGE),
])
def test_plan_refuses(bad, status):
    v = dict(offsets=1024, offset_bytes=4, n_experts=4, rows=100, chunk=8, plan=1024)
    v.update(bad)
    ptr = lambda p: None if p is None else ctypes.c_void_p(p)   # noqa: E731
    assert _lib.load().void_expert_plan(ptr(v["offsets"]), v["offset_bytes"], v["n_experts"], v["rows"], v["chunk"], ptr(v["plan"]), None, None) == status


def _linear(args=(), experts=(), tail=None, kind=_lib.KIND_F16):
    a = _lib.SpmmArgs()
    a.row_ptr, a.out, a.b, a.tiles, a.tile_cols = 1024, 1024, 1024, 1024, 1024
    a.nbr, a.nbc, a.nnz, a.M, a.K, a.N, a.ldb, a.ldc, a.transposed = 1, 1, 1, 32, 32, 4, 64, 32, 1
    for k, v in dict(args).items():
        setattr(a, k, v)
    x = _lib.Experts(plan=1024, n_experts=2, chunk=8)
    for k, v in dict(experts).items():
        setattr(x, k, v)
    e = None
    if tail is not None:
        e = _lib.Epilogue()
        for k, v in tail.items():
            setattr(e, k, v)
        e = ctypes.byref(e)
    return _lib.load().void_expert_linear(ctypes.byref(a), e, ctypes.byref(x), kind, None)


@pytest.mark.parametrize("kw, status", [
    (dict(kind=_lib.KIND_I8), BAD_ARG), (dict(kind=_lib.KIND_F8E4M3), BAD_ARG), (dict(args=dict(transposed=0)), BAD_ARG),
    (dict(args=dict(transposed=2)), BAD_ARG), (dict(args=dict(M=-1)), BAD_ARG), (dict(args=dict(out=None)), BAD_ARG),
    (dict(args=dict(b=None)), BAD_ARG), (dict(args=dict(act=4)), BAD_ARG), (dict(args=dict(out_dtype=3)), BAD_ARG),
    (dict(args=dict(col_scale=1024)), BAD_ARG), (dict(args=dict(row_scale=1024)), BAD_ARG), (dict(args=dict(bias=1024)), BAD_ARG),
    (dict(args=dict(segs=1024)), BAD_ARG), (dict(args=dict(acc_out=1024)), BAD_ARG), (dict(args=dict(tile_terms=2)), BAD_ARG),
    (dict(args=dict(n_peers=1)), BAD_ARG), (dict(args=dict(ldc=31)), SHAPE), (dict(args=dict(M=33, ldc=33)), SHAPE),
    (dict(args=dict(ldb=62)), ALIGN), (dict(args=dict(ldb=48)), ALIGN), (dict(args=dict(tiles=1040)), ALIGN), (dict(args=dict(b=1032)), ALIGN),
    (dict(experts=dict(n_experts=0)), BAD_ARG), (dict(experts=dict(chunk=48)), BAD_ARG), (dict(experts=dict(chunk=0)), BAD_ARG),
    (dict(experts=dict(plan=None)), BAD_ARG), (dict(experts=dict(plan=1032)), ALIGN),
    (dict(experts=dict(offset_bytes=3)), BAD_ARG), (dict(experts=dict(offset_bytes=4, n_experts=33)), BAD_ARG),
    (dict(experts=dict(offset_bytes=8, plan=1028)), ALIGN), (dict(experts=dict(offset_bytes=4, plan=1026)), ALIGN),
    (dict(tail=dict(residual=1024, ldr=32)), BAD_ARG), (dict(tail=dict(pre=1024, ldp=31)), BAD_ARG),
    (dict(args=dict(N=2 ** 30, nbr=2 ** 20, M=2 ** 25, ldc=2 ** 25)), TOO_LARGE),
])
def test_linear_refuses(kw, status):
    assert _linear(**kw) == status


def test_grouped_form_refuses():
    lib, a, x, g = _lib.load(), _lib.SpmmArgs(), _lib.Experts(plan=1024, n_experts=2, chunk=128), _lib.GroupStore()
    a.row_ptr, a.out, a.b, a.nbr, a.nbc, a.M, a.K, a.N, a.ldb, a.ldc, a.transposed = 1024, 1024, 1024, 1, 1, 32, 32, 4, 64, 32, 1

    def call(**kw):
        keep = {}
        for k, v in kw.items():
            if k != "kind":
                t = x if hasattr(_lib.Experts, k) else (g if hasattr(_lib.GroupStore, k) else a)
                keep[k] = (t, getattr(t, k))
                setattr(t, k, v)
        st = lib.void_expert_grouped(ctypes.byref(a), None, ctypes.byref(x), ctypes.byref(g), kw.get("kind", _lib.KIND_F16), None)
        for k, (t, v) in keep.items():
            setattr(t, k, v)
        return st
    assert lib.void_expert_grouped(None, None, ctypes.byref(x), ctypes.byref(g), _lib.KIND_F16, None) == BAD_ARG
    assert call() == BAD_ARG                                     # an empty store
    for bad in (dict(kind=_lib.KIND_I8), dict(chunk=32), dict(n_experts=0), dict(plan=None), dict(offset_bytes=4), dict(transposed=2), dict(col_scale=1024), dict(row_scale=1024)):
        assert call(**bad) == BAD_ARG, bad
    g.blob = g.records = g.stage_ptr = g.group_rows = 1024
    g.max_entries = g.max_tiles = 1
    assert call(n_groups=3) == BAD_ARG                           # not the same number for every expert
    p = ctypes.c_void_p(1024)
    assert lib.void_expert_group_build(p, None, p, p, 4, 3, 10, 2, 4, 1, 1, p, p, p, p, p, None) == BAD_ARG
    assert lib.void_expert_group_build(p, None, p, p, 100, 3, 10, 2, 3, 1, 1, p, p, p, p, p, None) == BAD_ARG     # more than eight rows in a group


def test_no_tokens_is_no_work():
    assert _linear(args=dict(N=0, out=None)) == 0
    assert _lib.load().void_expert_linear(None, None, None, _lib.KIND_F16, None) == BAD_ARG


@pytest.mark.parametrize("bad", [dict(x=None), dict(plan=None), dict(n_experts=0), dict(M=0), dict(N=0), dict(kind=_lib.KIND_I8), dict(out_dtype=5),
                                 dict(n_items=-1)])
def test_tile_gradient_refuses(bad):
    v = dict(M=32, N=4, kind=_lib.KIND_F16, plan=1024, n_experts=2, out_dtype=1, n_items=1, x=1)
    v.update(bad)
    x = _lib.Experts(plan=v["plan"], n_experts=v["n_experts"], chunk=8)
    p = ctypes.c_void_p(1024)
    assert _lib.load().void_expert_tile_grad(p, 64, p, 64, v["M"], 32, v["N"], v["kind"], ctypes.byref(x) if v["x"] else None, p, v["n_items"], p, p, p,
                                             v["out_dtype"], None, None) == BAD_ARG


@pytest.mark.parametrize("bad, status", [
    (dict(plan=None), BAD_ARG), (dict(n_experts=0), BAD_ARG), (dict(chunk=0), BAD_ARG), (dict(elem=5), BAD_ARG), (dict(rows=-1), BAD_ARG),
    (dict(act=4), BAD_ARG), (dict(ldg=7), BAD_ARG), (dict(ldz=7), BAD_ARG), (dict(lddz=7), BAD_ARG), (dict(be=2), BAD_ARG), (dict(g=None), BAD_ARG),
    (dict(z=None), BAD_ARG), (dict(dz=None), BAD_ARG), (dict(ws=None), WORKSPACE), (dict(ws_bytes=3), WORKSPACE), (dict(n_experts=70000, rows=10), TOO_LARGE),
    (dict(rows=2 ** 30), TOO_LARGE),
])
def test_activation_gradient_refuses(bad, status):
    v = dict(g=16, ldg=8, z=16, ldz=8, elem=1, rows=4, cols=8, act=2, dz=16, lddz=8, db=16, be=1, ws=16, ws_bytes=1 << 40, plan=1024, n_experts=2, chunk=8)
    v.update(bad)
    ptr = lambda p: None if p is None else ctypes.c_void_p(p)   # noqa: E731
    x = _lib.Experts(plan=v["plan"], n_experts=v["n_experts"], chunk=v["chunk"])
    assert _lib.load().void_expert_activation_grad(ptr(v["g"]), v["ldg"], ptr(v["z"]), v["ldz"], v["elem"], ctypes.byref(x), v["rows"], v["cols"], v["act"],
                                                   ptr(v["dz"]), v["lddz"], ptr(v["db"]), v["be"], ptr(v["ws"]), v["ws_bytes"], None) == status


def test_offsets_stand_for_a_plan_in_the_product_alone():
    lib, p = _lib.load(), ctypes.c_void_p(1024)
    x = _lib.Experts(plan=1024, n_experts=2, chunk=8, offset_bytes=4)
    assert lib.void_expert_tile_grad(p, 64, p, 64, 32, 32, 4, _lib.KIND_F16, ctypes.byref(x), p, 1, p, p, p, 1, None, None) == BAD_ARG
    assert lib.void_expert_activation_grad(p, 8, p, 8, 1, ctypes.byref(x), 4, 8, 2, p, 8, p, 1, p, 1 << 40, None) == BAD_ARG


def test_stacking_and_its_refusals():
    a, b = _cpu_weight(70, 96), _cpu_weight(70, 96, 5)
    e = void.stack_experts([a, b])
    assert e.n_experts == 2 and e.shape == (70, 96) and e.tile_rows == 3 and e.dtype == torch.float32
    assert e.tensor.shape == (192, 96) and e.tensor.n_blocks == a.n_blocks + b.n_blocks
    dense = e.tensor.to_dense()
    assert torch.equal(dense[:70], a.to_dense()) and torch.equal(dense[96:166], b.to_dense()) and not dense[70:96].any()
    assert e.to_dtype(torch.float16).dtype == torch.float16
    with pytest.raises(ValueError, match="at least one"):
        void.stack_experts([])
    with pytest.raises(ValueError, match="one shape"):
        void.stack_experts([a, _cpu_weight(64, 96)])
    with pytest.raises(ValueError, match="one shape"):
        void.stack_experts([a, b.half()])
    with pytest.raises(TypeError, match="VOIDTensors"):
        void.stack_experts([a, a.to_dense()])


def test_rows_by_length_is_a_permutation_of_every_expert():
    row_ptr = torch.tensor([0, 1, 4, 4, 6, 6, 9], dtype=torch.int32)
    assert rows_by_length(row_ptr, 2).tolist() == [1, 0, 2, 2, 0, 1]


def test_python_operators_refuse():
    e = void.stack_experts([_cpu_weight(64, 96), _cpu_weight(64, 96, 5)])
    x, offsets = torch.randn(4, 96), torch.tensor([0, 2, 4], dtype=torch.int32)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.void_expert_linear(e, x, offsets)
    with pytest.raises(AssertionError, match="Dimension mismatch"):
        void.void_expert_linear(e, x[:, :95], offsets)
    with pytest.raises(TypeError, match="VOIDExperts"):
        void.void_expert_linear(e.tensor, x, offsets)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.SparseExperts(e)(x, offsets)
    with pytest.raises(ValueError, match="unknown activation"):
        void.SparseExperts(e, activation="what")
