"""Dense 8-bit weights with scales of blocks, what needs no GPU: the tensor itself, and the refusals of the entry points and operators."""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import void_b200 as void
from void_b200 import _lib

BAD_ARG, ALIGN, SHAPE, TOO_LARGE = -1, -2, -3, -8
ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
E4M3 = torch.float8_e4m3fn


def test_mirror_matches_the_c_struct_layout(tmp_path):
    gcc = shutil.which("gcc")
    if gcc is None:
        pytest.skip("no C compiler")
    fields = [f for f, _ in _lib.Fp8Args._fields_]
    src = tmp_path / "layout.c"
    src.write_text('#include <stdio.h>\n#include <stddef.h>\n#include "void_b200.h"\nint main(void) {\n  printf("%zu\\n", sizeof(void_fp8_args));\n'
                   + "".join('  printf("%%zu\\n", offsetof(void_fp8_args, %s));\n' % f for f in fields) + "  return 0;\n}\n")
    exe = tmp_path / "layout"
    subprocess.run([gcc, "-std=c99", "-Wall", "-Werror", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    out = [int(x) for x in subprocess.run([str(exe)], check=True, capture_output=True, text=True).stdout.split()]
    assert out[0] == ctypes.sizeof(_lib.Fp8Args)
    assert out[1:] == [getattr(_lib.Fp8Args, f).offset for f in fields]


def _linear(experts=None, **bad):
    a = _lib.Fp8Args(a=4096, lda=256, expert_stride=256 * 64, a_scale=4096, a_scale_row=2, a_scale_col=1, x=4096, ldx=256, x_scale=4096, x_scale_row=1,
                     x_scale_col=8, out=4096, ldc=64, M=64, K=256, N=8)
    for k, v in bad.items():
        setattr(a, k, v)
    x = None if experts is None else ctypes.byref(_lib.Experts(**dict(dict(plan=4096, n_experts=2, chunk=32), **experts)))
    return _lib.load().void_fp8_linear(ctypes.byref(a), x, None)


@pytest.mark.parametrize("bad, status", [
    (dict(a=None), BAD_ARG), (dict(x=None), BAD_ARG), (dict(a_scale=None), BAD_ARG), (dict(x_scale=None), BAD_ARG), (dict(out=None), BAD_ARG),
    (dict(M=-1), BAD_ARG), (dict(K=0), BAD_ARG), (dict(act=4), BAD_ARG), (dict(out_elem=3), BAD_ARG), (dict(bias_elem=-1), BAD_ARG),
    (dict(residual_elem=3), BAD_ARG), (dict(ldc=63), SHAPE), (dict(residual=4096, ldr=63), SHAPE), (dict(a=4104), ALIGN), (dict(x=4104), ALIGN),
    (dict(lda=264), ALIGN), (dict(ldx=264), ALIGN), (dict(lda=240), ALIGN), (dict(ldx=240), ALIGN), (dict(N=0), 0), (dict(M=0), 0), (dict(K=2 ** 28 + 1), TOO_LARGE),
    (dict(experts=dict(chunk=48)), BAD_ARG), (dict(experts=dict(chunk=256)), BAD_ARG), (dict(experts=dict(plan=None)), BAD_ARG), (dict(experts=dict(n_experts=0)), BAD_ARG),
    (dict(experts=dict(offset_bytes=3)), BAD_ARG), (dict(experts=dict(offset_bytes=4, n_experts=33)), BAD_ARG),
    (dict(experts=dict(offset_bytes=8, plan=4100)), ALIGN), (dict(experts=dict(plan=4104)), ALIGN), (dict(experts={}, expert_stride=264), ALIGN),
])
def test_linear_refuses(bad, status):
    assert _linear(**bad) == status


@pytest.mark.parametrize("bad, status", [
    (dict(x=None), BAD_ARG), (dict(q=None), BAD_ARG), (dict(scales=None), BAD_ARG), (dict(elem=3), BAD_ARG), (dict(block=64), BAD_ARG), (dict(rows=-1), BAD_ARG),
    (dict(ldx=99), SHAPE), (dict(ldq=99), SHAPE), (dict(rows=0), 0), (dict(cols=0), 0),
])
def test_quantiser_refuses(bad, status):
    v = dict(x=4096, elem=0, ldx=100, rows=4, cols=100, block=1, q=4096, ldq=112, scales=4096, row=1, col=4)
    v.update(bad)
    assert _lib.load().void_quant_fp8_blocks(v["x"], v["elem"], v["ldx"], v["rows"], v["cols"], v["block"], v["q"], v["ldq"], v["scales"], v["row"], v["col"],
                                             None) == status


def test_tensor():
    w = void.FP8BlockTensor(torch.ones(200, 256).to(E4M3), torch.tensor([[1.0, 2.0], [4.0, 8.0]]))
    assert w.shape == (200, 256) and w.block_rows == 128 and w.n_experts is None and w.memory_bytes == 200 * 256 + 16
    d = w.dequantize()
    assert (d[127, 127], d[127, 128], d[128, 127], d[199, 255]) == (1.0, 2.0, 4.0, 8.0)
    x = void.FP8BlockTensor(torch.ones(3, 130).to(E4M3), torch.arange(6.0).view(3, 2))
    assert x.block_rows == 1 and x.dequantize()[2, 129] == 5.0 and x.dequantize()[2, 127] == 4.0
    e = void.FP8BlockTensor(torch.ones(5, 200, 256).to(E4M3), torch.ones(5, 2, 2))
    assert e.n_experts == 5 and e.to("cpu").shape == (5, 200, 256) and "128" in repr(e)


def test_rows_that_start_anywhere_are_copied():
    given = torch.randn(3, 130).to(E4M3)
    x = void.FP8BlockTensor(given, torch.ones(3, 2))
    assert x.values.stride() == (144, 1) and x.values.data_ptr() != given.data_ptr()
    assert torch.equal(x.values.view(torch.uint8), given.view(torch.uint8))
    whole = torch.randn(3, 256).to(E4M3)
    assert void.FP8BlockTensor(whole, torch.ones(3, 2)).values is whole


@pytest.mark.parametrize("values, scales, error", [
    (torch.ones(4, 4), torch.ones(1, 1), _lib.VoidB200Error), (torch.ones(4, 4).to(E4M3), torch.ones(1, 1, dtype=torch.float64), _lib.VoidB200Error),
    (torch.ones(4, 4).to(E4M3), torch.ones(2, 1), ValueError), (torch.ones(4, 4).to(E4M3), torch.ones(1), ValueError),
    (torch.ones(4).to(E4M3), torch.ones(1), ValueError), (torch.ones(0, 4).to(E4M3), torch.ones(0, 1), ValueError),
    (torch.ones(2, 4, 4).to(E4M3), torch.ones(2, 4, 1), ValueError), (torch.ones(4, 4).to(torch.float8_e5m2), torch.ones(1, 1), _lib.VoidB200Error),
])
def test_tensor_refuses(values, scales, error):
    with pytest.raises(error):
        void.FP8BlockTensor(values, scales)


def test_operators_refuse():
    w = void.FP8BlockTensor(torch.ones(256, 256).to(E4M3), torch.ones(2, 2))
    e = void.FP8BlockTensor(torch.ones(2, 256, 256).to(E4M3), torch.ones(2, 2, 2))
    tokens = void.FP8BlockTensor(torch.ones(256, 256).to(E4M3), torch.ones(256, 2))
    x, offsets = torch.ones(4, 256), torch.zeros(3, dtype=torch.int32)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.void_linear(w, x)
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.void_expert_linear(e, x, offsets)
    with pytest.raises(_lib.VoidB200Error, match="x_scale"):
        void.void_linear(w, x, x_scale=1.0)
    with pytest.raises(_lib.VoidB200Error, match="void_expert_linear"):
        void.void_linear(e, x)
    with pytest.raises(_lib.VoidB200Error, match="n_experts"):
        void.void_expert_linear(w, x, offsets)
    for bad in (dict(bias=torch.ones(255)), dict(residual=torch.ones(4, 255))):
        with pytest.raises(AssertionError):
            void.void_linear(w, x, **bad)
    with pytest.raises(AssertionError):
        void.void_linear(w, torch.ones(4, 255))
    with pytest.raises(AssertionError):
        void.void_expert_linear(e, x, offsets, bias=torch.ones(256))
    with pytest.raises(ValueError):
        void.quantize_fp8_blocks(x, 64)
    with pytest.raises(ValueError):
        void.quantize_fp8_blocks(torch.ones(4))
    with pytest.raises(_lib.VoidB200Error, match="no CPU path"):
        void.quantize_fp8_blocks(x)
