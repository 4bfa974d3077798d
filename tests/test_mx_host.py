"""Microscaled operators without a GPU: the host quantiser, the layout of the scales, the C ABI and the refusals."""

import ctypes
import os
import re
import subprocess

import numpy as np
import pytest
import torch

from oracle import mx as om

import qwen_image_kernel_amd as qik
from qwen_image_kernel_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(ROOT, "include", "qik_mx.h")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]
FORMATS = ["mxfp4", "mxfp8"]


def rows(M, K, dtype, seed=0):
    """Rows of many magnitudes, with the blocks that quantisers get wrong: zeros, minus zero, NaN, infinities,
    subnormals, the type's largest, and a block of every half step of its scale."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(M, K, generator=g) * torch.exp2(torch.randint(-9, 9, (M, K // 32), generator=g)
                                                    .float()).repeat_interleave(32, 1)
    x = x.to(dtype)
    b = x.view(-1, 32)
    special = [torch.zeros(32), -torch.zeros(32), torch.full((32,), float("nan")),
               torch.tensor([float("inf")] + [1.0] * 31), torch.tensor([1.0] * 31 + [float("-inf")]),
               torch.tensor([7.9, -7.9, 6.0, 5.0, -5.0, 3.5, 2.5, 1.75, 1.25, 0.75, 0.25, -0.25] + [0.1] * 20),
               torch.full((32,), torch.finfo(dtype).max), torch.full((32,), torch.finfo(dtype).smallest_normal / 4),
               torch.full((32,), 1e-38) * torch.arange(32), torch.tensor([480.0, 464.0, 450.0, 17.0, 18.0, 19.0] * 5 + [0.01] * 2),
               torch.tensor([torch.finfo(dtype).max] + [torch.finfo(dtype).smallest_normal] * 31)]
    for i, s in enumerate(special[:b.shape[0]]):
        b[(i * 7) % b.shape[0]] = s.to(dtype)
    return x


def expect(x, fmt):
    codes, scales = om.quantize(x.double().numpy(), fmt)
    return om.pack(codes, fmt), scales


def same_bytes(t, x):
    codes, scales = expect(x.reshape(-1, x.shape[-1]).cpu(), t.fmt)
    np.testing.assert_array_equal(t.codes.view(torch.uint8).reshape(codes.shape).cpu().numpy(), codes)
    np.testing.assert_array_equal(t.block_scales().reshape(scales.shape).cpu().numpy(), scales)
    np.testing.assert_array_equal(t.scales.cpu().numpy(), om.scale_layout(scales))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("M,K", [(1, 32), (3, 96), (33, 256), (32, 288), (70, 1504)])
def test_host_quantiser_gives_the_definitions_bytes(fmt, dtype, M, K):
    x = rows(M, K, dtype, seed=M)
    same_bytes(qik.quantize_mx(x, fmt), x)


@pytest.mark.parametrize("fmt", FORMATS)
def test_every_half_step_rounds_to_even(fmt):
    """Each midpoint of neighbouring magnitudes, and the values just beside it."""
    grid = om.GRID[fmt]
    mid = (grid[1:] + grid[:-1]) / 2
    a = np.concatenate([mid, np.nextafter(mid.astype(np.float32), np.float32(0)),
                        np.nextafter(mid.astype(np.float32), np.float32(1e9)), grid]).astype(np.float32)
    a = np.concatenate([a, -a])
    top = grid[-1]
    blocks = np.zeros((-(-len(a) // 31), 32), np.float32)
    blocks[:, 0] = top  # every block's scale is 1
    for i, v in enumerate(a):
        blocks[i // 31, 1 + i % 31] = v
    t = qik.quantize_mx(torch.from_numpy(blocks), fmt)
    assert (t.block_scales() == 127).all()
    same_bytes(t, torch.from_numpy(blocks))


@pytest.mark.parametrize("fmt", FORMATS)
def test_layouts_of_the_input(fmt):
    x = rows(24, 512, torch.bfloat16, seed=3)
    for v in (x[:, 64:320], x[::3], x.view(2, 12, 512), x.t().contiguous().t()[:, :96], x[0], x[:0], x[5:6, 32:96],
              x[:1].expand(4, 512), x.view(2, 12, 512).transpose(0, 1)):
        t = qik.quantize_mx(v, fmt)
        assert t.shape == v.shape
        same_bytes(t, v.contiguous())


def test_threads_do_not_change_the_bytes():
    x = rows(300, 1056, torch.float32, seed=9)
    n = torch.get_num_threads()
    try:
        torch.set_num_threads(1)
        one = qik.quantize_mx(x)
        torch.set_num_threads(7)
        many = qik.quantize_mx(x)
    finally:
        torch.set_num_threads(n)
    assert torch.equal(one.codes, many.codes) and torch.equal(one.scales, many.scales)


@pytest.mark.parametrize("shape", [(1, 32), (31, 224), (2, 17, 288), (64, 512), (0, 64)])
def test_block_scales_round_trip(shape):
    g = torch.Generator().manual_seed(1)
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g, dtype=torch.uint8)
    bs = torch.randint(0, 255, (*shape[:-1], shape[-1] // 32), generator=g, dtype=torch.uint8)
    t = qik.MXTensor.from_block_scales(codes, bs, "mxfp4")
    assert torch.equal(t.block_scales(), bs) and t.shape == shape
    np.testing.assert_array_equal(t.scales.numpy(), om.scale_layout(bs.reshape(-1, shape[-1] // 32).numpy()))
    n = ctypes.c_int64()
    rows_ = int(np.prod(shape[:-1]))
    assert _lib.load().qik_mx_scales_size(rows_, shape[-1], ctypes.byref(n)) == 0 and n.value == t.scales.numel()


@pytest.mark.parametrize("call,match", [
    (lambda: qik.quantize_mx(torch.zeros(4, 33)), "multiple of 32"),
    (lambda: qik.quantize_mx(torch.zeros(4, 0)), "multiple of 32"),
    (lambda: qik.quantize_mx(torch.zeros(1, 262144 + 32)), "multiple of 32"),
    (lambda: qik.quantize_mx(torch.tensor(1.0)), "dimension"),
    (lambda: qik.quantize_mx(torch.zeros(4, 32, dtype=torch.int32)), "bf16, fp16 or fp32"),
    (lambda: qik.quantize_mx(torch.zeros(4, 32), "mxfp6"), "format"),
    (lambda: qik.quantize_mx(torch.zeros(4, 32, device="meta")), "HIP or CPU"),
    (lambda: qik.MXTensor(torch.zeros(4, 16), torch.zeros(1, 1, 256, dtype=torch.uint8), "mxfp4"), "codes"),
    (lambda: qik.MXTensor(torch.zeros(4, 16, dtype=torch.uint8), torch.zeros(4, 1, dtype=torch.uint8), "mxfp4"), "scales"),
    (lambda: qik.MXTensor.from_block_scales(torch.zeros(4, 16, dtype=torch.uint8),
                                            torch.zeros(4, 2, dtype=torch.uint8), "mxfp4"), "block scales"),
    (lambda: qik.quantize_mx(torch.zeros(4, 32)).dequantize(), "HIP device"),
    (lambda: qik.quantize_mx(torch.zeros(4, 32)).dequantize(torch.float64), "dtype"),
    (lambda: qik.mx_linear(qik.quantize_mx(torch.zeros(4, 32)), qik.quantize_mx(torch.zeros(4, 32))), "HIP device"),
    (lambda: qik.mx_linear(torch.zeros(4, 32), qik.quantize_mx(torch.zeros(4, 32))), "MXTensor"),
    (lambda: qik.mx_linear(qik.quantize_mx(torch.zeros(4, 32)), qik.quantize_mx(torch.zeros(4, 32), "mxfp8")), "mxfp4"),
    (lambda: qik.mx_linear(qik.quantize_mx(torch.zeros(4, 32)), qik.quantize_mx(torch.zeros(4, 64))), "multiply"),
    (lambda: qik.mx_linear(qik.quantize_mx(torch.zeros(4, 32)), qik.quantize_mx(torch.zeros(4, 32)),
                           out_dtype=torch.float32), "out_dtype"),
    (lambda: qik.MXFP4Linear(48, 8), "multiple of 32"),
    (lambda: qik.MXFP4Linear(64, 0), "out_features"),
    (lambda: qik.MXFP4Linear(64, 8, activations="fp8"), "format"),
    (lambda: qik.MXFP4Linear(64, 8)(torch.zeros(2, 64)), "HIP device"),
    (lambda: qik.MXFP4Linear(64, 8)(torch.zeros(2, 32)), r"\[\.\.\., 64\]"),
    (lambda: qik.MXFP4Linear.from_quantized(qik.quantize_mx(torch.zeros(4, 32), "mxfp8")), "mxfp4"),
    (lambda: qik.MXFP4Linear.from_quantized(qik.quantize_mx(torch.zeros(4, 32)), torch.zeros(5)), "bias"),
    (lambda: qik.fused_residual_rms_norm(torch.zeros(2, 32), None, torch.ones(32), 1e-6), "device tensor"),
    (lambda: qik.fused_residual_rms_norm(torch.zeros(2, 32), None, torch.ones(32), 1e-6, "fp8"), "format"),
    (lambda: qik.fused_residual_rms_norm(torch.zeros(2, 32).long(), None, torch.ones(32), 1e-6), "bf16, fp16 or fp32"),
])
def test_refusals(call, match):
    with pytest.raises(ValueError, match=match):
        call()


class Net(torch.nn.Module):
    def __init__(self):
        super().__init__()
        self.proj = torch.nn.Linear(64, 40)
        self.odd = torch.nn.Linear(50, 8)  # not whole blocks: stays as it is
        self.inner = torch.nn.ModuleDict({"keep": torch.nn.Linear(32, 32), "go": torch.nn.Linear(96, 33, bias=False)})


def test_convert_linears_and_state_dict():
    torch.manual_seed(0)
    net = Net()
    w = net.inner["go"].weight.detach().clone()
    assert qik.convert_linears_mxfp4(net, skip_patterns=("keep",), activations="mxfp8") == ["proj", "inner.go"]
    assert isinstance(net.odd, torch.nn.Linear) and isinstance(net.inner["keep"], torch.nn.Linear)
    go = net.inner["go"]
    assert go.activations == "mxfp8" and go.bias is None
    same_bytes(go.mx_weight(), w)
    # the converted state loads into modules that were built empty
    fresh = qik.MXFP4Linear(64, 40, bias=True)
    fresh.load_state_dict(net.proj.state_dict())
    assert torch.equal(fresh.weight, net.proj.weight) and torch.equal(fresh.weight_scale, net.proj.weight_scale)
    assert torch.equal(fresh.bias, net.proj.bias) and fresh.bias.dtype == torch.bfloat16


# ---- C ABI -------------------------------------------------------------------

STRUCTS = [("qik_mx_quant_args", _lib.QikMxQuantArgs), ("qik_mx_dequant_args", _lib.QikMxDequantArgs),
           ("qik_residual_rms_norm_args", _lib.QikResidualRmsNormArgs), ("qik_mx_gemm_args", _lib.QikMxGemmArgs),
           ("qik_mx_linear_args", _lib.QikMxLinearArgs)]


def test_header_and_binding_name_the_same_functions():
    names = set(re.findall(r"^int (qik_\w+)\s*\(", open(HEADER).read(), flags=re.M))
    assert names == {n for n, _, _ in _lib.MX_EXPORTS}
    lib = _lib.load()
    for n in names:
        assert hasattr(lib, n)
    text = open(HEADER).read()
    for name, value in (("QIK_MX_NONE", _lib.MX_NONE), ("QIK_MXFP4", _lib.MXFP4), ("QIK_MXFP8", _lib.MXFP8)):
        assert re.search(rf"\b{name} = (\d+)", text).group(1) == str(value)


@pytest.mark.parametrize("cname,pytype", STRUCTS)
def test_struct_layout_matches_c_header(tmp_path, cname, pytype):
    fields = [f for f, _ in pytype._fields_]
    src = ["#include <stdio.h>", "#include <stddef.h>", '#include "qik_mx.h"', "int main(void) {",
           f'printf("sizeof %zu\\n", sizeof({cname}));']
    src += [f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields] + ["return 0; }"]
    c = tmp_path / "layout.c"
    c.write_text("\n".join(src))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{os.path.dirname(HEADER)}", str(c), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True,
                                                        check=True).stdout.splitlines())
    assert int(got["sizeof"]) == ctypes.sizeof(pytype)
    for f in fields:
        assert int(got[f]) == getattr(pytype, f).offset, f


AT = 0x10000  # an aligned address that no call here reads


def quant_args(**kw):
    a = _lib.QikMxQuantArgs(_lib.ABI_VERSION, _lib.DTYPE_BF16, _lib.MXFP4, 0, AT, AT, AT, 4, 64, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def norm_args(**kw):
    a = _lib.QikResidualRmsNormArgs(_lib.ABI_VERSION, _lib.DTYPE_BF16, _lib.MXFP8, _lib.DTYPE_FP32, AT, AT, AT, AT, AT,
                                    AT, 4, 64, 64, 64, 1e-6)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


def gemm_args(**kw):
    a = _lib.QikMxGemmArgs(_lib.ABI_VERSION, _lib.DTYPE_BF16, _lib.MXFP4, 0, AT, AT, AT, AT, None, AT, 4, 8, 64, 32, 32, 8)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -2), (dict(reserved0=1), -2), (dict(dtype=3), -3), (dict(format=0), -3), (dict(format=3), -3),
    (dict(M=-1), -5), (dict(M=2 ** 31), -5), (dict(K=48), -5), (dict(K=0), -5), (dict(K=262176), -5), (dict(ldx=63), -5),
    (dict(x=None), -1), (dict(codes=None), -1), (dict(scales=None), -1),
    (dict(x=AT + 1), -8), (dict(codes=AT + 8), -8), (dict(scales=AT + 2), -8), (dict(M=0, x=None), 0)])
def test_quantise_status_codes(kw, code):
    lib = _lib.load()
    assert lib.qik_mx_quantize(ctypes.byref(quant_args(**kw)), None) == code
    assert lib.qik_mx_quantize_host(ctypes.byref(quant_args(**kw)), 1) == code
    assert lib.qik_mx_quantize(None, None) == -1


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -2), (dict(dtype=3), -3), (dict(format=3), -3), (dict(weight_dtype=1), -3), (dict(M=-1), -5),
    (dict(D=0), -5), (dict(D=48), -5), (dict(D=32800), -5), (dict(ldx=63), -5), (dict(ldr=63), -5),
    (dict(residual=None), -1), (dict(sum=None), -1), (dict(x=None), -1), (dict(weight=None), -1), (dict(out=None), -1),
    (dict(scales=None), -1), (dict(x=AT + 1), -8), (dict(x=AT + 2), -8), (dict(ldx=68), -8), (dict(out=AT + 8), -8),
    (dict(scales=AT + 2), -8), (dict(weight=AT + 4), -8), (dict(M=0, x=None), 0)])
def test_norm_status_codes(kw, code):
    assert _lib.load().qik_residual_rms_norm(ctypes.byref(norm_args(**kw)), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -2), (dict(reserved0=1), -2), (dict(dtype=3), -3), (dict(format=0), -3), (dict(M=-1), -5),
    (dict(K=48), -5), (dict(codes=None), -1), (dict(scales=None), -1), (dict(out=None), -1), (dict(codes=AT + 8), -8),
    (dict(out=AT + 8), -8), (dict(scales=AT + 2), -8), (dict(M=0, out=None), 0)])
def test_dequantise_status_codes(kw, code):
    a = _lib.QikMxDequantArgs(_lib.ABI_VERSION, _lib.DTYPE_BF16, _lib.MXFP4, 0, AT, AT, AT, 4, 64)
    for k, v in kw.items():
        setattr(a, k, v)
    assert _lib.load().qik_mx_dequantize(ctypes.byref(a), None) == code


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -2), (dict(reserved0=1), -2), (dict(out_dtype=2), -3), (dict(a_format=0), -3), (dict(M=-1), -5),
    (dict(M=2 ** 31), -5), (dict(N=0), -5), (dict(N=2 ** 31), -5), (dict(K=48), -5), (dict(K=0), -5), (dict(lda=16), -5),
    (dict(ldw=16), -5), (dict(ldw=2 ** 24), -5), (dict(ldc=7), -5), (dict(a_format=_lib.MXFP8), -5), (dict(a=None), -1),
    (dict(a_scales=None), -1), (dict(w=None), -1), (dict(w_scales=None), -1), (dict(out=None), -1), (dict(a=AT + 8), -8),
    (dict(w=AT + 8), -8), (dict(a_scales=AT + 8), -8), (dict(w_scales=AT + 8), -8), (dict(lda=40), -8), (dict(ldw=40), -8),
    (dict(out=AT + 1), -8), (dict(bias=AT + 1), -8), (dict(bias=AT + 2), -8), (dict(M=0, a=None), 0)])
def test_gemm_status_codes(kw, code):
    lib = _lib.load()
    n = ctypes.c_int64(-1)
    assert lib.qik_mx_gemm(ctypes.byref(gemm_args(**kw)), None, 0, None) == code
    assert lib.qik_mx_gemm_workspace_size(ctypes.byref(gemm_args(**kw)), ctypes.byref(n)) == code
    assert code == 0 or n.value == 0


@pytest.mark.parametrize("kw", [
    dict(M=2 ** 30 + 1), dict(N=2 ** 28, ldc=2 ** 28), dict(M=2 ** 30, N=2 ** 20, ldc=2 ** 20)])
def test_products_beyond_a_launch_are_refused(kw):
    assert _lib.load().qik_mx_gemm(ctypes.byref(gemm_args(**kw)), None, 0, None) == -5


@pytest.mark.parametrize("kw,code", [
    (dict(x_dtype=3), -3), (dict(reserved0=1), -2), (dict(ldx=63), -5), (dict(x=None), -1), (dict(x=AT + 1), -8)])
def test_linear_status_codes(kw, code):
    lib = _lib.load()
    a = _lib.QikMxLinearArgs(gemm_args(a=None, a_scales=None, lda=0), AT, 64, _lib.DTYPE_BF16, 0)
    for k, v in kw.items():
        setattr(a, k, v)
    n = ctypes.c_int64(-1)
    assert lib.qik_mx_linear(ctypes.byref(a), None, 0, None) == code
    assert lib.qik_mx_linear_workspace_size(ctypes.byref(a), ctypes.byref(n)) == code and n.value == 0


def test_linear_wants_its_workspace():
    lib = _lib.load()
    a = _lib.QikMxLinearArgs(gemm_args(a=None, a_scales=None, lda=0, M=300), AT, 64, _lib.DTYPE_BF16, 0)
    n = ctypes.c_int64(-1)
    assert lib.qik_mx_linear_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value > 0
    assert lib.qik_mx_linear(ctypes.byref(a), None, 0, None) == -12
    assert lib.qik_mx_linear(ctypes.byref(a), AT, n.value - 1, None) == -12
    assert lib.qik_mx_linear(ctypes.byref(a), AT + 16, n.value, None) == -12
