"""The microscaled products' tests, on the CPU: their exact operands show a block that is lost, read twice or scaled by
another's byte, and their shapes take every launch."""

import ctypes

import numpy as np
import pytest
import torch

import qwen_image_kernel_amd as qik
from qwen_image_kernel_amd import _lib

from mx_exact import exact_operands, exact_sums
from oracle import mx as om


def rounded(sums, dtype):
    if dtype == "fp16":
        return sums.astype(np.float16).astype(np.float64)
    f = sums.astype(np.float32).view(np.uint32).astype(np.uint64)  # bf16: to nearest even
    return ((f + 0x7fff + ((f >> 16) & 1)) >> 16 << 16).astype(np.uint32).view(np.float32).astype(np.float64)


@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
@pytest.mark.parametrize("M,N,K", [(1, 65, 32768), (2, 33, 262144), (16, 40, 16416)])
def test_a_planted_mistake_shows(fmt, M, N, K):
    (ca, sa, a), (cw, sw, w), bias = exact_operands(M, N, K, fmt, 5)
    np.testing.assert_array_equal(om.values(ca, sa, fmt), a)
    np.testing.assert_array_equal(om.values(cw, sw, "mxfp4"), w)
    right = exact_sums(a, w, bias)
    rng = np.random.default_rng(7)
    B = K // 32
    places = {0, 1, B // 2 - 1, B // 2, B - 2, B - 1, *rng.integers(1, B - 1, 4).tolist()}
    for b in sorted(places):
        k = slice(32 * b, 32 * b + 32)
        part = a[:, k].astype(float) @ w[:, k].T.astype(float)
        other = sw[:, b - 1].astype(float) - sw[:, b]           # the byte of the block before
        mistakes = {"lost": -part, "twice": part, "scale": part * (2.0 ** other - 1)[None],
                    "half": -(a[:, k.start:k.start + 16].astype(float) @ w[:, k.start:k.start + 16].T.astype(float))}
        for name, off in mistakes.items():
            for dtype in ("bf16", "fp16"):
                # the product tests want every output equal, so one that differs is enough
                assert (rounded(right + off, dtype) != rounded(right, dtype)).any(), (name, b, dtype)


def plan(M, N, K, fmt, cus=0):
    """plan[0..5] and n1 of qik_mx_gemm_plan."""
    got, n1 = (ctypes.c_int32 * 6)(), ctypes.c_int64()
    assert _lib.load().qik_mx_gemm_plan(M, N, K, FMT[fmt], cus, got, ctypes.byref(n1)) == 0
    return list(got), n1.value


FMT = {"mxfp4": _lib.MXFP4, "mxfp8": _lib.MXFP8}


def kind(M, N, K, fmt, cus=0):
    """What runs: few rows (rows x columns, waves), a K split of a tile shape, one tile shape, or two in an order."""
    p, n1 = plan(M, N, K, fmt, cus)
    if p[5] == 0:
        return "rows {}x{} {}".format(*p)
    if p[5] > 1:
        return "split {}x{}".format(*p)
    if n1 in (0, N):
        return "tiles {}x{}".format(*(p[:2] if n1 else p[2:4]))
    return "{}x{} and {}x{}".format(*p) + (", small first" if p[4] else "")


# every launch of a product on 256 CUs, with its cheapest shapes of more than one stage or so; from a partial stage of
# K to more than a loop's turn of them
LAUNCHES = {
    "mxfp4": {
        (9, 41, 288): "rows 16x16 4", (16, 70, 1312): "rows 16x16 8", (9, 16500, 992): "rows 16x32 4",
        (12, 9000, 1824): "rows 16x16 4", (17, 41, 288): "rows 32x16 4", (31, 300, 1312): "rows 32x16 8",
        (33, 41, 288): "tiles 64x64", (65, 8490, 320): "tiles 64x128", (8202, 147, 288): "tiles 128x128",
        (810, 7009, 1824): "tiles 128x256", (268, 11316, 1824): "tiles 192x128", (810, 9344, 288): "tiles 192x256",
        (403, 11316, 288): "tiles 256x128", (8202, 1350, 288): "tiles 256x256",
        (602, 8490, 288): "128x256 and 128x128, small first", (1042, 14430, 8640): "128x256 and 128x128",
        (7454, 1048, 288): "192x256 and 192x128, small first", (1048, 10793, 5600): "192x256 and 192x128",
        (1087, 13702, 288): "256x256 and 128x128, small first", (5083, 3937, 288): "256x256 and 128x128",
        (7454, 1644, 1824): "256x256 and 256x128, small first", (1543, 9344, 288): "256x256 and 256x128",
        (9, 41, 12320): "split 64x64", (130, 257, 12320): "split 64x64", (65, 5000, 19424): "split 128x128"},
    "mxfp8": {
        (9, 41, 288): "rows 16x16 4", (16, 70, 1312): "rows 16x16 8", (9, 16500, 992): "rows 16x32 4",
        (12, 9000, 1824): "rows 16x16 4", (17, 41, 288): "rows 32x16 4", (31, 300, 1312): "rows 32x16 8",
        (33, 41, 288): "tiles 64x64", (65, 8490, 320): "tiles 64x128", (8202, 147, 288): "tiles 128x128",
        (810, 7009, 1824): "tiles 128x256", (268, 11316, 1824): "tiles 192x128", (810, 9344, 288): "tiles 192x256",
        (403, 11316, 288): "tiles 256x128", (810, 13702, 288): "tiles 256x256",
        (602, 8490, 288): "128x256 and 128x128, small first",
        (7454, 1048, 288): "192x256 and 192x128, small first", (2597, 9344, 288): "192x256 and 192x128",
        (1543, 11316, 288): "256x256 and 128x128, small first", (5083, 3937, 288): "256x256 and 128x128",
        (8202, 1350, 288): "256x256 and 256x128, small first", (1543, 9344, 288): "256x256 and 256x128",
        (17, 41, 4128): "split 64x64", (130, 257, 12320): "split 64x64", (2597, 71, 19424): "split 128x128"}}


@pytest.mark.parametrize("fmt,shape", [(f, s) for f in LAUNCHES for s in LAUNCHES[f]])
def test_launch_of_a_shape(fmt, shape):
    assert kind(*shape, fmt) == LAUNCHES[fmt][shape]


@pytest.mark.parametrize("fmt", LAUNCHES)
def test_no_launch_is_left_out(fmt):
    """Shapes at random take no launch that the table lacks (but a mix of the two smallest tile shapes, or of one that
    a shape here takes in the other order: the same kernel)."""
    rng = np.random.default_rng(3)
    have = {k.replace(", small first", "") for k in LAUNCHES[fmt].values()} | {"64x128 and 64x64"}
    for _ in range(20000):
        M, N, K = (int(lo * (hi / lo) ** rng.random()) for lo, hi in ((1, 9000), (1, 20000), (1, 700)))
        assert kind(M, N, 32 * K, fmt).replace(", small first", "") in have, (M, N, 32 * K, kind(M, N, 32 * K, fmt))


@pytest.mark.parametrize("fmt", LAUNCHES)
def test_plans_cover_the_output_and_fit_the_device(fmt):
    """Big tiles cover whole columns of theirs; a split's slices all run at once and take the scratch that the call asks
    for; no other launch takes any."""
    lib, n = _lib.load(), ctypes.c_int64()
    rng = np.random.default_rng(4)
    seen = 0
    for i in range(6000):
        M, N, K = (int(lo * (hi / lo) ** rng.random()) for lo, hi in ((1, 3000), (1, 9000), (4, 1000)))
        K *= 32
        for cus in (0, 128, 304):
            p, n1 = plan(M, N, K, fmt, cus)
            assert 0 <= n1 <= N and (n1 == N or n1 % p[1] == 0), (M, N, K, cus, p, n1)
            if p[5] > 1:
                seen += 1
                assert -(-(-(-M // p[0]) * -(-N // p[1])) // 8) * p[5] <= (cus or 256) // 8, (M, N, K, cus, p)
        p, n1 = plan(M, N, K, fmt)
        at = 1 << 20
        g = _lib.QikMxGemmArgs(_lib.ABI_VERSION, 0, FMT[fmt], 0, at, at, at, at, None, at, M, N, K,
                               K // 2 if fmt == "mxfp4" else K, K // 2, N)
        assert lib.qik_mx_gemm_workspace_size(ctypes.byref(g), ctypes.byref(n)) == 0
        assert n.value == (p[5] * M * -(-N // 4) * 16 if p[5] > 1 else 0)
    assert seen > 100


def test_plan_checks():
    lib, got, n1 = _lib.load(), (ctypes.c_int32 * 6)(), ctypes.c_int64()
    call = lambda M, N, K, f: lib.qik_mx_gemm_plan(M, N, K, f, 0, got, ctypes.byref(n1))  # noqa: E731
    assert call(1, 1, 32, 1) == 0 and call(1, 1, 32, 2) == 0
    assert call(1, 1, 32, 0) == -3 and call(1, 1, 32, 3) == -3
    for bad in ((0, 1, 32), (2 ** 30 + 1, 1, 32), (1, 0, 32), (1, 2 ** 28, 32), (1, 1, 0), (1, 1, 48), (1, 1, 262176)):
        assert call(*bad, 1) == -5, bad
    assert lib.qik_mx_gemm_plan(1, 1, 32, 1, 0, None, ctypes.byref(n1)) == -1
    assert lib.qik_mx_gemm_plan(1, 1, 32, 1, 0, got, None) == -1


@pytest.mark.parametrize("call", [
    lambda d: qik.MXFP4Linear(64, 8, out_dtype=d), lambda d: qik.MXFP4Linear.from_linear(torch.nn.Linear(64, 8), out_dtype=d),
    lambda d: qik.MXFP4Linear.from_quantized(qik.quantize_mx(torch.zeros(4, 32)), out_dtype=d),
    lambda d: qik.convert_linears_mxfp4(torch.nn.Sequential(torch.nn.Linear(64, 8)), out_dtype=d)])
def test_out_dtype_of_a_linear(call):
    for d in (torch.float32, torch.uint8, "fp16"):
        with pytest.raises(ValueError, match="out_dtype"):
            call(d)
    call(torch.bfloat16), call(torch.float16), call(None)


def test_bias_is_kept_in_the_out_dtype():
    lin = torch.nn.Linear(64, 8).half()
    lin.bias.data += 1
    for d in (torch.float16, torch.bfloat16, None):
        mod = qik.MXFP4Linear.from_linear(lin, out_dtype=d)
        assert mod.bias.dtype == (d or torch.bfloat16) and torch.equal(mod.bias, lin.bias.data.to(mod.bias.dtype))
        assert qik.MXFP4Linear(64, 8, bias=True, out_dtype=d).bias.dtype == mod.bias.dtype
        fresh = qik.MXFP4Linear(64, 8, bias=True, out_dtype=d)
        fresh.load_state_dict(mod.state_dict())
        assert torch.equal(fresh.bias, mod.bias)


def test_linear_finds_tensors_that_are_parameters():
    mod = qik.MXFP4Linear(64, 8)
    mod.weight = torch.nn.Parameter(mod.weight, requires_grad=False)
    with pytest.raises(ValueError, match="HIP device"):  # the refusal of a host tensor, not a lookup's error
        mod(torch.zeros(2, 64))
