"""GPU tests of RMSNorm + rotation by positions on several axes and its gradient, against the float64 oracle."""

import pytest
import torch

import qwen_image_kernel_amd as qik
from oracle import axial_rope as oa

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = 1e-6


def _axes(D):
    return (D // 8, D * 7 // 16, D * 7 // 16)


def _positions(g, B, S, how):
    if how == "grid":
        return torch.randint(-40, 60, (3, S), generator=g)
    if how == "far":
        return torch.randint(0, 1 << 22, (3, S), generator=g, dtype=torch.int32)
    return torch.rand(B, 3, S, generator=g) * 300 - 150   # fractional, each entry's own


def _within(got, want, bound):
    assert got.shape == want.shape
    off = (got.detach().cpu().double() - want.detach()).abs()
    worst = float((off / bound.detach()).max()) if off.numel() else 0.0
    assert worst <= 1.0, worst


def _inputs(g, B, S, Hq, Hk, D, dtype):
    x = [(torch.randn(B, S, H, D, generator=g) * torch.exp2(torch.randint(-4, 5, (B, S, H, 1), generator=g).float())).to(dtype)
         for H in (Hq, Hk)]
    w = [torch.rand(D, generator=g) + 0.5 for _ in range(2)]
    d = [torch.randn(t.shape, generator=g).to(dtype) for t in x]
    return x, w, d


CASES = [
    # B, S, Hq, Hk: one token, one head, runs that end inside a token, more tokens than a run's rows
    (1, 1, 1, 1), (1, 1, 32, 8), (2, 5, 3, 1), (1, 77, 24, 24), (3, 33, 7, 2), (2, 700, 1, 1), (1, 1031, 12, 4),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_forward_and_gradients(case, D, dtype, pairs):
    B, S, Hq, Hk = case
    g = torch.Generator().manual_seed(S + D)
    x, w, d = _inputs(g, B, S, Hq, Hk, D, dtype)
    how = ["grid", "far", "own"][(S + D // 32) % 3]
    spectrum = "shared" if D == 128 else "axis"
    pos = _positions(g, B, S, how)
    rope = qik.AxialRope(pos.to(DEV), _axes(D), (1e4, 500.0, 1e6), pairs=pairs, spectrum=spectrum)
    leaves = [t.to(DEV).requires_grad_() for t in (*x, *w)]
    out = qik.fused_qk_norm_rope(*leaves, rope, EPS, 1e-3)
    grads = torch.autograd.grad(out, leaves, [t.to(DEV) for t in d])
    angle = oa.angles(pos, _axes(D), (1e4, 500.0, 1e6), spectrum)
    for i, eps in enumerate((EPS, 1e-3)):
        xd, wd = x[i].double().requires_grad_(), w[i].double().requires_grad_()
        y = oa.forward(xd, wd, angle, pairs, eps)
        _within(out[i], y, oa.forward_bound(xd, wd, angle, pairs, eps, dtype))
        dx, dw = torch.autograd.grad(y, (xd, wd), d[i].double())
        _within(grads[i], dx, oa.dx_bound(xd, wd, d[i].double(), dx, pairs, eps, dtype))
        assert grads[2 + i].dtype == torch.float32
        _within(grads[2 + i], dw, oa.dw_bound(xd, d[i].double(), pairs, eps))
    # without gradients the same bits; one tensor alone too
    with torch.no_grad():
        again = qik.fused_qk_norm_rope(*leaves, rope, EPS, 1e-3)
        alone = qik.fused_rms_norm_rope(leaves[1], leaves[3], rope, 1e-3)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1]) and torch.equal(alone, out[1])
