"""Microscaled formats and the residual RMSNorm in numpy, from their definitions.

Independent of the product: quantisation picks the nearest of a format's
listed magnitudes in float64, the scale bytes come from ``frexp``.
"""

from __future__ import annotations

import numpy as np

BLOCK = 32
EMAX = {"mxfp4": 2, "mxfp8": 8}
E2M1 = np.array([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0])
# e4m3fn magnitudes by code 0..126: subnormals of 2^-9, then 8 steps to a power of two
E4M3 = np.array([c / 512 if c < 8 else (8 + c % 8) / 8 * 2.0 ** (c // 8 - 7) for c in range(127)])
GRID = {"mxfp4": E2M1, "mxfp8": E4M3}


def nearest_code(a: np.ndarray, grid: np.ndarray) -> np.ndarray:
    """Index of the grid value nearest to each a >= 0: halfway to the even index, past the end to the last."""
    hi = np.clip(np.searchsorted(grid, a), 1, len(grid) - 1)
    up, down = grid[hi] - a, a - grid[hi - 1]
    return np.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def quantize(x: np.ndarray, fmt: str) -> tuple[np.ndarray, np.ndarray]:
    """float64 x [M, K] -> (element codes uint8 [M, K], one per byte, and scale bytes uint8 [M, K/32])."""
    M, K = x.shape
    b = x.reshape(M, K // BLOCK, BLOCK)
    bad = ~np.isfinite(b).all(-1)
    top = np.where(bad, 0.0, np.abs(b).max(-1))
    e = np.where(top > 0, np.maximum(np.frexp(top)[1] - 1 - EMAX[fmt] + 127, 0), 0)
    with np.errstate(invalid="ignore"):
        q = np.where(bad[..., None], 0.0, b) * np.exp2(127.0 - e)[..., None]
    sign = np.signbit(q) & ~bad[..., None]
    codes = nearest_code(np.abs(q), GRID[fmt]) + np.where(sign, len(GRID[fmt]) + (fmt == "mxfp8") * 1, 0)
    return codes.reshape(M, K).astype(np.uint8), np.where(bad, 255, e).astype(np.uint8)


def pack(codes: np.ndarray, fmt: str) -> np.ndarray:
    """Element codes as a tensor keeps them: two E2M1 to a byte, the even one low."""
    return codes if fmt == "mxfp8" else (codes[:, 0::2] | (codes[:, 1::2] << 4)).astype(np.uint8)


def unpack(codes: np.ndarray, fmt: str) -> np.ndarray:
    if fmt == "mxfp8":
        return codes
    return np.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1)


def values(codes: np.ndarray, scales: np.ndarray, fmt: str) -> np.ndarray:
    """float64 values of element codes [M, K] (one per byte) and scale bytes [M, K/32]."""
    half = 8 if fmt == "mxfp4" else 128
    v = np.append(GRID[fmt], np.nan)[codes % half] * np.where(codes >= half, -1.0, 1.0)
    s = np.where(scales == 255, np.nan, np.exp2(scales.astype(np.float64) - 127))
    return (v.reshape(*scales.shape, BLOCK) * s[..., None]).reshape(codes.shape)


def scale_layout(scales: np.ndarray) -> np.ndarray:
    """Scale bytes [M, K/32] in the layout of the product, uint8 [ceil(M/32), ceil(K/256), 256]."""
    M, B = scales.shape
    C = (B + 7) // 8
    out = np.zeros(((M + 31) // 32, C, 256), np.uint8)
    for m in range(M):
        for b in range(B):
            out[m // 32, b // 8, (m % 32) * 8 + b % 8] = scales[m, b]
    return out


def rms_norm(h: np.ndarray, weight: np.ndarray, eps: float) -> np.ndarray:
    """fp32 y = (h * r) * weight, r = fp32(1 / sqrt(mean64(h^2) + eps)), each fp32 operation rounded."""
    with np.errstate(all="ignore"):
        ms = np.square(h.astype(np.float64)).mean(-1, keepdims=True)
        r = (1.0 / np.sqrt(ms + eps)).astype(np.float32)
        return (h.astype(np.float32) * r).astype(np.float32) * weight.astype(np.float32)
