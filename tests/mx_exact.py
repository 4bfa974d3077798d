"""Operands of microscaled products whose sums are exact in fp32, whatever their order and split.

Elements are -3 .. 3, scales 1, 2 or 4 for A and 1 or 2 for W, each block's its
own: every product is a whole number, and as long as the magnitudes of one
output's products and its bias add up to at most 2^24, so is every partial sum,
exactly.  A matrix core cuts nothing: the products of 8 elements of a block
differ by less than 2^4.  So a product is the exact sum rounded once, and a lost
or doubled block or a scale byte of another block shows in the result.
"""

import numpy as np

CODES = {"mxfp4": np.array([0, 2, 4, 5], np.uint8), "mxfp8": np.array([0, 0x38, 0x40, 0x44], np.uint8)}  # 0 1 2 3
SIGN = {"mxfp4": 8, "mxfp8": 128}


def exact_rows(M, K, fmt, scales, seed):
    """Codes uint8 [M, K] (one per byte), scale bytes [M, K/32], and the int64 values [M, K] they stand for."""
    rng = np.random.default_rng(seed)
    m = rng.integers(-3, 4, (M, K), dtype=np.int8)
    e = rng.integers(0, scales, (M, K // 32), dtype=np.uint8)
    codes = CODES[fmt][np.abs(m)] + np.where(m < 0, SIGN[fmt], 0).astype(np.uint8)
    return codes, e + np.uint8(127), m.astype(np.int64) << np.repeat(e, 32, -1).astype(np.int64)


def exact_operands(M, N, K, fmt, seed):
    """A's and W's (codes, scale bytes, values), and a bias of whole numbers [N]."""
    a = exact_rows(M, K, fmt, 3, seed)
    w = exact_rows(N, K, "mxfp4", 2, seed + 1)
    return a, w, np.random.default_rng(seed + 2).integers(-128, 129, N)


def exact_sums(a, w, bias):
    """The products' exact sums [M, N] in float64; asserts that no partial sum can leave fp32's whole numbers."""
    a, w = a.astype(np.float64), w.astype(np.float64)
    assert (np.abs(a) @ np.abs(w).T + np.abs(bias)).max() <= 2 ** 24
    return a @ w.T + bias
