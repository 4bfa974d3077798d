"""The exact operands of the product tests show a block that is lost, read twice or scaled by another's byte."""

import numpy as np
import pytest

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
