"""Microscaled operators at edges of what their calls allow."""

import pytest
import torch

import qwen_image_kernel_amd as qik

pytestmark = pytest.mark.gpu

DEV = "cuda"


def say(*a):
    print("case", *a, flush=True)


def test_norm_of_one_workgroup_less_than_two_full_rows_of_a_grid():
    """16 rows a workgroup of 256 threads: 2^25 - 1 workgroups, which two rows of a grid would hold only with 2^32
    threads in each."""
    M = 16 * (2 ** 25 - 1) - 3
    say("grid", M)
    x = torch.ones(M, 1, dtype=torch.bfloat16, device=DEV)
    x[-40:] = -3
    y = qik.fused_residual_rms_norm(x, None, torch.ones(1, device=DEV), 0.0)
    assert (y[:-40] == 1).all() and (y[-40:] == -1).all()
