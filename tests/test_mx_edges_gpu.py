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


@pytest.mark.parametrize("M", [1, 200])
def test_linear_follows_its_bias_to_another_dtype(M):
    """The bias's data replaced by another dtype's at the same address, which a prepared call must notice."""
    say("bias dtype", M)
    mod = qik.MXFP4Linear(64, 40, bias=True).to(DEV)
    x = torch.randn(M, 64, device=DEV).bfloat16()
    b = torch.randn(40, device=DEV).half()
    mod.bias.data = b.view(torch.bfloat16)
    assert torch.equal(mod(x), mod.bias.expand(M, 40)) and torch.equal(mod(qik.quantize_mx(x)), mod.bias.expand(M, 40))
    mod.bias.data = mod.bias.data.view(torch.float16)
    assert mod.bias.data_ptr() == b.data_ptr()
    assert torch.equal(mod(x), b.bfloat16().expand(M, 40)) and torch.equal(mod(qik.quantize_mx(x)), b.bfloat16().expand(M, 40))


def test_linear_whose_tensors_are_parameters():
    """Weight, scales and bias set to parameters (frozen, as loaders that know no buffers make them)."""
    say("parameters")
    ref = qik.MXFP4Linear.from_linear(torch.nn.Linear(288, 40, device=DEV))
    x = torch.randn(5, 288, device=DEV).bfloat16()
    want = ref(x)
    for names in (["weight"], ["weight_scale"], ["weight", "weight_scale", "bias"]):
        mod = qik.MXFP4Linear.from_quantized(ref.mx_weight(), ref.bias)
        for n in names:
            setattr(mod, n, torch.nn.Parameter(getattr(mod, n), requires_grad=False))
        assert torch.equal(mod(x), want) and torch.equal(mod(qik.quantize_mx(x)), ref(qik.quantize_mx(x)))
