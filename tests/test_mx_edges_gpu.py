"""Microscaled operators at edges of what their calls allow."""

from types import SimpleNamespace

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


@pytest.mark.parametrize("fused", [True, False])
@pytest.mark.parametrize("fmt", ["mxfp4", "mxfp8"])
def test_processor_takes_the_norms_microscaled_output(fmt, fused):
    """A layer whose residual norm writes the projections' input in their format: the processor's hidden_states are
    that MXTensor, read by one projection or by three."""
    say("processor", fmt, fused)
    B, S, H, D = 2, 150, 4, 128
    dim = H * D
    g = torch.Generator(device=DEV).manual_seed(6)
    torch.manual_seed(6)
    names = ["qkv", "out"] if fused else ["q", "k", "v", "out"]
    net = torch.nn.ModuleDict({n: torch.nn.Linear(dim, 3 * dim if n == "qkv" else dim) for n in names}).to(DEV)
    assert qik.convert_linears_mxfp4(net, activations=fmt) == names
    norm = SimpleNamespace(weight=torch.rand(D, generator=g, device=DEV) + 0.5, eps=1e-6)
    attn = SimpleNamespace(heads=H, to_out=[net["out"], torch.nn.Identity()], norm_q=norm, norm_k=norm)
    if fused:
        attn.fused_qkv = net["qkv"]
    else:
        attn.to_q, attn.to_k, attn.to_v = net["q"], net["k"], net["v"]
    x, res = (torch.randn(B, S, dim, generator=g, device=DEV).bfloat16() for _ in range(2))
    w = torch.rand(dim, generator=g, device=DEV) + 0.5
    ang = torch.rand(S, D // 2, generator=g, device=DEV)
    freqs = torch.polar(torch.ones_like(ang), ang)
    y, h = qik.fused_residual_rms_norm(x, res, w, 1e-6, out_format=fmt)
    got = qik.QwenImage21KernelProcessor()(attn, y, rotary_emb=freqs)
    assert got.shape == (B, S, dim) and got.dtype == torch.bfloat16

    def product(mod, t):
        t = t if isinstance(t, qik.MXTensor) else qik.quantize_mx(t, fmt)
        return qik.mx_linear(t, mod.mx_weight(), mod.bias)

    if fused:
        q, k, v = product(net["qkv"], y).unflatten(-1, (3 * H, D)).chunk(3, dim=-2)
    else:
        q, k, v = (product(net[n], y).unflatten(-1, (H, D)) for n in "qkv")
    q, k = (qik.fused_rms_norm_rope(t, norm.weight, freqs, norm.eps) for t in (q, k))
    o = qik.block_causal_flash_attention(q, k, v, None, None, uniform_full=True)
    assert torch.equal(got, product(net["out"], o.flatten(2, 3)))
    assert torch.equal(h, (x.float() + res.float()).bfloat16())


def test_dequantised_values_past_a_types_range():
    """Exact in bf16 and fp32 up to infinity from 2^128 on, and to bf16's least subnormal, 2^-133."""
    def value(code, e, fmt, dtype):
        codes = torch.full((1, 32 if fmt == "mxfp8" else 16), code, dtype=torch.uint8, device=DEV)
        scale = torch.full((1, 1), e, dtype=torch.uint8, device=DEV)
        t = qik.MXTensor.from_block_scales(codes.view(torch.float8_e4m3fn) if fmt == "mxfp8" else codes, scale, fmt)
        return t.dequantize(dtype)[0, 0].item()

    tiny = 2.0 ** -133
    for code, e, exact, rounded in ((1, 0, 2.0 ** -136, 0.0), (15, 0, 15 * 2.0 ** -136, 2 * tiny), (1, 2, 2.0 ** -134, 0.0),
                                    (3, 2, 1.5 * tiny, 2 * tiny), (1, 3, tiny, tiny), (7, 3, 7 * tiny, 7 * tiny)):
        assert value(code, e, "mxfp8", torch.float32) == exact and value(code, e, "mxfp8", torch.bfloat16) == rounded
    assert value(0x11, 0, "mxfp4", torch.bfloat16) == 2.0 ** -128  # 0.5 of the least scale
    for dtype in (torch.bfloat16, torch.float32):
        assert value(0x7e, 246, "mxfp8", dtype) == 448 * 2.0 ** 119 and value(0x7e, 247, "mxfp8", dtype) == float("inf")
        assert value(0x77, 252, "mxfp4", dtype) == 6 * 2.0 ** 125 and value(0xff, 253, "mxfp4", dtype) == float("-inf")
    # the largest values quantise to no larger a scale
    big = torch.full((1, 32), torch.finfo(torch.float32).max, device=DEV)
    assert qik.quantize_mx(big, "mxfp4").block_scales().item() == 252 and qik.quantize_mx(big, "mxfp8").block_scales().item() == 246


@pytest.mark.parametrize("M", [3, 90])
def test_linear_with_a_cast_bias_is_captured(M):
    """An fp16 result with a bias in bf16, cast within the call: captured, replayed between eager calls, with the bias
    changed in place in between."""
    say("captured cast", M)
    torch.manual_seed(2)
    mod = qik.MXFP4Linear.from_linear(torch.nn.Linear(1056, 300, device=DEV))
    mod.out_dtype = torch.float16
    x = torch.randn(M, 1056, device=DEV).half()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        mod(x)
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = mod(x)
    for i in range(4):
        mod.bias.fill_(float(i))
        got.zero_()
        graph.replay()
        want = mod(x)
        torch.cuda.synchronize()
        assert got.dtype == torch.float16 and torch.equal(got, want)
        if i:
            assert not torch.equal(want, before)
        before = want.clone()


@pytest.mark.parametrize("M", [1, 200])
def test_linear_follows_its_tensors_to_another_layout(M):
    """Data of another stride or size at the same address, which a prepared call must notice: a strided bias is read as
    it lies, a weight, scales or bias of another size is refused."""
    say("layout", M)
    x = torch.randn(M, 64, device=DEV).bfloat16()
    base = torch.randn(80, device=DEV).bfloat16()
    for arg in (x, qik.quantize_mx(x)):
        mod = qik.MXFP4Linear(64, 40, bias=True).to(DEV)
        mod.bias.data = base[:40]
        assert torch.equal(mod(arg), base[:40].expand(M, 40))
        mod.bias.data = base[::2]
        assert mod.bias.data_ptr() == base.data_ptr() and torch.equal(mod(arg), base[::2].expand(M, 40))
        mod.bias.data = base[:40]
        assert torch.equal(mod(arg), base[:40].expand(M, 40))
        for name in ("bias", "weight", "weight_scale"):
            t = getattr(mod, name)
            whole = t.data
            t.data = whole[:1]
            with pytest.raises(ValueError, match=name):
                mod(arg)
            t.data = whole
            assert torch.equal(mod(arg), base[:40].expand(M, 40))
