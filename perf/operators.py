"""The measured workload of the microscaled (MX) operators and the residual RMSNorm.

A case is one call through the public entry points, or in plain form (``own``
false) the same result from elementary torch operations.  Kinds:

* ``norm``     ``fused_residual_rms_norm``: h = x + residual, RMSNorm of h, the
               output in the element type or in a microscaled format
* ``quant``    ``quantize_mx`` of an activation or a weight, and its
               ``dequantize``: the values the codes stand for
* ``linear``   ``MXFP4Linear.forward``: dynamic quantisation of x and the
               product with the 4-bit weight
* ``product``  ``mx_linear`` of operands that are microscaled already (the
               output of a norm, say)

A microscaled row is cut into blocks of 32 along its last axis.  A block holds
one power-of-two scale, the byte e standing for 2^(e - 127), and 32 elements:
E2M1 (``mxfp4``: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; two to a byte, the
first in the low half) or E4M3 (``mxfp8``).  With E the fp32 exponent field of
the block's largest magnitude, e = max(E - emax, 0), emax 2 or 8; the elements
are x * 2^(127 - e) rounded to nearest, ties to even, saturated at 6 or 448.
"""

from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EMAX = {"mxfp4": 2, "mxfp8": 8}
BYTES = {"bf16": 2, "fp16": 2, "fp32": 4}
CODE_BYTES = {"mxfp4": 0.5 + 1 / 32, "mxfp8": 1 + 1 / 32}
EPS = 1e-6


def listed():
    return [
        # one token between two linears of a text model: the smallest call, where latency counts
        {"name": "norm_token", "kind": "norm", "M": 1, "D": 4096, "dtype": "bf16", "residual": True, "out": ""},
        # a prompt of 203 tokens, its normed hidden states in 8 bits for the linear that follows
        {"name": "norm_text_mxfp8", "kind": "norm", "M": 203, "D": 5120, "dtype": "bf16", "residual": True,
         "out": "mxfp8"},
        # the tokens of a 1024px layer (256 text + 4096 image) at 32 heads x 128, in 8 bits
        {"name": "norm_1024_mxfp8", "kind": "norm", "M": 4352, "D": 4096, "dtype": "bf16", "residual": True,
         "out": "mxfp8"},
        # an odd width and row count, fp16, no residual: the norm of a projected condition
        {"name": "norm_odd_fp16", "kind": "norm", "M": 9001, "D": 1111, "dtype": "fp16", "residual": False, "out": ""},
        # the activation of a 1024px layer to 4 bits and back
        {"name": "quant_act_1024", "kind": "quant", "M": 4352, "K": 4096, "dtype": "bf16", "out": "mxfp4"},
        # loading a model: an fp32 MLP weight to 4 bits, and what it then stands for
        {"name": "quant_weight", "kind": "quant", "M": 12288, "K": 4096, "dtype": "fp32", "out": "mxfp4"},
        # a short fp16 prompt of ragged width (47 blocks) to 8 bits and back
        {"name": "quant_small_mxfp8", "kind": "quant", "M": 77, "K": 1504, "dtype": "fp16", "out": "mxfp8"},
        # a single token through the MLP input: bound by the weight's 4-bit codes
        {"name": "linear_token", "kind": "linear", "M": 1, "K": 4096, "N": 12288, "bias": True, "act": "mxfp4"},
        # a few tokens, odd output width, 47 blocks of K, 8-bit activations
        {"name": "linear_ragged_w4a8", "kind": "linear", "M": 17, "K": 1504, "N": 5001, "bias": False,
         "act": "mxfp8"},
        # the text stream's MLP output, a prompt of 203 tokens: few tiles, a long K
        {"name": "linear_text_mlp", "kind": "linear", "M": 203, "K": 12288, "N": 4096, "bias": True, "act": "mxfp4"},
        # the MLP input of a 1024px layer on an activation that is in 4 bits already
        {"name": "product_mlp_in_1024", "kind": "product", "M": 4352, "K": 4096, "N": 12288, "bias": True,
         "act": "mxfp4"},
        # the MLP output of a guided (batch 2) 1024px layer, 8-bit activations: the largest
        {"name": "product_mlp_out_cfg_w4a8", "kind": "product", "M": 8704, "K": 12288, "N": 4096, "bias": True,
         "act": "mxfp8"},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["norm", "norm", "quant", "linear", "linear", "product"])
    if kind == "norm":
        out = rng.choice(["", "", "mxfp8", "mxfp8", "mxfp4"])
        D = 32 * _log(rng, 4, 256) if out else rng.choice([_log(rng, 64, 8192), 8 * _log(rng, 8, 1024)])
        M = _log(rng, 1, min(16384, 40_000_000 // D))
        return {"kind": kind, "M": M, "D": D, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "residual": rng.random() < 0.75, "out": out}
    if kind == "quant":
        K = 32 * _log(rng, 8, 512)
        return {"kind": kind, "M": _log(rng, 1, min(16384, 50_000_000 // K)), "K": K,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "out": rng.choice(["mxfp4", "mxfp4", "mxfp8"])}
    K, N = 32 * _log(rng, 8, 384), rng.choice([8 * _log(rng, 32, 1536), _log(rng, 200, 9000)])
    M = _log(rng, 1, 512) if kind == "linear" and rng.random() < 0.6 else _log(rng, 64, 8704)
    return {"kind": kind, "M": min(M, 8704 * 12288 * 4096 // (K * N)), "K": K, "N": N, "bias": rng.random() < 0.5,
            "act": rng.choice(["mxfp4", "mxfp4", "mxfp8"])}


# ---- the plain form --------------------------------------------------------

def _quantize(x, fmt):
    """fp32 x [M, K] -> the elements' values [M, K] (fp32) and the scale bytes [M, K/32] (int32)."""
    b = x.reshape(x.shape[0], -1, 32)
    E = (b.abs().amax(-1).view(torch.int32) >> 23) & 255
    e = torch.where(E == 255, E, (E - EMAX[fmt]).clamp_min(0))
    q = b * ((254 - e) << 23).view(torch.float32)[..., None]  # 2^(127 - e); where E is 255 the scale says NaN
    if fmt == "mxfp8":
        v = q.clamp(-448.0, 448.0).to(torch.float8_e4m3fn).float()
    else:
        a = q.abs().clamp_max(6.0)
        step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
        v = torch.copysign(torch.round(a / step) * step, q)
    return v.view(x.shape), e


def _values(v, e):
    """The values of elements v with scale bytes e."""
    # 2^(e - 127) from its bits: 2^-127 is a subnormal, 255 a NaN
    s = torch.where(e == 0, 0x400000, torch.where(e == 255, 0x7fc00000, e << 23)).to(torch.int32).view(torch.float32)
    return (v.view(v.shape[0], -1, 32) * s[..., None]).view(v.shape)


def _e2m1(codes):
    """Codes [N, K/2], two elements to a byte -> values [N, K], fp32."""
    c = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    m, x = c & 1, (c >> 1) & 3
    a = torch.where(x == 0, 0.5 * m, 0.25 * (2 + m) * (1 << x))
    return torch.where(c >= 8, -a, a)


def _decode(codes, scales, fmt):
    return _values(_e2m1(codes) if fmt == "mxfp4" else codes.float(), scales.int())


def _rms_norm(x, residual, weight, dtype):
    h = x if residual is None else (x.float() + residual.float()).to(dtype)
    r = 1.0 / torch.sqrt(h.double().square().mean(-1, keepdim=True) + EPS)
    return (h.float() * r.float()) * weight, h


# ---- inputs ----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _hidden(g, M, K, dtype):
    """Hidden states: normal, with one channel in 64 eight times larger, as transformer activations have."""
    x = torch.randn(M, K, generator=g, device="cuda")
    x[:, ::64] *= 8.0
    return x.to(DTYPES[dtype])


def _codes(x, fmt):
    """The codes a quantised tensor is kept in: mxfp4 uint8 [M, K/2], mxfp8 float8_e4m3fn [M, K]; scale bytes [M, K/32]."""
    v, e = _quantize(x, fmt)
    if fmt == "mxfp8":
        return v.to(torch.float8_e4m3fn), e.to(torch.uint8)
    a = (v.abs() * 2).int()  # twice the magnitude: 0 1 2 3 4 6 8 12
    c = torch.where(a < 4, a, torch.where(a < 8, 2 + a // 2, 4 + a // 4)) + 8 * (v < 0).int()
    return (c[:, 0::2] | (c[:, 1::2] << 4)).to(torch.uint8), e.to(torch.uint8)


def _weights(c, seed):
    g = _gen(seed)
    w = torch.randn(c["N"], c["K"], generator=g, device="cuda") * (c["K"] ** -0.5)
    b = torch.randn(c["N"], generator=g, device="cuda").bfloat16() if c["bias"] else None
    return g, *_codes(w, "mxfp4"), b


def prepare(case, seed):
    c = case
    s = SimpleNamespace(c=c)
    if c["kind"] == "norm":
        g = _gen(seed)
        s.x = _hidden(g, c["M"], c["D"], c["dtype"])
        s.res = _hidden(g, c["M"], c["D"], c["dtype"]) if c["residual"] else None
        s.w = torch.rand(c["D"], generator=g, device="cuda") + 0.5
    elif c["kind"] == "quant":
        s.x = _hidden(_gen(seed), c["M"], c["K"], c["dtype"])
    else:
        g, s.wc, s.ws, s.b = _weights(c, seed)
        s.x = _hidden(g, c["M"], c["K"], "bf16")
        if c["kind"] == "product":
            s.xc, s.xs = _codes(s.x.float(), c["act"])
        if own:  # the weight (and a product's activation) as a program keeps it: the module, the tensors in their layout
            import qwen_image_kernel_amd as qik
            w = qik.MXTensor.from_block_scales(s.wc, s.ws, "mxfp4")
            if c["kind"] == "linear":
                s.lin = qik.MXFP4Linear.from_quantized(w, s.b, activations=c["act"])
            else:
                s.w, s.a = w, qik.MXTensor.from_block_scales(s.xc, s.xs, c["act"])
    return s


def run(s):
    c = s.c
    if own:
        import qwen_image_kernel_amd as qik
        if c["kind"] == "norm":
            out = qik.fused_residual_rms_norm(s.x, s.res, s.w, EPS, out_format=c["out"] or None)
            y, h = out if c["residual"] else (out, None)
            y = y.dequantize(torch.bfloat16) if c["out"] else y
            return [y, h] if c["residual"] else [y]
        if c["kind"] == "quant":
            return qik.quantize_mx(s.x, c["out"]).dequantize(torch.bfloat16)
        if c["kind"] == "linear":
            return s.lin(s.x)
        return qik.mx_linear(s.a, s.w, s.b)
    if c["kind"] == "norm":
        dt = DTYPES[c["dtype"]]
        y, h = _rms_norm(s.x, s.res, s.w, dt)
        y = _values(*_quantize(y, c["out"])).bfloat16() if c["out"] else y.to(dt)
        return [y, h] if c["residual"] else [y]
    if c["kind"] == "quant":
        return _values(*_quantize(s.x.float(), c["out"])).bfloat16()
    if c["kind"] == "linear":
        x = _values(*_quantize(s.x.float(), c["act"]))
    else:
        x = _decode(s.xc, s.xs, c["act"])
    out = x @ _decode(s.wc, s.ws, "mxfp4").t()
    return (out if s.b is None else out + s.b.float()).bfloat16()


# ---- cost ------------------------------------------------------------------

def work(case):
    c = case
    M = c["M"]
    if c["kind"] == "norm":
        n, e = M * c["D"], BYTES[c["dtype"]]
        return {"bytes": n * e * (3 if c["residual"] else 1) + n * (2 if c["out"] else e) + 4 * c["D"], "flops": 6 * n}
    if c["kind"] == "quant":
        n = M * c["K"]
        return {"bytes": n * (BYTES[c["dtype"]] + 2), "flops": 3 * n}
    K, N = c["K"], c["N"]
    x = 2 if c["kind"] == "linear" else CODE_BYTES[c["act"]]
    return {"bytes": int(M * K * x + N * K * CODE_BYTES["mxfp4"]) + 2 * M * N + (2 * N if c["bias"] else 0),
            "flops": 2 * M * N * K}


# ---- the same results in 64 bits -------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _nearest64(a, grid):
    """The index of the grid value nearest to each a >= 0; halfway goes to the even index, past the end to the last."""
    hi = torch.searchsorted(grid, a).clamp(1, grid.numel() - 1)
    up, down = grid[hi] - a, a - grid[hi - 1]
    return torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)


def _mx64(x, fmt):
    """The values that x (fp64 [M, K]) is quantised to: the block's scale from the exponent of its largest
    magnitude, the nearest of the format's magnitudes."""
    if fmt == "mxfp4":
        grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    else:  # every E4M3 magnitude: 8 steps of 2^-9, then 8 to each power of two, up to 448
        k = torch.arange(127, device=x.device, dtype=torch.float64)
        grid = torch.where(k < 8, k / 512, (8 + k % 8) / 8 * torch.exp2((k // 8) - 7))
    out = torch.empty_like(x)
    for i in range(0, x.shape[0], 2048):
        b = x[i:i + 2048].unflatten(-1, (-1, 32))
        top = b.abs().amax(-1, keepdim=True)
        s = torch.exp2((torch.frexp(top)[1].double() - 1 - EMAX[fmt]).clamp_min(-127.0))
        s = torch.where(top == 0, 2.0 ** -127, s)
        out[i:i + 2048] = (grid[_nearest64((b / s).abs().contiguous(), grid)] * torch.sign(b) * s).flatten(-2)
    return out


def exact(case, seed):
    c = case
    if c["kind"] == "norm":
        g = _gen(seed)
        h = _hidden(g, c["M"], c["D"], c["dtype"]).double()
        if c["residual"]:
            h = h + _hidden(g, c["M"], c["D"], c["dtype"]).double()
        w = torch.rand(c["D"], generator=g, device="cuda") + 0.5
        # the norm is of the sum that is stored, in the element type
        hr = h.to(torch.float32).to(DTYPES[c["dtype"]]).double()
        y = hr / torch.sqrt((hr * hr).mean(-1, keepdim=True) + EPS) * w.double()
        y = _mx64(y, c["out"]) if c["out"] else y
        return [y, h] if c["residual"] else [y]
    if c["kind"] == "quant":
        return _mx64(_hidden(_gen(seed), c["M"], c["K"], c["dtype"]).double(), c["out"])
    g = _gen(seed)
    w = torch.randn(c["N"], c["K"], generator=g, device="cuda") * (c["K"] ** -0.5)
    b = torch.randn(c["N"], generator=g, device="cuda").bfloat16() if c["bias"] else None
    x = _hidden(g, c["M"], c["K"], "bf16")
    out = _mx64(x.double(), c["act"]) @ _mx64(w.double(), "mxfp4").t()
    return out if b is None else out + b.double()
