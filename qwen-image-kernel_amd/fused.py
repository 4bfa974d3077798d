"""Per-head RMSNorm + RoPE producing Q and K, same signature as the reference.

``fused_rms_norm_rope(x, weight, freqs_cis, eps)`` keeps the argument list and
result of ``qwen_image_kernel/triton_fused.py:75-105`` and runs the gfx950 HIP
kernel behind ``qik_rms_rope`` (include/qik_ops.h), asynchronously on the
current stream.

Per row of ``x [B, S, H, D]`` (fp32 arithmetic, triton_fused.py:48-69):
``n = round((x / sqrt(mean(x^2) + eps)) * weight)`` to the input dtype, then
each pair ``(n[2i], n[2i+1])`` is rotated by ``freqs_cis[s, i]`` and rounded to
the input dtype.  Differences from the reference, both on the safe side:

* a strided ``x`` (the q or k slice of a fused QKV output) is read in place
  instead of being copied to a contiguous tensor first (triton_fused.py:84-85);
* ``1 / sqrt`` is taken in fp64 and rounded once to fp32 (the reference uses the
  approximate fp32 ``rsqrt``), and every fp32 operation rounds on its own.

``fused_residual_rms_norm`` is the norm between a layer's linears: the residual
added, RMSNorm over the last dimension, the result in the element type or
microscaled for ``MXFP4Linear`` (qik_residual_rms_norm, include/qik_mx.h).

With an ``AxialRope`` in the place of ``freqs_cis`` the angles come from positions
on several axes (rope.py).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .mx import _DTYPES as _NORM_DTYPES
from .mx import MX_FORMATS, MXTensor, _as_rows, _check_format, _check_width, _CODE_DTYPE, _code_shape, _on_device, \
    _row_stride, _scales_shape
from .rope import AxialRope, fused_qk_norm_rope, norm_rope

__all__ = ["fused_rms_norm_rope", "fused_residual_rms_norm"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}

# cos/sin tables of recent freqs_cis tensors: Q and K of a layer, and every
# layer of a step, share one.  An entry keeps its freqs_cis alive, so a data
# pointer in a key can never be reused by another tensor; the version counter
# catches in-place updates.
_cos_sin_cache: dict = {}


def _cos_sin(freqs_cis: torch.Tensor, device: torch.device):
    key = (freqs_cis.data_ptr(), freqs_cis._version, tuple(freqs_cis.shape), freqs_cis.device, device)
    hit = _cos_sin_cache.get(key)
    if hit is None:
        cos = freqs_cis.real.float().contiguous().to(device)
        sin = freqs_cis.imag.float().contiguous().to(device)
        if len(_cos_sin_cache) > 8:
            _cos_sin_cache.clear()
        hit = _cos_sin_cache[key] = (freqs_cis, cos, sin)
    return hit[1], hit[2]


def fused_rms_norm_rope(
    x: torch.Tensor,           # [B, S, H, D] bf16 (or fp16)
    weight: torch.Tensor,      # [D] fp32
    freqs_cis: torch.Tensor | AxialRope,   # complex [S, D/2], or positions on several axes
    eps: float,
) -> torch.Tensor:
    """RMSNorm over D per (b, s, h), then complex RoPE by position s; returns [B, S, H, D].

    With an AxialRope the result is rounded once, weight may be None (no norm),
    and gradients are recorded."""
    if isinstance(freqs_cis, AxialRope):
        return norm_rope(x, weight, freqs_cis, eps)
    # One lookup per call: everything that only depends on the geometry, the
    # weight and freqs_cis tensors (and their in-place versions) and eps is
    # checked and prepared once per key -- the argument struct with the
    # weight and cos/sin pointers filled in, the output shape.  Only x's and
    # the output's data pointers change between calls.
    ent = _entry(x, weight, freqs_cis, eps)
    if ent.contig:
        x = x.clone(memory_format=torch.contiguous_format)
    out = x.new_empty(ent.shape)
    a = _lib.QikRmsRopeArgs.from_buffer_copy(ent.args)
    a.x = x.data_ptr()
    a.out = out.data_ptr()
    idx = ent.index
    if idx != torch.cuda.current_device():
        with torch.cuda.device(idx):
            _lib.check(ent.fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx)), "qik_rms_rope")
    else:
        _lib.check(ent.fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx)), "qik_rms_rope")
    return out


def _rms_rope_qk(query, key, norm_q, norm_k, freqs_cis):
    """fused_rms_norm_rope of a layer's Q and K (``norm_q`` and ``norm_k`` carry
    ``weight`` and ``eps``), in one launch when both are of one dtype, head dim
    and device, else in two."""
    if isinstance(freqs_cis, AxialRope):
        if query.dtype != key.dtype or query.shape[3] != key.shape[3]:
            return (norm_rope(query, norm_q.weight, freqs_cis, norm_q.eps),
                    norm_rope(key, norm_k.weight, freqs_cis, norm_k.eps))
        return fused_qk_norm_rope(query, key, norm_q.weight, norm_k.weight, freqs_cis, norm_q.eps, norm_k.eps)
    if query.dtype != key.dtype or query.shape[-1] != key.shape[-1] or query.device != key.device:
        return (fused_rms_norm_rope(query, norm_q.weight, freqs_cis, norm_q.eps),
                fused_rms_norm_rope(key, norm_k.weight, freqs_cis, norm_k.eps))
    # both entries are held here until the launch is enqueued: K's may clear Q's out
    # of the cache, and with it the last references to the fp32 weight, cos and sin
    # that Q's argument struct points to
    ents = [_entry(x, norm.weight, freqs_cis, norm.eps) for x, norm in ((query, norm_q), (key, norm_k))]
    args, outs, reads = [], [], []
    for x, ent in zip((query, key), ents):
        x = x.clone(memory_format=torch.contiguous_format) if ent.contig else x
        a = _lib.QikRmsRopeArgs.from_buffer_copy(ent.args)
        outs.append(x.new_empty(ent.shape))
        reads.append(x)
        a.x, a.out = x.data_ptr(), outs[-1].data_ptr()
        args.append(a)
    with torch.cuda.device(ent.index):
        _lib.check(_lib.load().qik_rms_rope_pair(ctypes.byref(args[0]), ctypes.byref(args[1]),
                                                 torch._C._cuda_getCurrentRawStream(ent.index)), "qik_rms_rope_pair")
    return outs


def _entry(x, weight, freqs_cis, eps) -> _Call:
    """The prepared call of a (geometry, weight, freqs_cis, eps) key."""
    key = (x.shape, x.stride(), x.data_ptr() & 15, x.dtype, x.device, eps,
           weight.data_ptr(), weight._version, weight.dtype, weight.shape, weight.stride(), weight.device,
           freqs_cis.data_ptr(), freqs_cis._version, freqs_cis.dtype, freqs_cis.shape, freqs_cis.stride(),
           freqs_cis.device)
    ent = _CALLS.get(key)
    if ent is None:
        ent = _prepare(x, weight, freqs_cis, eps)
        if len(_CALLS) >= 64:
            _CALLS.clear()
        _CALLS[key] = ent
    return ent


class _Call:
    """What one (geometry, weight, freqs_cis, eps) key needs at call time."""

    __slots__ = ("args", "shape", "contig", "index", "fn", "keep")


# Prepared calls by key (see fused_rms_norm_rope).  An entry keeps the weight
# and freqs_cis tensors it was built from alive, so the data pointers in a
# key can never be reused by other tensors while the key is cached; their
# version counters catch in-place updates.
_CALLS: dict = {}


def _prepare(x, weight, freqs_cis, eps) -> _Call:
    if x.dim() != 4:
        raise ValueError(f"x must be [B, S, H, D], got shape {tuple(x.shape)}")
    if x.dtype not in _DTYPES:
        raise ValueError(f"x must be bf16 or fp16, got {x.dtype}")
    if not x.is_cuda:
        raise ValueError("x must be a device tensor (the kernel runs on the GPU)")
    B, S, H, D = x.shape
    if tuple(freqs_cis.shape) != (S, D // 2):
        raise ValueError(f"freqs_cis must be [S, D/2] = {(S, D // 2)}, got {tuple(freqs_cis.shape)}")
    # the kernel reads 16-byte chunks in place from a 16-byte aligned base with
    # b/s/h strides in multiples of 8 elements and a unit D stride; any other
    # layout (the reference's kernel reads any strides) goes through a
    # contiguous copy made at each call
    sb, ss, sh, sd = x.stride()
    contig = ((D > 1 and sd != 1) or x.data_ptr() % 16 != 0 or (B > 1 and sb % 8 != 0)
              or (S > 1 and ss % 8 != 0) or (H > 1 and sh % 8 != 0))
    xs = x.clone(memory_format=torch.contiguous_format) if contig else x
    w = weight
    if w.dtype != torch.float32 or w.device != x.device or not w.is_contiguous():
        w = weight.to(device=x.device, dtype=torch.float32).contiguous()
    cos, sin = _cos_sin(freqs_cis, x.device)
    out = torch.empty((B, S, H, D), dtype=x.dtype, device=x.device)
    c = _Call()
    c.args = rms_rope_args(xs, w, cos, sin, out, eps)
    c.shape = (B, S, H, D)
    c.contig = contig
    c.index = x.device.index
    c.fn = _lib.load().qik_rms_rope
    c.keep = (weight, w, freqs_cis, cos, sin)
    return c


def rms_rope_args(x, weight, cos, sin, out, eps) -> _lib.QikRmsRopeArgs:
    """The qik_rms_rope argument struct for device tensors (no device work)."""
    B, S, H, D = x.shape
    a = _lib.QikRmsRopeArgs()
    a.abi_version = _lib.ABI_VERSION
    a.dtype = _DTYPES[x.dtype]
    a.x = x.data_ptr()
    a.out = out.data_ptr()
    a.weight = weight.data_ptr()
    a.cos = cos.data_ptr()
    a.sin = sin.data_ptr()
    a.B, a.S, a.H, a.D = B, S, H, D
    a.stride_x = _lib._i64x3(x.stride(0), x.stride(1), x.stride(2))
    a.stride_out = _lib._i64x3(out.stride(0), out.stride(1), out.stride(2))
    a.eps = float(eps)
    return a


_MAX_NORM_WIDTH = 32768


def fused_residual_rms_norm(
    x: torch.Tensor,                   # [..., D] bf16, fp16 or fp32
    residual: torch.Tensor | None,     # x's shape and dtype, or None
    weight: torch.Tensor,              # [D] fp32, or x's dtype
    eps: float,
    out_format: str | None = None,     # None, "mxfp8" or "mxfp4"
):
    """RMSNorm over the last dimension of ``h = x + residual``.

    Returns ``(out, h)``, or ``out`` alone where residual is None (h is x).  h
    is rounded to x's dtype, and the norm is of the rounded h: ``y = (h * r) *
    weight`` in fp32 with ``r = 1 / sqrt(mean(h^2) + eps)`` taken in fp64 and
    rounded to fp32.  ``out`` is y rounded to x's dtype, or with ``out_format`` y
    in that microscaled format (an MXTensor, D a multiple of 32), with no
    rounding in between.  Asynchronous on the current stream; records no
    gradients."""
    # one lookup per call: what depends on the operands' geometry alone (the
    # checks, the argument struct without addresses) is prepared once per key
    r, eps = residual, float(eps)
    key = (x.shape, x.stride(), x.dtype, x.device, weight.shape, weight.stride(), weight.dtype, weight.device, eps,
           out_format, x.data_ptr() & 15, weight.data_ptr() & 15,
           None if r is None else (r.shape, r.stride(), r.dtype, r.device, r.data_ptr() & 15))
    ent = _NORM_CALLS.get(key)
    if ent is None:
        ent = _prepare_norm(x, r, weight, eps, out_format)
        if len(_NORM_CALLS) >= 64:
            _NORM_CALLS.clear()
        _NORM_CALLS[key] = ent
    a = _lib.QikResidualRmsNormArgs.from_buffer_copy(ent.args)
    h = scales = None
    if ent.like:
        out = torch.empty_like(x)
        if r is not None:
            a.residual = r.data_ptr()
            h = torch.empty_like(x)
            a.sum = h.data_ptr()
        a.x, a.weight, a.out = x.data_ptr(), weight.data_ptr(), out.data_ptr()
    else:
        xs, rs, ws = (x, r, weight) if not ent.copy else _norm_copies(x, r, weight, ent.fmt)
        out = x.new_empty(ent.out_shape, dtype=ent.out_dtype)
        if r is not None:
            a.residual = rs.data_ptr()
            h = x.new_empty(x.shape)
            a.sum = h.data_ptr()
        if ent.fmt:
            scales = x.new_empty(ent.scales_shape, dtype=torch.uint8)
            a.scales = scales.data_ptr()
        a.x, a.weight, a.out = xs.data_ptr(), ws.data_ptr(), out.data_ptr()
    idx = ent.index
    if idx != torch._C._cuda_getDevice():
        with torch.cuda.device(idx):
            _lib.check(ent.fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx)), "qik_residual_rms_norm")
    else:
        st = ent.fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx))
        if st:
            _lib.check(st, "qik_residual_rms_norm")
    if scales is not None:
        out = MXTensor._make(out, scales, out_format, x.shape)
    return out if r is None else (out, h)


class _NormCall:
    """What one geometry of fused_residual_rms_norm needs at call time; no tensor."""

    __slots__ = ("args", "fn", "index", "fmt", "like", "copy", "out_shape", "out_dtype", "scales_shape")


# Prepared calls by the operands' geometry (shapes, strides, types, devices and
# alignments: see fused_residual_rms_norm).
_NORM_CALLS: dict = {}


def _prepare_norm(x, residual, weight, eps, out_format) -> _NormCall:
    fmt = _lib.MX_NONE if out_format is None else MX_FORMATS[_check_format(out_format)]
    if x.dtype not in _NORM_DTYPES:
        raise ValueError(f"x must be bf16, fp16 or fp32, got {x.dtype}")
    if x.dim() < 1:
        raise ValueError("x must have at least one dimension")
    if not x.is_cuda:
        raise ValueError("x must be a device tensor (the kernel runs on the GPU)")
    D = x.shape[-1]
    if not 1 <= D <= _MAX_NORM_WIDTH:
        raise ValueError(f"the last dimension must be 1 to {_MAX_NORM_WIDTH}, got {D}")
    if fmt:
        _check_width(D)
    if residual is not None and (residual.shape != x.shape or residual.dtype != x.dtype or residual.device != x.device):
        raise ValueError(f"residual must be {tuple(x.shape)} {x.dtype} on {x.device}, "
                         f"got {tuple(residual.shape)} {residual.dtype} on {residual.device}")
    if weight.shape != (D,) or weight.device != x.device:
        raise ValueError(f"weight must be [{D}] on {x.device}, got {tuple(weight.shape)} on {weight.device}")
    if weight.dtype != torch.float32 and weight.dtype != x.dtype:
        raise ValueError(f"weight must be fp32 or {x.dtype}, got {weight.dtype}")
    xs, rs, ws = _norm_copies(x, residual, weight, fmt)
    M = xs.shape[0]
    c = _NormCall()
    c.fn = _lib.load().qik_residual_rms_norm
    c.index, c.fmt = x.device.index, fmt
    # a view of an operand at the operand's own address needs no work per call
    c.copy = M > 0 and (xs.data_ptr() != x.data_ptr() or ws.data_ptr() != weight.data_ptr()
                        or (rs is not None and rs.data_ptr() != residual.data_ptr()))
    c.like = not fmt and not c.copy and x.is_contiguous()
    c.out_shape = _code_shape(x.shape, out_format) if fmt else x.shape
    c.out_dtype = _CODE_DTYPE[out_format] if fmt else x.dtype
    c.scales_shape = _scales_shape(M, D) if fmt else None
    c.args = _lib.QikResidualRmsNormArgs(
        _lib.ABI_VERSION, _NORM_DTYPES[x.dtype], fmt, _NORM_DTYPES[weight.dtype], None, None, None, None, None, None, M, D,
        _row_stride(xs), D if rs is None else _row_stride(rs), eps)
    return c


def _norm_copies(x, residual, weight, fmt: int):
    """The operands as rows in a layout that the kernel takes: copies where they have another."""
    w = weight
    if not w.is_contiguous() or (fmt and w.data_ptr() % 16 != 0):
        w = w.clone(memory_format=torch.contiguous_format)
    return _norm_rows(x, fmt), None if residual is None else _norm_rows(residual, fmt), w


def _norm_rows(t: torch.Tensor, fmt: int) -> torch.Tensor:
    """t as rows; a microscaled output reads them in 16-byte vectors, so rows at other addresses are copied."""
    t2 = _as_rows(t)
    if fmt and (t2.data_ptr() % 16 != 0 or (t2.shape[0] > 1 and t2.stride(0) * t2.element_size() % 16 != 0)):
        t2 = t2.clone(memory_format=torch.contiguous_format)
    return t2
