"""Attention over a 4-bit slab and fresh keys: ``block_causal_flash_attention`` with ``MXSlab`` caches.

Row q of batch entry b attends key kv iff kv <= L[b, q] (every key where L is None,
or with ``uniform_full`` and no mask) and key_valid[b, kv] says so; the slab's rows are
keys 0 .. P - 1, of which entry b has ``lengths[b]``, and fresh key n is key P +
n.  Rows that attend nothing are zeros.  Softmax statistics and sums are fp32,
the probabilities are rounded to the query's type for the second product, as in
the attention over a 16-bit slab.  Keys that key_valid hides and slab rows
behind ``lengths`` may hold anything; a value row that only L hides from a row
has to be finite.  Few query rows run a kernel that splits the keys over the
device (include/qik_mx_attn.h).  Records no gradients.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from . import attention as _attn
from .mx_slab import _DTYPES, MXSlab

__all__ = ["mx_slab_attention"]


class _Call:
    """What one geometry of mx_slab_attention needs at call time; no tensor."""

    __slots__ = ("args", "ws_bytes", "index", "device", "copy", "slab_copy", "L", "valid", "shape", "like")

    # args: without the number of slab rows; ws_bytes: by that number


# Prepared calls by the operands' geometry (shapes, strides, types, devices and alignments), of which
# the number of slab rows is no part: a serving step's call has a row more than the last one's.
_CALLS: dict = {}
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


def mx_slab_attention(query, key, value, prefix_lengths, key_valid, cache_k, cache_v, uniform_full) -> torch.Tensor:
    if not isinstance(cache_k, MXSlab) or not isinstance(cache_v, MXSlab):
        raise ValueError("cache_k and cache_v must both be MXSlab, or neither")
    uniform = prefix_lengths is None or (uniform_full and key_valid is None)
    L = None if uniform else prefix_lengths
    q, k, v = query.data_ptr(), key.data_ptr(), value.data_ptr()
    gkey = (query.shape, query.stride(), query.dtype, query.device, key.shape, key.stride(), key.dtype, key.device,
            value.shape, value.stride(), value.dtype, value.device, (q & 15, k & 15, v & 15) if (q | k | v) & 15 else 0,
            cache_k._layout, cache_v._layout, uniform,
            None if L is None else (L.shape, L.stride(), L.dtype, L.device),
            None if key_valid is None else (key_valid.shape, key_valid.stride(), key_valid.dtype, key_valid.device))
    c = _CALLS.get(gkey)
    if c is None:
        c = _prepare(query, key, value, L, key_valid, cache_k, cache_v, uniform)
        if len(_CALLS) >= 256:
            _CALLS.clear()
        _CALLS[gkey] = c
    P = cache_k._shape[1]
    ws_bytes = c.ws_bytes.get(P)
    if ws_bytes is None or cache_v._shape[1] != P:
        ws_bytes = _rows(c, P, query, key, key_valid, cache_v)
    out = torch.empty_like(query) if c.like else query.new_empty(c.shape)
    if c.args is None:
        return out
    if c.copy is not None:
        query, key, value = (t.clone(memory_format=torch.contiguous_format) if f else t
                             for f, t in zip(c.copy, (query, key, value)))
        q, k, v = query.data_ptr(), key.data_ptr(), value.data_ptr()
    x = _lib.QikMxAttnArgs.from_buffer_copy(c.args)
    if c.slab_copy:  # (dense copies, whose strides go by the rows)
        cache_k, cache_v = cache_k.readable(), cache_v.readable()
        x.k_slab, x.v_slab = cache_k.struct(), cache_v.struct()
    a = x.a
    a.P = P
    a.q, a.k_new, a.v_new, a.out = q, k, v, out.data_ptr()
    if L is not None:
        if c.L:
            L = _attn._int32(L)
        a.prefix_lengths = L.data_ptr()
    if key_valid is not None:
        key_valid = _valid_bytes(key_valid, c.valid)
        a.key_valid = key_valid.data_ptr()
    s = x.k_slab
    s.codes, s.scales = cache_k._codes.data_ptr(), cache_k._scales.data_ptr()
    s = x.v_slab
    s.codes, s.scales = cache_v._codes.data_ptr(), cache_v._scales.data_ptr()
    if cache_k._lengths is not None:
        x.lengths = cache_k._lengths.data_ptr()
    if c.index != _current_device():
        with torch.cuda.device(c.index):
            st = _launch(c, x, ws_bytes)
    else:
        st = _launch(c, x, ws_bytes)
    if st:
        _lib.check(st, "qik_mx_attn_fwd")
    return out


def _launch(c: _Call, x: _lib.QikMxAttnArgs, ws_bytes: int) -> int:
    handle = _raw_stream(c.index)
    ws = _attn._workspace(c.device, handle, ws_bytes).data_ptr() if ws_bytes else None
    return _lib.load().qik_mx_attn_fwd(ctypes.byref(x), ws, ws_bytes, handle)


def _rows(c: _Call, P: int, query, key, key_valid, cache_v) -> int:
    """What depends on the number of slab rows, checked; the workspace's bytes."""
    if cache_v.shape[1] != P:
        raise ValueError(f"cache_k has {P} rows, cache_v {cache_v.shape[1]}")
    if query.numel() == 0:
        c.ws_bytes[P] = 0
        return 0
    if key_valid is not None:
        assert key_valid.shape[1] >= P + key.shape[1], "key_valid must be [B, KV_TOTAL]"
    x = _lib.QikMxAttnArgs.from_buffer_copy(c.args)
    x.a.P = P
    nbytes = ctypes.c_int64(0)
    with torch.cuda.device(c.device):
        _lib.check(_lib.load().qik_mx_attn_workspace_size(ctypes.byref(x), ctypes.byref(nbytes)), "qik_mx_attn_fwd")
    if len(c.ws_bytes) >= 64:
        c.ws_bytes.clear()
    c.ws_bytes[P] = nbytes.value
    return nbytes.value


def _valid_bytes(key_valid: torch.Tensor, how: str) -> torch.Tensor:
    """key_valid as bytes, zero for a hidden key, with a dense last dimension."""
    return key_valid.view(torch.uint8) if how == "view" else key_valid if how == "" else (key_valid != 0).contiguous().view(torch.uint8)


def _prepare(query, key, value, L, key_valid, cache_k, cache_v, uniform) -> _Call:
    assert query.dtype in _DTYPES, "fp16/bf16 only"
    assert key.dtype == query.dtype and value.dtype == query.dtype, "q/k/v dtypes must match"
    for name, t in (("query", query), ("key", key), ("value", value)):
        _attn._check_rows(name, t)
    B, SQ, H, D = query.shape
    Bk, SN, HKV, Dk = key.shape
    if value.shape != key.shape:
        raise ValueError(f"key is {tuple(key.shape)}, value {tuple(value.shape)}")
    if Bk != B or Dk != D:
        raise ValueError(f"key must be [{B}, SN, HKV, {D}], got {tuple(key.shape)}")
    if HKV == 0 and H != 0 or (HKV and H % HKV != 0):
        raise ValueError(f"{H} query heads do not share {HKV} key heads evenly")
    for name, t in (("cache_k", cache_k), ("cache_v", cache_v)):
        if t.shape[0] != B or tuple(t.shape[2:]) != (HKV, D):
            raise ValueError(f"{name} must be [{B}, P, {HKV}, {D}], got {tuple(t.shape)}")
    if (cache_k.lengths is None) != (cache_v.lengths is None):
        raise ValueError("cache_k and cache_v must both have lengths, or neither")
    dev = query.device
    for name, t in (("key", key), ("value", value), ("cache_k", cache_k), ("cache_v", cache_v)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, query on {dev}")
    c = _Call()
    c.index, c.device = dev.index, dev
    c.shape = tuple(query.shape)
    c.like = torch.empty_like(query, device="meta").is_contiguous()
    c.args, c.ws_bytes, c.copy, c.slab_copy, c.L, c.valid = None, {}, None, False, False, ""
    if query.numel() == 0:
        return c
    x = _lib.QikMxAttnArgs()
    a = x.a
    stride_L = 0
    if not uniform:
        _attn._check_aux("prefix_lengths", L, dev)
        if L.dim() == 2:
            assert L.shape[0] in (1, B) and L.shape[1] == SQ, "prefix_lengths must be [SQ] or [B, SQ]"
            stride_L = SQ if L.shape[0] > 1 else 0
        else:
            assert L.dim() == 1 and L.numel() >= SQ, "prefix_lengths must be [SQ] or [B, SQ]"
        c.L = L.dtype != torch.int32 or not L.is_contiguous()
        a.prefix_lengths = L.data_ptr()
    flags = _lib.UNIFORM_L if uniform else 0
    if cache_k.shape[1] > 0:
        flags |= _lib.HAS_CACHE
    if key_valid is not None:
        _attn._check_aux("key_valid", key_valid, dev)
        assert key_valid.dim() == 2, "key_valid must be [B, KV_TOTAL]"
        if key_valid.shape[0] not in (1, B):
            raise ValueError(f"key_valid batch dim must be 1 or B={B}, got {key_valid.shape[0]}")
        flags |= _lib.HAS_KEY_VALID
        dense = key_valid.shape[1] <= 1 or key_valid.stride(1) == 1
        c.valid = "view" if dense and key_valid.dtype == torch.bool else "" if dense and key_valid.dtype == torch.uint8 else "test"
        kb = _valid_bytes(key_valid, c.valid)
        a.key_valid = kb.data_ptr()
        a.stride_valid_b = kb.stride(0) if key_valid.shape[0] > 1 else 0
    # operands that the kernel cannot read in place go through dense copies, at each call
    laid = [_attn._kernel_layout(t) for t in (query, key, value)]
    copies = tuple(u is not t for u, t in zip(laid, (query, key, value)))
    c.copy = copies if any(copies) else None
    slabs = [t.readable() for t in (cache_k, cache_v)]
    c.slab_copy = slabs[0] is not cache_k or slabs[1] is not cache_v
    a.abi_version, a.dtype, a.flags = _lib.ABI_VERSION, _DTYPES[query.dtype], flags
    a.q, a.k_new, a.v_new = (t.data_ptr() for t in laid)
    a.out = laid[0].data_ptr()
    a.B, a.SQ, a.SN, a.H, a.D = B, SQ, SN, H, D
    a.stride_q = _lib._i64x3(*laid[0].stride()[:3])
    a.stride_k_new = _lib._i64x3(*laid[1].stride()[:3])
    a.stride_v_new = _lib._i64x3(*laid[2].stride()[:3])
    a.stride_out = _lib._i64x3(SQ * H * D, H * D, D)
    a.sm_scale = float(D) ** -0.5
    x.k_slab, x.v_slab = (t.struct() for t in slabs)
    x.HKV, x.stride_lengths_b = HKV, stride_L
    if cache_k.lengths is not None:  # (the plan goes by whether there are lengths)
        x.lengths = cache_k.lengths.data_ptr()
    c.args = x
    return c
