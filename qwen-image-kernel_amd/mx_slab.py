"""Rows of a 4-bit K or V slab as the attention reads them.

``MXSlab`` is what ``MXKVCache`` layers hand to ``block_causal_flash_attention``
in the place of a cache tensor: the codes and block scales of ``[B, P, H, D]``
rows in MXFP4 (blocks of 32 along D, the format of ``quantize_mx``), as strided
views, and optionally how many of the P rows each batch entry has.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib

__all__ = ["MXSlab"]

HEAD_DIMS = (32, 64, 128, 256)
_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}


class MXSlab:
    """Rows ``[B, P, H, D]`` of a slab in 4 bits.

    ``codes`` uint8 ``[B, P, H, D / 2]`` (two elements to a byte, the even one in
    the low half) and ``scales`` uint8 ``[B, P, H, D / 32]`` (E8M0), any strides
    with the last dimension dense; a layout that the kernels cannot read in
    place is copied at each call.  ``lengths`` int32 ``[B]`` on the same device:
    rows from ``lengths[b]`` on are not part of entry b (None: all P are); the
    two slabs of a call have the same (K's are read)."""

    __slots__ = ("_codes", "_scales", "_lengths", "_shape", "_layout")

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, lengths: torch.Tensor | None = None):
        for name, t in (("codes", codes), ("scales", scales)):
            if t.dim() != 4 or t.dtype != torch.uint8:
                raise ValueError(f"{name} must be uint8 [B, P, H, ...], got {t.dtype} {tuple(t.shape)}")
        D = codes.shape[-1] * 2
        if D not in HEAD_DIMS:
            raise ValueError(f"the head dim must be one of {HEAD_DIMS}, got {D}")
        if tuple(scales.shape) != (*codes.shape[:3], D // 32):
            raise ValueError(f"scales must be {(*codes.shape[:3], D // 32)}, got {tuple(scales.shape)}")
        if scales.device != codes.device:
            raise ValueError(f"codes are on {codes.device}, scales on {scales.device}")
        if lengths is not None:
            if tuple(lengths.shape) != (codes.shape[0],) or lengths.dtype != torch.int32:
                raise ValueError(f"lengths must be int32 [{codes.shape[0]}], got {lengths.dtype} {tuple(lengths.shape)}")
            if lengths.device != codes.device:
                raise ValueError(f"codes are on {codes.device}, lengths on {lengths.device}")
            if not lengths.is_contiguous():
                raise ValueError("lengths must be contiguous")
        self._codes, self._scales, self._lengths = codes, scales, lengths
        self._shape = torch.Size((*codes.shape[:3], D))
        # what a prepared call depends on, beside the number of rows
        B, P, H, _ = codes.shape
        self._layout = (codes.stride(), scales.stride(), codes.data_ptr() % 16, scales.data_ptr() % 8, lengths is None,
                        B, H, D, codes.device, min(P, 2))

    def first(self, P: int) -> "MXSlab":
        """The slab's first P rows: the same memory and lengths, no tensor operation."""
        s = MXSlab.__new__(MXSlab)
        s._codes, s._scales, s._lengths = self._codes, self._scales, self._lengths
        B, own, H, D = self._shape
        if not 0 <= P <= own:
            raise ValueError(f"{P} rows of a slab of {own}")
        s._shape = torch.Size((B, P, H, D))
        few = min(P, 2)
        s._layout = self._layout if self._layout[-1] == few else (*self._layout[:-1], few)
        return s

    @property
    def codes(self) -> torch.Tensor:
        return self._codes[:, :self._shape[1]]

    @property
    def scales(self) -> torch.Tensor:
        return self._scales[:, :self._shape[1]]

    @property
    def lengths(self) -> torch.Tensor | None:
        return self._lengths

    @property
    def shape(self) -> torch.Size:
        return self._shape

    @property
    def device(self) -> torch.device:
        return self._codes.device

    def in_place(self) -> bool:
        """Whether the kernels read this layout as it is (include/qik_mx_attn.h)."""
        B, P, H, D = self._shape
        (cb, cp, ch, cd), (eb, ep, eh, ed), cbase, ebase = self._layout[:4]
        n = D // 32
        return (cd == 1 and (ed == 1 or n == 1) and cbase == 0 and ebase % n == 0
                and (B == 1 or (cb % 16 == 0 and eb % n == 0)) and (H == 1 or (ch % 16 == 0 and eh % n == 0))
                and (P == 1 or (cp % 16 == 0 and ep % n == 0 and cp >= D // 2 and ep >= n)))

    def readable(self) -> "MXSlab":
        """This slab, or a dense copy of it where the kernels cannot read its layout in place."""
        if self.in_place():
            return self
        return MXSlab(*(t.clone(memory_format=torch.contiguous_format) for t in (self.codes, self.scales)), self._lengths)

    def struct(self) -> _lib.QikMxSlab:
        """The argument struct of a slab that is ``in_place``."""
        c, e = self._codes, self._scales
        return _lib.QikMxSlab(c.data_ptr(), e.data_ptr(), _lib._i64x3(*c.stride()[:3]), _lib._i64x3(*e.stride()[:3]))

    def __repr__(self) -> str:
        return f"MXSlab({tuple(self._shape)}, lengths={self._lengths is not None}, device={str(self.device)!r})"


def load_args(k: MXSlab, v: MXSlab, dtype: torch.dtype) -> _lib.QikMxSlabLoadArgs:
    """The argument struct of ``slab_values``, without the outputs' addresses and the number of rows."""
    if dtype not in _DTYPES:
        raise ValueError(f"dtype must be bf16 or fp16, got {dtype}")
    if not k.codes.is_cuda:
        raise ValueError("a slab is read on a HIP device")
    return _lib.QikMxSlabLoadArgs(_lib.ABI_VERSION, _DTYPES[dtype], k.struct(), v.struct(),
                                  None if k.lengths is None else k.lengths.data_ptr(), None, None, *k.shape)


def slab_values(args: _lib.QikMxSlabLoadArgs, like: torch.Tensor, shape, dtype) -> tuple[torch.Tensor, torch.Tensor]:
    """The values of both slabs' rows, ``[B, P, H, D]`` in dtype on like's device, zeros behind the lengths."""
    a = _lib.QikMxSlabLoadArgs.from_buffer_copy(args)
    a.P = shape[1]
    k, v = like.new_empty(shape, dtype=dtype), like.new_empty(shape, dtype=dtype)
    a.k, a.v = k.data_ptr(), v.data_ptr()
    idx = like.device.index
    fn = _lib.load().qik_mx_slab_load
    if idx != torch._C._cuda_getDevice():
        with torch.cuda.device(idx):
            st = fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx))
    else:
        st = fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx))
    if st:
        _lib.check(st, "qik_mx_slab_load")
    return k, v
