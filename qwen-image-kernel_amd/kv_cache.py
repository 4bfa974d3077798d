"""Contiguous prefix-KV slab, same attributes and layout as the reference.

``ContiguousKVCache`` / ``_LayerView`` keep the API of
``qwen_image_kernel/kv_cache.py:23-95``: one preallocated slab for all layers,
K ``[L, B, H, P_max, D]`` in the model dtype, V the same or fp8e4m3fn with one
fp32 scale per (layer, b, h), and ``lengths [L]`` int64 on the device.  Each
head's prefix tokens are dense (256 B rows of bf16 K, 128 B rows of fp8 V), and
``views()`` returns ``[B, P, H, D]`` strided views that the attention kernel
reads in place.

``store`` on a HIP device is one call of ``qik_slab_store_ws`` (include/qik_ops.h):
the transposed copy of K (and of a bf16 V) and, for an fp8 slab, the per-(b, h)
amax, scale and e4m3fn codes of V, bit-identical to the torch ops of
kv_cache.py:36-42 run on the same device, in two launches with a small
workspace that the cache keeps per (device, stream).  A slab on the CPU (the
reference's own CPU-runnable case) runs those torch ops.

Difference from the reference: the prefix length of each layer is also kept on
the host, so ``get()``/``views()`` do not synchronise the device
(the reference reads ``int(lengths[layer])``, kv_cache.py:49, 56).

``MXKVCache`` (no counterpart in the reference) is a slab with K and V in 4
bits, 272 bytes a token and head at D = 128 where the bf16 slab has 1024 and the
fp8-V one 768, with a length for each batch entry and tokens appended behind it
(include/qik_mx_attn.h).
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .attention import _kernel_layout
from .mx_slab import _DTYPES, HEAD_DIMS, MXSlab, load_args, slab_values

FP8_E4M3_MAX = 448.0


class _SlabLayer:
    """A layer whose store copies what it is given (a cache that keeps the tensors themselves is none)."""


class _LayerView(_SlabLayer):
    """Per-layer store/get interface compatible with the stock cache."""

    def __init__(self, cache: "ContiguousKVCache", layer: int):
        self._c = cache
        self._layer = layer

    def store(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v: [B, P, H, D] post-RoPE; V is quantised per (b, h) when the slab is fp8.

        Quantisation (kv_cache.py:36-42): scale = max(amax|v| / 448, 1e-12) in
        fp32, code = e4m3fn(clamp(v / scale, +-448)) with a true fp32 division
        and round-to-nearest-even.
        """
        c = self._c
        P = k.shape[1]
        if P > c.capacity:
            raise ValueError(f"prefix of {P} tokens exceeds the slab capacity {c.capacity}")
        if c.k_buf.is_cuda and P > 0 and k.shape[0] > 0 and k.shape[2] > 0:
            # the store's launch that copies K also writes lengths[layer] = P
            self._store_device(k, v, P)
        else:
            if c.k_buf.is_cuda:
                self._store_device(k, v, P)
            else:
                self._store_torch(k, v, P)
            # a fill kernel: assigning a Python int to one element is a
            # host-to-device copy, which a stream under graph capture rejects
            c.lengths[self._layer:self._layer + 1].fill_(P)
        c._host_lengths[self._layer] = P

    def _store_device(self, k: torch.Tensor, v: torch.Tensor, P: int) -> None:
        c = self._c
        kd = c.k_buf
        # inputs the kernels cannot read in place (a base off 16 bytes, odd
        # strides) go through contiguous copies; other dtypes or devices are
        # converted (into fresh tensors) by store_args
        if k.dim() == 4 and k.device == kd.device and k.dtype == kd.dtype:
            k = _kernel_layout(k)
        if v.dim() == 4 and v.device == kd.device and v.dtype == kd.dtype:
            v = _kernel_layout(v)
        a, keep, nbytes = self._cached_store_args(k, v, P)
        lib = _lib.load()
        idx = kd.device.index
        if idx != torch.cuda.current_device():
            with torch.cuda.device(kd.device):
                self._launch_store(lib, a, nbytes, idx)
        else:
            self._launch_store(lib, a, nbytes, idx)
        del keep

    def _launch_store(self, lib, a, nbytes: int, idx: int) -> None:
        handle = torch._C._cuda_getCurrentRawStream(idx)
        ws = self._c._workspace(idx, handle, nbytes)
        _lib.check(lib.qik_slab_store_ws(ctypes.byref(a), ws, nbytes, ctypes.c_void_p(handle)), "qik_slab_store_ws")

    def _cached_store_args(self, k: torch.Tensor, v: torch.Tensor, P: int):
        """store_args with the struct and its workspace size kept per geometry (layer, shapes, strides)."""
        c = self._c
        gkey = (self._layer, P, tuple(k.shape), k.stride(), v.stride(), k.dtype, v.dtype, k.device, v.device)
        hit = c._args_cache.get(gkey)
        if hit is None:
            a, keep = self.store_args(k, v, P)
            nbytes = ctypes.c_int64(0)
            with torch.cuda.device(c.k_buf.device):
                _lib.check(_lib.load().qik_slab_store_workspace_size(ctypes.byref(a), ctypes.byref(nbytes)),
                           "qik_slab_store_workspace_size")
            if len(c._args_cache) >= 4 * max(c.num_layers, 1):
                c._args_cache.clear()
            # only inputs already in the slab's dtype, device and a unit D stride are
            # launched from the cached struct; others are converted per call
            if keep[0] is k and keep[1] is v:
                c._args_cache[gkey] = (_lib.QikSlabStoreArgs.from_buffer_copy(a), nbytes.value)
            return a, keep, nbytes.value
        a = _lib.QikSlabStoreArgs.from_buffer_copy(hit[0])
        a.k = k.data_ptr()
        a.v = v.data_ptr()
        return a, (k, v), hit[1]

    def store_args(self, k: torch.Tensor, v: torch.Tensor, P: int):
        """(qik_slab_store argument struct, tensors it points into) for a device slab."""
        c = self._c
        if k.shape != v.shape or k.dim() != 4 or tuple(k.shape[2:]) != tuple(c.k_buf.shape[2:3] + c.k_buf.shape[4:]):
            raise ValueError(f"k, v must be [B, P, H, D] matching the slab, got {tuple(k.shape)}, {tuple(v.shape)}")
        if k.shape[0] != c.batch_size:
            raise ValueError(f"batch {k.shape[0]} != slab batch {c.batch_size}")
        k = k.to(device=c.k_buf.device, dtype=c.k_buf.dtype)
        v = v.to(device=c.k_buf.device, dtype=c.k_buf.dtype)
        if k.stride(-1) != 1:
            k = k.contiguous()
        if v.stride(-1) != 1:
            v = v.contiguous()
        kd = c.k_buf[self._layer]
        vd = c.v_buf[self._layer]
        a = _lib.QikSlabStoreArgs()
        a.abi_version = _lib.ABI_VERSION
        a.dtype = _lib.DTYPE_BF16 if c.k_buf.dtype == torch.bfloat16 else _lib.DTYPE_FP16
        a.v_fp8 = 1 if c.v_fp8 else 0
        a.k = k.data_ptr()
        a.v = v.data_ptr()
        a.k_dst = kd.data_ptr()
        a.v_dst = vd.data_ptr()
        a.v_scale = c.v_scale[self._layer].data_ptr() if c.v_fp8 else None
        a.B, a.P, a.H, a.D = k.shape[0], P, k.shape[2], k.shape[3]
        a.stride_k = _lib._i64x3(k.stride(0), k.stride(1), k.stride(2))
        a.stride_v = _lib._i64x3(v.stride(0), v.stride(1), v.stride(2))
        a.stride_k_dst = _lib._i64x3(kd.stride(0), kd.stride(1), kd.stride(2))
        a.stride_v_dst = _lib._i64x3(vd.stride(0), vd.stride(1), vd.stride(2))
        a.length_dst = c.lengths.data_ptr() + c.lengths.element_size() * self._layer
        return a, (k, v)

    def _store_torch(self, k: torch.Tensor, v: torch.Tensor, P: int) -> None:
        c = self._c
        c.k_buf[self._layer, :, :, :P, :].copy_(k.transpose(1, 2))
        if c.v_fp8:
            vt = v.transpose(1, 2).float()
            scale = vt.abs().amax(dim=(2, 3)).float() / FP8_E4M3_MAX
            scale = scale.clamp_min(1e-12)
            vq = (vt / scale[:, :, None, None]).clamp(-FP8_E4M3_MAX, FP8_E4M3_MAX).to(torch.float8_e4m3fn)
            c.v_buf[self._layer, :, :, :P, :].copy_(vq)
            c.v_scale[self._layer].copy_(scale)
        else:
            c.v_buf[self._layer, :, :, :P, :].copy_(v.transpose(1, 2))

    def get(self):
        """(k, v) as [B, P, H, D] strided views."""
        c = self._c
        P = c._host_lengths[self._layer]
        return self._prefix(c.k_buf, P), self._prefix(c.v_buf, P)

    def _prefix(self, buf: torch.Tensor, P: int) -> torch.Tensor:
        """``buf[layer, :, :, :P, :].transpose(1, 2)`` in one view op (1.7 us of host time for
        the chain's 5.6, of which a store and its views have two)."""
        sl, sb, sh, sp, sd = buf.stride()
        n, B, H, cap, D = buf.shape
        i = self._layer
        if not -n <= i < n:  # as_strided checks the storage only, and takes no negative index
            raise IndexError(f"layer {i} is out of range for a slab of {n} layers")
        return buf.as_strided((B, P if P < cap else cap, H, D), (sb, sp, sh, sd),
                              buf.storage_offset() + (i if i >= 0 else i + n) * sl)

    def views(self):
        """(k, v, v_scale_or_None) for block_causal_flash_attention."""
        k, v = self.get()
        return k, v, (self._c.v_scale[self._layer] if self._c.v_fp8 else None)


class ContiguousKVCache:
    """Single-slab prefix KV cache: one allocation per buffer for all layers.

    K layout: [L, B, H, P_max, D] (dtype).  V layout: same (dtype) or fp8e4m3fn
    with per-head fp32 scales [L, B, H].  Per prefix token across 32 layers at
    H*D = 3072: K+V bf16 = 384 KB, K bf16 + V fp8 = 288 KB.
    """

    def __init__(
        self,
        num_layers: int,
        batch: int,
        prefix_max: int,
        num_heads: int,
        head_dim: int,
        v_fp8: bool = False,
        device: torch.device | str = "cuda",
        dtype: torch.dtype = torch.bfloat16,
    ):
        if torch.device(device).type != "cpu" and dtype not in (torch.bfloat16, torch.float16):
            # the device store and the attention kernel read 2-byte K/V
            # elements; a CPU slab (stored by torch's ops, as the reference's
            # cache does) takes any dtype
            raise ValueError(f"a device slab's dtype must be bfloat16 or float16, got {dtype}")
        self.v_fp8 = v_fp8
        self.num_layers = num_layers
        self.capacity = prefix_max
        self.batch_size = batch
        self.k_buf = torch.empty(num_layers, batch, num_heads, prefix_max, head_dim, dtype=dtype, device=device)
        v_dtype = torch.float8_e4m3fn if v_fp8 else dtype
        self.v_buf = torch.empty(num_layers, batch, num_heads, prefix_max, head_dim, dtype=v_dtype, device=device)
        self.v_scale = torch.empty(num_layers, batch, num_heads, dtype=torch.float32, device=device)
        self.lengths = torch.zeros(num_layers, dtype=torch.int64, device=device)
        self._host_lengths = [0] * num_layers
        self._ws: dict = {}   # (device index, stream) -> store workspace (fp8 slab)
        self._args_cache: dict = {}  # store geometry -> (argument struct, workspace bytes)
        self.layers = [_LayerView(self, i) for i in range(num_layers)]

    def _workspace(self, device_index: int, stream: int, nbytes: int):
        """Device pointer of this cache's store workspace for `stream` (None when none is needed).

        Its contents never need clearing: every store writes what it reads.
        Stores on different streams get different workspaces.
        """
        if nbytes <= 0:
            return None
        key = (device_index, stream)
        ws = self._ws.get(key)
        if ws is None or ws.numel() < nbytes:
            if ws is None and len(self._ws) >= 16:
                self._ws.pop(next(iter(self._ws)))
            ws = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", device_index))
            self._ws[key] = ws
        return ws.data_ptr()

    def get_layer(self, i: int) -> _LayerView:
        return self.layers[i]


class _MXLayerView(_SlabLayer):
    """One layer of an ``MXKVCache``: store / append / get / views."""

    def __init__(self, cache: "MXKVCache", layer: int):
        self._c = cache
        self._layer = layer
        self._lengths = cache.lengths[layer]
        self._index = self._lengths.device.index
        self._calls: dict = {}  # store geometry -> (argument struct, operands that need a copy)
        self._full = None       # (k, v MXSlab views of the whole capacity, argument struct of get)
        self._rows, self._views = -1, None  # what views() gave last, and for how many rows

    def store(self, k: torch.Tensor, v: torch.Tensor) -> None:
        """k, v ``[B, P, H, D]`` post-RoPE become rows 0 .. P - 1 of every batch entry, whose length is then P."""
        c = self._c
        P = k.shape[1] if k.dim() == 4 else 0
        call = self._call(k, v)
        if P > c.capacity:
            raise ValueError(f"prefix of {P} tokens exceeds the slab capacity {c.capacity}")
        if P == 0 or call is None:
            c._write_lengths(self._lengths.fill_, P)
        else:
            self._launch(call, k, v, None, False)
        self._note(P, True, P)

    def append(self, k: torch.Tensor, v: torch.Tensor, at: torch.Tensor | int | None = None) -> None:
        """k, v ``[B, S, H, D]`` become rows ``at[b]`` .. ``at[b] + S - 1`` of batch entry b, whose length is then
        ``at[b] + S``, clamped to 0 .. capacity.

        ``at``: None (behind each entry's present length), an int, or an int32
        ``[B]`` device tensor, which must not overlap the layer's ``lengths``
        unless it is them.  Rows past the capacity are not written; where the
        host knows the lengths (they came from ``store``, or from appends with
        None or an int, no store or append of the layer was ever captured into a
        graph, and the program never wrote into ``lengths`` itself) that is a
        ValueError instead."""
        c, i, lengths = self._c, self._layer, self._lengths
        S = k.shape[1] if k.dim() == 4 else 0
        call = self._call(k, v)
        grow = True
        if isinstance(at, torch.Tensor):
            if at.shape != lengths.shape or at.dtype != torch.int32 or at.device != lengths.device:
                raise ValueError(f"at must be int32 [{c.batch_size}] on {lengths.device}, "
                                 f"got {at.dtype} {tuple(at.shape)} on {at.device}")
            first, here = lengths.data_ptr(), at.data_ptr()
            grow = here == first and at.is_contiguous()
            if not grow and (not at.is_contiguous() or abs(here - first) < 4 * c.batch_size):
                at = at.clone(memory_format=torch.contiguous_format)
            n, exact, most = c.capacity, False, c.capacity
        elif at is not None:
            at = int(at)
            if at < 0 or at + S > c.capacity:
                raise ValueError(f"{S} tokens at {at} exceed the slab capacity {c.capacity}")
            c._write_lengths(lengths.fill_, at)
            n, exact, most, at = at + S, True, at + S, lengths
        else:
            n, exact, most, at = c._host_lengths[i], c._exact[i] and not c._lengths_written(), c.capacity, lengths
            if exact and n + S > c.capacity:
                raise ValueError(f"{S} tokens behind {n} exceed the slab capacity {c.capacity}")
            n = min(n + S, c.capacity)
        if call is not None:
            self._launch(call, k, v, at, grow)
        elif S or not grow:
            c._write_lengths(lengths.copy_, (at + S).clamp_(0, c.capacity))
        self._note(n, exact, most)

    def _note(self, n: int, exact: bool, most: int) -> None:
        """Keep what the host knows after a call: no entry is longer than n, and with `exact` each is that long; `most`: how
        long replays of the call may leave one."""
        c, i = self._c, self._layer
        if self._capturing():
            # nothing has run yet, and a replay comes when the program likes, unseen by the host
            n, c._captured[i] = c._host_lengths[i], max(most, c._captured[i] or 0)
        if c._captured[i] is not None:
            n, exact = max(n, c._captured[i]), False
        c._host_lengths[i], c._exact[i] = n, exact

    def _capturing(self) -> bool:
        if self._index == torch._C._cuda_getDevice():
            return torch.cuda.is_current_stream_capturing()
        with torch.cuda.device(self._index):
            return torch.cuda.is_current_stream_capturing()

    def _call(self, k: torch.Tensor, v: torch.Tensor):
        """The prepared store of operands like these; None where there are no rows."""
        key = (k.shape, k.stride(), k.dtype, k.device, k.data_ptr() & 15,
               v.shape, v.stride(), v.dtype, v.device, v.data_ptr() & 15)
        hit = self._calls.get(key)
        if hit is None:
            hit = self._prepare(k, v)
            if len(self._calls) >= 8:
                self._calls.clear()
            self._calls[key] = hit
        return hit[0]

    def _prepare(self, k: torch.Tensor, v: torch.Tensor):
        c = self._c
        H, D = c.num_heads, c.head_dim
        if k.shape != v.shape or k.dim() != 4 or tuple(k.shape[2:]) != (H, D):
            raise ValueError(f"k, v must be [B, P, {H}, {D}] matching the slab, got {tuple(k.shape)}, {tuple(v.shape)}")
        if k.shape[0] != c.batch_size:
            raise ValueError(f"batch {k.shape[0]} != slab batch {c.batch_size}")
        if k.numel() == 0:
            return (None,)
        laid = [self._readable(t) for t in (k, v)]
        full = self._slabs()
        a = _lib.QikMxSlabStoreArgs(_lib.ABI_VERSION, _DTYPES[c.dtype], None, None, full[0].struct(), full[1].struct(),
                                    None, self._lengths.data_ptr(), None, *k.shape, c.capacity,
                                    *(_lib._i64x3(*t.stride()[:3]) for t in laid))
        return ((a, laid[0] is not k or laid[1] is not v),)

    def _readable(self, t: torch.Tensor) -> torch.Tensor:
        """t in the cache's dtype, on its device, in a layout that the kernel reads in place."""
        t = t.to(device=self._lengths.device, dtype=self._c.dtype)
        return _kernel_layout(t if t.stride(-1) == 1 else t.contiguous())

    def _launch(self, call, k, v, at, grow: bool) -> None:
        a, copy = call
        if copy:
            k, v = self._readable(k), self._readable(v)
        a = _lib.QikMxSlabStoreArgs.from_buffer_copy(a)
        a.k, a.v = k.data_ptr(), v.data_ptr()
        if at is not None:
            a.at = at.data_ptr()
            if grow:
                a.arrivals = self._c._arrivals.data_ptr() + 4 * self._layer
        idx = self._index
        fn = _lib.load().qik_mx_slab_store
        if idx != torch._C._cuda_getDevice():
            with torch.cuda.device(idx):
                st = fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx))
        else:
            st = fn(ctypes.byref(a), torch._C._cuda_getCurrentRawStream(idx))
        if st:
            _lib.check(st, "qik_mx_slab_store")

    def _slabs(self):
        if self._full is None:
            c, i = self._c, self._layer
            k, v = (MXSlab(codes[i].transpose(1, 2), scales[i].transpose(1, 2), self._lengths)
                    for codes, scales in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales)))
            self._full = (k, v, load_args(k, v, c.dtype))
        return self._full

    def get(self):
        """(k, v): the values of the layer's rows, ``[B, P, H, D]`` in the cache's dtype, zeros behind each entry's
        length; P as in ``views()``."""
        c = self._c
        args = self._slabs()[2]
        return slab_values(args, self._lengths, (c.batch_size, c._host_lengths[self._layer], c.num_heads, c.head_dim), c.dtype)

    def views(self, P: int | None = None):
        """(k, v, None) for block_causal_flash_attention: ``MXSlab`` views of the first P rows, with the entries'
        lengths.  P by default is the longest length as far as the host knows it (the capacity after an append whose
        places only the device knows, and from the first captured append on, whose replays the host does not see); fewer
        rows plan a call for fewer keys, and leave out what lies behind them."""
        c = self._c
        if P is None:
            P = c._host_lengths[self._layer]
        elif not 0 <= P <= c.capacity:
            raise ValueError(f"{P} rows of a slab of {c.capacity}")
        if P != self._rows:
            k, v, _ = self._slabs()
            self._rows, self._views = P, (k.first(P), v.first(P), None)
        return self._views


class MXKVCache:
    """Single-slab prefix KV cache with K and V in MXFP4: one allocation for all layers' codes and scales.

    Codes ``k_codes``, ``v_codes`` uint8 ``[L, B, H, P_max, D / 2]`` and block
    scales ``k_scales``, ``v_scales`` uint8 ``[L, B, H, P_max, D / 32]``, the
    format of ``quantize_mx`` (an infinity or NaN makes its block NaN);
    ``lengths`` int32 ``[L, B]``, kept on the device by ``store`` and ``append``.  A
    program may lower lengths itself (an entry that ends and starts anew), by
    torch's in-place operations; they grow through ``append`` alone.  ``append``
    then no longer says when an entry is full.  ``num_heads`` counts the keys'
    heads, which may be fewer than the queries'.  HIP devices only."""

    def __init__(
        self,
        num_layers: int,
        batch: int,
        prefix_max: int,
        num_heads: int,
        head_dim: int,
        device: torch.device | str = "cuda",
        dtype: torch.dtype = torch.bfloat16,
    ):
        if torch.device(device).type != "cuda":
            raise ValueError(f"a 4-bit slab lives on a HIP device, got {device}")
        if dtype not in _DTYPES:
            raise ValueError(f"the model's dtype must be bfloat16 or float16, got {dtype}")
        if head_dim not in HEAD_DIMS:
            raise ValueError(f"the head dim must be one of {HEAD_DIMS}, got {head_dim}")
        self.num_layers, self.batch_size, self.capacity = num_layers, batch, prefix_max
        self.num_heads, self.head_dim, self.dtype = num_heads, head_dim, dtype
        shape = (num_layers, batch, num_heads, prefix_max)
        rows = num_layers * batch * num_heads * prefix_max
        widths = (head_dim // 2, head_dim // 2, head_dim // 32, head_dim // 32)
        # (the codes first: their part is a multiple of 16 bytes long, the scales' of what their rows need)
        parts = torch.zeros(rows * sum(widths), dtype=torch.uint8, device=device).split([rows * w for w in widths])
        self.k_codes, self.v_codes, self.k_scales, self.v_scales = (t.view(*shape, w) for t, w in zip(parts, widths))
        with torch.inference_mode(False):  # (an inference tensor does not say whether it was written to)
            counts = torch.zeros(num_layers * (batch + 1), dtype=torch.int32, device=device)
        self.lengths = counts[:num_layers * batch].view(num_layers, batch)
        self._arrivals = counts[num_layers * batch:]
        self._host_lengths = [0] * num_layers   # no entry of the layer is longer
        self._exact = [True] * num_layers       # ... and every one is that long, if the program changed none
        self._captured: list = [None] * num_layers  # the longest that replays of captured calls may leave, None without such
        # `lengths` counts torch's writes into it, whatever view they go through; the kernels' are no such
        self._version, self._program_writes = self.lengths._version, False
        self.layers = [_MXLayerView(self, i) for i in range(num_layers)]

    def _lengths_written(self) -> bool:
        """Whether the program ever wrote into ``lengths`` itself."""
        if self.lengths._version != self._version:
            self._program_writes = True
        return self._program_writes

    def _write_lengths(self, write, value) -> None:
        """A write of the cache's own by torch."""
        self._lengths_written()
        write(value)
        self._version = self.lengths._version

    def get_layer(self, i: int) -> _MXLayerView:
        return self.layers[i]
