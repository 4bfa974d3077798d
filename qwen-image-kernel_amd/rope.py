"""Rotary positions on several axes (time, height, width), with the RMSNorm of Q and K.

``AxialRope`` holds a step's positions and the frequencies of the pairs; it
takes the place of the complex table in ``fused_rms_norm_rope`` and in the
processor's ``rotary_emb``, and ``fused_qk_norm_rope`` is the call for a layer's Q
and K together.  The angles are computed on the device as they are needed, D / 2
a token for all heads of Q and K (include/qik_rope.h): position times frequency
and its fraction of a turn in fp64, sine and cosine in fp32.  The norm and the
rotation are fp32 and the result is rounded once, where the call with a table
rounds between them as well.  These calls record gradients (backward; a
forward-mode derivative is refused).
"""

from __future__ import annotations

import ctypes
import math
import threading
import weakref

import torch
from torch.autograd import forward_ad

from . import _lib
from .attention import _kernel_layout

__all__ = ["AxialRope", "fused_qk_norm_rope"]

_DTYPES = {torch.bfloat16: _lib.DTYPE_BF16, torch.float16: _lib.DTYPE_FP16}
_HEAD_DIMS = (32, 64, 128, 256)
_current_device, _raw_stream = torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream


class _Spectrum:
    """The frequencies of a head's pairs and the axis of each on a device, and the calls prepared with them; one for
    all AxialRopes of the same parameters, which a program makes anew at every step."""

    __slots__ = ("freq", "axis", "plans")


_SPECTRA: dict = {}  # by the axes' dimensions, theta, the kind of spectrum and the device


def _spectrum(axes_dims, thetas, spectrum, device) -> _Spectrum:
    key = (axes_dims, thetas, spectrum, device)
    s = _SPECTRA.get(key)
    if s is None:
        D = sum(axes_dims)
        freq, axis = [], []
        for a, d in enumerate(axes_dims):
            for i in range(d // 2):
                power = 2 * len(freq) / D if spectrum == "shared" else 2 * i / d
                freq.append(thetas[a] ** -power / (2 * math.pi))  # turns per unit
                axis.append(a)
        s = _Spectrum()
        s.freq = torch.tensor(freq, dtype=torch.float64, device=device)
        s.axis = torch.tensor(axis, dtype=torch.int32, device=device)
        s.plans = {}  # prepared calls by the operands' geometry, forward and backward
        if len(_SPECTRA) >= 64:
            _SPECTRA.clear()
        _SPECTRA[key] = s
    return s


class AxialRope:
    """Positions of a step's tokens on several axes, and the pairs' frequencies.

    ``positions``: ``[A, S]``, or ``[B, A, S]`` with positions of each batch entry's
    own, any integer or floating dtype (negative and fractional ones too), on a
    HIP device.  ``axes_dims``: how many of the head's D dimensions each axis
    turns, even numbers that add up to D (0 for an axis that turns none).
    Pair i of axis a's d dimensions turns by ``position[a] * theta ** (-2 i / d)``
    (``spectrum="axis"``), or the head's pair j by ``position[axis of j] * theta **
    (-2 j / D)`` (``"shared"``: one spectrum, cut among the axes).  ``theta`` is one
    number or one for each axis.  ``pairs``: "interleaved" (dimensions 2j and 2j +
    1) or "halves" (j and j + D / 2).

    The positions are kept as fp64 in ``positions`` (the given tensor itself if it
    is dense fp64): a program that replays a captured step copies the next
    step's into it."""

    def __init__(self, positions: torch.Tensor, axes_dims, theta=10000.0, *, pairs: str = "interleaved",
                 spectrum: str = "axis"):
        axes_dims = tuple(int(d) for d in axes_dims)
        D = sum(axes_dims)
        if not axes_dims or any(d < 0 or d % 2 for d in axes_dims) or D not in _HEAD_DIMS:
            raise ValueError(f"axes_dims must be even and add up to one of {_HEAD_DIMS}, got {axes_dims}")
        if positions.dim() not in (2, 3) or positions.shape[-2] != len(axes_dims):
            raise ValueError(f"positions must be [{len(axes_dims)}, S] or [B, {len(axes_dims)}, S], got {tuple(positions.shape)}")
        if positions.is_complex() or positions.dtype == torch.bool:
            raise ValueError(f"positions must be numbers, got {positions.dtype}")
        if not positions.is_cuda:
            raise ValueError("positions must be a device tensor (the kernel runs on the GPU)")
        if pairs not in ("interleaved", "halves"):
            raise ValueError(f"pairs must be 'interleaved' or 'halves', got {pairs!r}")
        if spectrum not in ("axis", "shared"):
            raise ValueError(f"spectrum must be 'axis' or 'shared', got {spectrum!r}")
        thetas = tuple(float(t) for t in theta) if isinstance(theta, (tuple, list)) else (float(theta),) * len(axes_dims)
        if len(thetas) != len(axes_dims) or not all(math.isfinite(t) and t > 0 for t in thetas):
            raise ValueError(f"theta must be positive, one or {len(axes_dims)}, got {theta}")
        self._positions = positions.detach().to(torch.float64).contiguous()
        self.axes_dims, self.head_dim, self.theta = axes_dims, D, thetas
        self.pairs, self.spectrum = pairs, spectrum
        self._spectrum = _spectrum(axes_dims, thetas, spectrum, positions.device)
        self._shape = tuple(self._positions.shape)

    @property
    def positions(self) -> torch.Tensor:
        """fp64 ``[A, S]`` or ``[B, A, S]``; may be written to, not replaced."""
        return self._positions

    @property
    def device(self) -> torch.device:
        return self._positions.device

    def __repr__(self) -> str:
        return (f"AxialRope(positions={self._shape}, axes_dims={self.axes_dims}, theta={self.theta}, "
                f"pairs={self.pairs!r}, spectrum={self.spectrum!r}, device={str(self.device)!r})")


class _Plan:
    """What one geometry needs at call time; no tensor."""

    __slots__ = ("args", "index", "copies", "casts", "norm", "shapes", "like", "ws_bytes")


def _plan(rope: AxialRope, xs, ws, eps, grads=None) -> _Plan:
    q, k, wq, wk = xs[0], xs[-1], ws[0], ws[-1]
    key = (rope._shape, rope.pairs, len(xs), q.shape, q.stride(), q.dtype, q.device, q.data_ptr() & 15,
           k.shape, k.stride(), k.dtype, k.device, k.data_ptr() & 15, eps,
           None if wq is None else (wq.shape, wq.stride(), wq.dtype, wq.device, wq.data_ptr() & 15),
           None if wk is None else (wk.shape, wk.stride(), wk.dtype, wk.device, wk.data_ptr() & 15),
           None if grads is None else tuple((g.stride(), g.data_ptr() & 15) for g in grads))
    plans = rope._spectrum.plans
    p = plans.get(key)
    if p is None:
        p = _prepare(rope, xs, ws, eps, grads)
        if len(plans) >= 64:
            plans.clear()
        plans[key] = p
    return p


def _prepare(rope: AxialRope, xs, ws, eps, grads) -> _Plan:
    x0 = xs[0]
    for name, x in zip(("query", "key"), xs):
        if x.dim() != 4:
            raise ValueError(f"{name} must be [B, S, H, D], got shape {tuple(x.shape)}")
        if x.dtype not in _DTYPES:
            raise ValueError(f"{name} must be bf16 or fp16, got {x.dtype}")
        if x.dtype != x0.dtype or x.shape[:2] != x0.shape[:2] or x.shape[3] != x0.shape[3]:
            raise ValueError(f"query is {tuple(x0.shape)} {x0.dtype}, key {tuple(x.shape)} {x.dtype}: "
                             "they differ in more than their heads")
        if x.device != rope.device:
            raise ValueError(f"{name} is on {x.device}, the positions on {rope.device}")
    B, S, _, D = x0.shape
    if D != rope.head_dim:
        raise ValueError(f"the head dim is {D}, the axes' dimensions add up to {rope.head_dim}")
    if rope._shape[-1] != S or (len(rope._shape) == 3 and rope._shape[0] not in (1, B)):
        raise ValueError(f"positions {rope._shape} do not fit {B} entries of {S} tokens")
    if any((w is None) != (ws[0] is None) for w in ws):
        raise ValueError("both weights or neither")
    for w in ws:
        if w is not None and (tuple(w.shape) != (D,) or w.device != x0.device):
            raise ValueError(f"a weight must be [{D}] on {x0.device}, got {tuple(w.shape)} on {w.device}")
    p = _Plan()
    p.index = x0.device.index
    p.shapes = [tuple(x.shape) for x in xs]
    groups = (xs,) if grads is None else (xs, grads)
    laid = [[_layout(t) for t in g] for g in groups]
    # operands that the kernel cannot read in place go through dense copies, at each call
    p.copies = [c if any(c) else None for c in (tuple(u is not t for u, t in zip(l, g)) for l, g in zip(laid, groups))]
    p.like = all(x.is_contiguous() for x in xs)
    p.norm = ws[0] is not None
    p.casts = p.norm and any(w.dtype != torch.float32 or not w.is_contiguous() or w.data_ptr() % 16 != 0 for w in ws)
    a = _lib.QikAxialRopeArgs()
    a.abi_version, a.dtype = _lib.ABI_VERSION, _DTYPES[x0.dtype]
    a.halves, a.naxes = int(rope.pairs == "halves"), len(rope.axes_dims)
    a.stride_pos_a = rope._shape[-1]
    a.stride_pos_b = rope._shape[-1] * len(rope.axes_dims) if len(rope._shape) == 3 and rope._shape[0] > 1 else 0
    a.B, a.S, a.D = B, S, D
    for i, x in enumerate(laid[0]):
        t = a.t[i]
        H = x.shape[2]
        t.H, t.eps = H, eps[i]
        t.stride_x = _lib._i64x3(*x.stride()[:3])
        t.stride_out = _lib._i64x3(S * H * D, H * D, D)
        if grads is not None:
            t.stride_dy = _lib._i64x3(*laid[1][i].stride()[:3])
    p.args, p.ws_bytes = a, 0
    if grads is not None and ws[0] is not None and x0.shape[0] * S and any(s[2] for s in p.shapes):
        # sized with any addresses that pass the checks
        any_ptr = rope._spectrum.freq.data_ptr()
        q = _lib.QikAxialRopeArgs.from_buffer_copy(a)
        q.positions = q.freq = q.axis = any_ptr
        for t in q.t:
            t.x = t.weight = t.dy = t.dx = t.dw = any_ptr
        n = ctypes.c_int64(0)
        _lib.check(_lib.load().qik_axial_rope_bwd_workspace_size(ctypes.byref(q), ctypes.byref(n)), "qik_axial_rope_bwd")
        p.ws_bytes = n.value
    return p


def _layout(t: torch.Tensor) -> torch.Tensor:
    """t, or a dense copy where the kernel cannot read it in place."""
    if t.shape[-1] > 1 and t.stride(-1) != 1:
        return t.clone(memory_format=torch.contiguous_format)
    return _kernel_layout(t)


def _dense(ts, copies):
    if copies is None:
        return ts
    return [t.clone(memory_format=torch.contiguous_format) if c else t for t, c in zip(ts, copies)]


def _fp32(w: torch.Tensor) -> torch.Tensor:
    w = w.to(torch.float32).contiguous()
    return w if w.data_ptr() % 16 == 0 else w.clone()


def _call(index: int, fn, name: str, *args) -> None:
    if index != _current_device():
        with torch.cuda.device(index):
            st = fn(*args, _raw_stream(index))
    else:
        st = fn(*args, _raw_stream(index))
    if st:
        _lib.check(st, name)


def _struct(p: _Plan, rope: AxialRope) -> _lib.QikAxialRopeArgs:
    a = _lib.QikAxialRopeArgs.from_buffer_copy(p.args)
    s = rope._spectrum
    a.positions, a.freq, a.axis = rope._positions.data_ptr(), s.freq.data_ptr(), s.axis.data_ptr()
    return a


def _forward(rope: AxialRope, xs, ws, eps):
    p = _plan(rope, xs, ws, eps)
    xs = _dense(xs, p.copies[0])
    if p.casts:
        ws = [_fp32(w) for w in ws]
    a = _struct(p, rope)
    outs = []
    for t, x, w, shape in zip(a.t, xs, ws, p.shapes):
        out = torch.empty_like(x) if p.like else x.new_empty(shape)
        t.x, t.out = x.data_ptr(), out.data_ptr()
        if p.norm:
            t.weight = w.data_ptr()
        outs.append(out)
    _call(p.index, _lib.load().qik_axial_rope, "qik_axial_rope", ctypes.byref(a))
    return outs


def _backward(rope: AxialRope, xs, ws, eps, grads):
    """(dx of each, dw of each in fp32 or None)."""
    p = _plan(rope, xs, ws, eps, grads)
    xs, grads = _dense(xs, p.copies[0]), _dense(grads, p.copies[1])
    if p.casts:
        ws = [_fp32(w) for w in ws]
    a = _struct(p, rope)
    dx, dw = [], []
    for t, x, w, g in zip(a.t, xs, ws, grads):
        d = torch.empty_like(x) if p.like else x.new_empty(x.shape)
        t.x, t.dy, t.dx = x.data_ptr(), g.data_ptr(), d.data_ptr()
        dx.append(d)
        if p.norm:
            # (with no rows nothing is launched: the sums are zeros)
            d = (torch.empty_like if p.ws_bytes and x.shape[2] else torch.zeros_like)(w)
            t.weight, t.dw = w.data_ptr(), d.data_ptr()
            dw.append(d)
        else:
            dw.append(None)
    mem = xs[0].new_empty(p.ws_bytes, dtype=torch.uint8) if p.ws_bytes else None
    _call(p.index, _lib.load().qik_axial_rope_bwd, "qik_axial_rope_bwd", ctypes.byref(a),
          None if mem is None else mem.data_ptr(), p.ws_bytes)
    return dx, dw


# A leaf's node of the backward pass belongs to the stream on which the first graph
# that is still alive was recorded, also when that graph's own backward pass is over,
# and the backward pass ties that stream to its own by waits.  So a captured pass
# takes another stream (a warm-up's) into the capture.  The default stream cannot be
# captured: the process would end, so the capture is refused while it can be.  By
# leaf: the kind of that stream, and the recorded calls.
_LEAVES: dict = {}
_LEAVES_LOCK = threading.RLock()  # threads may share leaves; a finalizer may run a call while this one is noted


def _record(call, leaves, stream: int, capturing: bool) -> None:
    """Note that `call` (its ctx) is recorded on `stream` (any value that tells apart what a capture cannot join);
    RuntimeError if a capture could not run its backward pass."""
    with _LEAVES_LOCK:
        for t in leaves:
            here = _LEAVES.get(id(t))
            alive = [] if here is None else [r for r in here[1] if r() is not None]
            if alive and capturing and here[0] != stream:
                raise RuntimeError("a graph of the same leaves, recorded on the default stream, is alive: its outputs have to "
                                   "be dropped before a call with gradients is captured")
            if not alive and len(_LEAVES) >= 4096:
                for k in [k for k, (_, refs) in _LEAVES.items() if all(r() is None for r in refs)]:
                    del _LEAVES[k]
            _LEAVES[id(t)] = (here[0] if alive else stream, [*alive, weakref.ref(call)])


class _NormRope(torch.autograd.Function):
    """One or two tensors: (rope, eps, n, x.., w..) -> y.."""

    @staticmethod
    def forward(ctx, rope, eps, n, *ts):
        xs, ws = list(ts[:n]), list(ts[n:])
        ctx.rope, ctx.eps, ctx.n = rope, eps, n
        leaves = [t for t in ts if t is not None and t.requires_grad and t.is_leaf]
        if leaves and xs[0].is_cuda:
            # (the default stream's handle is 0; a capture is never on it)
            side = int(_raw_stream(xs[0].device.index) != 0)
            _record(ctx, leaves, side, torch.cuda.is_current_stream_capturing())
        # the positions are saved with the inputs: a change before the backward pass is an error there
        ctx.save_for_backward(rope._positions, *ts)
        return tuple(_forward(rope, xs, ws, eps))

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, *grads):
        _, *ts = ctx.saved_tensors  # (and the positions are the saved ones)
        xs, ws = ts[:ctx.n], ts[ctx.n:]
        dx, dw = _backward(ctx.rope, xs, ws, ctx.eps, grads)
        dw = [d if d is None or d.dtype == w.dtype else d.to(w.dtype) for d, w in zip(dw, ws)]
        return (None, None, None, *dx, *dw)


def _run(rope: AxialRope, xs, ws, eps):
    # (a dual tensor need not require gradients: inside a forward-mode level the Function refuses it by itself)
    if forward_ad._current_level >= 0 or torch.is_grad_enabled() and (xs[0].requires_grad or xs[-1].requires_grad
                                                                      or (ws[0] is not None and ws[0].requires_grad)
                                                                      or (ws[-1] is not None and ws[-1].requires_grad)):
        return _NormRope.apply(rope, eps, len(xs), *xs, *ws)
    return _forward(rope, xs, ws, eps)


def norm_rope(x, weight, rope: AxialRope, eps: float) -> torch.Tensor:
    """``fused_rms_norm_rope`` with an AxialRope."""
    return _run(rope, (x,), (weight,), (float(eps),))[0]


def fused_qk_norm_rope(
    query: torch.Tensor,                # [B, S, H, D] bf16 or fp16
    key: torch.Tensor,                  # [B, S, HKV, D], query's dtype
    weight_q: torch.Tensor | None,      # [D], or None for both: the rotation alone
    weight_k: torch.Tensor | None,
    rope: AxialRope,
    eps: float,
    eps_k: float | None = None,         # of the key's norm; None: eps
) -> tuple[torch.Tensor, torch.Tensor]:
    """A layer's Q and K: RMSNorm over each head, then the rotation by the tokens' positions.

    ``y = rotate((x * r) * weight)`` with ``r = 1 / sqrt(mean(x^2) + eps)``, in fp32
    and rounded once.  One launch for both, the angles of a token computed once
    for all its heads; strided inputs are read in place.  Records the
    gradients of query, key and the weights (whose sums over the rows are fp32, in
    an order that depends on the sizes alone)."""
    if not isinstance(rope, AxialRope):
        raise ValueError(f"rope must be an AxialRope, got {type(rope).__name__}")
    eps = float(eps)
    q, k = _run(rope, (query, key), (weight_q, weight_k), (eps, eps if eps_k is None else float(eps_k)))
    return q, k
