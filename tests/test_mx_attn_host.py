"""The 4-bit slab, its attention and the rotary positions without a GPU: C ABI, plans, refusals."""

import ctypes
import os
import re
import subprocess

import pytest
import torch

from oracle import axial_rope as oa
from oracle import mx_slab as om

import qwen_image_kernel_amd as qik
from qwen_image_kernel_amd import _lib

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
INCLUDE = os.path.join(ROOT, "include")
FAKE = 0x100000  # an address that passes the alignment checks and is never read


@pytest.mark.parametrize("header,exports", [("qik_mx_attn.h", _lib.MX_ATTN_EXPORTS), ("qik_rope.h", _lib.ROPE_EXPORTS)])
def test_header_and_binding_name_the_same_functions(header, exports):
    names = set(re.findall(r"^int (qik_\w+)\s*\(", open(os.path.join(INCLUDE, header)).read(), flags=re.M))
    assert names == {n for n, _, _ in exports}
    for n in names:
        assert hasattr(_lib.load(), n)


@pytest.mark.parametrize("cname,pytype", [("qik_mx_slab", _lib.QikMxSlab), ("qik_mx_slab_store_args", _lib.QikMxSlabStoreArgs),
                                          ("qik_mx_slab_load_args", _lib.QikMxSlabLoadArgs),
                                          ("qik_mx_attn_args", _lib.QikMxAttnArgs), ("qik_rope_tensor", _lib.QikRopeTensor),
                                          ("qik_axial_rope_args", _lib.QikAxialRopeArgs)])
def test_struct_layout_matches_c_header(tmp_path, cname, pytype):
    fields = [f for f, _ in pytype._fields_]
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "qik_mx_attn.h"', '#include "qik_rope.h"', "int main(void) {",
             f'printf("sizeof %zu\\n", sizeof({cname}));', *(f'printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields),
             "return 0; }"]
    (tmp_path / "layout.c").write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-std=c99", f"-I{INCLUDE}", str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    got = dict(line.split() for line in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines())
    assert int(got["sizeof"]) == ctypes.sizeof(pytype)
    for f in fields:
        assert int(got[f]) == getattr(pytype, f).offset, f


# ---- attention -------------------------------------------------------------

def _slab(B=2, P=100, H=2, D=128):
    return _lib.QikMxSlab(FAKE, FAKE, _lib._i64x3(H * P * D // 2, D // 2, P * D // 2), _lib._i64x3(H * P * D // 32, D // 32, P * D // 32))


def _attn(**kw):
    x = _lib.QikMxAttnArgs()
    a = x.a
    B, SQ, SN, P, H, D = 2, 3, 3, 100, 8, 128
    x.HKV = 2
    a.abi_version, a.flags = _lib.ABI_VERSION, _lib.HAS_CACHE
    a.q = a.k_new = a.v_new = a.out = a.prefix_lengths = FAKE
    a.B, a.SQ, a.SN, a.P, a.H, a.D = B, SQ, SN, P, H, D
    a.stride_q = a.stride_out = _lib._i64x3(SQ * H * D, H * D, D)
    a.stride_k_new = a.stride_v_new = _lib._i64x3(SN * 2 * D, 2 * D, D)
    a.sm_scale = D ** -0.5
    x.k_slab, x.v_slab = _slab(), _slab()
    for k, v in kw.items():
        setattr(x if hasattr(x, k) else a, k, v)
    return x


def _status(x):
    return _lib.load().qik_mx_attn_validate(ctypes.byref(x))


def test_attention_arguments_in_order():
    assert _status(_attn()) == 0
    assert _status(_attn(P=0, flags=0)) == 0
    assert _status(_attn(SN=0, k_new=None, v_new=None)) == 0
    assert _status(_attn(flags=_lib.HAS_CACHE | _lib.UNIFORM_L, prefix_lengths=None)) == 0
    assert _status(_attn(SQ=0)) == 0 and _status(_attn(B=0)) == 0


def _bad_slab(**kw):
    s = _slab()
    for k, v in kw.items():
        setattr(s, k, v)
    return s


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=9), -2), (dict(reserved0=1), -2), (dict(dtype=2), -3), (dict(D=96), -4), (dict(D=512), -4),
    (dict(SQ=-1), -5), (dict(B=1 << 40), -5), (dict(HKV=3), -5), (dict(HKV=0), -5), (dict(HKV=-1), -5), (dict(P=1 << 31), -5),
    (dict(SQ=1 << 30), -5),                                     # rows of a KV head past 2^31
    (dict(flags=_lib.HAS_CACHE | _lib.V_CACHE_FP8), -5), (dict(flags=0), -6), (dict(P=0), -6), (dict(k_cache=FAKE), -6),
    (dict(v_scale=FAKE), -7), (dict(key_valid=FAKE), -1), (dict(flags=_lib.HAS_CACHE | _lib.HAS_KEY_VALID), -1),
    (dict(debug_tiles=FAKE), -1), (dict(q=None), -1), (dict(out=None), -1), (dict(k_new=None), -1), (dict(prefix_lengths=None), -1),
    (dict(q=FAKE + 8), -8), (dict(v_new=FAKE + 2), -8), (dict(stride_q=_lib._i64x3(3 * 1024, 1020, 128)), -8),
    (dict(stride_k_new=_lib._i64x3(768, 64, 128)), -8), (dict(stride_v_new=_lib._i64x3(768, 1 << 27, 128)), -5),
    (dict(k_slab=_bad_slab(codes=None)), -1), (dict(v_slab=_bad_slab(scales=None)), -1), (dict(k_slab=_bad_slab(codes=FAKE + 8)), -8),
    (dict(k_slab=_bad_slab(scales=FAKE + 2)), -8), (dict(v_slab=_bad_slab(stride_codes=_lib._i64x3(12800, 72, 6400))), -8),
    (dict(v_slab=_bad_slab(stride_codes=_lib._i64x3(12800, 48, 6400))), -8),   # rows overlap
    (dict(v_slab=_bad_slab(stride_scales=_lib._i64x3(800, 6, 400))), -8),
    (dict(k_slab=_bad_slab(stride_codes=_lib._i64x3(12800, 1 << 25, 6400))), -5),
])
def test_attention_refusals(kw, code):
    x = _attn(**kw)
    assert _status(x) == code
    lib = _lib.load()
    n = ctypes.c_int64(-1)
    assert lib.qik_mx_attn_workspace_size(ctypes.byref(x), ctypes.byref(n)) == code
    assert lib.qik_mx_attn_fwd(ctypes.byref(x), None, 0, None) == code


def test_attention_without_work_touches_no_device():
    lib = _lib.load()
    for kw in (dict(SQ=0), dict(B=0), dict(H=0, HKV=0)):
        x = _attn(**kw)
        assert lib.qik_mx_attn_fwd(ctypes.byref(x), None, 0, None) == 0


def _plan(B, SQ, SN, P, H, HKV, D=128, ragged=0, cus=256):
    few, tiles, pieces = (ctypes.c_int32() for _ in range(3))
    assert _lib.load().qik_mx_attn_plan(B, SQ, SN, P, H, HKV, D, ragged, cus, ctypes.byref(few), ctypes.byref(tiles),
                                        ctypes.byref(pieces)) == 0
    return few.value, tiles.value, pieces.value


def test_attention_plan():
    """A token runs the kernel of few rows and is spread over the CUs; an image's rows run the other."""
    assert _plan(1, 1, 1, 131072, 32, 8) == (1, 1, 32)
    assert _plan(1, 1, 0, 40, 32, 8) == (1, 1, 1)
    assert _plan(1, 4096, 4096, 2560, 24, 24)[0] == 0
    assert _plan(1, 16, 16, 30000, 32, 8)[:2] == (1, 4)
    for case in ((24, 1, 0, 8192, 32, 8), (1, 1, 1, 1, 1, 1), (1, 1, 0, 0, 4, 4), (70000, 1, 1, 64, 4, 4), (3, 64, 64, 1 << 20, 64, 1),
                 (9000, 1, 1, 4096, 1, 1), (1, 1, 1, (1 << 31) - 2, 1, 1)):
        for D in (32, 64, 128, 256):
            for cus in (1, 256):
                few, tiles, pieces = _plan(*case, D=D, cus=cus)
                steps = max(-(-case[3] // 32) + -(-case[2] // 32), 1)
                assert pieces >= 1 or not few
                assert pieces <= min(steps, 65535)
    assert _plan(70000, 1, 1, 64, 4, 4)[0] == 0   # more entries than a grid has rows
    assert _plan(9000, 1, 1, 4096, 1, 1)[2] == 1  # more items than control words: none is cut
    lib = _lib.load()
    n = ctypes.c_int32()
    assert lib.qik_mx_attn_plan(1, 1, 1, 1, 4, 3, 128, 0, 256, ctypes.byref(n), ctypes.byref(n), ctypes.byref(n)) == -5
    assert lib.qik_mx_attn_plan(1, 1, 1, 1, 4, 4, 100, 0, 256, ctypes.byref(n), ctypes.byref(n), ctypes.byref(n)) == -4
    assert lib.qik_mx_attn_plan(1, 1, 1, 1, 4, 4, 128, 0, 256, None, ctypes.byref(n), ctypes.byref(n)) == -1


# ---- store and load --------------------------------------------------------

def _store(**kw):
    a = _lib.QikMxSlabStoreArgs()
    B, S, H, D = 2, 5, 2, 128
    a.abi_version, a.k, a.v = _lib.ABI_VERSION, FAKE, FAKE
    a.k_dst, a.v_dst = _slab(), _slab()
    a.B, a.S, a.H, a.D, a.capacity = B, S, H, D, 100
    a.stride_k = a.stride_v = _lib._i64x3(S * H * D, H * D, D)
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -2), (dict(dtype=2), -3), (dict(D=48), -4), (dict(S=-1), -5), (dict(capacity=-1), -5),
    (dict(B=1 << 20, S=1 << 20), -5), (dict(k=None), -1), (dict(v=FAKE + 4), -8),
    (dict(stride_v=_lib._i64x3(1280, 250, 128)), -8), (dict(k_dst=_bad_slab(codes=FAKE + 4)), -8),
    (dict(v_dst=_bad_slab(scales=None)), -1), (dict(at=FAKE, lengths=FAKE), -1),   # grows without the arrivals word
])
def test_store_refusals(kw, code):
    assert _lib.load().qik_mx_slab_store(ctypes.byref(_store(**kw)), None) == code


def test_store_and_load_without_rows_touch_no_device():
    lib = _lib.load()
    for kw in (dict(B=0), dict(S=0), dict(H=0)):
        assert lib.qik_mx_slab_store(ctypes.byref(_store(**kw)), None) == 0
    a = _lib.QikMxSlabLoadArgs()
    a.abi_version, a.D, a.B, a.H = _lib.ABI_VERSION, 64, 2, 2
    assert lib.qik_mx_slab_load(ctypes.byref(a), None) == 0
    a.P = 3
    assert lib.qik_mx_slab_load(ctypes.byref(a), None) == -1
    a.D = 65
    assert lib.qik_mx_slab_load(ctypes.byref(a), None) == -4


# ---- rotary positions ------------------------------------------------------

def _rope(**kw):
    a = _lib.QikAxialRopeArgs()
    a.abi_version, a.naxes = _lib.ABI_VERSION, 3
    a.positions = a.freq = a.axis = FAKE
    a.B, a.S, a.D = 1, 5, 128
    a.stride_pos_a = 5
    for t in a.t:
        t.x = t.out = t.weight = t.dy = t.dx = t.dw = FAKE
        t.H = 2
        t.stride_x = t.stride_out = t.stride_dy = _lib._i64x3(1280, 256, 128)
    for k, v in kw.items():
        if hasattr(a, k):
            setattr(a, k, v)
        else:
            setattr(a.t[1], k, v)
    return a


@pytest.mark.parametrize("kw,code", [
    (dict(abi_version=1), -2), (dict(reserved0=1), -2), (dict(dtype=2), -3), (dict(D=96), -4), (dict(B=-1), -5), (dict(naxes=0), -5),
    (dict(halves=2), -5), (dict(H=-1), -5), (dict(S=1 << 30), -5), (dict(positions=None), -1), (dict(axis=None), -1),
    (dict(weight=None), -1),                                   # one weight of two
    (dict(weight=FAKE + 4), -8), (dict(stride_x=_lib._i64x3(1280, 252, 128)), -8),
    (dict(stride_out=_lib._i64x3(1280, 1 << 40, 128)), -5), (dict(dy=None), -1), (dict(dx=None), -1), (dict(dw=None), -1),
])
def test_rope_refusals(kw, code):
    lib = _lib.load()
    a = _rope(**kw)
    n = ctypes.c_int64()
    assert lib.qik_axial_rope_bwd(ctypes.byref(a), FAKE, 1 << 30, None) == code
    assert lib.qik_axial_rope_bwd_workspace_size(ctypes.byref(a), ctypes.byref(n)) == code
    if not set(kw) & {"dy", "dx", "dw"}:
        assert lib.qik_axial_rope(ctypes.byref(a), None) == code


def test_rope_without_rows_touches_no_device():
    lib = _lib.load()
    for kw in (dict(B=0), dict(S=0)):
        assert lib.qik_axial_rope(ctypes.byref(_rope(**kw)), None) == 0
        assert lib.qik_axial_rope_bwd(ctypes.byref(_rope(**kw)), None, 0, None) == 0


def test_rope_workspace_is_checked():
    lib = _lib.load()
    a, n = _rope(), ctypes.c_int64()
    assert lib.qik_axial_rope_bwd_workspace_size(ctypes.byref(a), ctypes.byref(n)) == 0 and n.value >= 2 * 128 * 4
    assert lib.qik_axial_rope_bwd(ctypes.byref(a), None, n.value, None) == -12
    assert lib.qik_axial_rope_bwd(ctypes.byref(a), FAKE + 8, n.value, None) == -12
    assert lib.qik_axial_rope_bwd(ctypes.byref(a), FAKE, n.value - 1, None) == -12


# ---- Python refusals -------------------------------------------------------

def test_python_objects_refuse():
    c, s = torch.zeros(1, 4, 2, 64, dtype=torch.uint8), torch.zeros(1, 4, 2, 4, dtype=torch.uint8)
    assert qik.MXSlab(c, s).shape == (1, 4, 2, 128)
    for bad in ((c[0], s), (c.int(), s), (c, s[..., :3]), (c[..., :40], s), (c, s, torch.zeros(2, dtype=torch.int32)),
                (c, s, torch.zeros(1, dtype=torch.int64)), (c, s, torch.zeros(2, dtype=torch.int32)[::2][:1].expand(1)[:0])):
        with pytest.raises(ValueError):
            qik.MXSlab(*bad)
    for kw in (dict(device="cpu"), dict(dtype=torch.float32), dict(head_dim=96)):
        with pytest.raises(ValueError):
            qik.MXKVCache(**{**dict(num_layers=1, batch=1, prefix_max=4, num_heads=1, head_dim=64, device="cuda"), **kw})
    pos = torch.zeros(3, 5)
    for args, kw in (((pos, (16, 56, 56)), {}), ((pos, (15, 57, 56)), {}), ((pos, (16, 16, 16)), {}), ((pos, (64, 64)), {}),
                     ((pos[0], (128,)), {}), ((pos, (16, 56, 56)), dict(pairs="x")), ((pos, (16, 56, 56)), dict(theta=0.0))):
        with pytest.raises(ValueError):   # the first for the CPU tensor alone
            qik.AxialRope(*args, **kw)
    with pytest.raises(ValueError):
        qik.fused_qk_norm_rope(pos, pos, None, None, torch.zeros(5, 64), 1e-6)
    q = torch.zeros(1, 1, 2, 128, dtype=torch.bfloat16)
    m = qik.MXSlab(c, s)
    for kw in (dict(cache_k=m, cache_v=q), dict(cache_k=q, cache_v=m), dict(cache_k=m, cache_v=m, split_tail=False),
               dict(cache_k=m, cache_v=m, cache_v_scale=s), dict(cache_k=m, cache_v=m, debug_tiles=s),
               dict(cache_k=m, cache_v=m)):   # the last for the CPU tensors alone
        with pytest.raises(ValueError):
            qik.block_causal_flash_attention(q, q, q, None, None, uniform_full=True, **kw)


def test_slab_layouts_read_in_place():
    c, s = torch.zeros(2, 3, 8, 64, dtype=torch.uint8), torch.zeros(2, 3, 8, 4, dtype=torch.uint8)   # [B, H, P, ..]
    assert qik.MXSlab(c.transpose(1, 2), s.transpose(1, 2)).in_place()
    assert qik.MXSlab(c[:, :, :5].transpose(1, 2), s[:, :, :5].transpose(1, 2)).in_place()
    odd = torch.zeros(2 * 3 * 8 * 64 + 1, dtype=torch.uint8)[1:].view(2, 3, 8, 64)
    slab = qik.MXSlab(odd.transpose(1, 2), s.transpose(1, 2))
    assert not slab.in_place() and slab.readable().in_place()
    wide = torch.zeros(2, 8, 3, 8, dtype=torch.uint8)[..., ::2]   # scales that are not dense
    assert not qik.MXSlab(c.transpose(1, 2), wide).in_place()


# ---- the oracles themselves ------------------------------------------------

def test_slab_oracle_round_trip_and_attention():
    g = torch.Generator().manual_seed(1)
    x = torch.randn(3, 64, generator=g, dtype=torch.float64) * 10.0
    codes, scales = om.encode(x)
    v = om.decode(codes, scales)
    again = om.encode(v)
    assert torch.equal(om.decode(*again), v)
    top = x.unflatten(-1, (2, 32)).abs().amax(-1, keepdim=True)
    # half of E2M1's widest step (2), or saturation from below 8 to 6, at a scale of at most top / 4
    assert ((v - x).unflatten(-1, (2, 32)).abs() <= top / 4 * 2 + 1e-12).all()
    bad = torch.ones(1, 32, dtype=torch.float64)
    bad[0, 3] = torch.nan
    assert om.encode(bad)[1].item() == 255 and om.decode(*om.encode(bad)).isnan().all()
    q, k, w = (torch.randn(1, 5, 2, 32, generator=g, dtype=torch.float64) for _ in range(3))
    ok = om.allowed(1, 5, 2, 3, L=torch.tensor([-1, 0, 1, 4, 2], dtype=torch.int32))
    parts = om.attention(q, k, w, ok)
    assert (parts["out"][0, 0] == 0).all()
    assert torch.allclose(parts["out"][0, 1], w[0, 0])
    s = (q[0, 3, 1] @ k[0, :, 1].t()) / 32 ** 0.5
    assert torch.allclose(parts["out"][0, 3, 1], torch.softmax(s, -1) @ w[0, :, 1])


@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_rope_oracle_gradient_against_differences(pairs):
    g = torch.Generator().manual_seed(2)
    x = torch.randn(2, 3, 2, 32, generator=g, dtype=torch.float64).requires_grad_()
    w = torch.randn(32, generator=g, dtype=torch.float64).requires_grad_()
    angle = oa.angles(torch.randn(3, 3, generator=g) * 30, (4, 14, 14), 1e4, "axis")
    assert torch.autograd.gradcheck(lambda a, b: oa.forward(a, b, angle, pairs, 1e-3), (x, w))


def test_leaves_of_a_live_graph():
    """A capture is refused while a graph of the same leaves from another stream is alive, and only then."""
    from qwen_image_kernel_amd import rope as R

    class Call:
        pass

    a, b = torch.ones(2, requires_grad=True), torch.ones(2, requires_grad=True)
    eager = Call()
    R._record(eager, [a], 1, False)
    R._record(Call(), [a, b], 2, False)          # dropped at once; a's first graph is still stream 1's
    with pytest.raises(RuntimeError):
        R._record(Call(), [b, a], 2, True)
    R._record(Call(), [b], 2, True)
    R._record(Call(), [a], 1, True)              # the same stream
    later = Call()
    R._record(later, [a], 2, False)
    del eager
    with pytest.raises(RuntimeError):            # `later` keeps the node of stream 1
        R._record(Call(), [a], 2, True)
    del later
    R._record(Call(), [a], 2, True)


# ---- what the host knows of a cache's lengths ------------------------------

@pytest.fixture
def cache_on_the_host(monkeypatch):
    """MXKVCache with its buffers in host memory and the store's effect on the lengths in the launch's place; a call made
    while `capturing[0]` changes nothing and is appended to `recorded`, which a replay runs."""
    from qwen_image_kernel_amd import kv_cache as K

    zeros, capturing, recorded = torch.zeros, [False], []
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: None, raising=False)

    def launch(layer, call, k, v, at, grow):
        def run():
            lengths = layer._lengths.data     # as a kernel does: no version moves
            first = torch.zeros_like(lengths) if at is None else at
            lengths.copy_((first + k.shape[1]).clamp(0, layer._c.capacity))
        recorded.append(run) if capturing[0] else run()

    monkeypatch.setattr(K._MXLayerView, "_launch", launch)
    monkeypatch.setattr(K, "load_args", lambda *a: None)

    def make(layers=1, batch=2, capacity=100):
        with monkeypatch.context() as m:
            m.setattr(torch, "zeros", lambda *a, device=None, **kw: zeros(*a, **kw))
            return qik.MXKVCache(layers, batch, capacity, 1, 32)

    return make, capturing, recorded


def _states(n, batch=2):
    return [torch.zeros(batch, n, 1, 32, dtype=torch.bfloat16) for _ in range(2)]


def test_replays_of_captured_steps_are_reckoned_with(cache_on_the_host):
    """However a layer is filled after its step was captured, its default views hold what replays appended."""
    make, capturing, recorded = cache_on_the_host
    for fill in (lambda layer: layer.store(*_states(50)), lambda layer: layer.append(*_states(5), 45),
                 lambda layer: layer.store(*_states(0))):
        cache = make()
        layer = cache.get_layer(0)
        layer.store(*_states(80))
        del recorded[:]
        capturing[0] = True
        layer.append(*_states(1))
        capturing[0] = False
        assert cache.lengths[0].tolist() == [80, 80] and layer.views()[0].shape[1] == 100
        fill(layer)
        start = int(cache.lengths[0, 0])
        for i in range(10):
            recorded[0]()
            assert int(cache.lengths[0, 0]) == start + i + 1 <= layer.views()[0].shape[1]
        layer.append(*_states(3))
        assert int(cache.lengths[0, 0]) == start + 13 <= layer.views()[0].shape[1]
        layer.append(*_states(60))               # (no ValueError by a count that is not theirs)
        layer.append(*_states(60))
        assert cache.lengths[0].tolist() == [100, 100]


def test_captured_stores_and_places_are_no_present_lengths(cache_on_the_host):
    """A captured call moves no length before it is replayed, and any time after."""
    make, capturing, recorded = cache_on_the_host
    cache = make(2)
    layer, other = cache.get_layer(0), cache.get_layer(1)
    layer.store(*_states(60))
    other.store(*_states(7))
    del recorded[:]
    capturing[0] = True
    layer.store(*_states(20))
    capturing[0] = False
    assert layer.views()[0].shape[1] == 60
    recorded[0]()
    layer.append(*_states(90))                   # behind 20, not 60: some rows do not fit, and none is refused
    layer.store(*_states(3))
    assert layer.views()[0].shape[1] == 20       # what a replay may leave
    recorded[0]()
    assert cache.lengths[0].tolist() == [20, 20]
    capturing[0] = True
    layer.append(*_states(2), 70)
    capturing[0] = False
    assert layer.views()[0].shape[1] == 72
    cache.lengths.data[0] = 20                   # (the capture wrote none)
    recorded[1]()
    assert layer.views()[0].shape[1] >= 72
    # the other layer's lengths are still known
    assert other.views()[0].shape[1] == 7
    other.append(*_states(93))
    with pytest.raises(ValueError):
        other.append(*_states(1))


@pytest.mark.parametrize("inference", [False, True])
def test_entries_that_start_anew_are_not_refused(cache_on_the_host, inference):
    """append(None) goes by the entries' lengths where the program lowered them, whichever way it wrote."""
    make = cache_on_the_host[0]
    with torch.inference_mode(inference):
        for lower in (lambda c: c.lengths[0].zero_(), lambda c: c.lengths.fill_(1), lambda c: c.lengths[0, :].sub_(8),
                      lambda c: c.get_layer(0).views()[0].lengths.zero_(), lambda c: c.lengths.view(-1)[:2].copy_(torch.zeros(2))):
            cache = make(capacity=9)
            layer = cache.get_layer(0)
            layer.store(*_states(8))
            lower(cache)
            for _ in range(20):
                before = cache.lengths[0].clone()
                layer.append(*_states(2))
                assert torch.equal(cache.lengths[0], (before + 2).clamp(max=9)) and layer.views()[0].shape[1] == 9
                cache.lengths[0, 0] = 0
        # an entry of the other layer, and what the cache writes itself
        cache = make(2, capacity=9)
        layer, other = cache.get_layer(0), cache.get_layer(1)
        layer.store(*_states(3))
        layer.append(*_states(1), 4)
        other.store(*_states(0))
        other.append(*_states(0))
        with pytest.raises(ValueError):
            layer.append(*_states(5))
        with pytest.raises(ValueError):
            other.append(*_states(10))
        cache.lengths[1].zero_()
        other.store(*_states(9))
        layer.append(*_states(5))
        other.append(*_states(1))
        assert cache.lengths.tolist() == [[9, 9], [9, 9]]


def test_forward_mode_derivatives_are_refused(monkeypatch):
    """A dual tensor is refused whether or not it requires gradients, and is not taken for a plain one."""
    from torch.autograd import forward_ad

    from qwen_image_kernel_amd import rope as R

    class Rope:
        _positions = torch.zeros(1)

    monkeypatch.setattr(R, "_forward", lambda rope, xs, ws, eps: [torch.zeros_like(x) for x in xs])
    x, w = torch.ones(1, 1, 1, 32), torch.ones(32)
    with forward_ad.dual_level():
        dual, dual_w = (forward_ad.make_dual(t, torch.ones_like(t)) for t in (x, w))
        for xs, ws in (((dual,), (w,)), ((x, dual), (w, w)), ((x,), (dual_w,)), ((dual, x), (None, None)),
                       ((forward_ad.make_dual(x.clone().requires_grad_(), x),), (w,))):
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    R._run(Rope, xs, ws, (1e-6, 1e-6))
        assert R._run(Rope, (x,), (w,), (1e-6,))[0].shape == x.shape


def test_two_threads_record_calls_of_one_leaf(monkeypatch):
    """A call noted while another thread notes one of the same leaf is not lost, and a capture is refused for it."""
    import threading

    from qwen_image_kernel_amd import rope as R

    class Call:
        pass

    calls, leaf = [Call(), Call()], torch.ones(2, requires_grad=True)
    other = threading.Thread(target=lambda: R._record(calls[1], [leaf], 1, False))

    class Leaves(dict):
        def get(self, key):
            here = super().get(key)
            if threading.current_thread() is not other:   # the other thread's turn, between this one's look and its note
                if not other.ident:
                    other.start()
                other.join(0.5)
            return here

    monkeypatch.setattr(R, "_LEAVES", Leaves())
    R._record(calls[0], [leaf], 1, False)
    other.join()
    assert len(R._LEAVES[id(leaf)][1]) == 2
    del calls[0]
    with pytest.raises(RuntimeError):
        R._record(Call(), [leaf], 2, True)
