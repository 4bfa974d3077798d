"""GPU tests of the 4-bit slab where it can go wrong: hidden values, layouts, lengths, places, streams, graphs, the
processor's path."""

import ctypes

import pytest
import torch

import qwen_image_kernel_amd as qik
from oracle import mx_slab as om
from qwen_image_kernel_amd import _lib
from test_mx_attn_gpu import DEV, _check, _few, _mx, _randn, _slab

pytestmark = pytest.mark.gpu

FEW = (2, 2, 3, 150, 8, 2)      # B, SQ, SN, P, H, HKV: the kernel of few rows
MANY = (1, 700, 700, 150, 24, 24)  # the kernel of many rows


def _inputs(shape, D=128, dtype=torch.bfloat16, seed=1, pad=3):
    B, SQ, SN, P, H, HKV = shape
    g = torch.Generator().manual_seed(seed)
    q = _randn(g, B, SQ, H, D).to(dtype)
    k, v = (_randn(g, B, SN, HKV, D).to(dtype) for _ in range(2))
    return q, k, v, _slab(g, B, P, HKV, D, pad), _slab(g, B, P, HKV, D, pad)


def _call(q, k, v, ck, cv, L=None, valid=None, uniform=False):
    return qik.block_causal_flash_attention(q.to(DEV), k.to(DEV), v.to(DEV), None if L is None else L.to(DEV),
                                            None if valid is None else valid.to(DEV), cache_k=ck, cache_v=cv, uniform_full=uniform)


def test_shapes_run_the_kernels_they_stand_for():
    assert _few(FEW) and not _few(MANY)


def _parts(q, k, v, kc, vc, P, ok):
    keys, values = (torch.cat((om.decode(c[:, :, :P], s[:, :, :P]).transpose(1, 2), t.double()), 1)
                    for (c, s), t in ((kc, k), (vc, v)))
    return om.attention(q.double(), keys, values, ok)


@pytest.mark.parametrize("shape", [FEW, MANY, (1, 1, 40, 3000, 4, 1), (1, 140, 140, 64, 2, 2), (2, 700, 690, 150, 24, 12)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_hidden_keys_may_hold_anything(shape, dtype):
    """NaN blocks and values behind a mask, and bytes of any kind behind a length, change nothing."""
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape, dtype=dtype)
    g = torch.Generator().manual_seed(9)
    valid = torch.rand(B, P + SN, generator=g) < 0.6
    lengths = torch.tensor([P - 7] + [P // 3] * (B - 1), dtype=torch.int32)
    L = torch.full((SQ,), P + SN - 1, dtype=torch.int32)
    ok = om.allowed(B, SQ, P, SN, L, valid, lengths)
    hidden = ~ok[:, 0]                                                # [B, P + SN], the same for every row
    want = _call(q, k, v, _mx(*kc, P, lengths.to(DEV)), _mx(*vc, P, lengths.to(DEV)), L, valid)
    for t, (codes, scales) in ((k, kc), (v, vc)):
        t[hidden[:, P:]] = torch.tensor([torch.nan, torch.inf, -torch.inf, 1e4]).to(dtype).repeat(t.shape[-1] // 4)
        bad = hidden[:, None, :P].expand(-1, HKV, -1)
        scales[:, :, :P][bad] = 255
        codes[:, :, :P][bad] = 0x7f
    out = _call(q, k, v, _mx(*kc, P, lengths.to(DEV)), _mx(*vc, P, lengths.to(DEV)), L, valid)
    assert torch.equal(out, want)
    zero = [torch.where(hidden[:, P:, None, None], 0.0, t.double()) for t in (k, v)]
    _check(out, _parts(q, *zero, kc, vc, P, ok), 128, dtype)


@pytest.mark.parametrize("shape", [FEW, MANY])
def test_visible_nan_reaches_its_rows(shape):
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape)
    kc[1][0, 1, 5] = 255        # entry 0, KV head 1: every row of its query heads sees key 5
    out = _call(q, k, v, _mx(*kc, P), _mx(*vc, P), uniform=True)
    G = H // HKV
    assert out[0, :, G:2 * G].isnan().all()
    rest = torch.cat((out[0, :, :G].flatten(), out[0, :, 2 * G:].flatten(), out[1:].flatten()))
    assert torch.isfinite(rest).all()


@pytest.mark.parametrize("shape", [FEW, MANY])
def test_masks_of_every_kind(shape):
    """bool, bytes, numbers, one row for all entries, a wider mask, gaps between its rows; L as int64, longer, [1, SQ]."""
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape)
    ck, cv = _mx(*kc, P), _mx(*vc, P)
    g = torch.Generator().manual_seed(3)
    valid = (torch.rand(1, P + SN, generator=g) < 0.7).to(DEV)
    L = torch.randint(-1, P + SN + 40, (SQ,), generator=g, dtype=torch.int32).to(DEV)
    want = _call(q, k, v, ck, cv, L, valid)
    wide = torch.ones(B, P + SN + 13, dtype=torch.bool, device=DEV)
    wide[:, :P + SN] = valid
    for m in (valid.expand(B, -1), valid.expand(B, -1).contiguous().to(torch.uint8) * 7, valid.float() * 0.25,
              valid.long() * 256, wide, wide[:, :P + SN], valid.expand(B, -1).contiguous().t().contiguous().t()):
        assert torch.equal(_call(q, k, v, ck, cv, L, m), want)
    for l in (L.long(), torch.cat((L, L)), L[None], L.expand(B, -1), L.repeat(2).view(2, -1).t().contiguous().t()[0]):
        assert torch.equal(_call(q, k, v, ck, cv, l, valid), want)
    none = torch.zeros(B, P + SN, dtype=torch.bool, device=DEV)
    assert (_call(q, k, v, ck, cv, L, none) == 0).all()
    assert (_call(q, k, v, ck, cv, torch.full_like(L, -1)) == 0).all()


@pytest.mark.parametrize("shape", [FEW, MANY, (3, 1, 0, 40, 6, 3)])
def test_lengths_of_any_value(shape):
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape)
    for lengths in ([P] * B, [P + 100, -5, 0][:B], [0] * B, [1, 31, 32][:B], [33, 2 ** 31 - 1, -2 ** 31][:B]):
        ln = torch.tensor(lengths, dtype=torch.int64).to(torch.int32)
        out = _call(q, k, v, _mx(*kc, P, ln.to(DEV)), _mx(*vc, P, ln.to(DEV)), uniform=True)
        ok = om.allowed(B, SQ, P, SN, None, None, ln)
        _check(out, _parts(q, k, v, kc, vc, P, ok), 128, torch.bfloat16)
        assert (out.cpu()[~ok.any(-1)] == 0).all()


def test_no_keys_no_rows_no_heads():
    for shape in ((2, 3, 0, 0, 4, 2), (1, 200, 0, 0, 4, 4)):
        q, k, v, kc, vc = _inputs(shape, pad=1)
        assert (_call(q, k, v, _mx(*kc, 0), _mx(*vc, 0), uniform=True) == 0).all()
    for shape in ((2, 0, 4, 9, 4, 2), (0, 3, 4, 9, 4, 2)):
        q, k, v, kc, vc = _inputs(shape)
        assert _call(q, k, v, _mx(*kc, 9), _mx(*vc, 9), uniform=True).shape == q.shape
    # an empty slab leaves the fresh keys, which the bf16 call attends too
    q, k, v, kc, vc = _inputs((1, 200, 200, 0, 4, 4), pad=1)
    L = torch.arange(200, dtype=torch.int32)
    _check(_call(q, k, v, _mx(*kc, 0), _mx(*vc, 0), L), _parts(q, k, v, kc, vc, 0, om.allowed(1, 200, 0, 200, L)), 128, torch.bfloat16)


@pytest.mark.parametrize("shape", [FEW, (2, 130, 40, 150, 8, 4), MANY])
def test_layouts(shape):
    """Slices of a fused projection, operands off their alignment, slabs in other orders: the same bits."""
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape)
    ck, cv = _mx(*kc, P), _mx(*vc, P)
    want = _call(q, k, v, ck, cv, uniform=True)
    qd, kd, vd = q.to(DEV), k.to(DEV), v.to(DEV)

    def strided(t, pad, off):   # the same values, rows `pad` elements further apart, `off` elements into the buffer
        buf = torch.full((t.numel() // 128 * (128 + pad) + off,), torch.nan, dtype=t.dtype, device=DEV)
        out = buf[off:].as_strided(t.shape, tuple(s // 128 * (128 + pad) for s in t.stride()[:3]) + (1,))
        return out.copy_(t)

    for pad, off in ((8, 0), (3, 0), (0, 1), (5, 3)):
        for which in range(3):
            ts = [strided(t, pad, off) if i == which else t for i, t in enumerate((qd, kd, vd))]
            assert torch.equal(_call(*ts, ck, cv, uniform=True), want), (pad, off, which)
    both = torch.cat((kd, vd), 2)
    assert torch.equal(_call(qd, both[:, :, :HKV], both[:, :, HKV:], ck, cv, uniform=True), want)
    transposed = qd.transpose(1, 2).contiguous().transpose(1, 2)   # [B, H, SQ, D] in memory
    assert torch.equal(_call(transposed, kd, vd, ck, cv, uniform=True), want)
    for slab, other in ((0, cv), (1, ck)):
        me = (ck, cv)[slab]
        dense = qik.MXSlab(me.codes.contiguous(), me.scales.contiguous())
        odd = torch.zeros(me.codes.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(me.codes.shape).copy_(me.codes)
        odde = torch.zeros(me.scales.numel() + 1, dtype=torch.uint8, device=DEV)[1:].view(me.scales.shape).copy_(me.scales)
        for alt in (dense, qik.MXSlab(odd, me.scales), qik.MXSlab(me.codes, odde)):
            pair = (alt, other) if slab == 0 else (other, alt)
            assert torch.equal(_call(qd, kd, vd, *pair, uniform=True), want)


@pytest.mark.parametrize("pad", [0, 8])
def test_row_counts_share_a_prepared_call(pad):
    """One geometry with another number of rows at each call, in place and (scales at odd strides) through copies."""
    B, SN, H, HKV, D = 2, 2, 4, 2, 64
    q, k, v, kc, vc = _inputs((B, SN, SN, 200, H, HKV), D, pad=0)

    def slab(codes, scales):
        wide = torch.zeros(*scales.shape[:-1], 3, dtype=torch.uint8)
        wide[..., :2] = scales
        s = wide[..., :2].to(DEV) if not pad else wide.to(DEV)[..., :2]
        return qik.MXSlab(codes.to(DEV).transpose(1, 2), s.transpose(1, 2))

    ck, cv = slab(*kc), slab(*vc)
    assert ck.in_place() == (pad == 0)
    for P in (200, 199, 3, 2, 1, 0, 64, 200):
        L = P + torch.arange(SN, dtype=torch.int32)
        for mask in (None, torch.rand(B, P + SN, generator=torch.Generator().manual_seed(P)) > 0.2):
            a, b = ck.first(P), cv.first(P)
            assert a.shape == (B, P, HKV, D) and a.codes.shape == (B, P, HKV, D // 2) and a.scales.shape == (B, P, HKV, D // 32)
            _check(_call(q, k, v, a, b, L, mask), _parts(q, k, v, kc, vc, P, om.allowed(B, SN, P, SN, L, mask)), D, torch.bfloat16)
            if mask is not None and P:
                with pytest.raises(AssertionError):
                    _call(q, k, v, a, b, L, mask[:, 1:])
    with pytest.raises(ValueError):
        _call(q, k, v, ck.first(3), cv.first(4), torch.arange(SN, dtype=torch.int32))
    with pytest.raises(ValueError):
        ck.first(201)


def test_shared_slab():
    """One prefix for every entry of a batch: a slab expanded over the batch is read in place."""
    q, k, v, kc, vc = _inputs((3, 4, 4, 70, 4, 2))
    one = [_mx(c[:1], s[:1], 70) for c, s in (kc, vc)]
    shared = [qik.MXSlab(t.codes.expand(3, -1, -1, -1), t.scales.expand(3, -1, -1, -1)) for t in one]
    assert all(t.in_place() for t in shared)
    kc, vc = ((c[:1].expand(3, -1, -1, -1), s[:1].expand(3, -1, -1, -1)) for c, s in (kc, vc))
    out = _call(q, k, v, *shared, uniform=True)
    _check(out, _parts(q, k, v, kc, vc, 70, om.allowed(3, 4, 70, 4)), 128, torch.bfloat16)


@pytest.mark.parametrize("SQ", [1, 150, 30000])
def test_offsets_past_32_bits(SQ):
    """Rows 33 MB apart and entries 7 GB apart."""
    B, SN, P, H, D = 2, 1, 200, 1, 128
    q, k, v, kc, vc = _inputs((B, SQ, SN, P, H, H))
    far, ends = 33_000_000 // 16 * 16, 33_000_000 * P // 16 * 16
    buf = torch.zeros(ends + far * (P - 1) + 128, dtype=torch.uint8, device=DEV)
    slabs = []
    for i, (c, s) in enumerate((kc, vc)):   # K and V interleaved in one buffer
        codes = buf[64 * i:].as_strided((B, P, H, 64), (ends, far, 64, 1))
        codes.copy_(c[:, :, :P].transpose(1, 2))
        slabs.append(qik.MXSlab(codes, s[:, :, :P].transpose(1, 2).contiguous().to(DEV)))
    out = _call(q, k, v, *slabs, uniform=True)
    assert _few((B, SQ, SN, P, H, H)) == (SQ < 1000)
    assert torch.equal(out, _call(q, k, v, _mx(*kc, P), _mx(*vc, P), uniform=True))
    _check(out[:, :200], _parts(q[:, :200], k, v, kc, vc, P, om.allowed(B, min(SQ, 200), P, SN)), D, torch.bfloat16)


@pytest.mark.parametrize("shape", [(2, 1, 1, 9000, 8, 2), (1, 20, 20, 5000, 8, 2), (1, 700, 700, 900, 6, 6), (1, 2816, 70, 500, 24, 24),
                                   MANY])
def test_the_same_bits_every_time_and_on_every_stream(shape):
    """Pieces that arrive in any order, two calls at once on two streams."""
    q, k, v, kc, vc = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in _inputs(shape))
    ck, cv = _mx(*kc, shape[3]), _mx(*vc, shape[3])
    want = _call(q, k, v, ck, cv, uniform=True)
    streams = [torch.cuda.Stream() for _ in range(3)]
    outs = []
    torch.cuda.synchronize()
    for i in range(24):
        with torch.cuda.stream(streams[i % 3]):
            outs.append(_call(q, k, v, ck, cv, uniform=True))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_workspace_is_shared_with_the_16_bit_call():
    """Both kinds of call in turn on one stream leave the workspace's control words zero for each other."""
    shape = (1, 3, 3, 4000, 8, 8)
    q, k, v, kc, vc = (t.to(DEV) if isinstance(t, torch.Tensor) else t for t in _inputs(shape))
    ck, cv = _mx(*kc, 4000), _mx(*vc, 4000)
    big = [t.to(DEV) for t in _inputs((1, 3000, 3000, 1, 8, 8))[:3]]
    a, b = _call(q, k, v, ck, cv, uniform=True), qik.block_causal_flash_attention(*big, None, None, uniform_full=True)
    for _ in range(3):
        assert torch.equal(_call(q, k, v, ck, cv, uniform=True), a)
        assert torch.equal(qik.block_causal_flash_attention(*big, None, None, uniform_full=True), b)


# ---- store and append ------------------------------------------------------

def _states(seed, B, S, H, D, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return [_randn(g, B, S, H, D).to(dtype).to(DEV) for _ in range(2)]


def _bytes_of(x):
    codes, scales = om.encode(x)
    return codes.transpose(1, 2), scales.transpose(1, 2)   # [B, H, S, ..]


@pytest.mark.parametrize("D", [32, 128, 256])
@pytest.mark.parametrize("S", [1, 5, 130])
def test_append_at_places(D, S):
    """Each entry's own place, some outside of the slab in part or whole: what does not fit is not written, nothing else
    changes, and the lengths are clamped."""
    B, H, cap = 5, 3, 160
    cache = qik.MXKVCache(2, B, cap, H, D, device=DEV)
    for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
        t.copy_(torch.randint(0, 250, t.shape, dtype=torch.uint8))
    before = [t.clone().cpu() for t in (cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales)]
    k, v = _states(S, B, S, H, D)
    at = torch.tensor([0, 17, cap - 2, cap, -3], dtype=torch.int32)
    cache.get_layer(1).append(k, v, at.to(DEV))
    want = [t.clone() for t in before]
    for x, (codes, scales) in ((k, (want[0], want[1])), (v, (want[2], want[3]))):
        nc, ne = _bytes_of(x)
        for b in range(B):
            for s in range(S):
                p = int(at[b]) + s
                if 0 <= p < cap:
                    codes[1, b, :, p], scales[1, b, :, p] = nc[b, :, s], ne[b, :, s]
    for t, w in zip((cache.k_codes, cache.k_scales, cache.v_codes, cache.v_scales), want):
        assert torch.equal(t.cpu(), w)
    assert cache.lengths[1].tolist() == [max(0, min(cap, int(a) + S)) for a in at]
    assert cache.lengths[0].tolist() == [0] * B
    k2, v2, _ = cache.get_layer(1).views()
    assert k2.shape == v2.shape == (B, cap, H, D)


def test_append_grows():
    """Behind the present lengths: from store, one by one, several at once, at an int, and with the lengths as places."""
    B, H, D, cap = 3, 2, 64, 40
    cache = qik.MXKVCache(1, B, cap, H, D, device=DEV)
    layer = cache.get_layer(0)
    steps = [_states(i, B, n, H, D) for i, n in enumerate((7, 1, 4, 1))]
    layer.store(*steps[0])
    layer.append(*steps[1])
    layer.append(*steps[2], None)
    layer.append(*steps[3], cache.lengths[0])
    assert cache.lengths[0].tolist() == [13] * B and int(cache._arrivals[0]) == 0
    want = qik.MXKVCache(1, B, cap, H, D, device=DEV)
    want.get_layer(0).store(*(torch.cat(t, 1) for t in zip(*steps)))
    for n in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(getattr(cache, n), getattr(want, n))
    layer.append(*steps[2], 30)
    assert cache.lengths[0].tolist() == [34] * B and layer.views()[0].shape[1] == 34
    with pytest.raises(ValueError):
        layer.append(*steps[0])
    layer.append(*_states(9, B, 6, H, D))
    with pytest.raises(ValueError):
        layer.append(*steps[1])
    with pytest.raises(ValueError):
        layer.append(*steps[1], cap)
    with pytest.raises(ValueError):
        layer.append(*steps[1], -1)
    with pytest.raises(ValueError):
        layer.store(*_states(1, B, cap + 1, H, D))
    for bad in (torch.zeros(B, dtype=torch.int64, device=DEV), torch.zeros(B + 1, dtype=torch.int32, device=DEV),
                torch.zeros(B, dtype=torch.int32)):
        with pytest.raises(ValueError):
            layer.append(*steps[1], bad)
    for bad in (_states(1, B, 1, H, 128), _states(1, B + 1, 1, H, D), [steps[1][0], steps[2][1]]):
        with pytest.raises(ValueError):
            layer.append(*bad)
    assert cache.lengths[0].tolist() == [40] * B
    # places that overlap the lengths otherwise are copied first
    two = qik.MXKVCache(2, B, cap, H, D, device=DEV)
    two.lengths.copy_(torch.tensor([[1, 2, 3], [4, 5, 6]], dtype=torch.int32))
    two.get_layer(1).append(*steps[1], two.lengths.view(-1)[2:5])
    assert two.lengths.tolist() == [[1, 2, 3], [4, 5, 6]]   # 3, 4, 5, and one more each
    two.get_layer(1).append(*_states(3, B, 0, H, D))
    assert two.lengths.tolist() == [[1, 2, 3], [4, 5, 6]]


def test_store_of_empty_and_lowered_lengths():
    B, H, D = 2, 2, 64
    cache = qik.MXKVCache(1, B, 9, H, D, device=DEV)
    layer = cache.get_layer(0)
    layer.store(*_states(1, B, 8, H, D))
    cache.lengths[0, 1] = 3     # entry 1 is shorter: a padded batch
    k, v = layer.get()
    assert (k[1, 3:] == 0).all() and (v[1, 3:] == 0).all() and k[1, 2].any() and k[0, 7].any()
    ck, cv, _ = layer.views()
    q, nk, nv = (_randn(torch.Generator().manual_seed(5), B, 1, n, D).to(torch.bfloat16).to(DEV) for n in (4, H, H))
    out = qik.block_causal_flash_attention(q, nk, nv, None, None, cache_k=ck, cache_v=cv, uniform_full=True)
    ok = om.allowed(B, 1, 8, 1, lengths=torch.tensor([8, 3]))
    keys = [torch.cat((om.decode(c[0, :, :, :8], s[0, :, :, :8]).transpose(1, 2), t.cpu().double()), 1)
            for c, s, t in ((cache.k_codes, cache.k_scales, nk), (cache.v_codes, cache.v_scales, nv))]
    _check(out, om.attention(q.cpu().double(), *keys, ok), D, torch.bfloat16)
    layer.store(*_states(2, B, 0, H, D))
    assert cache.lengths[0].tolist() == [0, 0] and layer.get()[0].shape == (B, 0, H, D)


def test_infinities_make_their_block_nan():
    k, v = _states(1, 1, 3, 1, 64)
    k[0, 1, 0, 40], v[0, 2, 0, 3] = torch.inf, torch.nan
    cache = qik.MXKVCache(1, 1, 3, 1, 64, device=DEV)
    cache.get_layer(0).store(k, v)
    gk, gv = cache.get_layer(0).get()
    assert gk[0, 1, 0, 32:].isnan().all() and torch.isfinite(gk[0, 1, 0, :32]).all() and torch.isfinite(gk[0, [0, 2]]).all()
    assert gv[0, 2, 0, :32].isnan().all() and torch.isfinite(gv[0, :2]).all()


def test_store_converts_and_copies():
    """Other types, other layouts, the CPU: as the values say, whatever layout came before."""
    B, S, H, D = 2, 6, 2, 64
    k, v = _states(4, B, S, H, D)
    cache = qik.MXKVCache(1, B, S, H, D, device=DEV)
    layer = cache.get_layer(0)
    layer.store(k, v)
    want = [t.clone() for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales)]
    odd = torch.zeros(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape)
    off = torch.zeros(k.numel() + 1, dtype=k.dtype, device=DEV)[1:].view(k.shape)
    wide = torch.zeros(B, S, H, D + 8, dtype=k.dtype, device=DEV)[..., :D]
    for a, b in ((k.float(), v.double()), (k.cpu(), v), (odd.copy_(k), v), (k, off.copy_(v)),
                 (wide.copy_(k), v), (k.transpose(2, 3).contiguous().transpose(2, 3), v), (k, v)):
        for t in (cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales):
            t.zero_()
        layer.store(a, b)
        for t, w in zip((cache.k_codes, cache.v_codes, cache.k_scales, cache.v_scales), want):
            assert torch.equal(t, w)


def test_store_of_many_heads():
    """More (entry, head) pairs than a grid has rows."""
    B, H, D = 40, 1700, 32
    x = torch.randn(B, 1, H, D, device=DEV, dtype=torch.bfloat16)
    cache = qik.MXKVCache(1, B, 2, H, D, device=DEV)
    cache.get_layer(0).append(x, -x, torch.ones(B, dtype=torch.int32, device=DEV))
    wc, we = _bytes_of(x)
    assert torch.equal(cache.k_codes[0, :, :, 1:].cpu(), wc) and torch.equal(cache.k_scales[0, :, :, 1:].cpu(), we)
    cache.get_layer(0).append(x, -x)
    assert cache.lengths[0].tolist() == [2] * B and int(cache._arrivals[0]) == 0
    k, v = cache.get_layer(0).get()
    assert torch.equal(k, -v) and torch.equal(k[:, 1:].cpu().double(), om.decode(wc, we).transpose(1, 2))


# ---- graphs and the processor ----------------------------------------------

@pytest.mark.parametrize("S", [1, 6])
def test_captured_step_grows_with_every_replay(S):
    """append + attention captured once; each replay is the next step, as eager steps on another cache say."""
    B, H, HKV, D, cap, start = 3, 8, 2, 128, 3000, 2500
    caches = [qik.MXKVCache(1, B, cap, HKV, D, device=DEV) for _ in range(2)]
    prefix = _states(1, B, start, HKV, D)
    for c in caches:
        c.get_layer(0).store(*prefix)
        c.lengths[0, 1] = 1200
    q = torch.empty(B, S, H, D, dtype=torch.bfloat16, device=DEV)
    k, v = (torch.empty(B, S, HKV, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    L = torch.empty(B, S, dtype=torch.int32, device=DEV)

    def step(cache):
        layer = cache.get_layer(0)
        torch.add(cache.lengths[0][:, None], torch.arange(S, device=DEV, dtype=torch.int32), out=L)
        layer.append(k, v)
        ck, cv, _ = layer.views(cap)
        return qik.block_causal_flash_attention(q, k[:, :0], v[:, :0], L, None, cache_k=ck, cache_v=cv)

    def fill(i):
        g = torch.Generator().manual_seed(100 + i)
        for t in (q, k, v):
            t.copy_(_randn(g, *t.shape).to(torch.bfloat16))

    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    fill(0)
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        saved = caches[0].lengths.clone()
        step(caches[0])                      # warm-up
        caches[0].lengths.copy_(saved)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        out = step(caches[0])
    for i in range(5):
        fill(i)
        graph.replay()
        got = out.clone()
        want = step(caches[1])
        torch.cuda.synchronize()
        assert torch.equal(got, want), i
        assert torch.equal(caches[0].lengths, caches[1].lengths)
        for n in ("k_codes", "v_scales"):
            assert torch.equal(getattr(caches[0], n), getattr(caches[1], n))
    assert caches[0].lengths[0].tolist() == [start + 5 * S, 1200 + 5 * S, start + 5 * S]
    assert caches[0].get_layer(0).views()[0].shape[1] == cap   # the host no longer knows them


def test_two_graphs_on_one_stream():
    shape = (1, 1, 1, 20000, 8, 2)
    data = [[t.to(DEV) if isinstance(t, torch.Tensor) else t for t in _inputs(shape, seed=s)] for s in (1, 2)]
    slabs = [(_mx(*d[3], 20000), _mx(*d[4], 20000)) for d in data]
    want = [_call(*d[:3], *s, uniform=True) for d, s in zip(data, slabs)]
    stream, graphs, outs = torch.cuda.Stream(), [], []
    torch.cuda.synchronize()
    for d, s in zip(data, slabs):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=stream):
            outs.append(_call(*d[:3], *s, uniform=True))
        graphs.append(g)
    for _ in range(4):
        for o in outs:
            o.zero_()
        for g in graphs:
            g.replay()
        eager = [_call(*d[:3], *s, uniform=True) for d, s in zip(data, slabs)]
        torch.cuda.synchronize()
        for o, e, w in zip(outs, eager, want):
            assert torch.equal(o, w) and torch.equal(e, w)


class _Lin(torch.nn.Linear):
    def __init__(self, i, o):
        super().__init__(i, o, device=DEV, dtype=torch.bfloat16)


class _Attn:
    """What the processor reads from an attention module."""

    def __init__(self, dim, H, D):
        self.heads = H
        self.to_q, self.to_k, self.to_v = (_Lin(dim, H * D).requires_grad_(False) for _ in range(3))
        self.norm_q, self.norm_k = (type("Norm", (), {"weight": torch.rand(D, device=DEV) + 0.5, "eps": e})() for e in (1e-6, 1e-5))
        self.to_out = [torch.nn.Identity(), torch.nn.Identity()]


@pytest.mark.parametrize("key_mask", [False, True])
def test_processor_with_axes_and_a_4bit_slab(key_mask):
    """The whole layer: projections, norm and rotation, the slab, prefill and decode, as the public calls compose."""
    torch.manual_seed(1)
    B, H, D, dim, text, img, T = 2, 4, 128, 256, 40, 150, 130
    P = text + img
    attn, proc = _Attn(dim, H, D), qik.QwenImage21KernelProcessor()
    pos = torch.randint(0, 90, (3, P + T), device=DEV)
    axes = (16, 56, 56)
    rope_p, rope_t = qik.AxialRope(pos[:, :P], axes), qik.AxialRope(pos[:, P:], axes)
    cache = qik.MXKVCache(1, B, P + 8, H, D, device=DEV)
    x, y = (torch.randn(B, n, dim, device=DEV, dtype=torch.bfloat16) for n in (P, T))
    segments = [(0, text, True), (text, P, False)]
    out = proc(attn, x, rotary_emb=rope_p, layer_cache=cache.get_layer(0), kv_cache_mode="extract", cache_write_slice=slice(0, P),
               segments=segments)
    q, k, v = (m(x).unflatten(-1, (H, D)) for m in (attn.to_q, attn.to_k, attn.to_v))
    q, k = qik.fused_qk_norm_rope(q, k, attn.norm_q.weight, attn.norm_k.weight, rope_p, 1e-6, 1e-5)
    L = qik.build_prefix_lengths(segments, P, P, torch.device(DEV, torch.cuda.current_device()))
    assert torch.equal(out, qik.block_causal_flash_attention(q, k, v, L, None).flatten(2, 3))
    for codes, scales, t in ((cache.k_codes, cache.k_scales, k), (cache.v_codes, cache.v_scales, v)):
        wc, we = _bytes_of(t)
        assert torch.equal(codes[0, :, :, :P].cpu(), wc) and torch.equal(scales[0, :, :, :P].cpu(), we)
    mask = None
    if key_mask:
        mask = torch.rand(B, P + T, device=DEV) < 0.8
    out = proc(attn, y, attention_mask=mask, rotary_emb=rope_t, layer_cache=cache.get_layer(0), kv_cache_mode="cached")
    q, k, v = (m(y).unflatten(-1, (H, D)) for m in (attn.to_q, attn.to_k, attn.to_v))
    q, k = qik.fused_qk_norm_rope(q, k, attn.norm_q.weight, attn.norm_k.weight, rope_t, 1e-6, 1e-5)
    ok = om.allowed(B, T, P, T, None, None if mask is None else mask.cpu())
    keys = [torch.cat((om.decode(c[0, :, :, :P], s[0, :, :, :P]).transpose(1, 2), t.cpu().double()), 1)
            for c, s, t in ((cache.k_codes, cache.k_scales, k), (cache.v_codes, cache.v_scales, v))]
    _check(out.unflatten(-1, (H, D)), om.attention(q.cpu().double(), *keys, ok), D, torch.bfloat16)


def test_refusals_on_the_device():
    q, k, v, kc, vc = _inputs((2, 3, 3, 20, 4, 2))
    ck, cv = _mx(*kc, 20), _mx(*vc, 20)
    q, k, v = q.to(DEV), k.to(DEV), v.to(DEV)
    L = torch.zeros(3, dtype=torch.int32, device=DEV)

    def refused(*a, error=(ValueError, AssertionError), **kw):
        with pytest.raises(error):
            qik.block_causal_flash_attention(*a, **{**dict(cache_k=ck, cache_v=cv), **kw})

    refused(q, k[..., :64], v[..., :64], L, None)
    refused(q, k[:1], v[:1], L, None)
    refused(q, k[:, :2], v, L, None)
    refused(q[:, :, :3], k, v, L, None)
    refused(q.float(), k.float(), v.float(), L, None)
    refused(q.half(), k, v, L, None)
    refused(q, k, v, L[:2], None)
    refused(q, k, v, L[None].expand(3, -1), None)
    refused(q, k, v, L.cpu(), None)
    refused(q, k, v, L, torch.ones(2, 22, dtype=torch.bool, device=DEV))
    refused(q, k, v, L, torch.ones(3, 23, dtype=torch.bool, device=DEV))
    refused(q, k, v, L, torch.ones(2, 23, dtype=torch.bool))
    refused(q, k, v, L, None, cache_v=_mx(vc[0], vc[1], 19))
    refused(q, k, v, L, None, cache_k=_mx(kc[0][:1], kc[1][:1], 20))
    refused(q, k, v, L, None, cache_k=_mx(kc[0][:, :1], kc[1][:, :1], 20))
    refused(q, k, v, L, None, cache_v=k)
    ln = torch.tensor([20, 3], dtype=torch.int32, device=DEV)
    refused(q, k, v, L, None, cache_k=_mx(*kc, 20, ln))
    refused(q, k, v, L, None, cache_v=_mx(*vc, 20, ln))


@pytest.mark.parametrize("shape", [FEW, MANY, (2, 40, 40, 64, 6, 3)])
def test_without_lengths_every_key_counts(shape):
    """prefix_lengths None, with and without a mask and slab lengths: as full lengths, to the bit."""
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape, seed=23)
    valid = torch.rand(B, P + SN, generator=torch.Generator().manual_seed(23)) > 0.3
    full = torch.full((SQ,), P + SN - 1, dtype=torch.int32)
    ln = torch.tensor([P // 3] * (B - 1) + [P], dtype=torch.int32, device=DEV)
    for mask in (None, valid):
        for lengths in (None, ln):
            ck, cv = (_mx(*t, P, lengths) for t in (kc, vc))
            want = _call(q, k, v, ck, cv, full, mask)
            for uniform in (False, True):
                assert torch.equal(_call(q, k, v, ck, cv, None, mask, uniform), want)


@pytest.mark.parametrize("B,S,P,H,HKV,D,dtype", [(2, 1, 2000, 8, 2, 128, torch.bfloat16), (7, 3, 900, 4, 4, 64, torch.float16),
                                                 (64, 1, 300, 4, 1, 128, torch.bfloat16), (65, 2, 257, 2, 1, 32, torch.bfloat16),
                                                 (130, 1, 700, 1, 1, 64, torch.bfloat16), (3, 1, 1500, 4, 4, 256, torch.float16),
                                                 (300, 1, 100, 2, 2, 64, torch.bfloat16)])
@pytest.mark.parametrize("how", ["spread", "one long", "none", "negative and past the end", "all"])
def test_entries_of_many_lengths(B, S, P, H, HKV, D, dtype, how):
    """The pieces of all entries together: none lost, none read twice, whatever the lengths sum up to."""
    q, k, v, kc, vc = _inputs((B, S, S, P, H, HKV), D, dtype, pad=0)
    g = torch.Generator().manual_seed(B)
    ln = torch.randint(0, P + 1, (B,), generator=g, dtype=torch.int32)
    if how == "one long":
        ln = ln.clamp_max(3)
        ln[B - 1] = P
    elif how == "none":
        ln.zero_()
    elif how == "all":
        ln.fill_(P)
    elif how != "spread":
        ln = torch.where(torch.rand(B, generator=g) < 0.5, ln - P, ln + P // 2)
    slabs = [_mx(*t, P, ln.to(DEV)) for t in (kc, vc)]
    ok = om.allowed(B, S, P, S, None, None, ln)
    _check(_call(q, k, v, *slabs), _parts(q, k, v, kc, vc, P, ok), D, dtype)
    out = _call(q, k[:, :0], v[:, :0], *slabs)   # the slab alone
    _check(out, _parts(q, k[:, :0], v[:, :0], kc, vc, P, ok[..., :P]), D, dtype)
    assert (out[(ln <= 0).to(DEV)] == 0).all()
    assert torch.equal(out, _call(q, k[:, :0], v[:, :0], *slabs))


@pytest.mark.parametrize("S", [1, 3])
def test_lengths_of_a_slab_without_rows(S):
    """Entries with lengths over no slab row: the fresh keys alone, also where they are cut into pieces."""
    B, SN, H, HKV, D = 3, 2000, 4, 2, 128
    q, k, v, kc, vc = _inputs((B, S, SN, 0, H, HKV), D, pad=4)
    ln = torch.tensor([0, 7, -2], dtype=torch.int32, device=DEV)
    slabs = [_mx(*t, 0, ln) for t in (kc, vc)]
    _check(_call(q, k, v, *slabs), _parts(q, k, v, kc, vc, 0, om.allowed(B, S, 0, SN)), D, torch.bfloat16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("shape", [FEW, (1, 40, 40, 400, 2, 2), MANY])
def test_causal_lengths_far_below_zero(shape, D, dtype):
    """Rows of length -2^31 and the like, next to rows that see keys, see nothing."""
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape, D, dtype, seed=31)
    ck, cv = _mx(*kc, P), _mx(*vc, P)
    g = torch.Generator().manual_seed(31)
    L = torch.randint(0, P + SN, (B, SQ), generator=g, dtype=torch.int32)
    none = torch.rand(B, SQ, generator=g) < 0.4
    none[:, 1] = True
    none[:, 0], L[:, 0] = False, P + SN - 1
    valid = torch.rand(B, P + SN, generator=g) < 0.8
    for mask in (None, valid):
        want = _call(q, k, v, ck, cv, torch.where(none, -1, L), mask)
        assert (want.cpu()[none] == 0).all()
        for low in (-2 ** 31, -2 ** 31 + 3, -2):
            assert torch.equal(_call(q, k, v, ck, cv, torch.where(none, low, L), mask), want), low


@pytest.mark.parametrize("shape", [FEW, MANY])
def test_causal_lengths_in_64_bits(shape):
    """Past 32 bits a length is as its nearest one: no key, or every one."""
    B, SQ, SN, P, H, HKV = shape
    q, k, v, kc, vc = _inputs(shape, seed=37)
    ck, cv = _mx(*kc, P), _mx(*vc, P)
    g = torch.Generator().manual_seed(37)
    L = torch.randint(-1, P + SN, (SQ,), generator=g)
    far = torch.tensor([-2 ** 63, -2 ** 40, -2 ** 32, 2 ** 31, 2 ** 32, 2 ** 40, 2 ** 63 - 1])
    where = torch.rand(SQ, generator=g) < 0.5
    where[0] = True
    pick = far[torch.randint(0, far.numel(), (SQ,), generator=g)]
    near = torch.where(pick < 0, -1, P + SN - 1)
    want = _call(q, k, v, ck, cv, torch.where(where, near, L).to(torch.int32))
    assert torch.equal(_call(q, k, v, ck, cv, torch.where(where, pick, L)), want)
    assert torch.equal(_call(q, k, v, ck, cv, torch.where(where, pick, L)[None].expand(B, -1)), want)


def _spreads(B, SQ, SN, P, H, HKV, D) -> bool:
    """Whether the kernel deals out the keys of all entries together: the plan then aims at more pieces than an entry alone
    is ever cut into (a piece has a step of 32 keys for each of 8 waves, two from 8 pieces on)."""
    few, tiles, pieces = (ctypes.c_int32() for _ in range(3))
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.load().qik_mx_attn_plan(B, SQ, SN, P, H, HKV, D, 1, cus, ctypes.byref(few), ctypes.byref(tiles),
                                        ctypes.byref(pieces)) == 0
    steps = max((-(-P // 32) + -(-SN // 32)) // 8, 1)
    return few.value == 1 and tiles.value == 1 and pieces.value > max(steps // 2, min(steps, 8))


# B, SQ, SN, P, H, HKV, D, dtype: entries below, at and past a wave's 64, past two and four times that
TOGETHER = [(24, 1, 1, 4000, 16, 4, 128, torch.bfloat16), (64, 1, 2, 1100, 4, 1, 128, torch.bfloat16),
            (65, 1, 0, 1100, 4, 1, 128, torch.float16), (65, 2, 2, 4500, 4, 2, 32, torch.bfloat16),
            (128, 1, 1, 1100, 4, 1, 128, torch.bfloat16), (130, 1, 0, 1100, 8, 2, 64, torch.float16),
            (129, 3, 3, 1100, 4, 1, 256, torch.bfloat16), (200, 1, 2, 1600, 4, 1, 128, torch.bfloat16),
            (300, 1, 0, 620, 2, 2, 256, torch.bfloat16), (300, 1, 2, 1558, 4, 1, 32, torch.float16)]


@pytest.mark.parametrize("case", TOGETHER)
def test_entries_dealt_out_together(case):
    """Pieces over all entries, in chunks of a wave's lanes: no key lost, none read twice, with and without masks."""
    B, SQ, SN, P, H, HKV, D, dtype = case
    assert _spreads(*case[:-1])
    g = torch.Generator().manual_seed(B + D)
    q, k, v = (_randn(g, B, n, h, D).to(dtype) for n, h in ((SQ, H), (SN, HKV), (SN, HKV)))
    kc, vc = ((torch.randint(0, 256, (B, HKV, P, D // 2), generator=g, dtype=torch.uint8),
               torch.randint(123, 127, (B, HKV, P, D // 32), generator=g, dtype=torch.uint8)) for _ in range(2))
    every = torch.randint(0, P + 1, (B,), generator=g, dtype=torch.int32)
    one = every.clamp_max(3)
    one[B * 2 // 3] = P
    few = torch.where(torch.arange(B) < B - 3, 0, every)
    ends = torch.where(torch.rand(B, generator=g) < 0.5, every - P, every + P // 2)
    L = torch.randint(-1, P + SN, (B, SQ), generator=g, dtype=torch.int32)
    valid = torch.rand(B, P + SN, generator=g) < 0.8
    keys, values = (torch.cat((om.decode(c, s).transpose(1, 2).to(DEV), t.to(DEV).double()), 1) for (c, s), t in ((kc, k), (vc, v)))
    for ln, lengths, mask in ((every, None, None), (every, L, None), (every, None, valid), (every, L, valid), (one, None, None),
                              (one, L, valid), (few, None, None), (few, None, valid), (torch.full_like(every, P), None, None),
                              (torch.zeros_like(every), None, None), (ends, None, None), (ends, L, valid)):
        slabs = [_mx(*t, P, ln.to(DEV)) for t in (kc, vc)]
        out = _call(q, k, v, *slabs, lengths, mask)
        ok = om.allowed(B, SQ, P, SN, lengths, mask, ln).to(DEV)
        _check(out, om.attention(q.to(DEV).double(), keys, values, ok), D, dtype)
        assert (out[~ok.any(-1)] == 0).all()
        assert torch.equal(out, _call(q, k, v, *slabs, lengths, mask))


def test_store_and_read_past_32_bits():
    """Rows of a slab and of the states behind 4 GB; an entry's last rows, which alone are not zeros."""
    B, H, D, cap, S = 2, 16, 256, 1_200_000, 3
    assert H * B * cap * D // 2 > 2 ** 32
    cache = qik.MXKVCache(1, B, cap, H, D, device=DEV)
    buf = torch.zeros(2_300_000_000 + 2 * S * H * D, dtype=torch.bfloat16, device=DEV)
    x = _states(3, B, S, H, D)
    far = [buf[i * S * H * D:].as_strided((B, S, H, D), (2_300_000_000 // 8 * 8, H * D, D, 1)).copy_(t) for i, t in enumerate(x)]
    layer = cache.get_layer(0)
    layer.append(*far, cap - S)
    assert cache.lengths[0].tolist() == [cap] * B
    got = layer.get()
    for t, g, codes, scales in zip(x, got, (cache.k_codes, cache.v_codes), (cache.k_scales, cache.v_scales)):
        wc, we = _bytes_of(t)
        assert torch.equal(codes[0, :, :, -S:].cpu(), wc) and torch.equal(scales[0, :, :, -S:].cpu(), we)
        assert not codes[0, -1, -1, :-S].any() and not codes[0, 0, 0, :-S].any()
        assert torch.equal(g[:, -S:].cpu().double(), om.decode(wc, we).transpose(1, 2))
        assert not g[-1, -1000:-S].any()


@pytest.mark.parametrize("fill", ["store", "append at an int", "append"])
def test_a_cache_filled_anew_after_its_step_was_captured(fill):
    """get() and the default views hold what replays appended behind an eager store or append, as an eager cache's do."""
    B, H, HKV, D, cap = 2, 4, 2, 64, 300
    caches = [qik.MXKVCache(1, B, cap, HKV, D, device=DEV) for _ in range(2)]
    for c in caches:
        c.get_layer(0).store(*_states(1, B, 80, HKV, D))
    k, v = (torch.empty(B, 1, HKV, D, dtype=torch.bfloat16, device=DEV) for _ in range(2))
    graph, stream = torch.cuda.CUDAGraph(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        caches[0].get_layer(0).append(k, v)
    for c in caches:
        layer = c.get_layer(0)
        if fill == "store":
            layer.store(*_states(2, B, 50, HKV, D))
        elif fill == "append":
            layer.append(*_states(2, B, 50, HKV, D))
        else:
            layer.append(*_states(2, B, 10, HKV, D), 40)
    for i in range(10):
        k.copy_(_states(10 + i, B, 1, HKV, D)[0])
        v.copy_(_states(30 + i, B, 1, HKV, D)[1])
        graph.replay()
        caches[1].get_layer(0).append(k, v)
    torch.cuda.synchronize()
    n = int(caches[1].lengths[0, 0])
    assert torch.equal(caches[0].lengths, caches[1].lengths) and n == (140 if fill == "append" else 60)
    q = _randn(torch.Generator().manual_seed(3), B, 1, H, D).to(torch.bfloat16).to(DEV)
    for c in caches:
        ck, cv, _ = c.get_layer(0).views()
        keys = [om.decode(x[0, :, :, :n], e[0, :, :, :n]).transpose(1, 2) for x, e in ((c.k_codes, c.k_scales), (c.v_codes, c.v_scales))]
        _check(_call(q, k[:, :0], v[:, :0], ck, cv), om.attention(q.cpu().double(), *keys, om.allowed(B, 1, n, 0)), D, torch.bfloat16)
        for got, want in zip(c.get_layer(0).get(), keys):
            assert torch.equal(got[:, :n].cpu().double(), want) and not got[:, n:].any()
    for t in ("k_codes", "k_scales", "v_codes", "v_scales"):
        assert torch.equal(*(getattr(c, t)[:, :, :, :n] for c in caches))


@pytest.mark.parametrize("inference", [False, True])
def test_an_entry_that_starts_anew(inference):
    """Entries set back by the program take tokens again, in every entry up to the slab's last row and no further."""
    B, H, D, cap = 3, 2, 64, 9
    with torch.inference_mode(inference):
        cache = qik.MXKVCache(1, B, cap, H, D, device=DEV)
        layer = cache.get_layer(0)
        layer.store(*_states(1, B, 8, H, D))
        cache.lengths[0, 1:] = torch.tensor([0, 3], dtype=torch.int32, device=DEV)
        k, v = _states(2, B, 4, H, D)
        layer.append(k, v)
        assert cache.lengths[0].tolist() == [9, 4, 7] and int(cache._arrivals[0]) == 0
        for t, codes, scales in ((k, cache.k_codes, cache.k_scales), (v, cache.v_codes, cache.v_scales)):
            wc, we = _bytes_of(t)
            for b, at in enumerate((8, 0, 3)):
                n = min(4, cap - at)
                assert torch.equal(codes[0, b, :, at:at + n].cpu(), wc[b, :, :n])
                assert torch.equal(scales[0, b, :, at:at + n].cpu(), we[b, :, :n])
        layer.append(*_states(3, B, 9, H, D))
        assert cache.lengths[0].tolist() == [9] * B
