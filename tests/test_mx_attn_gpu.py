"""GPU tests of the 4-bit slab and of ``block_causal_flash_attention`` over it, against the float64 oracle."""

import ctypes

import pytest
import torch

import qwen_image_kernel_amd as qik
from oracle import mx_slab as om
from qwen_image_kernel_amd import _lib

pytestmark = pytest.mark.gpu

DEV = "cuda"


def _randn(g, *shape):
    x = torch.randn(*shape, generator=g)
    x[..., 3::32] *= 4.0
    return x


def _slab(g, B, P, H, D, pad=0):
    """A slab of P rows in a buffer of P + pad (garbage behind), [B, H, P, D] in memory; its bytes."""
    codes, scales = om.encode(_randn(g, B, H, P + pad, D))
    scales[:, :, P:] = 255
    return codes, scales


def _mx(codes, scales, P, lengths=None):
    c, s = codes.to(DEV), scales.to(DEV)
    return qik.MXSlab(c[:, :, :P].transpose(1, 2), s[:, :, :P].transpose(1, 2), lengths)


def _check(out, parts, D, dtype):
    want, lim = parts["out"], om.bound(parts, D, dtype)
    off = (out.to(want.device).double() - want).abs()
    assert torch.isfinite(out).all()
    worst = float((off / lim).max()) if off.numel() else 0.0
    assert worst <= 1.0, worst


def _case(B, SQ, SN, P, H, HKV, D, dtype, seed, L=None, valid=None, lengths=None, uniform=False, pad=5):
    g = torch.Generator().manual_seed(seed)
    q = _randn(g, B, SQ, H, D).to(dtype)
    k, v = (_randn(g, B, SN, HKV, D).to(dtype) for _ in range(2))
    kc, vc = _slab(g, B, P, HKV, D, pad), _slab(g, B, P, HKV, D, pad)
    ln = None if lengths is None else torch.tensor(lengths, dtype=torch.int32)
    ck, cv = (_mx(*t, P, None if ln is None else ln.to(DEV)) for t in (kc, vc))
    dev = [None if t is None else t.to(DEV) for t in (L, valid)]
    out = qik.block_causal_flash_attention(q.to(DEV), k.to(DEV), v.to(DEV), dev[0], dev[1], cache_k=ck, cache_v=cv,
                                           uniform_full=uniform)
    ok = om.allowed(B, SQ, P, SN, None if uniform else L, valid, ln)
    keys, values = (torch.cat((om.decode(c[:, :, :P], s[:, :, :P]).transpose(1, 2), t.double()), 1)
                    for (c, s), t in ((kc, k), (vc, v)))
    on = DEV if SQ * (P + SN) * H > 2_000_000 else "cpu"   # where the oracle computes
    parts = om.attention(*(t.to(on) for t in (q.double(), keys, values, ok)))
    _check(out, parts, D, dtype)
    return out, ok


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("e", [1, 64, 100, 126, 127, 130, 200, 254])
def test_every_code_at_a_scale(dtype, e):
    """get() gives every element at a scale byte exactly (in fp16 rounded once)."""
    cache = qik.MXKVCache(1, 1, 4, 2, 32, device=DEV, dtype=dtype)
    codes = torch.arange(16, dtype=torch.uint8)
    row = (codes | (codes.flip(0) << 4))
    cache.k_codes[0] = row.to(DEV)
    cache.v_codes[0] = row.flip(0).to(DEV)
    cache.k_scales.fill_(e)
    cache.v_scales.fill_(e)
    cache.lengths.fill_(4)
    cache._host_lengths[0] = 4
    got = cache.get_layer(0).get()
    for t, c in zip(got, (cache.k_codes, cache.v_codes)):
        want = om.decode(c[0].transpose(1, 2), torch.full((1, 4, 2, 1), e, dtype=torch.uint8))
        assert torch.equal(t.cpu().double(), want.to(torch.float32).to(dtype).double())


@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("P", [1, 33, 203])
def test_store_bytes(D, dtype, P):
    """store writes the format's bytes, from strided rows, and get gives their values."""
    B, H = 2, 3
    g = torch.Generator().manual_seed(D + P)
    qkv = (_randn(g, B, P, 3 * H, D) * torch.exp2(torch.randint(-9, 6, (B, P, 3 * H, 1), generator=g).float())).to(dtype)
    cache = qik.MXKVCache(2, B, P + 7, H, D, device=DEV, dtype=dtype)
    d = qkv.to(DEV)
    cache.get_layer(1).store(d[:, :, H:2 * H], d[:, :, 2 * H:])
    for codes, scales, x in ((cache.k_codes, cache.k_scales, qkv[:, :, H:2 * H]),
                             (cache.v_codes, cache.v_scales, qkv[:, :, 2 * H:])):
        wc, we = om.encode(x)
        assert torch.equal(codes[1, :, :, :P].cpu().transpose(1, 2), wc)
        assert torch.equal(scales[1, :, :, :P].cpu().transpose(1, 2), we)
        assert not codes[0].any() and not codes[1, :, :, P:].any() and not scales[1, :, :, P:].any()
    assert cache.lengths.tolist() == [[0] * B, [P] * B]
    k, v = cache.get_layer(1).get()
    assert k.shape == (B, P, H, D)
    assert torch.equal(k.cpu().double(), om.decode(cache.k_codes[1, :, :, :P], cache.k_scales[1, :, :, :P]).transpose(1, 2)
                       .float().to(dtype).double())


SHAPES = [
    # B, SQ, SN, P, H, HKV: tokens, drafted tokens, row tiles, steps that end inside a tile, fresh keys alone
    (1, 1, 0, 1, 1, 1), (1, 1, 1, 31, 4, 1), (2, 1, 1, 1000, 8, 2), (1, 1, 0, 4097, 32, 8), (3, 5, 5, 129, 12, 4),
    (1, 8, 8, 300, 8, 1), (1, 1, 1, 3, 64, 1), (2, 3, 70, 32, 6, 6), (1, 2, 64, 65, 3, 3), (1, 1, 9, 20000, 2, 1),
]
# the kernel of many rows in each of its forms: a row block for a workgroup of two
# groups, two such workgroups for a row block, the queue, the queue with items of
# eight pieces; grouped heads
MANY = [(1, 700, 700, 150, 24, 24), (2, 1024, 1000, 300, 8, 8), (2, 700, 690, 150, 48, 24), (1, 2816, 70, 500, 24, 24)]
# more rows than a tile, few enough for the other
MORE = [(1, 65, 65, 70, 2, 2), (2, 130, 40, 333, 4, 2), (1, 300, 300, 64, 7, 1), (1, 257, 0, 1500, 3, 3)]


def _few(shape, D=128, ragged=False):
    """Whether a call of this shape runs the kernel of few rows on this device."""
    B, SQ, SN, P, H, HKV = shape
    few, tiles, pieces = (ctypes.c_int32() for _ in range(3))
    cus = torch.cuda.get_device_properties(0).multi_processor_count
    assert _lib.load().qik_mx_attn_plan(B, SQ, SN, P, H, HKV, D, int(ragged), cus, ctypes.byref(few), ctypes.byref(tiles),
                                        ctypes.byref(pieces)) == 0
    return bool(few.value)


def test_both_kernels_are_covered():
    assert all(_few(s) for s in SHAPES + MORE) and not any(_few(s) for s in MANY)


@pytest.mark.parametrize("shape", SHAPES + MORE + MANY)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_uniform(shape, D, dtype):
    _case(*shape, D, dtype, 7 + D, uniform=True)


@pytest.mark.parametrize("shape", SHAPES[2:6] + MORE[:2] + MANY[:2])
@pytest.mark.parametrize("D", [32, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_other_head_dims(shape, D, dtype):
    B, SQ, SN, P, _, _ = shape
    _case(*shape, D, dtype, 11 + D, uniform=True)
    g = torch.Generator().manual_seed(2)
    _case(*shape, D, dtype, 13 + D, L=torch.randint(-1, P + SN, (SQ,), generator=g, dtype=torch.int32),
          valid=torch.rand(B, P + SN, generator=g) < 0.7)


@pytest.mark.parametrize("shape", SHAPES + MORE + MANY)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_masks_and_lengths(shape, dtype):
    """Ragged lengths (one empty), causal limits of each entry, rows and keys that see nothing."""
    B, SQ, SN, P, H, HKV = shape
    g = torch.Generator().manual_seed(SQ + P)
    lengths = torch.randint(0, P + 1, (B,), generator=g).tolist()
    lengths[-1] = 0 if B > 1 else P
    L = torch.randint(-1, P + SN, (B, SQ), generator=g, dtype=torch.int32)
    L[:, 0] = -1
    valid = torch.rand(B, P + SN, generator=g) < 0.8
    _case(*shape, 128, dtype, 3, uniform=True, lengths=lengths)
    out, ok = _case(*shape, 128, dtype, 4, L=L, lengths=lengths)
    assert (out.cpu()[~ok.any(-1)] == 0).all()
    _case(*shape, 128, dtype, 5, L=L[0], valid=valid)
    out, ok = _case(*shape, 128, dtype, 6, L=L, valid=valid, lengths=lengths)
    assert (out.cpu()[~ok.any(-1)] == 0).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("e", [0, 255])
def test_every_code_at_the_ends_of_the_scale(dtype, e):
    """Scale byte 0 is 2^-127, also for elements that are not zero; 255 makes its block NaN."""
    cache = qik.MXKVCache(1, 1, 4, 2, 32, device=DEV, dtype=dtype)
    codes = torch.arange(16, dtype=torch.uint8)
    cache.k_codes[0] = (codes | (codes.flip(0) << 4)).to(DEV)
    cache.v_codes[0] = (codes.flip(0) | (codes << 4)).to(DEV)
    cache.k_scales.fill_(e)
    cache.v_scales.fill_(e)
    cache.lengths.fill_(4)
    cache._host_lengths[0] = 4
    for t, c in zip(cache.get_layer(0).get(), (cache.k_codes, cache.v_codes)):
        want = om.decode(c[0].transpose(1, 2), torch.full((1, 4, 2, 1), e, dtype=torch.uint8)).to(dtype)
        if e == 255:
            assert t.isnan().all() and want.isnan().all()
        else:
            assert torch.equal(t.cpu().double(), want.double())
            assert dtype == torch.float16 or (t != 0).sum() == t.numel() * 14 // 16
