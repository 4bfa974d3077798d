"""Float64 oracle of the 4-bit slab and of the attention over it.

``decode`` gives a slab's values from its bytes, ``attention`` the result of
``block_causal_flash_attention`` with ``MXSlab`` caches (qwen-image-kernel_amd/mx_attention.py),
and ``bound`` how far a kernel with fp32 sums and statistics may be from it that
rounds the probabilities and the output to ``dtype``.
"""

from __future__ import annotations

import torch

E2M1 = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0, -0.0, -0.5, -1.0, -1.5, -2.0, -3.0, -4.0, -6.0],
                    dtype=torch.float64)


def decode(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """Values (float64) of codes [..., D / 2] and scale bytes [..., D / 32]; byte 255 is NaN."""
    codes, scales = codes.cpu(), scales.cpu()
    v = torch.stack((E2M1[(codes & 15).long()], E2M1[(codes >> 4).long()]), -1).flatten(-2)
    s = torch.where(scales == 255, torch.nan, torch.exp2(scales.double() - 127))
    return (v.unflatten(-1, (-1, 32)) * s[..., None]).flatten(-2)


def encode(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Codes and scale bytes of rows [..., D] by the format's definition: the nearest element, halfway to the even code."""
    b = x.cpu().double().unflatten(-1, (-1, 32))
    top = b.abs().amax(-1)
    e = torch.where(top == 0, 0.0, torch.frexp(top)[1].double() - 1 + 127 - 2).clamp_min(0)
    bad = ~torch.isfinite(b).all(-1)
    e = torch.where(bad, 255.0, e)
    a = torch.where(bad[..., None], 0.0, b) / torch.exp2(torch.where(bad, 127.0, e) - 127)[..., None]
    grid = E2M1[:8]
    m = a.abs()
    hi = torch.searchsorted(grid, m.contiguous()).clamp(1, 7)
    up, down = grid[hi] - m, m - grid[hi - 1]
    c = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    # the sign of a negative zero is kept
    c = (c + 8 * torch.signbit(a).long()).flatten(-2).to(torch.uint8)
    return c[..., 0::2] | (c[..., 1::2] << 4), e.to(torch.uint8)


def allowed(B, SQ, P, SN, L=None, key_valid=None, lengths=None) -> torch.Tensor:
    """bool [B, SQ, P + SN]: which keys each query position sees."""
    kv = torch.arange(P + SN)
    ok = torch.ones(B, SQ, P + SN, dtype=torch.bool)
    if lengths is not None:
        ok &= ((kv[None] >= P) | (kv[None] < lengths.cpu().clamp(0, P)[:, None]))[:, None]
    if L is not None:
        L = L.cpu()
        L = L[:, :SQ] if L.dim() == 2 else L[None, :SQ]
        ok &= kv <= L[..., None]
    if key_valid is not None:
        ok &= (key_valid.cpu() != 0)[:, None, :P + SN]
    return ok


def attention(q, k, v, ok):
    """q [B, SQ, H, D], k, v [B, N, HKV, D] float64, ok [B, SQ, N] -> out and bound's parts (float64).

    Values of keys that nobody sees count as zeros, whatever they are."""
    B, SQ, H, D = q.shape
    G = H // k.shape[2]
    seen = ok.any(1)[..., None, None]
    k, v = torch.where(seen, k, 0.0), torch.where(seen, v, 0.0)
    kh, vh = (t.repeat_interleave(G, 2).permute(0, 2, 1, 3) for t in (k, v))
    qh = q.permute(0, 2, 1, 3)
    s = qh @ kh.transpose(-1, -2) / D ** 0.5
    s = s.masked_fill(~ok[:, None], -torch.inf)
    top = s.amax(-1, keepdim=True)
    p = torch.exp(s - torch.where(top == -torch.inf, 0.0, top))
    w = p / p.sum(-1, keepdim=True).clamp_min(1e-300)
    mass = qh.abs() @ kh.abs().transpose(-1, -2) / D ** 0.5
    parts = {
        "out": w @ vh,
        "weighted": w @ vh.abs(),                                     # sum p |v| / l
        "seen": ok[:, None].double() @ vh.abs(),                      # sum of |v| over the keys seen
        "mass": torch.where(ok[:, None], mass, 0.0).amax(-1, keepdim=True),  # largest sum of |q k| / sqrt(D)
    }
    return {n: t.permute(0, 2, 1, 3) for n, t in parts.items()}


def bound(parts, D: int, dtype: torch.dtype) -> torch.Tensor:
    """Elementwise |kernel - out| for fp32 sums and a probability and an output rounded to dtype.

    With u = 2^-24 and h = eps(dtype) / 2.  The score of a key is a sum of D
    exact products in fp32, scaled and set against the reference point: off by at
    most (D + 4) u mass in the exponent's natural unit, so its probability by that
    factor, twice (once over the row sum); the exp2 instruction and the fp32 sums
    of up to 2^17 terms in at most 2^10 chains add less than 2^-12 altogether.
    Rounding the probability is h of it, rounding the output h of |out| <=
    weighted.  fp16 probabilities below 2^-14 are subnormal: off by at most
    2^-25 each, of a row sum of at least 1."""
    u, h = 2.0 ** -24, torch.finfo(dtype).eps / 2
    rel = 2 * (D + 4) * u * parts["mass"] + 2.0 ** -12
    b = parts["weighted"] * (rel + h) * (1 + h) + parts["out"].abs() * h
    if dtype == torch.float16:
        b = b + 2.0 ** -25 * parts["seen"] + 2.0 ** -25
    return b + 1e-30
