"""Float64 oracle of RMSNorm + rotation by positions on several axes (qwen-image-kernel_amd/rope.py).

``forward`` is written as complex numbers from the definition; its gradients are
autograd's, in float64.  ``forward_bound``, ``dx_bound`` and ``dw_bound`` say how
far a kernel in fp32 that rounds its results to ``dtype`` may be from them.
"""

from __future__ import annotations

import torch


def angles(positions, axes_dims, theta, spectrum) -> torch.Tensor:
    """Angles [.., S, D / 2] (float64) of positions [.., A, S]."""
    D, out = sum(axes_dims), []
    thetas = theta if isinstance(theta, (tuple, list)) else [theta] * len(axes_dims)
    for a, d in enumerate(axes_dims):
        for i in range(d // 2):
            power = 2 * len(out) / D if spectrum == "shared" else 2 * i / d
            out.append(positions[..., a, :].double() / float(thetas[a]) ** power)
    return torch.stack(out, -1)


def pair_up(x, pairs):
    """[..., D] -> the two elements of each pair, [..., D / 2] each."""
    return x.chunk(2, -1) if pairs == "halves" else (x[..., 0::2], x[..., 1::2])


def unpair(a, b, pairs):
    return torch.cat((a, b), -1) if pairs == "halves" else torch.stack((a, b), -1).flatten(-2)


def normed(x, w, eps):
    return x if w is None else x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w


def turn(x, angle, pairs):
    """x [B, S, H, D] turned by angle [.., S, D / 2]."""
    z = torch.complex(*pair_up(x, pairs)) * torch.polar(torch.ones_like(angle), angle)[..., None, :]
    return unpair(z.real, z.imag, pairs)


def forward(x, w, angle, pairs, eps):
    return turn(normed(x, w, eps), angle, pairs)


def _pair_mass(x, pairs):
    a, b = pair_up(x.abs(), pairs)
    return unpair(a + b, a + b, pairs)


def _floor(dtype):
    # half of fp16's smallest step; bf16's is far below any value here
    return 2.0 ** -25 if dtype == torch.float16 else 1e-37


def forward_bound(x, w, angle, pairs, eps, dtype):
    """u = 2^-24: the mean of D squares is off by at most (D + 1) u of it, so r with its root and quotient by (D / 2 +
    4) u, n by two more; a cosine or sine by the fraction's rounding (pi u / 2) and the function's (2 ulp), together 6
    u; the two products and their sum by 3 u: in all less than (D / 2 + 16) u of |n0| + |n1|, and h of |y|."""
    u, h, D = 2.0 ** -24, torch.finfo(dtype).eps / 2, x.shape[-1]
    n = normed(x, w, eps)
    return h * turn(n, angle, pairs).abs() + (D / 2 + 16) * u * (1 + h) * _pair_mass(n, pairs) + _floor(dtype)


def _dn_mass(g, w, pairs):
    m = _pair_mass(g, pairs)
    return m if w is None else m * w.abs()


def dx_bound(x, w, g, dx, pairs, eps, dtype):
    """dn is off by 9 u of |g0| + |g1| (as above), w dn by one more; the mean of D products by D + 12 u of the mean of
    their magnitudes, r^2 by D + 8 u, the rest by 4: less than (2 D + 40) u of r (w |dn| + |x| r^2 mean |x w dn|)."""
    u, h, D = 2.0 ** -24, torch.finfo(dtype).eps / 2, x.shape[-1]
    m = _dn_mass(g, w, pairs)
    if w is not None:
        r2 = 1.0 / ((x * x).mean(-1, keepdim=True) + eps)
        m = r2.sqrt() * (m + x.abs() * r2 * (x.abs() * m).mean(-1, keepdim=True))
    return h * dx.abs() + (2 * D + 40) * u * (1 + h) * m + _floor(dtype)


def dw_bound(x, g, pairs, eps):
    """Each row's dn x r is off by (D / 2 + 16) u of its magnitude; N rows are added in chains of at most N / 32 + 112
    (a lane group's, the groups', the workgroups'), u each of the magnitudes' sum."""
    u, D = 2.0 ** -24, x.shape[-1]
    r = 1.0 / torch.sqrt((x * x).mean(-1, keepdim=True) + eps)
    m = (_pair_mass(g, pairs) * x.abs() * r).flatten(0, -2)
    return (D / 2 + 16 + m.shape[0] / 32 + 112) * u * m.sum(0) + 1e-30
