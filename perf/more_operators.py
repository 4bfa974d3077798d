"""The measured workload of the 4-bit prefix slab and of rotary positions with several axes.

A case is one call (or the calls of one step) through the public entry points,
or in plain form (``own`` false) the same result from elementary torch
operations.  Kinds:

* ``rope``   ``fused_qk_norm_rope``: a layer's Q and K, RMSNorm over each head,
             then the rotation by positions on several axes (time, height,
             width); with ``train`` also the gradients of Q, K and both weights
* ``store``  ``MXKVCache`` layer's ``store`` of a prefix's K and V in 4 bits, and
             ``get``: the values that the slab then stands for
* ``step``   a serving step: ``append`` of the new tokens' K and V at each
             sequence's length, then ``block_causal_flash_attention`` of their
             queries over the slab
* ``attn``   ``block_causal_flash_attention`` of queries over a 4-bit prefix and
             fresh keys

A slab row (one token's head) is cut into blocks of 32; a block holds one scale
byte e, standing for 2^(e - 127), and 32 E2M1 elements (0, 0.5, 1, 1.5, 2, 3, 4,
6 and a sign), two to a byte, the first in the low half.  With E the fp32
exponent field of the block's largest magnitude, e = max(E - 2, 0); the
elements are x * 2^(127 - e) rounded to nearest, ties to even, saturated at 6.
Pair i of axis a's d dimensions turns by position[a] * theta^(-2 i / d)
(``spectrum`` "axis"); with "shared" the pairs take theta^(-2 i / D) over the whole
head.  A pair is two neighbours ("interleaved") or the same place of the head's
two halves ("halves").  Query row q of sequence b attends key j iff j <= L[b, q],
where the slab's keys come first and end at that sequence's length, and
``key_valid`` has not masked it; a row that attends nothing gives zeros.
"""

from types import SimpleNamespace

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def listed():
    return [
        # one token of a text model with grouped heads: the smallest call, where latency counts
        {"name": "rope_token", "kind": "rope", "B": 1, "T": 1, "F": 0, "gh": 0, "gw": 0, "Hq": 32, "Hk": 8, "D": 128,
         "dtype": "bf16", "pairs": "halves", "spectrum": "shared", "per_sample": False, "train": False},
        # a 1024px layer: 256 text tokens, then 64 x 64 image tokens
        {"name": "rope_1024", "kind": "rope", "B": 1, "T": 256, "F": 1, "gh": 64, "gw": 64, "Hq": 24, "Hk": 24, "D": 128,
         "dtype": "bf16", "pairs": "interleaved", "spectrum": "axis", "per_sample": False, "train": False},
        # two videos of 17 frames, an odd grid, narrow heads, positions of their own for each
        {"name": "rope_video_fp16", "kind": "rope", "B": 2, "T": 41, "F": 17, "gh": 15, "gw": 26, "Hq": 12, "Hk": 12,
         "D": 64, "dtype": "fp16", "pairs": "interleaved", "spectrum": "axis", "per_sample": True, "train": False},
        # a training step of two 512px-and-more samples: outputs and gradients
        {"name": "rope_train", "kind": "rope", "B": 2, "T": 77, "F": 1, "gh": 41, "gw": 43, "Hq": 24, "Hk": 24, "D": 128,
         "dtype": "bf16", "pairs": "interleaved", "spectrum": "axis", "per_sample": False, "train": True},
        # the prefix of a 768px edit (256 text + 48 x 48 condition tokens) into the slab
        {"name": "store_edit_768", "kind": "store", "B": 1, "P": 2560, "H": 24, "D": 128, "dtype": "bf16"},
        # three short fp16 prompts, narrow heads
        {"name": "store_prompt_fp16", "kind": "store", "B": 3, "P": 77, "H": 8, "D": 64, "dtype": "fp16"},
        # one token against a short cache: latency
        {"name": "step_token", "kind": "step", "B": 1, "S": 1, "cap": 2048, "top": 1501, "Hq": 32, "Hk": 8, "D": 128,
         "dtype": "bf16"},
        # a serving batch of ragged lengths: bound by the slab's bytes
        {"name": "step_batch", "kind": "step", "B": 24, "S": 1, "cap": 8192, "top": 8191, "Hq": 32, "Hk": 8, "D": 128,
         "dtype": "bf16"},
        # four drafted tokens a sequence, causal among themselves, as many KV heads as query heads
        {"name": "step_drafted_fp16", "kind": "step", "B": 5, "S": 4, "cap": 3000, "top": 2993, "Hq": 16, "Hk": 16,
         "D": 64, "dtype": "fp16"},
        # one token against a long cache
        {"name": "attn_token_long", "kind": "attn", "B": 1, "SQ": 1, "SN": 1, "P": 131072, "Hq": 32, "Hk": 8, "D": 128,
         "dtype": "bf16", "mask": False, "causal": False},
        # the target rows of a 768px edit against its prefix and themselves: the largest
        {"name": "attn_edit_768", "kind": "attn", "B": 1, "SQ": 4096, "SN": 4096, "P": 2560, "Hq": 24, "Hk": 24, "D": 128,
         "dtype": "bf16", "mask": False, "causal": False},
        # a causal continuation of two prompts, padded keys, rows that see nothing
        {"name": "attn_prompt_masked", "kind": "attn", "B": 2, "SQ": 1031, "SN": 1031, "P": 1777, "Hq": 24, "Hk": 8,
         "D": 128, "dtype": "fp16", "mask": True, "causal": True},
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    kind = rng.choice(["rope", "rope", "store", "step", "step", "attn", "attn"])
    dtype, D = rng.choice(["bf16", "bf16", "fp16"]), rng.choice([64, 128, 128])
    Hk = rng.choice([1, 4, 8, 8, 12, 24])
    Hq = Hk * rng.choice([1, 1, 2, 4, 7] if Hk < 12 else [1, 1, 2])
    if kind == "rope":
        F = rng.choice([0, 1, 1, _log(rng, 2, 24)])
        gh, gw = (_log(rng, 4, 64), _log(rng, 4, 64)) if F else (0, 0)
        F = min(F, max(1, 16384 // (gh * gw))) if F else 0
        return {"kind": kind, "B": rng.choice([1, 1, 2, 3]), "T": _log(rng, 1, 600), "F": F, "gh": gh, "gw": gw,
                "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype, "pairs": rng.choice(["interleaved", "interleaved", "halves"]),
                "spectrum": rng.choice(["axis", "shared"]), "per_sample": rng.random() < 0.3, "train": rng.random() < 0.4}
    if kind == "store":
        return {"kind": kind, "B": rng.choice([1, 1, 2, 5]), "P": _log(rng, 1, 6000), "H": Hk, "D": D, "dtype": dtype}
    if kind == "step":
        B = _log(rng, 1, 40)
        cap = _log(rng, 64, min(40000, 4_000_000 // (B * Hk)))
        S = min(rng.choice([1, 1, 1, 2, 5, 9]), cap - 1)
        return {"kind": kind, "B": B, "S": S, "cap": cap, "top": max(1, cap - S - rng.randrange(0, cap // 3)), "Hq": Hq,
                "Hk": Hk, "D": D, "dtype": dtype}
    B = rng.choice([1, 1, 2])
    most = 4096 * 6656 * 24 // (B * Hq)  # (query, key) pairs of a head, for the largest listed case's cost
    SQ = _log(rng, 1, min(4096, int(most ** 0.5) - 64))
    causal = rng.random() < 0.5
    SN = SQ if causal or rng.random() < 0.5 else _log(rng, 1, min(4096, most // SQ - 64))
    P = min(_log(rng, 16, 60000), most // SQ - SN, 8_000_000 // (B * Hk))
    return {"kind": kind, "B": B, "SQ": SQ, "SN": SN, "P": P, "Hq": Hq, "Hk": Hk, "D": D, "dtype": dtype,
            "mask": rng.random() < 0.4, "causal": causal}


# ---- inputs ----------------------------------------------------------------

def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _states(g, shape, dtype=None):
    """Projected states: normal, with one channel in 32 four times larger, as keys have."""
    x = torch.randn(shape, generator=g, device="cuda")
    x[..., 5::32] *= 4.0
    return x if dtype is None else x.to(DTYPES[dtype])


def _codes(x):
    """fp32 rows [..., D] in 4 bits: codes uint8 [..., D/2] and scale bytes uint8 [..., D/32]."""
    b = x.unflatten(-1, (-1, 32))
    E = (b.abs().amax(-1).view(torch.int32) >> 23) & 255
    e = (E - 2).clamp_min(0)
    q = b * ((254 - e) << 23).view(torch.float32)[..., None]
    a = q.abs().clamp_max(6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = (torch.round(a / step) * step * 2).int()  # twice the magnitude: 0 1 2 3 4 6 8 12
    c = torch.where(a < 4, a, torch.where(a < 8, 2 + a // 2, 4 + a // 4)) + 8 * (q < 0).int()
    c = c.flatten(-2)
    return (c[..., 0::2] | (c[..., 1::2] << 4)).to(torch.uint8), e.to(torch.uint8)


def _positions(c):
    """[3, S] or [B, 3, S], float64: text tokens at (i, i, i), then frames of a grid centred on zero (as a model
    lays an image of any size around the same middle), in half steps along the height (a grid scaled to another's)."""
    T, F, gh, gw = c["T"], c["F"], c["gh"], c["gw"]
    t = torch.arange(T, device="cuda", dtype=torch.float64)
    f, h, w = torch.meshgrid(*(torch.arange(n, device="cuda", dtype=torch.float64) for n in (F, gh, gw)), indexing="ij")
    grid = torch.stack((T + f, 0.5 * (h - gh // 2), w - gw // 2)).flatten(1)
    p = torch.cat((t.expand(3, T), grid), 1)
    if c["T"] == 1 and not F:
        p = p + 20017.0  # a token far into a text
    return p + 1000.0 * torch.arange(c["B"], device="cuda").view(-1, 1, 1) if c["per_sample"] else p


def _axes(D):
    return (D // 8, D * 7 // 16, D * 7 // 16)


def _theta(c):
    return 1e6 if c["spectrum"] == "shared" else 1e4


def _rope_inputs(c, seed):
    g = _gen(seed)
    S = c["T"] + c["F"] * c["gh"] * c["gw"]
    s = SimpleNamespace(c=c, S=S, pos=_positions(c))
    s.x = [_states(g, (c["B"], S, H, c["D"]), c["dtype"]) for H in (c["Hq"], c["Hk"])]
    s.w = [torch.rand(c["D"], generator=g, device="cuda") + 0.5 for _ in range(2)]
    s.g = [torch.randn(x.shape, generator=g, device="cuda").to(x.dtype) for x in s.x] if c["train"] else None
    return s


def _store_inputs(c, seed):
    g = _gen(seed)
    return [_states(g, (c["B"], c["P"], c["H"], c["D"]), c["dtype"]) for _ in range(2)]


def _step_inputs(c, seed):
    """Queries, the new tokens' keys and values, the sequences' lengths (the first one the longest, one empty where
    there are four or more), and the slabs' codes and scale bytes."""
    g = _gen(seed)
    B, S, Hk, D = c["B"], c["S"], c["Hk"], c["D"]
    q = _states(g, (B, S, c["Hq"], D), c["dtype"])
    k, v = (_states(g, (B, S, Hk, D), c["dtype"]) for _ in range(2))
    at = torch.randint(max(1, c["top"] // 8), c["top"] + 1, (B,), generator=g, device="cuda", dtype=torch.int32)
    at[0] = c["top"]
    if B >= 4:
        at[B // 2] = 0
    return q, k, v, at, _codes(_states(g, (B, Hk, c["cap"], D))), _codes(_states(g, (B, Hk, c["cap"], D)))


def _attn_inputs(c, seed):
    g = _gen(seed)
    B, SQ, SN, P, Hk, D = (c[n] for n in ("B", "SQ", "SN", "P", "Hk", "D"))
    q = _states(g, (B, SQ, c["Hq"], D), c["dtype"])
    k, v = (_states(g, (B, SN, Hk, D), c["dtype"]) for _ in range(2))
    valid = None
    if c["mask"]:  # the second half of the batch is padded: its first keys and a stretch before its fresh ones
        valid = torch.ones(B, P + SN, dtype=torch.bool, device="cuda")
        valid[B // 2:, :P // 5] = False
        valid[B // 2:, P - P // 16:P] = False
    L = None
    if c["causal"]:
        L = P + torch.arange(SQ, device="cuda", dtype=torch.int32)
        if c["mask"] and SQ > 4:
            L[:3] = -1  # rows of padding see nothing
    return q, k, v, L, valid, _codes(_states(g, (B, Hk, P, D))), _codes(_states(g, (B, Hk, P, D)))


def prepare(case, seed):
    c = case
    s = SimpleNamespace(c=c)
    if c["kind"] == "rope":
        s = _rope_inputs(c, seed)
        if own:  # the plan of a step's positions, as every layer of the step uses it
            import qwen_image_kernel_amd as qik
            s.rope = qik.AxialRope(s.pos, _axes(c["D"]), _theta(c), pairs=c["pairs"], spectrum=c["spectrum"])
            if c["train"]:
                for t in s.x + s.w:
                    t.requires_grad_()
        return s
    if c["kind"] == "store":
        s.k, s.v = _store_inputs(c, seed)
        if own:
            import qwen_image_kernel_amd as qik
            s.layer = qik.MXKVCache(1, c["B"], c["P"], c["H"], c["D"], device="cuda", dtype=DTYPES[c["dtype"]]).get_layer(0)
        return s
    if c["kind"] == "step":
        s.q, s.k, s.v, s.at, s.kc, s.vc = _step_inputs(c, seed)
        s.L = s.at[:, None] + torch.arange(c["S"], device="cuda", dtype=torch.int32)
        if own:
            import qwen_image_kernel_amd as qik
            cache = qik.MXKVCache(1, c["B"], c["cap"], c["Hk"], c["D"], device="cuda", dtype=DTYPES[c["dtype"]])
            for buf, t in ((cache.k_codes, s.kc[0]), (cache.k_scales, s.kc[1]), (cache.v_codes, s.vc[0]),
                           (cache.v_scales, s.vc[1])):
                buf[0].copy_(t)
            s.cache, s.layer = cache, cache.get_layer(0)
        return s
    s.q, s.k, s.v, s.L, s.valid, s.kc, s.vc = _attn_inputs(c, seed)
    if own:
        import qwen_image_kernel_amd as qik
        s.slabs = [qik.MXSlab(*(t.transpose(1, 2) for t in kv)) for kv in (s.kc, s.vc)]
    return s


# ---- the plain form --------------------------------------------------------

def _values(codes, e):
    """fp32 values of codes [..., D/2] with scale bytes [..., D/32]."""
    n = torch.stack((codes & 15, codes >> 4), -1).flatten(-2).int()
    m, x = n & 1, (n >> 1) & 3
    a = torch.where(x == 0, 0.5 * m, 0.25 * (2 + m) * (1 << x))
    v = torch.where(n >= 8, -a, a).unflatten(-1, (-1, 32))
    # 2^(e - 127) from its bits: 2^-127 is a subnormal
    s = torch.where(e == 0, 0x400000, e.int() << 23).to(torch.int32).view(torch.float32)
    return (v * s[..., None]).flatten(-2)


def _frequencies(c, device="cuda"):
    """theta^(-2 i / d) of each of the D/2 pairs, and the pair's axis."""
    D, axes = c["D"], _axes(c["D"])
    axis = torch.repeat_interleave(torch.arange(3, device=device), torch.tensor([d // 2 for d in axes], device=device))
    i = torch.arange(D // 2, device=device, dtype=torch.float64)
    if c["spectrum"] == "shared":
        return _theta(c) ** (-2 * i / D), axis
    first = torch.tensor([0, axes[0] // 2, (axes[0] + axes[1]) // 2], device=device, dtype=torch.float64)
    return _theta(c) ** (-2 * (i - first[axis]) / torch.tensor(axes, device=device, dtype=torch.float64)[axis]), axis


def _turn(c, x, cos, sin):
    if c["pairs"] == "halves":
        a, b = x.chunk(2, -1)
        return torch.cat((a * cos - b * sin, a * sin + b * cos), -1)
    a, b = x[..., 0::2], x[..., 1::2]
    return torch.stack((a * cos - b * sin, a * sin + b * cos), -1).flatten(-2)


def _rope(s):
    c = s.c
    f, axis = _frequencies(c)
    angle = (s.pos.index_select(-2, axis) * f[:, None]).transpose(-1, -2)  # [.., S, D/2], in 64 bits: far positions
    cos, sin = torch.cos(angle).float()[..., None, :], torch.sin(angle).float()[..., None, :]
    xs = [x.float() for x in s.x]
    rs = [1.0 / torch.sqrt(x.square().mean(-1, keepdim=True) + EPS) for x in xs]
    out = [_turn(c, x * r * w, cos, sin).to(t.dtype) for x, r, w, t in zip(xs, rs, s.w, s.x)]
    if not c["train"]:
        return out
    dn = [_turn(c, g.float(), cos, -sin) for g in s.g]
    hat = [x * r for x, r in zip(xs, rs)]
    dh = [d * w for d, w in zip(dn, s.w)]
    dx = [(r * (d - h * (d * h).mean(-1, keepdim=True))).to(t.dtype) for r, d, h, t in zip(rs, dh, hat, s.x)]
    return out + dx + [(d * h).flatten(0, -2).sum(0) for d, h in zip(dn, hat)]


def _attend(q, keys, values, allowed):
    """fp32 q [B, SQ, Hq, D], keys and values [B, Hk, N, D], allowed [B or 1, SQ, N] or None -> [B, SQ, Hq, D]."""
    B, SQ, Hq, D = q.shape
    Hk, N = keys.shape[1:3]
    G = Hq // Hk
    x = q.view(B, SQ, Hk, G, D).permute(0, 2, 3, 1, 4).reshape(B * Hk, G * SQ, D)
    s = torch.bmm(x, keys.reshape(B * Hk, N, D).transpose(1, 2)) * D ** -0.5
    if allowed is not None:
        s = s.view(B, Hk * G, SQ, N).masked_fill_(~allowed[:, None], -torch.inf).view(B * Hk, G * SQ, N)
    s = s.sub_(s.amax(-1, keepdim=True).clamp_min(-1e30)).exp_()
    total = s.sum(-1, keepdim=True)
    o = torch.bmm(s, values.reshape(B * Hk, N, D)) / torch.where(total > 0, total, 1.0)
    return o.view(B, Hk, G, SQ, D).permute(0, 3, 1, 2, 4).reshape(B, SQ, Hq, D)


def _put(slab, new, rows):
    """The new tokens [B, S, Hk, D] into the slab's rows [B, S]."""
    b = torch.arange(rows.shape[0], device="cuda")[:, None]
    codes, e = _codes(new.float())
    slab[0][b, :, rows], slab[1][b, :, rows] = codes, e


def _plain_step(s):
    c = s.c
    _put(s.kc, s.k, s.L.long())
    _put(s.vc, s.v, s.L.long())
    allowed = torch.arange(c["cap"], device="cuda") <= s.L[..., None]
    out = _attend(s.q.float(), _values(*s.kc), _values(*s.vc), allowed)
    return [out.to(s.q.dtype), s.at + c["S"]]


def _plain_attn(s):
    c = s.c
    keys = torch.cat((_values(*s.kc), s.k.float().transpose(1, 2)), 2)
    values = torch.cat((_values(*s.vc), s.v.float().transpose(1, 2)), 2)
    allowed = None
    if s.L is not None:
        allowed = (torch.arange(c["P"] + c["SN"], device="cuda") <= s.L[:, None])[None]
    if s.valid is not None:
        allowed = s.valid[:, None] if allowed is None else allowed & s.valid[:, None]
        allowed = allowed.expand(-1, c["SQ"], -1)
    return _attend(s.q.float(), keys, values, allowed).to(s.q.dtype)


def run(s):
    c = s.c
    if own:
        import qwen_image_kernel_amd as qik
        if c["kind"] == "rope":
            out = qik.fused_qk_norm_rope(s.x[0], s.x[1], s.w[0], s.w[1], s.rope, EPS)
            return [*out, *torch.autograd.grad(out, s.x + s.w, s.g)] if c["train"] else list(out)
        if c["kind"] == "store":
            s.layer.store(s.k, s.v)
            return list(s.layer.get())
        if c["kind"] == "step":
            s.layer.append(s.k, s.v, s.at)
            k, v, _ = s.layer.views(c["top"] + c["S"])
            out = qik.block_causal_flash_attention(s.q, s.k[:, :0], s.v[:, :0], s.L, None, cache_k=k, cache_v=v,
                                                   uniform_full=c["S"] == 1)
            return [out, s.cache.lengths[0]]
        return qik.block_causal_flash_attention(s.q, s.k, s.v, s.L, s.valid, cache_k=s.slabs[0], cache_v=s.slabs[1],
                                                uniform_full=not c["causal"] and s.valid is None)
    if c["kind"] == "rope":
        return _rope(s)
    if c["kind"] == "store":
        return [_values(*_codes(t.float())).to(t.dtype) for t in (s.k, s.v)]
    return _plain_step(s) if c["kind"] == "step" else _plain_attn(s)


# ---- cost ------------------------------------------------------------------

def _pairs(c):
    """Allowed (query, key) pairs of one query head, of the whole batch (key masks apart), and the slab rows read."""
    if c["kind"] == "step":  # the lengths are drawn: their middle
        n = c["B"] * ((c["top"] + c["top"] // 8) // 2 + c["S"])
        return c["S"] * n, n
    n = c["B"] * c["P"]
    own_keys = c["B"] * c["SQ"] * (c["SQ"] + 1) // 2 if c["causal"] else c["B"] * c["SQ"] * c["SN"]
    return c["SQ"] * n + own_keys, n


def work(case):
    c = case
    if c["kind"] == "rope":
        tokens = c["B"] * (c["T"] + c["F"] * c["gh"] * c["gw"])
        n = tokens * (c["Hq"] + c["Hk"]) * c["D"]
        return {"bytes": n * 2 * (4 if c["train"] else 2) + 24 * tokens, "flops": n * (25 if c["train"] else 8)}
    if c["kind"] == "store":
        n = 2 * c["B"] * c["P"] * c["H"] * c["D"]
        return {"bytes": 4 * n, "flops": 3 * n}
    pairs, rows = _pairs(c)
    fresh = c["B"] * (c["S"] if c["kind"] == "step" else c["SN"]) * c["Hk"] * c["D"] * 2 * 2
    ends = c["B"] * (c["S"] if c["kind"] == "step" else c["SQ"]) * c["Hq"] * c["D"] * 2 * 2
    return {"bytes": 2 * rows * c["Hk"] * (c["D"] // 2 + c["D"] // 32) + fresh + ends, "flops": 4 * c["D"] * c["Hq"] * pairs}


# ---- the same results in 64 bits -------------------------------------------

_E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _mx64(x):
    """The values that fp64 rows are stored as: the block's scale from the exponent of its largest magnitude, the
    nearest of the eight magnitudes, halfway to the even one, past the end the last."""
    grid = torch.tensor(_E2M1, dtype=torch.float64, device=x.device)
    b = x.unflatten(-1, (-1, 32))
    top = b.abs().amax(-1, keepdim=True)
    s = torch.where(top == 0, 2.0 ** -127, torch.exp2((torch.frexp(top)[1].double() - 3).clamp_min(-127.0)))
    a = (b / s).abs().contiguous()
    hi = torch.searchsorted(grid, a).clamp(1, 7)
    up, down = grid[hi] - a, a - grid[hi - 1]
    at = torch.where((up < down) | ((up == down) & (hi % 2 == 0)), hi, hi - 1)
    return (grid[at] * torch.sign(b) * s).flatten(-2)


def _read64(codes, e):
    """The fp64 values of a slab's codes and scale bytes, by a table of the sixteen elements."""
    table = torch.tensor(_E2M1 + tuple(-m for m in _E2M1), dtype=torch.float64, device=codes.device)
    pair = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), -1).flatten(-2)
    return (pair.unflatten(-1, (-1, 32)) * torch.exp2(e.double() - 127)[..., None]).flatten(-2)


def _exact_rope(c, seed):
    s = _rope_inputs(c, seed)
    D, axes, angle = c["D"], _axes(c["D"]), []
    for a, d in enumerate(axes):
        first = sum(axes[:a])
        for i in range(0, d, 2):
            power = (first + i) / D if c["spectrum"] == "shared" else i / d
            angle.append(s.pos[..., a, :] / _theta(c) ** power)
    angle = torch.stack(angle, -1)
    z = torch.polar(torch.ones_like(angle), angle)[..., None, :]

    def pairs(x):
        return torch.complex(*((x[..., :D // 2], x[..., D // 2:]) if c["pairs"] == "halves"
                               else (x[..., 0::2], x[..., 1::2])))

    def flat(y):
        return torch.cat((y.real, y.imag), -1) if c["pairs"] == "halves" else torch.view_as_real(y).flatten(-2)

    out, dx, dw = [], [], []
    for i, x in enumerate(s.x):
        x, w = x.double(), s.w[i].double()
        r = torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS)
        out.append(flat(pairs(x * r * w) * z))
        if c["train"]:
            d = flat(pairs(s.g[i].double()) * z.conj())
            dw.append((d * x * r).sum((0, 1, 2)))
            dx.append(r * d * w - x * r ** 3 * (d * w * x).mean(-1, keepdim=True))
    return out + dx + dw


def _exact_attend(q, k, v, allowed):
    """q [SQ, D], k, v [N, D] of one head in 64 bits."""
    s = q @ k.t() / q.shape[-1] ** 0.5
    if allowed is not None:
        s = torch.where(allowed, s, -torch.inf)
    return torch.nan_to_num(torch.softmax(s, -1)) @ v


def exact(case, seed):
    c = case
    if c["kind"] == "rope":
        return _exact_rope(c, seed)
    if c["kind"] == "store":
        return [_mx64(t.double()) for t in _store_inputs(c, seed)]
    G = c["Hq"] // c["Hk"]
    if c["kind"] == "step":
        q, k, v, at, kc, vc = _step_inputs(c, seed)
        out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
        k, v = _mx64(k.double()), _mx64(v.double())
        for b, n in enumerate(at.tolist()):
            rows = torch.arange(n + c["S"], device="cuda") <= n + torch.arange(c["S"], device="cuda")[:, None]
            for h in range(c["Hk"]):
                kh = torch.cat((_read64(kc[0][b, h, :n], kc[1][b, h, :n]), k[b, :, h]))
                vh = torch.cat((_read64(vc[0][b, h, :n], vc[1][b, h, :n]), v[b, :, h]))
                for g in range(h * G, h * G + G):
                    out[b, :, g] = _exact_attend(q[b, :, g].double(), kh, vh, rows)
        return [out, None]
    q, k, v, L, valid, kc, vc = _attn_inputs(c, seed)
    out = torch.zeros(q.shape, dtype=torch.float64, device="cuda")
    for b in range(c["B"]):
        allowed = None
        if L is not None or valid is not None:
            allowed = torch.ones(c["SQ"], c["P"] + c["SN"], dtype=torch.bool, device="cuda")
            if L is not None:
                allowed &= torch.arange(c["P"] + c["SN"], device="cuda")[None] <= L[:, None]
            if valid is not None:
                allowed &= valid[b][None]
        for h in range(c["Hk"]):
            kh = torch.cat((_read64(kc[0][b, h], kc[1][b, h]), k[b, :, h].double()))
            vh = torch.cat((_read64(vc[0][b, h], vc[1][b, h]), v[b, :, h].double()))
            for g in range(h * G, h * G + G):
                out[b, :, g] = _exact_attend(q[b, :, g].double(), kh, vh, allowed)
    return out
