"""GPU tests of RMSNorm + rotation by positions on several axes and its gradient, against the float64 oracle."""

import pytest
import torch

import qwen_image_kernel_amd as qik
from oracle import axial_rope as oa

pytestmark = pytest.mark.gpu

DEV = "cuda"
EPS = 1e-6


def _axes(D):
    return (D // 8, D * 7 // 16, D * 7 // 16)


def _positions(g, B, S, how):
    if how == "grid":
        return torch.randint(-40, 60, (3, S), generator=g)
    if how == "far":
        return torch.randint(0, 1 << 22, (3, S), generator=g, dtype=torch.int32)
    return torch.rand(B, 3, S, generator=g) * 300 - 150   # fractional, each entry's own


def _within(got, want, bound):
    assert got.shape == want.shape
    off = (got.detach().cpu().double() - want.detach()).abs()
    worst = float((off / bound.detach()).max()) if off.numel() else 0.0
    assert worst <= 1.0, worst


def _inputs(g, B, S, Hq, Hk, D, dtype):
    x = [(torch.randn(B, S, H, D, generator=g) * torch.exp2(torch.randint(-4, 5, (B, S, H, 1), generator=g).float())).to(dtype)
         for H in (Hq, Hk)]
    w = [torch.rand(D, generator=g) + 0.5 for _ in range(2)]
    d = [torch.randn(t.shape, generator=g).to(dtype) for t in x]
    return x, w, d


CASES = [
    # B, S, Hq, Hk: one token, one head, runs that end inside a token, more tokens than a run's rows
    (1, 1, 1, 1), (1, 1, 32, 8), (2, 5, 3, 1), (1, 77, 24, 24), (3, 33, 7, 2), (2, 700, 1, 1), (1, 1031, 12, 4),
]


@pytest.mark.parametrize("case", CASES)
@pytest.mark.parametrize("D", [32, 64, 128, 256])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("pairs", ["interleaved", "halves"])
def test_forward_and_gradients(case, D, dtype, pairs):
    B, S, Hq, Hk = case
    g = torch.Generator().manual_seed(S + D)
    x, w, d = _inputs(g, B, S, Hq, Hk, D, dtype)
    how = ["grid", "far", "own"][(S + D // 32) % 3]
    spectrum = "shared" if D == 128 else "axis"
    pos = _positions(g, B, S, how)
    rope = qik.AxialRope(pos.to(DEV), _axes(D), (1e4, 500.0, 1e6), pairs=pairs, spectrum=spectrum)
    leaves = [t.to(DEV).requires_grad_() for t in (*x, *w)]
    out = qik.fused_qk_norm_rope(*leaves, rope, EPS, 1e-3)
    grads = torch.autograd.grad(out, leaves, [t.to(DEV) for t in d])
    angle = oa.angles(pos, _axes(D), (1e4, 500.0, 1e6), spectrum)
    for i, eps in enumerate((EPS, 1e-3)):
        xd, wd = x[i].double().requires_grad_(), w[i].double().requires_grad_()
        y = oa.forward(xd, wd, angle, pairs, eps)
        _within(out[i], y, oa.forward_bound(xd, wd, angle, pairs, eps, dtype))
        dx, dw = torch.autograd.grad(y, (xd, wd), d[i].double())
        _within(grads[i], dx, oa.dx_bound(xd, wd, d[i].double(), dx, pairs, eps, dtype))
        assert grads[2 + i].dtype == torch.float32
        _within(grads[2 + i], dw, oa.dw_bound(xd, d[i].double(), pairs, eps))
    # without gradients the same bits; one tensor alone too
    with torch.no_grad():
        again = qik.fused_qk_norm_rope(*leaves, rope, EPS, 1e-3)
        alone = qik.fused_rms_norm_rope(leaves[1], leaves[3], rope, 1e-3)
    assert torch.equal(again[0], out[0]) and torch.equal(again[1], out[1]) and torch.equal(alone, out[1])


def _one(B=2, S=9, Hq=3, Hk=2, D=64, dtype=torch.bfloat16, seed=5):
    g = torch.Generator().manual_seed(seed)
    x, w, d = _inputs(g, B, S, Hq, Hk, D, dtype)
    pos = _positions(g, B, S, "grid")
    rope = qik.AxialRope(pos.to(DEV), _axes(D))
    return [t.to(DEV) for t in x], [t.to(DEV) for t in w], [t.to(DEV) for t in d], pos, rope


def test_without_a_weight_it_is_the_rotation():
    x, _, d, pos, rope = _one()
    angle = oa.angles(pos, _axes(64), 1e4, "axis")
    leaves = [t.requires_grad_() for t in x]
    out = qik.fused_qk_norm_rope(*leaves, None, None, rope, 0.0)
    grads = torch.autograd.grad(out, leaves, d)
    for i in range(2):
        xd, g = x[i].detach().cpu().double(), d[i].cpu().double()
        mass = oa._pair_mass(xd, "interleaved")
        _within(out[i], oa.turn(xd, angle, "interleaved"), (2.0 ** -8 + 2.0 ** -20) * mass + 1e-30)
        # 2^-8 of the result, at most the pair's mass, and the fp32 terms as in the oracle's bounds
        _within(grads[i], oa.turn(g, -angle, "interleaved"), oa.dx_bound(xd, None, g, oa.turn(g, -angle, "interleaved"), "interleaved",
                                                                        0.0, torch.bfloat16))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_agrees_with_the_table(dtype):
    """A table of the same angles, rounded once more between norm and rotation: within that rounding of each other."""
    x, w, _, pos, rope = _one(B=1, S=200, Hq=5, D=128, dtype=dtype)
    angle = oa.angles(pos, _axes(128), 1e4, "axis")
    table = torch.polar(torch.ones_like(angle), angle).to(torch.complex64).to(DEV)
    for t, v in zip(x, w):
        a = qik.fused_rms_norm_rope(t, v, rope, EPS).cpu().double()
        b = qik.fused_rms_norm_rope(t, v, table, EPS).cpu().double()
        n = oa.normed(t.cpu().double(), v.cpu().double(), EPS)
        h = torch.finfo(dtype).eps / 2
        # one rounding of each result, one of n in the table's call, its cosines and sines in fp32
        lim = h * (a.abs() + b.abs()) + (h + 2.0 ** -15) * oa._pair_mass(n, "interleaved") + 2.0 ** -23
        assert ((a - b).abs() <= lim).all()


def test_layouts_types_and_parameters():
    """Slices of a fused projection, odd addresses and strides, other weight types, positions of every kind."""
    x, w, d, pos, rope = _one(B=2, S=9, Hq=3, Hk=3)
    want = qik.fused_qk_norm_rope(*x, *w, rope, EPS)
    qkv = torch.cat((*x, x[0]), 2)
    assert all(torch.equal(a, b) for a, b in zip(qik.fused_qk_norm_rope(qkv[:, :, :3], qkv[:, :, 3:6], *w, rope, EPS), want))
    odd = torch.zeros(x[0].numel() + 1, dtype=x[0].dtype, device=DEV)[1:].view(x[0].shape).copy_(x[0])
    wide = torch.zeros(2, 9, 3, 69, dtype=x[0].dtype, device=DEV)[..., :64].copy_(x[0])
    for alt in (odd, wide, x[0].transpose(1, 2).contiguous().transpose(1, 2), x[0].transpose(2, 3).contiguous().transpose(2, 3)):
        assert all(torch.equal(a, b) for a, b in zip(qik.fused_qk_norm_rope(alt, x[1], *w, rope, EPS), want))
        assert torch.equal(qik.fused_qk_norm_rope(x[0], alt, *w, rope, EPS)[0], want[0])
    w16 = [t.bfloat16() for t in w]
    ref = qik.fused_qk_norm_rope(*x, *(t.float() for t in w16), rope, EPS)
    shifted = [torch.zeros(65, device=DEV)[1:].copy_(t) for t in w16]
    gaps = [torch.zeros(64, 2, device=DEV)[:, 0].copy_(t) for t in w16]
    for ws in (w16, shifted, gaps, [w16[0], shifted[1]]):
        assert all(torch.equal(a, b) for a, b in zip(qik.fused_qk_norm_rope(*x, *ws, rope, EPS), ref))
    for p in (pos, pos.int(), pos.float(), pos.half(), pos.double(), pos[None].expand(2, -1, -1), pos[None], pos.t().contiguous().t()):
        r = qik.AxialRope(p.to(DEV), _axes(64))
        assert all(torch.equal(a, b) for a, b in zip(qik.fused_qk_norm_rope(*x, *w, r, EPS), want))
    # gradients: of some, of 16-bit weights, broadcast and strided incoming gradients
    leaves = [t.clone().requires_grad_() for t in (*x, *w16)]
    out = qik.fused_qk_norm_rope(*leaves, rope, EPS)
    got = torch.autograd.grad(out, leaves, d)
    assert got[2].dtype == torch.bfloat16
    only = qik.fused_qk_norm_rope(leaves[0], x[1], *w16, rope, EPS)
    assert torch.equal(torch.autograd.grad(only[0], leaves[0], d[0])[0], got[0])
    out = qik.fused_qk_norm_rope(*leaves, rope, EPS)
    broad = torch.autograd.grad(out[0].sum() + 2 * out[1].sum(), leaves)
    ones = torch.autograd.grad(qik.fused_qk_norm_rope(*leaves, rope, EPS), leaves, [torch.ones_like(x[0]), 2 * torch.ones_like(x[1])])
    assert all(torch.equal(a, b) for a, b in zip(broad, ones))
    strided = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in d]
    assert all(torch.equal(a, b) for a, b in zip(torch.autograd.grad(qik.fused_qk_norm_rope(*leaves, rope, EPS), leaves, strided), got))


def test_broadcast_inputs_and_shared_weights():
    """One key head expanded to all, one weight for both: autograd adds the parts."""
    x, w, d, pos, rope = _one(Hq=3, Hk=1)
    k1, w1 = x[1].clone().requires_grad_(), w[0].clone().requires_grad_()
    d3 = torch.randn(2, 9, 3, 64, generator=torch.Generator().manual_seed(1)).bfloat16().to(DEV)
    out = qik.fused_qk_norm_rope(x[0], k1.expand(-1, -1, 3, -1), w1, w1, rope, EPS)
    dk, dw = torch.autograd.grad(out, (k1, w1), (d[0], d3))
    parts = [torch.autograd.grad(qik.fused_rms_norm_rope(t, v, rope, EPS), (t, v), g)
             for t, v, g in ((x[0].clone().requires_grad_(), w[0].clone().requires_grad_(), d[0]),
                             (x[1].expand(-1, -1, 3, -1).contiguous().requires_grad_(), w[0].clone().requires_grad_(), d3))]
    assert torch.equal(dk, parts[1][0].sum(2, keepdim=True))
    assert torch.equal(dw, parts[0][1] + parts[1][1]) or torch.allclose(dw, parts[0][1] + parts[1][1], rtol=0, atol=float(2 ** -23 * dw.abs().max()))


def test_gradient_against_differences():
    """The kernel's gradients along random directions against differences of the float64 oracle."""
    x, w, d, pos, rope = _one(B=1, S=40, Hq=4, Hk=4, D=128)
    leaves = [t.requires_grad_() for t in (*x, *w)]
    grads = torch.autograd.grad(qik.fused_qk_norm_rope(*leaves, rope, EPS), leaves, d)
    angle = oa.angles(pos, _axes(128), 1e4, "axis")
    for i in range(2):
        xd, wd, g = x[i].detach().cpu().double(), w[i].detach().cpu().double(), d[i].cpu().double()
        gen = torch.Generator().manual_seed(i)
        for which in range(2):
            v = torch.randn((xd, wd)[which].shape, generator=gen, dtype=torch.float64)
            step = 1e-6
            f = [(oa.forward(*((xd + s * v, wd) if which == 0 else (xd, wd + s * v)), angle, "interleaved", EPS) * g).sum()
                 for s in (step, -step)]
            slope = (f[0] - f[1]) / (2 * step)
            got = (grads[i + 2 * which].cpu().double() * v).sum()
            # dx is rounded to bf16: 2^-8 of each term at most; differences lose about 1e-16 / 1e-6 of the sum's terms
            scale = (grads[i + 2 * which].cpu().double() * v).abs().sum()
            assert abs(got - slope) <= (2.0 ** -8 if which == 0 else 1e-5) * scale


def test_positions_that_change():
    """A plan's positions may be written to between calls (a captured step's), not between a call and its backward."""
    x, w, d, pos, rope = _one()
    first = qik.fused_qk_norm_rope(*x, *w, rope, EPS)
    other = qik.AxialRope((pos + 3).to(DEV), _axes(64))
    want = qik.fused_qk_norm_rope(*x, *w, other, EPS)
    rope.positions.copy_(other.positions)
    assert all(torch.equal(a, b) for a, b in zip(qik.fused_qk_norm_rope(*x, *w, rope, EPS), want))
    assert not torch.equal(first[0], want[0])
    leaf = x[0].clone().requires_grad_()
    out = qik.fused_rms_norm_rope(leaf, w[0], rope, EPS)
    rope.positions.add_(1)
    with pytest.raises(RuntimeError):
        out.sum().backward()
    leaf = x[0].clone().requires_grad_()
    (g,) = torch.autograd.grad(qik.fused_rms_norm_rope(leaf, w[0], rope, EPS).float().square().sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_odd_positions_stay_with_their_token():
    x, w, _, pos, _ = _one()
    p = pos.double()
    p[1, 4], p[0, 6] = torch.nan, torch.inf
    out = qik.fused_qk_norm_rope(*x, *w, qik.AxialRope(p.to(DEV), _axes(64)), EPS)
    want = qik.fused_qk_norm_rope(*x, *w, qik.AxialRope(pos.to(DEV), _axes(64)), EPS)
    keep = [i for i in range(9) if i not in (4, 6)]
    for a, b in zip(out, want):
        assert torch.equal(a[:, keep], b[:, keep]) and a[:, 4].isnan().any() and a[:, 6].isnan().any()


def test_no_rows():
    for B, S, Hq, Hk in ((0, 3, 2, 2), (2, 0, 2, 2), (2, 3, 2, 0), (2, 3, 0, 2)):
        x = [torch.randn(B, S, H, 64, device=DEV).bfloat16().requires_grad_() for H in (Hq, Hk)]
        w = [torch.ones(64, device=DEV, requires_grad=True) for _ in range(2)]
        rope = qik.AxialRope(torch.zeros(3, S, device=DEV), _axes(64))
        out = qik.fused_qk_norm_rope(*x, *w, rope, EPS)
        assert out[0].shape == x[0].shape and out[1].shape == x[1].shape
        grads = torch.autograd.grad([o for o in out], x + w, [torch.ones_like(o) for o in out])
        for t, g in zip(x + w, grads):
            assert g.shape == t.shape
        for i in range(2):
            if x[i].numel() == 0:
                assert (grads[2 + i] == 0).all()


def test_the_same_bits_every_time_and_on_every_stream():
    x, w, d, _, rope = _one(B=3, S=700, Hq=5, Hk=3, D=128)
    leaves = [t.requires_grad_() for t in (*x, *w)]

    def both():
        out = qik.fused_qk_norm_rope(*leaves, rope, EPS)
        return [*out, *torch.autograd.grad(out, leaves, d)]

    want = both()
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for i in range(8):
        with torch.cuda.stream(streams[i % 2]):
            got = both()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_captured_forward_and_backward():
    """Replays with new inputs and positions, with eager work between them, give the eager results."""
    B, S, Hq, Hk, D = 2, 60, 4, 2, 128
    x, w, d, pos, rope = _one(B, S, Hq, Hk, D)
    stat = [t.clone().requires_grad_() for t in (*x, *w)]
    sd = [t.clone() for t in d]

    def both(leaves, grads, r):
        out = qik.fused_qk_norm_rope(*leaves, r, EPS)
        return [*out, *torch.autograd.grad(out, leaves, grads)]

    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.stream(stream):
        both(stat, sd, rope)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        outs = both(stat, sd, rope)
    for i in range(4):
        fresh = _one(B, S, Hq, Hk, D, seed=50 + i)
        with torch.no_grad():
            for t, v in zip((*stat, *sd), (*fresh[0], *fresh[1], *fresh[2])):
                t.copy_(v)
        rope.positions.copy_(fresh[4].positions)
        graph.replay()
        got = [t.clone() for t in outs]
        want = both([t.requires_grad_() for t in (*fresh[0], *fresh[1])], fresh[2], fresh[4])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, want)), i


def test_refusals_on_the_device():
    x, w, _, pos, rope = _one()
    bad = [(x[0][0], x[1], *w, rope), (x[0].float(), x[1].float(), *w, rope), (x[0], x[1].half(), *w, rope), (x[0], x[1][:, :5], *w, rope),
           (x[0][..., :32], x[1][..., :32], w[0][:32], w[1][:32], rope), (x[0][:, :5], x[1][:, :5], *w, rope),
           (x[0], x[1], w[0], None, rope), (x[0], x[1], w[0][:32], w[1], rope), (x[0], x[1], w[0].cpu(), w[1], rope),
           (x[0].cpu(), x[1].cpu(), *w, rope)]
    for q, k, wq, wk, r in bad:
        with pytest.raises(ValueError):
            qik.fused_qk_norm_rope(q, k, wq, wk, r, EPS)
    with pytest.raises(ValueError):
        qik.fused_qk_norm_rope(*x, *w, qik.AxialRope(torch.zeros(3, 3, 9, device=DEV), _axes(64)), EPS)
    for p in (torch.zeros(3, 9, dtype=torch.bool, device=DEV), torch.zeros(3, 9, dtype=torch.complex64, device=DEV)):
        with pytest.raises(ValueError):
            qik.AxialRope(p, _axes(64))


def test_plans_made_anew_share_their_frequencies():
    """Objects of the same parameters, of other positions, lengths, batch forms and pairings, used in turn."""
    B, H, D = 2, 2, 64
    g = torch.Generator().manual_seed(9)
    cases = []
    for S, per, pairs in ((5, False, "interleaved"), (5, False, "halves"), (5, True, "interleaved"), (8, False, "interleaved")):
        x, w, _ = _inputs(g, B, S, H, H, D, torch.bfloat16)
        cases.append((x, w, torch.randint(-50, 50, (B, 3, S) if per else (3, S), generator=g), pairs))
    for _ in range(2):
        for x, w, pos, pairs in cases:
            rope = qik.AxialRope(pos.to(DEV), _axes(D), pairs=pairs)
            out = qik.fused_qk_norm_rope(*(t.to(DEV) for t in (*x, *w)), rope, EPS)
            angle = oa.angles(pos, _axes(D), 1e4, "axis")
            for i in range(2):
                xd, wd = x[i].double(), w[i].double()
                _within(out[i], oa.forward(xd, wd, angle, pairs, EPS), oa.forward_bound(xd, wd, angle, pairs, EPS, torch.bfloat16))


def test_a_capture_beside_a_live_graph_is_refused():
    x, w, d, _, rope = _one()
    leaves = [t.requires_grad_() for t in (*x, *w)]
    alive = qik.fused_qk_norm_rope(*leaves, rope, EPS)
    stream, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=stream):
        with pytest.raises(RuntimeError, match="alive"):
            qik.fused_qk_norm_rope(*leaves, rope, EPS)
        with torch.no_grad():
            free = qik.fused_qk_norm_rope(*leaves, rope, EPS)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(alive, free))
    want = [t.clone() for t in torch.autograd.grad(alive, leaves, d)]
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        got = torch.autograd.grad(qik.fused_qk_norm_rope(*leaves, rope, EPS), leaves, d)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(p, q) for p, q in zip(got, want))


def test_offsets_past_32_bits():
    """Entries, then tokens, behind 4 GB of each other, in the inputs and in the gradients that come in."""
    B, S, Hq, Hk, D = 2, 5, 3, 2, 64
    x, w, d, _, rope = _one(B, S, Hq, Hk, D)
    buf = torch.zeros(2_400_000_000, dtype=torch.bfloat16, device=DEV)

    def both(xs, ds):
        leaves = [t.detach().requires_grad_() for t in (*xs, *w)]
        out = qik.fused_qk_norm_rope(*leaves, rope, EPS)
        return [*out, *torch.autograd.grad(out, leaves, ds)]

    want = both(x, d)
    for strides in ((2_300_000_000, 512, 64, 1), (512, 550_000_000, 64, 1)):
        def put(t, i):   # in turn within the 512 elements of a row of tokens
            return buf[4096 * i:].as_strided(t.shape, strides).copy_(t)

        for which in ((0,), (1,), (2, 3)):
            ts = [put(t, i) if i in which else t for i, t in enumerate((*x, *d))]
            assert all(torch.equal(a, b) for a, b in zip(both(ts[:2], ts[2:]), want)), (strides, which)


def test_a_capture_beside_a_warm_up_that_lives_on():
    """Warm up on a side stream, keep its outputs and loss, capture on the graph's own stream: as torch's own recipe goes."""
    x, w, d, _, rope = _one(B=2, S=40)
    leaves = [t.requires_grad_() for t in (*x, *w)]

    def loss_of(outs):
        return sum((o.float() * g.float()).sum() for o, g in zip(outs, d))

    side, stream = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        kept = qik.fused_qk_norm_rope(*leaves, rope, EPS)
        kept_loss = loss_of(kept)
        kept_loss.backward()
        never_run = qik.fused_qk_norm_rope(*leaves, rope, EPS)
    torch.cuda.synchronize()
    want = [*(t.detach().clone() for t in kept), *(t.grad.clone() for t in leaves)]
    for t in leaves:
        t.grad = None
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        outs = qik.fused_qk_norm_rope(*leaves, rope, EPS)
        loss_of(outs).backward()
    got = [*outs, *(t.grad for t in leaves)]
    for _ in range(4):
        for t in got:
            t.detach().zero_()
        graph.replay()
        again = torch.autograd.grad(never_run, leaves, d, retain_graph=True)   # the other stream's graph, between the replays
        torch.cuda.synchronize()
        assert all(torch.equal(a.detach(), b) for a, b in zip(got, want))
        assert all(torch.equal(a, b) for a, b in zip(again, want[2:]))
    del kept, kept_loss, never_run
