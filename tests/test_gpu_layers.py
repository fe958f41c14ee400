"""GPU tests of rotary positions and of the root-mean-square norm, against plain implementations in 64 bits.

Tolerances on the 2-norm of the difference over that of the result: bf16 2^-8 and one part in a thousand of it (one
rounding to 8 bits: half of a spacing of 2^-7), fp32 2e-6 (angles and sums of a row at a few 2^-24; a weight's gradient, a
sum over rows whose terms may cancel, against the sum of their magnitudes), e4m3 2^-4 (half a step of 3 bits) and as much
of 2^-9 for each scale's smallest step.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

F32, BF16 = torch.float32, torch.bfloat16
TOL = {BF16: 2.0 ** -8 * 1.001, F32: 2e-6}


def fss():
    import fast_sequential_scan_b200 as pkg
    return pkg


def relative(x, y):
    x, y = x.double(), y.double()
    assert x.shape == y.shape and torch.isfinite(x).all()
    n = y.norm()
    return ((x - y).norm() / n).item() if n > 0 else x.norm().item()


# ------------------------------------------------------------------ rotary positions
def turned(x, positions, frequencies, layout, magnitude=1.0, sign=1.0):
    x = x.double()
    r = 2 * len(frequencies)
    angle = positions.double()[..., None] * frequencies * sign
    cos, sin = (magnitude * f(angle)[..., None, :] for f in (torch.cos, torch.sin))
    if positions.dim() == 1:
        cos, sin = cos[None], sin[None]
    y = x.clone()
    a, b = (slice(0, r, 2), slice(1, r, 2)) if layout == "interleaved" else (slice(0, r // 2), slice(r // 2, r))
    y[..., a], y[..., b] = x[..., a] * cos - x[..., b] * sin, x[..., a] * sin + x[..., b] * cos
    return y


def frequencies(r, base=10000.0):
    return torch.tensor([base ** (-2.0 * j / r) for j in range(r // 2)], dtype=torch.float64, device="cuda")


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
@pytest.mark.parametrize("D,r", [(128, 128), (128, 64), (64, 32), (96, 96), (80, 20), (34, 34), (7, 2), (256, 250), (16, 16)])
@pytest.mark.parametrize("B,T,H,Hk", [(2, 65, 4, 2), (3, 1, 20, 4), (1, 700, 3, 3)])
def test_rotary(B, T, H, Hk, D, r, layout, dtype):
    gen = torch.Generator(device="cuda").manual_seed(D + r)
    q, k = (torch.randn(B, T, h, D, generator=gen, device="cuda").to(dtype) for h in (H, Hk))
    turns, magnitude = fss().rotary_turns(r, device="cuda")
    assert magnitude == 1.0
    positions = torch.randint(0, 50_000, (B, T), generator=gen, device="cuda")
    got = fss().rotary(q, k, positions, turns, layout=layout)
    for x, y in zip((q, k), got):
        assert relative(y, turned(x, positions, frequencies(r), layout)) <= TOL[dtype]
        assert torch.equal(y[..., r:], x[..., r:])
    alone = fss().rotary(q, None, positions[0], turns, layout=layout, magnitude=1.25)
    assert relative(alone[..., :r], turned(q, positions[0], frequencies(r), layout, 1.25)[..., :r]) <= TOL[dtype]


@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_far_positions(layout):
    """Angles stay exact where the product of position and frequency has long left fp32 (and fp64) behind."""
    q = torch.randn(1, 4, 2, 64, device="cuda")
    turns, _ = fss().rotary_turns(64, device="cuda")
    positions = torch.tensor([10_000_019, 2 ** 40 + 3, -5, 2 ** 62 - 1], device="cuda")
    words = [int(w) for w in turns.cpu()]
    angle = torch.tensor([[((p * w) % 2 ** 64) / 2 ** 64 * 2 * math.pi for w in words] for p in positions.tolist()], dtype=torch.float64, device="cuda")
    cos, sin = angle.cos()[None, :, None], angle.sin()[None, :, None]
    got = fss().rotary(q, None, positions, turns, layout=layout)
    x = q.double()
    a, b = (x[..., 0::2], x[..., 1::2]) if layout == "interleaved" else (x[..., :32], x[..., 32:])
    y = (a * cos - b * sin, a * sin + b * cos)
    want = torch.stack(y, -1).flatten(-2) if layout == "interleaved" else torch.cat(y, -1)
    assert relative(got, want) <= TOL[F32]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["half", "interleaved"])
def test_rotary_strides_and_gradients(layout, dtype):
    row = torch.randn(2, 50, 6 * 64 + 3, device="cuda").to(dtype)
    turns, _ = fss().rotary_turns(48, device="cuda")
    positions = torch.arange(50, device="cuda", dtype=torch.int32) + 7
    for start in (0, 8, 3):      # wide and narrow accesses
        q, k = row[..., start:start + 256].unflatten(-1, (4, 64)), row[..., :128].unflatten(-1, (2, 64))
        assert relative(fss().rotary(q, k, positions, turns, layout=layout)[0], turned(q, positions, frequencies(48), layout)) <= TOL[dtype]
    q = torch.randn(2, 4, 50, 64, device="cuda").to(dtype).transpose(1, 2).requires_grad_()
    k = torch.randn(2, 50, 2, 64, device="cuda").to(dtype).requires_grad_()
    out = fss().rotary(q, k, positions, turns, layout=layout, magnitude=1.5)
    up = [torch.randn(t.shape, device="cuda").to(dtype) for t in out]
    for g, u, x in zip(torch.autograd.grad(out, [q, k], up), up, (q, k)):
        want = turned(u, positions, frequencies(48), layout, 1.5, -1.0)
        assert relative(g[..., :48], want[..., :48]) <= TOL[dtype] and torch.equal(g[..., 48:], u[..., 48:])


def test_rotary_gradient_against_differences():
    """The rotation is linear, so a difference over a step of 1 has no curvature error: what is left is rounding, 2^-22 of sums
    of a few thousand terms."""
    q = torch.randn(1, 9, 3, 32, device="cuda").requires_grad_()
    turns, _ = fss().rotary_turns(32, device="cuda")
    up, step, positions = torch.randn(1, 9, 3, 32, device="cuda"), torch.randn(1, 9, 3, 32, device="cuda"), torch.arange(9, device="cuda")
    g, = torch.autograd.grad(fss().rotary(q, None, positions, turns), q, up)
    value = lambda x: (fss().rotary(x, None, positions, turns).double() * up).sum().item()
    with torch.no_grad():
        moved = value(q + step) - value(q - step)
    assert abs(moved / 2 - (g.double() * step).sum().item()) <= 1e-4


def test_rotary_empty_and_refusals():
    f = fss().rotary
    turns, _ = fss().rotary_turns(16, device="cuda")
    q, p = torch.randn(2, 5, 2, 32, device="cuda"), torch.arange(5, device="cuda")
    assert f(q[:, :0], None, p[:0], turns).shape == (2, 0, 2, 32)
    for args, kw in (((q.cpu(), None, p, turns), {}), ((q.half(), None, p, turns), {}), ((q, q[:, :4], p, turns), {}), ((q, q[..., :16], p, turns), {}),
                     ((q, q.to(BF16), p, turns), {}), ((q, None, p.float(), turns), {}), ((q, None, p[:4], turns), {}), ((q, None, p, turns.float()), {}),
                     ((q[..., :8], None, p, turns), {}), ((q, None, p, turns[:0]), {}), ((q, None, p, turns), {"layout": "pairs"}),
                     ((q, None, p, turns.cpu()), {}), ((q[:, :, 0], None, p, turns), {})):
        with pytest.raises((RuntimeError, TypeError, ValueError)):
            f(*args, **kw)


# ------------------------------------------------------------------ root-mean-square norm
def norm64(x, w, residual=None, eps=1e-6):
    s = x if residual is None else (x.double() + residual.double()).to(x.dtype)
    f = s.double()
    return f / (f.square().mean(-1, keepdim=True) + eps).sqrt() * w.double(), s


WIDTHS = [1, 3, 8, 64, 100, 128, 250, 768, 1000, 1024, 1025, 2048, 2560, 4096, 8192, 16384, 40000]


def norm_case(shape, dtype, wide, residual, seed=0):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x = rnd(*shape).to(dtype)
    return x, (1 + 0.2 * rnd(shape[-1])).to(F32 if wide else dtype), (2 * rnd(*shape)).to(dtype) if residual else None


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", WIDTHS)
@pytest.mark.parametrize("residual", [False, True])
def test_norm(D, dtype, residual):
    for shape, wide in (((2, 9, D), False), ((1, D), True), ((D,), True), ((2, 3, 5, D), False)):
        x, w, r = norm_case(shape, dtype, wide, residual, D)
        y, s = norm64(x, w, r)
        got = fss().rms_norm(x, w, residual=r)
        if residual:
            assert torch.equal(got[1], s)
            got = got[0]
        assert relative(got, y) <= TOL[dtype]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D", WIDTHS)
def test_norm_gradients(D, dtype):
    for rows, wide, residual in ((9, False, True), (1, True, False), (700, True, True)):
        if rows * D > 4_000_000:
            continue
        x, w, r = norm_case((1, rows, D), dtype, wide, residual, D)
        leaves = [t.requires_grad_() for t in (x, w, r) if t is not None]
        out = fss().rms_norm(x, w, residual=r)
        out = list(out) if residual else [out]
        up = [torch.randn(x.shape, device="cuda").to(dtype) for _ in out]
        got = torch.autograd.grad(out, leaves, up)
        # the oracle normalises the stored sum, as the definition says
        s = norm64(x.detach(), w.detach(), r.detach() if residual else None)[1].double().requires_grad_()
        w64 = w.detach().double().requires_grad_()
        y = s / (s.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w64
        ds, dw = torch.autograd.grad([y] + ([s * 1.0] if residual else []), [s, w64], [u.double() for u in up])
        # one channel: dx is a difference of two equal terms; what is left is eps's share and rounding of the terms
        scale = up[0].double().norm().item() if D == 1 else 0.0
        assert (got[0].double() - ds).norm().item() <= TOL[dtype] * ds.norm().item() + 1e-6 * scale
        terms = (up[0].double() * s * (s.square().mean(-1, keepdim=True) + 1e-6).rsqrt()).abs().sum((0, 1))
        assert (got[1].double() - dw).norm().item() <= (TOL[BF16] * dw.norm().item() if got[1].dtype == BF16 else 0.0) + TOL[F32] * terms.norm().item()
        if residual:
            assert torch.equal(got[2], got[0])


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("D,group", [(128, None), (100, None), (2560, None), (40000, None), (1024, 128), (2560, 64), (96, 32), (4096, 128), (40064, 128), (64, 32)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm_quantized(D, group, residual, dtype):
    x, w, r = norm_case((2, 7, D), dtype, D % 3 == 0, residual, D)
    x[0, 1] = 0.0
    if residual:
        r[0, 1] = 0.0
    y, s = norm64(x, w, r)
    out = fss().rms_norm_quantized(x, w, residual=r, group=group)
    held, scales = out[:2]
    assert held.dtype == torch.float8_e4m3fn and scales.dtype == F32
    if residual:
        assert torch.equal(out[2], s)
    groups = y.unflatten(-1, (-1, group)) if group else y[..., None, :]
    most = groups.abs().amax(-1)
    want_scales = most / 448.0
    assert relative(scales, want_scales if group else want_scales[..., 0]) <= 2e-6
    # half a step of 3 bits relative to the value, or half of the smallest step (2^-9) of the scale
    back = held.float().double().unflatten(-1, (-1, group)) if group else held.float().double()[..., None, :]
    back = back * want_scales[..., None]
    limit = groups.abs() * (2.0 ** -4 + 1e-5) + want_scales[..., None] * 2.0 ** -10 * 1.001
    assert ((back - groups).abs() <= limit).all()
    assert not held[0, 1].float().any() and not scales[0, 1].any()


def test_norm_quantized_extremes():
    """Rows of tiny values, a NaN in one row and an infinity in another stay in their rows."""
    x = torch.randn(6, 256, device="cuda")
    clean = x.clone()
    w = torch.ones(256, device="cuda")
    x[1, 5], x[3, 9], x[4] = math.nan, math.inf, 1e-38 * x[4]
    for group in (None, 128):
        held, scales = fss().rms_norm_quantized(x, w, group=group)
        want, want_scales = fss().rms_norm_quantized(clean, w, group=group)
        for row in (0, 2, 5):
            assert torch.equal(held[row].float(), want[row].float()) and torch.equal(scales[row], want_scales[row])
        assert held[1].float().isnan().any() and held[3].float().isnan().any()
        assert torch.isfinite(held[4].float()).all()


@pytest.mark.parametrize("D", [64, 250, 2048])
def test_norm_strides(D):
    x, w, r = norm_case((4, 6, 2 * D + 8), BF16, False, True)
    w = w[:D].contiguous()
    for start in (0, 8, 5):
        a, b = x[..., start:start + D], r[:, :, start:start + D]
        y, s = norm64(a, w, b)
        got = fss().rms_norm(a, w, residual=b)
        assert relative(got[0], y) <= TOL[BF16] and torch.equal(got[1], s)
    a = x[..., :D].transpose(0, 1)
    assert relative(fss().rms_norm(a, w), norm64(a, w)[0]) <= TOL[BF16]
    a = x[:1, :1, :D].expand(3, 6, D)
    assert relative(fss().rms_norm(a, w), norm64(a, w)[0]) <= TOL[BF16]


def test_norm_repeats_bit_for_bit_and_in_a_graph():
    x, w, r = norm_case((8, 300, 1024), BF16, False, True)
    leaves = [t.requires_grad_() for t in (x, w, r)]
    up = [torch.randn(x.shape, device="cuda").to(BF16) for _ in range(2)]
    grads = lambda: torch.autograd.grad(fss().rms_norm(x, w, residual=r), leaves, up)
    first = grads()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, grads()))
    with torch.no_grad():
        want = fss().rms_norm_quantized(x, w, residual=r)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = fss().rms_norm_quantized(x, w, residual=r)
        graph.replay()
        torch.cuda.synchronize()
    assert torch.equal(got[0].float(), want[0].float()) and torch.equal(got[1], want[1]) and torch.equal(got[2], want[2])


def test_norm_gradient_against_differences():
    """Central differences along random directions, step 2^-7: curvature 6e-5 and rounding 2^-24 * 2^7 (8e-6) of the value's
    scale, so 1e-3 of the largest derivative."""
    x, w, r = norm_case((2, 5, 96), F32, True, True)
    up = [torch.randn(x.shape, device="cuda") for _ in range(2)]
    leaves = [t.requires_grad_() for t in (x, w, r)]

    def value(ts):
        y, s = fss().rms_norm(ts[0], ts[1], residual=ts[2])
        return (y.double() * up[0]).sum() + (s.double() * up[1]).sum()

    grads, found = torch.autograd.grad(value(leaves), leaves), []
    for i, d in enumerate(grads):
        direction = torch.randn_like(leaves[i])
        direction /= direction.abs().max()
        with torch.no_grad():
            at = [[t.detach() + e * direction if j == i else t.detach() for j, t in enumerate(leaves)] for e in (2.0 ** -7, -2.0 ** -7)]
            found.append(((d.double() * direction).sum().item(), (value(at[0]) - value(at[1])).item() / 2.0 ** -6))
    largest = max(abs(a) for a, _ in found)
    assert all(abs(a - b) <= 1e-3 * largest for a, b in found), found


def test_norm_empty_and_refusals():
    x, w, r = norm_case((2, 3, 64), BF16, False, True)
    assert fss().rms_norm(x[:, :0], w).shape == (2, 0, 64)
    held, scales, s = fss().rms_norm_quantized(x[:0], w, residual=r[:0])
    assert held.shape == (0, 3, 64) and scales.shape == (0, 3) and s.shape == (0, 3, 64)
    z = x[:0].clone().requires_grad_()
    wz = w.clone().requires_grad_()
    assert not torch.autograd.grad(fss().rms_norm(z, wz).sum(), wz)[0].any()
    for args, kw in (((x.cpu(), w), {}), ((x.half(), w.half()), {}), ((x, w[:32]), {}), ((x, w.half()), {}), ((x.float(), w), {}), ((x, w[None]), {}),
                     ((x, w), {"residual": r[:1]}), ((x, w), {"residual": r.float()}), ((x, w.cpu()), {})):
        with pytest.raises((RuntimeError, TypeError)):
            fss().rms_norm(*args, **kw)
    for kw in ({"group": 48}, {"group": 256}, {"group": 0}):
        with pytest.raises(ValueError):
            fss().rms_norm_quantized(x, w, **kw)
    with pytest.raises(ValueError):
        fss().rms_norm_quantized(x[..., :40].contiguous(), w[:40].contiguous(), group=32)
    with pytest.raises(RuntimeError):
        fss().rms_norm_quantized(x.clone().requires_grad_(), w)
