"""GPU tests of linear attention: whole sequences, their gradients, single tokens.

The oracle is the recurrence itself, token by token in 64 bits, and autograd through it.  Tolerances, on the 2-norm of the
difference over that of the result:
    fp32  1e-5: sums of at most a few thousand products of fp32 values, rounded at 2^-24 each, with room for states that
          decay over a thousand tokens;
    bf16  3 * 2^-9: at most three roundings to 8 bits on the way of a value (a score or a state that enters a matrix
          product, the output), each at most 2^-9 of it.
States and the gradients of decays are fp32 whatever the inputs' type.
"""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

TOL = {torch.float32: 1e-5, torch.bfloat16: 3 * 2.0 ** -9}
F32, BF16 = torch.float32, torch.bfloat16


def fss():
    import fast_sequential_scan_b200 as pkg
    return pkg


def oracle(q, k, v, g, scale, h0=None, lengths=None):
    """(o, state behind the last token) in 64 bits, differentiable."""
    B, T = q.shape[:2]
    H = max(q.shape[2], k.shape[2], v.shape[2])
    q, k, v = (t.double().repeat_interleave(H // t.shape[2], 2) for t in (q, k, v))
    g = g.double().expand(B, T, H)
    S = h0.double() if h0 is not None else q.new_zeros(B, H, q.shape[3], v.shape[3])
    o = []
    for t in range(T):
        live = torch.ones(B, dtype=torch.bool, device=q.device) if lengths is None else t < lengths
        m = live[:, None, None]
        kt, vt, qt = (torch.where(m, x[:, t], 0.0) for x in (k, v, q))
        a = torch.where(live[:, None], g[:, t], 0.0).exp()
        S = a[..., None, None] * S + kt[..., :, None] * vt[..., None, :]
        o.append(scale * (qt[..., None, :] @ S)[..., 0, :])
    return (torch.stack(o, 1) if o else v), S


def relative(x, y):
    x, y = x.double(), y.double()
    assert x.shape == y.shape
    assert torch.isfinite(x).all()
    n = y.norm()
    return ((x - y).norm() / n).item() if n > 0 else x.norm().item()


def make(B, T, H, K, V, dtype, Hk=None, Hv=None, decay="gated", state=True, ragged=False, seed=0, layout="plain"):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    Hk, Hv = Hk or H, Hv or H
    if layout == "fused":
        row = rnd(B, T, H * K + Hk * K + Hv * V).to(dtype)
        q, k, v = row.split([H * K, Hk * K, Hv * V], -1)
        q, k, v = q.unflatten(-1, (H, K)), k.unflatten(-1, (Hk, K)), v.unflatten(-1, (Hv, V))
    elif layout == "heads_first":
        q, k, v = (rnd(B, h, T, d).to(dtype).transpose(1, 2) for h, d in ((H, K), (Hk, K), (Hv, V)))
    elif layout == "unaligned":
        q, k, v = (rnd(B, T, h, d + 1).to(dtype)[..., 1:] for h, d in ((H, K), (Hk, K), (Hv, V)))
    elif layout == "channels_apart":
        q, k, v = (rnd(B, T, d, h).to(dtype).transpose(2, 3) for h, d in ((H, K), (Hk, K), (Hv, V)))
    elif layout == "broadcast":
        q, k, v = (rnd(1, T, h, d).to(dtype).expand(B, T, h, d) for h, d in ((H, K), (Hk, K), (Hv, V)))
    else:
        q, k, v = (rnd(B, T, h, d).to(dtype) for h, d in ((H, K), (Hk, K), (Hv, V)))
    if decay == "gated":
        g = -torch.rand(B, T, H, generator=gen, device="cuda") ** 3 * 2
        g = torch.where(torch.rand(B, T, H, generator=gen, device="cuda") < 0.03, torch.full_like(g, -math.inf), g)
    elif decay == "strong":
        g = -30.0 * torch.rand(B, T, H, generator=gen, device="cuda")
    elif decay == "none":
        g = torch.zeros(H, device="cuda")
    else:
        g = -0.2 * torch.rand(H, generator=gen, device="cuda")
    h0 = rnd(B, H, K, V) if state else None
    lengths = None
    if ragged:
        lengths = torch.randint(0, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
        lengths[0] = 0
        if B > 1:
            lengths[1] = T
    return q, k, v, g, h0, lengths


LENGTHS = [1, 2, 17, 31, 32, 33, 63, 64, 65, 127, 128, 129, 190, 257]
DIMS = [(128, 128), (64, 64), (64, 128), (128, 64), (32, 32), (16, 80), (96, 40), (1, 3), (33, 7), (72, 130), (256, 256), (200, 64)]


def check_forward(case, scale=None):
    q, k, v, g, h0, lengths = case
    o, last = fss().linear_attention(q, k, v, g, h0=h0, return_final_state=True, lengths=lengths, scale=scale)
    ro, rlast = oracle(q, k, v, g, scale or q.shape[-1] ** -0.5, h0, lengths)
    fss().check_status()
    assert relative(o, ro) <= TOL[q.dtype]
    assert last.dtype == F32 and relative(last, rlast) <= TOL[F32]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", LENGTHS)
def test_forward_lengths(T, dtype):
    check_forward(make(2, T, 3, 64, 64, dtype, seed=T))
    check_forward(make(3, T, 2, 128, 128, dtype, ragged=True, seed=T + 1, state=T % 2 == 0, decay="fixed"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K,V", DIMS)
def test_forward_dimensions(K, V, dtype):
    check_forward(make(2, 150, 2, K, V, dtype, seed=K + V))
    check_forward(make(1, 70, 4, K, V, dtype, Hk=1, Hv=2, seed=K + V, state=False, decay="fixed"))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["fused", "heads_first", "unaligned", "channels_apart", "broadcast"])
def test_forward_layouts(layout, dtype):
    check_forward(make(2, 150, 4, 64, 128, dtype, Hk=2, layout=layout))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("decay", ["strong", "none", "fixed"])
def test_forward_decays(decay, dtype):
    check_forward(make(2, 200, 2, 128, 128, dtype, decay=decay, seed=5))
    check_forward(make(2, 200, 2, 64, 64, dtype, decay=decay, seed=6), scale=0.7)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_long_sequences_are_cut_into_segments(dtype):
    """A few states and many tokens: the segments' own sums, folded, have to be the sequential state."""
    check_forward(make(1, 3000, 1, 128, 128, dtype, decay="fixed", seed=9))
    check_forward(make(2, 2113, 2, 64, 64, dtype, ragged=True, seed=10))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K,V", [(64, 64), (128, 128), (40, 24)])
def test_rows_behind_a_sequence_are_not_read(K, V, dtype):
    q, k, v, g, h0, _ = make(3, 140, 2, K, V, dtype)
    lengths = torch.tensor([0, 77, 140], dtype=torch.int32, device="cuda")
    want = fss().linear_attention(q, k, v, g, h0=h0, lengths=lengths, return_final_state=True)
    behind = torch.arange(140, device="cuda")[None, :] >= lengths[:, None]
    for bad in (math.nan, math.inf):
        dirty = [torch.where(behind[..., None, None], torch.full_like(t, bad), t) for t in (q, k, v)]
        dirty_g = torch.where(behind[..., None], torch.full_like(g, bad), g)
        got = fss().linear_attention(*dirty, dirty_g, h0=h0, lengths=lengths, return_final_state=True)
        for x, y in zip(got, want):
            assert torch.equal(x, y)
    assert torch.equal(want[1][0], h0[0])
    assert not want[0][behind].any()
    for out_of_range in ([-5, 77, 140], [0, 77, 4000]):      # clamped
        got = fss().linear_attention(q, k, v, g, h0=h0, lengths=torch.tensor(out_of_range, dtype=torch.int32, device="cuda"))
        assert torch.equal(got, want[0])


def gradients(case, seed=1, scale=None, f=None):
    q, k, v, g, h0, lengths = case
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g)] + ([h0.detach().requires_grad_()] if h0 is not None else [])
    gen = torch.Generator(device="cuda").manual_seed(seed)
    o, last = f(*leaves[:4], leaves[4] if h0 is not None else None, lengths)
    upstream = [torch.randn(x.shape, generator=gen, device="cuda").to(q.dtype if i == 0 else F32) for i, x in enumerate((o, last))]
    if f is not own_call:
        upstream = [u.double() for u in upstream]
    return torch.autograd.grad([o, last], leaves, upstream)


def own_call(q, k, v, g, h0, lengths):
    return fss().linear_attention(q, k, v, g, h0=h0, return_final_state=True, lengths=lengths)


def oracle_call(q, k, v, g, h0, lengths):
    return oracle(q, k, v, g, q.shape[-1] ** -0.5, h0, lengths)


def check_gradients(case):
    got, want = gradients(case, f=own_call), gradients(case, f=oracle_call)
    fss().check_status()
    names = ["dq", "dk", "dv", "dlog_decay", "dh0"]
    for name, x, y in zip(names, got, want):
        assert relative(x, y) <= TOL[x.dtype], (name, relative(x, y))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("T", [1, 2, 31, 33, 64, 65, 128, 129, 200])
def test_gradient_lengths(T, dtype):
    check_gradients(make(2, T, 2, 64, 64, dtype, seed=T))
    check_gradients(make(3, T, 2, 128, 128, dtype, seed=T, ragged=True, decay="fixed", state=T % 2 == 1))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K,V", [(64, 128), (128, 64), (16, 80), (1, 3), (33, 7), (72, 130), (256, 200)])
def test_gradient_dimensions(K, V, dtype):
    check_gradients(make(2, 90, 2, K, V, dtype, seed=K))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("H,Hq,Hk,Hv", [(4, 4, 2, 4), (4, 4, 1, 2), (6, 2, 3, 6), (4, 1, 4, 1)])
def test_gradients_of_shared_heads(H, Hq, Hk, Hv, dtype):
    q, k, v, g, h0, lengths = make(2, 100, H, 64, 32, dtype, Hk=Hk, Hv=Hv, ragged=True)
    check_gradients((q[:, :, :Hq], k, v, g, h0, lengths))
    fixed = make(2, 100, H, 64, 64, dtype, Hk=Hk, Hv=Hv, decay="fixed")
    check_gradients((fixed[0][:, :, :Hq], *fixed[1:]))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("layout", ["fused", "heads_first", "unaligned", "channels_apart", "broadcast"])
def test_gradient_layouts(layout, dtype):
    check_gradients(make(2, 100, 2, 64, 64, dtype, layout=layout, decay="fixed"))


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_gradients_of_long_sequences(dtype):
    check_gradients(make(1, 1500, 1, 64, 64, dtype, seed=3))
    check_gradients(make(1, 1500, 2, 128, 128, dtype, seed=4, decay="fixed", state=False))


@pytest.mark.parametrize("want", [("q",), ("k",), ("v",), ("g",), ("h0",), ("q", "v"), ("k", "g")])
def test_only_the_gradients_that_are_asked_for(want):
    q, k, v, g, h0, _ = make(2, 80, 2, 64, 64, BF16)
    named = dict(q=q, k=k, v=v, g=g, h0=h0)
    everything = {n: t.detach().requires_grad_() for n, t in named.items()}
    some = {n: t.detach().requires_grad_(n in want) for n, t in named.items()}
    up = torch.randn(2, 80, 2, 64, device="cuda").to(BF16)
    run = lambda d: fss().linear_attention(d["q"], d["k"], d["v"], d["g"], h0=d["h0"])
    full = dict(zip(named, torch.autograd.grad(run(everything), list(everything.values()), up)))
    got = torch.autograd.grad(run(some), [some[n] for n in want], up)
    for n, x in zip(want, got):
        assert relative(x, full[n]) <= TOL[x.dtype]


def test_gradient_against_differences():
    """Central differences of the fp32 operator itself along random directions.  A step of 2^-6 of an input of order 1 leaves a
    curvature error of its square (2.4e-4) and rounding errors of 2^-24 * 2^6 (4e-6) of the function's scale, so 2e-3 of the
    largest directional derivative.  A constant decay acts once for each of the 40 tokens, so it moves by a fortieth."""
    q, k, v, g, h0, _ = make(2, 40, 2, 16, 24, F32, decay="fixed")
    up, up_last = torch.randn(2, 40, 2, 24, device="cuda"), torch.randn(2, 2, 16, 24, device="cuda")
    leaves = [t.detach().requires_grad_() for t in (q, k, v, g, h0)]

    def value(ts):
        o, last = own_call(*ts, None)
        return (o.double() * up).sum() + (last.double() * up_last).sum()

    grads = torch.autograd.grad(value(leaves), leaves)
    found = []
    for i, d in enumerate(grads):
        direction = torch.randn_like(leaves[i])
        direction /= direction.abs().max() * (40 if leaves[i] is leaves[3] else 1)
        moved = []
        with torch.no_grad():
            for e in (2.0 ** -6, -2.0 ** -6):
                ts = [t.detach() for t in leaves]
                ts[i] = ts[i] + e * direction
                moved.append(value(ts).item())
        found.append(((d.double() * direction).sum().item(), (moved[0] - moved[1]) / 2.0 ** -5))
    largest = max(abs(a) for a, _ in found)
    for a, b in found:
        assert abs(a - b) <= 2e-3 * largest, found


def test_empty_calls():
    q, k, v, g, h0, _ = make(2, 4, 2, 64, 64, BF16, decay="fixed")
    o, last = fss().linear_attention(q[:, :0], k[:, :0], v[:, :0], g, h0=h0, return_final_state=True)
    assert o.shape == (2, 0, 2, 64) and torch.equal(last, h0)
    o, last = fss().linear_attention(q[:, :0], k[:, :0], v[:, :0], g, return_final_state=True)
    assert not last.any()
    o, last = fss().linear_attention(q[:0], k[:0], v[:0], g, return_final_state=True)
    assert o.shape == (0, 4, 2, 64) and last.shape == (0, 2, 64, 64)
    h0 = h0.requires_grad_()
    _, last = fss().linear_attention(q[:, :0], k[:, :0], v[:, :0], g, h0=h0, return_final_state=True)
    assert torch.equal(torch.autograd.grad(last.sum(), h0)[0], torch.ones_like(h0))


def test_a_sequence_in_two_calls():
    q, k, v, g, h0, _ = make(2, 200, 2, 128, 128, BF16, decay="fixed")
    o, last = fss().linear_attention(q, k, v, g, h0=h0, return_final_state=True)
    o1, mid = fss().linear_attention(q[:, :77], k[:, :77], v[:, :77], g, h0=h0, return_final_state=True)
    o2, last2 = fss().linear_attention(q[:, 77:], k[:, 77:], v[:, 77:], g, h0=mid, return_final_state=True)
    assert relative(torch.cat([o1, o2], 1), o) <= TOL[BF16]
    assert relative(last2, last) <= TOL[F32]


def test_repeated_calls_give_the_same_bits():
    case = make(2, 700, 4, 128, 128, BF16, Hk=2)
    first = gradients(case, f=own_call)
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, gradients(case, f=own_call)))


def test_on_another_stream_and_in_a_graph():
    q, k, v, g, h0, _ = make(2, 300, 2, 128, 128, BF16)
    want = fss().linear_attention(q, k, v, g, h0=h0, return_final_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = fss().linear_attention(q, k, v, g, h0=h0, return_final_state=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fss().linear_attention(q, k, v, g, h0=h0, return_final_state=True)
    for t in got:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    fss().check_status()


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K,V", [(129, 64), (144, 144), (160, 20), (161, 161), (192, 130), (193, 65)])
def test_wide_keys(K, V, dtype):
    check_forward(make(2, 77, 2, K, V, dtype, ragged=True, seed=K))
    check_gradients(make(1, 50, 2, K, V, dtype, Hk=1, seed=V))


@pytest.mark.parametrize("T", [70, 128])
@pytest.mark.parametrize("V,pitch", [(52, 64), (64, 72), (40, 41)])
def test_outputs_between_other_data(V, pitch, T):
    """Rows of outputs with a gap behind each: nothing else is written (through the C entry; the Python functions make contiguous ones)."""
    import ctypes
    from fast_sequential_scan_b200 import _lib, attention_cuda, workspace
    q, k, v, g, _, _ = make(2, T, 2, 64, V, BF16, decay="fixed", state=False)
    v = torch.nn.functional.pad(v, (0, 64 - V))[..., :V]      # rows of 128 bytes
    room = torch.full((2, T, 2, pitch), 7.0, device="cuda", dtype=BF16)
    p = attention_cuda._problem(q, k, v, g, None, None, 0.125, 2, T)
    out = _lib.Heads(room.data_ptr(), T * 2 * pitch, 2 * pitch, pitch, 2, V)
    ctx = workspace.call_context(q.device, attention_cuda._scratch(p, 0, q.device))
    _lib.check(_lib.lib().fss_linear_attention_forward(ctypes.byref(ctx), ctypes.byref(p), ctypes.byref(out), None), "forward")
    fss().check_status()
    assert relative(room[..., :V], oracle(q, k, v, g, 0.125)[0]) <= TOL[BF16]
    assert (room[..., V:] == 7.0).all()


# ------------------------------------------------------------------ single tokens
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("K,V", DIMS)
@pytest.mark.parametrize("slots", [False, True])
def test_step(K, V, dtype, slots):
    q, k, v, g, _, _ = make(5, 1, 4, K, V, dtype, Hk=2, Hv=1, seed=K)
    q, k, v, g = q[:, 0], k[:, 0], v[:, 0], g[:, 0]
    pool = torch.randn(9, 4, K, V, device="cuda")
    where = torch.tensor([7, 0, 3, 8, 2], dtype=torch.int32, device="cuda")
    rows = where.long() if slots else torch.arange(5, device="cuda")
    ro, rs = oracle(q[:, None], k[:, None], v[:, None], g[:, None], K ** -0.5, pool[rows])
    want = pool.double()
    want[rows] = rs
    o = fss().linear_attention_step(q, k, v, g, pool, slots=where if slots else None)
    assert relative(o, ro[:, 0]) <= TOL[dtype]
    assert relative(pool, want) <= TOL[F32]
    untouched = torch.ones(9, dtype=torch.bool, device="cuda")
    untouched[rows] = False
    assert torch.equal(pool[untouched], want[untouched].float())


def test_step_leaves_padding_alone():
    q, k, v, g, _, _ = make(4, 1, 2, 64, 64, BF16)
    q, k, v, g = q[:, 0], k[:, 0], v[:, 0], g[:, 0]
    k = torch.where(torch.tensor([0, 1, 1, 0], device="cuda", dtype=torch.bool)[:, None, None], torch.full_like(k, math.nan), k)
    pool = torch.randn(3, 2, 64, 64, device="cuda")
    before = pool.clone()
    o = fss().linear_attention_step(q, k, v, g, pool, slots=torch.tensor([2, -1, 3, 0], dtype=torch.int32, device="cuda"))
    assert torch.equal(pool[1], before[1]) and not torch.equal(pool[0], before[0]) and not torch.equal(pool[2], before[2])
    assert not o[1].any() and not o[2].any() and torch.isfinite(o.float()).all()
    o = fss().linear_attention_step(q[:0], k[:0], v[:0], g[:0], pool)
    assert o.shape == (0, 2, 64)


def test_step_continues_a_sequence():
    q, k, v, g, h0, _ = make(3, 40, 2, 128, 64, F32)
    o, last = fss().linear_attention(q, k, v, g, h0=h0, return_final_state=True)
    state = h0.clone()
    outs = [fss().linear_attention_step(q[:, t], k[:, t], v[:, t], g[:, t], state) for t in range(40)]
    assert relative(torch.stack(outs, 1), o) <= TOL[F32] and relative(state, last) <= TOL[F32]


def test_step_strides():
    """States inside a larger allocation, unaligned states, a constant decay, heads of one projection's output."""
    row = torch.randn(3, 4 * 64 * 3, device="cuda").to(BF16)
    q, k, v = (t.unflatten(-1, (4, 64)) for t in row.split(256, -1))
    g = -torch.rand(4, device="cuda")
    for offset, gap in ((0, 8), (1, 3)):
        store = torch.randn(3 * (4 * 64 * 64 + gap) + offset, device="cuda")
        state = store[offset:].view(3, -1)[:, :4 * 64 * 64].unflatten(1, (4, 64, 64))
        ro, rs = oracle(q[:, None], k[:, None], v[:, None], g, 0.125, state)
        o = fss().linear_attention_step(q, k, v, g, state)
        assert relative(o, ro[:, 0]) <= TOL[BF16] and relative(state, rs) <= TOL[F32]


# ------------------------------------------------------------------ refusals
def test_refusals():
    q, k, v, g, h0, _ = make(2, 8, 4, 16, 16, BF16)
    f, step = fss().linear_attention, fss().linear_attention_step
    for bad in (dict(q=q.cpu()), dict(q=q.half(), k=k.half(), v=v.half()), dict(k=k.float()), dict(k=k[:, :7]), dict(k=k[..., :8]), dict(k=k[:, :, :3]),
                dict(q=q[0]), dict(log_decay=g.to(BF16)), dict(log_decay=g[:, :, :3]), dict(log_decay=g[:, 0]), dict(h0=h0[:1]),
                dict(h0=h0.long()), dict(lengths=torch.tensor([1, 2], device="cuda")), dict(lengths=torch.tensor([1], device="cuda", dtype=torch.int32)),
                dict(v=torch.zeros(2, 8, 4, 300, device="cuda", dtype=BF16)), dict(q=q[:, :, :0])):
        args = dict(dict(q=q, k=k, v=v, log_decay=g), **bad)
        with pytest.raises((RuntimeError, TypeError)):
            f(args.pop("q"), args.pop("k"), args.pop("v"), args.pop("log_decay"), **args)
    state = torch.zeros(2, 4, 16, 16, device="cuda")
    q, k, v, g = q[:, 0], k[:, 0], v[:, 0], g[:, 0]
    for bad in (dict(state=state[:1]), dict(state=state.double()), dict(state=state.transpose(2, 3)), dict(state=state[:, :2]),
                dict(slots=torch.zeros(2, device="cuda", dtype=torch.int64)), dict(slots=torch.zeros(3, device="cuda", dtype=torch.int32)),
                dict(state=torch.zeros(1, 4, 16, 16, device="cuda").expand(2, 4, 16, 16)), dict(q=q.clone().requires_grad_())):
        args = dict(dict(q=q, k=k, v=v, log_decay=g, state=state), **bad)
        with pytest.raises((RuntimeError, TypeError)):
            step(args.pop("q"), args.pop("k"), args.pop("v"), args.pop("log_decay"), args.pop("state"), **args)
