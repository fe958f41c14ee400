"""The operators of recurrent layers with a matrix state, as measurable cases: linear attention with a decay for each head (prompts,
training and single tokens), rotary positions, and the root-mean-square norm between layers.

A case is a dict of plain values.  Common keys:

``op``              ``"attend"`` (:func:`linear_attention`), ``"step"`` (:func:`linear_attention_step`), ``"rotate"`` (:func:`rotary`) or
                    ``"norm"`` (:func:`rms_norm`, :func:`rms_norm_quantized`)
``dtype``           ``"bf16"`` or ``"f32"``, the type of the tensors; states, decays and scales are fp32
``batch, seq``      sequences and tokens of each
``grad``            a training step (forward, then the gradients of every input) or a forward alone under ``no_grad``

``attend`` and ``step``: ``heads`` states a sequence, each ``key_dim`` x ``value_dim``; ``key_heads`` and ``value_heads`` keys and values,
shared by groups of heads; ``decay``: ``"fixed"`` a constant for each head, ``"learned"`` the same with a gradient, ``"gated"`` a value for
each token and head, with the state emptied where a document starts; ``state``: start from a given state and return the last one;
``ragged``: sequences of different lengths, some empty; ``fused``: q, k and v are slices of one projection's output; ``slots``: the
sequences' states lie anywhere in a larger pool.
``rotate``: ``rotary_dim`` of the ``dim`` channels of each head are turned, ``layout`` says which make a pair.
``norm``: ``residual``: the residual stream is added first and returned; ``quant``: ``"none"``, or an e4m3 output with a scale for each
``"row"`` or each ``"group"`` of 128 channels.
"""
import math

import torch

own = False

_DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
EPS = 1e-6
GROUP = 128
CHUNK = 64          # tokens a chunk of the plain form
DOCUMENT = 700      # tokens of a document on the average, where a sequence holds several


def _attend(dtype="bf16", grad=True, decay="fixed", state=False, ragged=False, fused=False, key_heads=None, value_heads=None, value_dim=None,
            *, batch, seq, heads, key_dim, **more):
    return dict(more, op="attend", dtype=dtype, grad=grad, decay=decay, state=state, ragged=ragged, fused=fused, batch=batch, seq=seq,
                heads=heads, key_heads=key_heads or heads, value_heads=value_heads or heads, key_dim=key_dim, value_dim=value_dim or key_dim)


def _step(dtype="bf16", decay="fixed", slots=False, key_heads=None, value_dim=None, *, batch, heads, key_dim, **more):
    return dict(more, op="step", dtype=dtype, grad=False, decay=decay, slots=slots, batch=batch, seq=1, heads=heads,
                key_heads=key_heads or heads, value_heads=heads, key_dim=key_dim, value_dim=value_dim or key_dim)


def _rotate(dtype="bf16", grad=False, layout="half", key_heads=None, rotary_dim=None, *, batch, seq, heads, dim, **more):
    return dict(more, op="rotate", dtype=dtype, grad=grad, layout=layout, batch=batch, seq=seq, heads=heads, key_heads=key_heads or heads,
                dim=dim, rotary_dim=rotary_dim or dim)


def _norm(dtype="bf16", grad=False, residual=True, quant="none", *, batch, seq, width, **more):
    return dict(more, op="norm", dtype=dtype, grad=grad, residual=residual, quant=quant, batch=batch, seq=seq, width=width)


def listed():
    return [
        # a token for every sequence of a small serving batch: nothing but latency
        _step(name="step", batch=16, heads=20, key_dim=128),
        # decoding of a large batch whose states lie in a pool
        _step(name="step_pool", batch=256, heads=32, key_heads=8, key_dim=128, decay="gated", slots=True),
        # chunked prefill: prompts of different lengths, each continuing its own state
        _attend(name="prompt", batch=4, seq=1000, heads=16, key_dim=128, grad=False, state=True, ragged=True, fused=True),
        # one long prompt
        _attend(name="prompt_long", batch=1, seq=65536, heads=32, key_dim=128, grad=False, state=True),
        # the headline training shape, 16 heads of 64
        _attend(name="train", batch=8, seq=2048, heads=16, key_dim=64),
        # training with decays that depend on the token, several documents in a sequence, a length that fits no tile
        _attend(name="train_gated", batch=4, seq=3000, heads=16, key_dim=128, decay="gated"),
        # fp32 training with learned decays, truncated back-propagation through the state
        _attend(name="train_f32", batch=2, seq=1024, heads=12, key_dim=64, dtype="f32", decay="learned", state=True),
        # a large layer's training step, keys shared by groups of heads
        _attend(name="train_large", batch=16, seq=4096, heads=20, key_heads=4, key_dim=128),
        # positions of one token for every sequence of a serving batch
        _rotate(name="rotate_step", batch=16, seq=1, heads=20, key_heads=4, dim=128),
        # positions in training, interleaved pairs, half of each head
        _rotate(name="rotate_train", batch=8, seq=2048, heads=16, dim=128, rotary_dim=64, layout="interleaved", grad=True),
        # the norm before an 8-bit projection, one token for every sequence
        _norm(name="norm_step", batch=16, seq=1, width=2560, quant="row"),
        # the norm of a large layer's training step
        _norm(name="norm_train", batch=16, seq=4096, width=2560, grad=True),
    ]


def _log_uniform(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def _head_dim(rng):
    return rng.choice([64, 64, 128, 128, 128, 96, 80, 256, rng.randint(8, 200)])


def _groups(rng, heads):
    return rng.choice([heads, heads] + [h for h in range(1, heads + 1) if heads % h == 0])


def draw(rng):
    kind = rng.choice(["step", "prompt", "prompt", "train", "train", "gated", "f32", "rotate", "norm"])
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    if kind == "step":
        heads, dim = rng.choice([4, 8, 12, 16, 20, 32]), _head_dim(rng)
        batch = max(1, min(_log_uniform(rng, 1, 400), (256 * 32 * 128 * 128) // (heads * dim * dim)))
        return _step(dtype=dtype, batch=batch, heads=heads, key_heads=_groups(rng, heads), key_dim=dim, value_dim=rng.choice([dim, dim, 64, 128]),
                     decay=rng.choice(["fixed", "gated"]), slots=rng.random() < 0.5)
    if kind == "rotate":
        heads, dim = rng.choice([4, 8, 12, 16, 20, 32]), 2 * _log_uniform(rng, 16, 128)
        tokens = _log_uniform(rng, 1, (1 << 27) // (heads * dim))
        batch = min(tokens, _log_uniform(rng, 1, 32))
        return _rotate(dtype=dtype, batch=batch, seq=tokens // batch, heads=heads, key_heads=_groups(rng, heads), dim=dim,
                       rotary_dim=rng.choice([dim, dim, 2 * rng.randint(1, dim // 2)]), layout=rng.choice(["half", "interleaved"]),
                       grad=rng.random() < 0.4)
    if kind == "norm":
        width = rng.choice([768, 1024, 2048, 2560, 4096, _log_uniform(rng, 64, 8192)])
        tokens = _log_uniform(rng, 1, (1 << 27) // width)
        batch = min(tokens, _log_uniform(rng, 1, 32))
        grad = rng.random() < 0.5
        return _norm(dtype=dtype, batch=batch, seq=tokens // batch, width=width, residual=rng.random() < 0.7, grad=grad,
                     quant="none" if grad else rng.choice(["none", "row", "group"]) if width % GROUP == 0 else rng.choice(["none", "row"]))
    heads, dim = rng.choice([4, 8, 12, 16, 20, 32]), _head_dim(rng)
    # tokens times heads: from a small prompt's to half of the largest training case's
    work = _log_uniform(rng, 1 << 8, 1 << (18 if kind == "f32" else 19))
    work = max(heads, int(work * min(1.0, (128 / dim) ** 2)))
    batch = max(1, min(_log_uniform(rng, 1, 32), work // heads))
    seq = max(1, min(32768, work // (heads * batch)))
    more = dict(batch=batch, seq=seq, heads=heads, key_dim=dim, key_heads=_groups(rng, heads), value_heads=_groups(rng, heads),
                value_dim=rng.choice([dim, dim, dim, 64, 128]), fused=rng.random() < 0.3)
    if kind == "prompt":
        return _attend(dtype=dtype, grad=False, decay=rng.choice(["fixed", "gated"]), state=rng.random() < 0.8, ragged=rng.random() < 0.6, **more)
    if kind == "gated":
        return _attend(dtype=rng.choice(["bf16", "bf16", "f32"]), decay="gated", state=rng.random() < 0.3, ragged=rng.random() < 0.3, **more)
    if kind == "f32":
        return _attend(dtype="f32", decay=rng.choice(["fixed", "learned", "gated"]), state=rng.random() < 0.5, **more)
    return _attend(dtype="bf16", decay=rng.choice(["fixed", "fixed", "learned"]), state=rng.random() < 0.3, ragged=rng.random() < 0.3, **more)


# ------------------------------------------------------------------ inputs
def _normal(gen, *shape, dtype=torch.float32):
    return torch.randn(shape, generator=gen, device="cuda").to(dtype)


def _uniform(gen, *shape):
    return torch.rand(shape, generator=gen, device="cuda")


def _log_decay(case, gen):
    heads = case["heads"]
    if case["decay"] != "gated":
        # memories from 32 to 4,096 tokens, spread over the heads
        away = 5.0 + 7.0 * torch.arange(heads, device="cuda") / max(1, heads - 1) + 0.2 * _uniform(gen, heads)
        return torch.log1p(-torch.exp2(-away))
    shape = (case["batch"], heads) if case["op"] == "step" else (case["batch"], case["seq"], heads)
    lam = -4.3 + 3.8 * _uniform(gen, heads)
    g = -8.0 * torch.log1p(torch.exp(lam)) * torch.sigmoid(_normal(gen, *shape))
    if case["op"] == "attend":
        starts = _uniform(gen, case["batch"], case["seq"], 1) < 1.0 / DOCUMENT
        g = torch.where(starts, torch.full_like(g, -math.inf), g)
    return g


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype, B, T = _DTYPES[case["dtype"]], case["batch"], case["seq"]
    s = {"case": case}
    if case["op"] in ("attend", "step"):
        H, Hk, Hv, K, V = (case[n] for n in ("heads", "key_heads", "value_heads", "key_dim", "value_dim"))
        lead = (B,) if case["op"] == "step" else (B, T)
        if case.get("fused"):
            row = _normal(gen, *lead, H * K + Hk * K + Hv * V, dtype=dtype)
            q, k, v = row.split([H * K, Hk * K, Hv * V], dim=-1)
            q, k, v = q.unflatten(-1, (H, K)), k.unflatten(-1, (Hk, K)), v.unflatten(-1, (Hv, V))
        else:
            q, k, v = (_normal(gen, *lead, *e, dtype=dtype) for e in ((H, K), (Hk, K), (Hv, V)))
        s |= {"q": q, "k": k, "v": v, "log_decay": _log_decay(case, gen)}
        if case["op"] == "step":
            pool = B + (B + 1) // 2 if case["slots"] else B
            s["state"] = _normal(gen, pool, H, K, V)
            s["slots"] = torch.randperm(pool, generator=gen, device="cuda")[:B].to(torch.int32) if case["slots"] else None
            return s
        s["h0"] = _normal(gen, B, H, K, V) if case["state"] else None
        s["lengths"] = None
        if case["ragged"]:
            lengths = torch.randint(0, T + 1, (B,), generator=gen, device="cuda", dtype=torch.int32)
            lengths[0] = T
            s["lengths"] = lengths
        if case["grad"]:
            s["grads"] = [_normal(gen, B, T, H, V, dtype=dtype)] + ([_normal(gen, B, H, K, V)] if case["state"] else [])
            s["wanted"] = ["q", "k", "v"] + (["log_decay"] if case["decay"] != "fixed" else []) + (["h0"] if case["state"] else [])
            for name in s["wanted"]:
                s[name] = s[name].detach().requires_grad_()
    elif case["op"] == "rotate":
        s["q"], s["k"] = (_normal(gen, B, T, case[n], case["dim"], dtype=dtype) for n in ("heads", "key_heads"))
        start = torch.randint(0, 100_000, (B, 1), generator=gen, device="cuda")
        s["positions"] = start + torch.arange(T, device="cuda")
        # the angle of pair j grows by 10000^(-2j/r) a position; kept as a 64-bit fraction of a turn
        pairs = torch.arange(case["rotary_dim"] // 2, device="cuda", dtype=torch.float64)
        s["turns"] = torch.round(10000.0 ** (-2.0 * pairs / case["rotary_dim"]) / (2 * math.pi) * 2.0**64).to(torch.int64)
        if case["grad"]:
            s["grads"] = [_normal(gen, *s[n].shape, dtype=dtype) for n in ("q", "k")]
            s["wanted"] = ["q", "k"]
            s["q"].requires_grad_()
            s["k"].requires_grad_()
    else:
        D = case["width"]
        s["x"] = _normal(gen, B, T, D, dtype=dtype)
        s["residual"] = (3.0 * _normal(gen, B, T, D)).to(dtype) if case["residual"] else None
        s["weight"] = (1.0 + 0.1 * _normal(gen, D)).to(dtype)
        if case["grad"]:
            s["grads"] = [_normal(gen, B, T, D, dtype=dtype) for _ in range(2 if case["residual"] else 1)]
            s["wanted"] = ["x", "weight"] + (["residual"] if case["residual"] else [])
            for name in s["wanted"]:
                s[name].requires_grad_()
    return s


# ------------------------------------------------------------------ plain forms, in 32 bits
def _per_head(t, heads, dim):
    return t.float().repeat_interleave(heads // t.shape[dim], dim)


def _segments(x):
    """exp of the sums of x over s in (j, i], for every i >= j of the last dimension; 0 above the diagonal."""
    n = x.shape[-1]
    at = torch.arange(n, device=x.device)
    terms = torch.where(at[:, None] > at[None, :], x[..., :, None], torch.zeros((), device=x.device))
    sums = torch.where(at[:, None] >= at[None, :], terms.cumsum(-2), torch.full((), -math.inf, device=x.device))
    return sums.exp()


def _attend_plain(s):
    case = s["case"]
    B, T, H = case["batch"], case["seq"], case["heads"]
    C = min(CHUNK, T)
    N = -(-T // C)
    q, k, v = (_per_head(s[n], H, 2) for n in ("q", "k", "v"))
    g = s["log_decay"].expand(B, T, H)
    valid = None
    if s["lengths"] is not None:
        valid = torch.arange(T, device=g.device)[None, :] < s["lengths"][:, None]
        zero = torch.zeros((), device=g.device)
        k, v = (torch.where(valid[..., None, None], t, zero) for t in (k, v))
        g = torch.where(valid[..., None], g, zero)

    def chunks(t):      # [B, T, H, ...] -> [B, H, N, C, ...]
        pad = [0, 0] * (t.dim() - 2) + [0, N * C - T]
        return torch.nn.functional.pad(t, pad).unflatten(1, (N, C)).movedim(3, 1)

    q, k, v, g = chunks(q) * case["key_dim"] ** -0.5, chunks(k), chunks(v), chunks(g)
    inside = _segments(g)
    added = (k * inside[..., -1, :, None]).transpose(-1, -2) @ v                       # what each chunk adds to the state
    first = s["h0"][:, :, None] if s["h0"] is not None else torch.zeros_like(added[:, :, :1])
    total = torch.nn.functional.pad(g.sum(-1), [1, 0])
    states = (_segments(total) @ torch.cat([first, added], 2).flatten(3)).unflatten(-1, added.shape[-2:])
    o = ((q @ k.transpose(-1, -2)) * inside) @ v + (q * g.cumsum(-1).exp()[..., None]) @ states[:, :, :-1]
    o = o.movedim(1, 3).flatten(1, 2)[:, :T]
    if valid is not None:
        o = torch.where(valid[..., None, None], o, torch.zeros((), device=o.device))
    o = o.to(s["v"].dtype)
    return [o, states[:, :, -1]] if case["state"] else [o]


def _step_plain(s):
    case = s["case"]
    q, k, v = (_per_head(s[n], case["heads"], 1) for n in ("q", "k", "v"))
    slots = s["slots"].long() if s["slots"] is not None else torch.arange(case["batch"], device=q.device)
    decay = s["log_decay"].exp().expand(case["batch"], case["heads"])[..., None, None]
    new = s["state"][slots] * decay + k[..., :, None] * v[..., None, :]
    s["state"][slots] = new
    o = (q[..., None, :] * case["key_dim"] ** -0.5 @ new)[..., 0, :]
    return [o.to(s["v"].dtype), s["state"]]


def _rotate_plain(s):
    case = s["case"]
    r, interleaved = case["rotary_dim"], case["layout"] == "interleaved"
    angle = ((s["positions"][..., None] * s["turns"]) >> 40).float() * (2 * math.pi / 2**24)      # (whole turns wrap away)
    cos, sin = angle.cos()[:, :, None], angle.sin()[:, :, None]

    def turn(x):
        y, rest = x[..., :r].float(), x[..., r:]
        a, b = (y[..., 0::2], y[..., 1::2]) if interleaved else (y[..., : r // 2], y[..., r // 2:])
        a, b = a * cos - b * sin, a * sin + b * cos
        y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
        return torch.cat([y.to(x.dtype), rest], -1)

    return [turn(s["q"]), turn(s["k"])]


def _norm_plain(s):
    case, x = s["case"], s["x"]
    total = (x.float() + s["residual"].float()).to(x.dtype) if case["residual"] else x
    f = total.float()
    y = f * torch.rsqrt((f * f).mean(-1, keepdim=True) + EPS) * s["weight"].float()
    if case["quant"] == "none":
        out = [y.to(x.dtype)]
    else:
        g = y.unflatten(-1, (-1, GROUP)) if case["quant"] == "group" else y[..., None, :]
        most = g.abs().amax(-1, keepdim=True)
        held = (g * (448.0 / torch.clamp(most, min=1e-30))).clamp(-448.0, 448.0).to(torch.float8_e4m3fn)
        out = [held.reshape(y.shape), (most / 448.0)[..., 0]]
        out[1] = out[1] if case["quant"] == "group" else out[1][..., 0]
    return out + [total] if case["residual"] else out


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    import fast_sequential_scan_b200 as fss
    case = s["case"]
    if case["op"] == "attend":
        out = fss.linear_attention(s["q"], s["k"], s["v"], s["log_decay"], h0=s["h0"], return_final_state=case["state"], lengths=s["lengths"])
        return list(out) if case["state"] else [out]
    if case["op"] == "step":
        return [fss.linear_attention_step(s["q"], s["k"], s["v"], s["log_decay"], s["state"], slots=s["slots"]), s["state"]]
    if case["op"] == "rotate":
        return list(fss.rotary(s["q"], s["k"], s["positions"], s["turns"], layout=case["layout"]))
    if case["quant"] == "none":
        out = fss.rms_norm(s["x"], s["weight"], residual=s["residual"], eps=EPS)
        return list(out) if case["residual"] else [out]
    return list(fss.rms_norm_quantized(s["x"], s["weight"], residual=s["residual"], eps=EPS, group=GROUP if case["quant"] == "group" else None))


_PLAIN = {"attend": _attend_plain, "step": _step_plain, "rotate": _rotate_plain, "norm": _norm_plain}


def run(state):
    forward = _own if own else _PLAIN[state["case"]["op"]]
    if not state["case"]["grad"]:
        with torch.no_grad():
            return forward(state)
    out = forward(state)
    return [o.detach() for o in out] + list(torch.autograd.grad(out, [state[n] for n in state["wanted"]], state["grads"]))


# ------------------------------------------------------------------ what a pass cannot do without
def work(case):
    size, tokens = (2 if case["dtype"] == "bf16" else 4), case["batch"] * case["seq"]
    if case["op"] == "step":
        states = case["batch"] * case["heads"]
        K, V = case["key_dim"], case["value_dim"]
        rows = case["batch"] * (case["heads"] * (K + V) + case["key_heads"] * K + case["value_heads"] * V)
        return {"bytes": float(8 * states * K * V + size * rows), "flops": 5.0 * states * K * V}
    if case["op"] == "rotate":
        n = tokens * (case["heads"] + case["key_heads"]) * case["dim"]
        passes = 2 if case["grad"] else 1
        return {"bytes": float(passes * (2 * n * size + 8 * tokens)), "flops": 3.0 * passes * n}
    if case["op"] == "norm":
        n = tokens * case["width"]
        out = size if case["quant"] == "none" else 1
        if not case["grad"]:
            return {"bytes": float(n * (size + out + (2 * size if case["residual"] else 0))), "flops": 5.0 * n}
        # the backward reads what was normalised and the gradients, and writes one gradient
        return {"bytes": float(n * size * (4 + 4 if case["residual"] else 2 + 3)), "flops": 15.0 * n}
    if case["ragged"]:
        tokens = case["seq"] + (case["batch"] - 1) * case["seq"] / 2
    H, Hk, Hv, K, V = (case[n] for n in ("heads", "key_heads", "value_heads", "key_dim", "value_dim"))
    q, k, v, o = H * K, Hk * K, Hv * V, H * V
    gates = 4 * tokens * H if case["decay"] == "gated" else 4 * H
    states = 4 * case["batch"] * H * K * V if case["state"] else 0
    # chunks as long as make the work least: about sqrt(K V) tokens; the state's product and update, the chunk's own two
    least = 4.0 * K * V + 2.0 * min(case["seq"], 64) * (K + V) / 2
    bytes_ = size * tokens * (q + k + v + o) + gates + 2 * states
    flops = tokens * H * least
    if case["grad"]:
        bytes_ += size * tokens * (2 * (q + k + v) + o) + 2 * gates + 2 * states
        flops *= 3.5
    return {"bytes": float(bytes_), "flops": float(flops)}


# ------------------------------------------------------------------ the same from the definitions, in 64 bits
def _exact_attend(s):
    case = s["case"]
    B, T, H, K, V = (case[n] for n in ("batch", "seq", "heads", "key_dim", "value_dim"))
    wide = {n: s[n].detach().double() for n in ("q", "k", "v", "log_decay")}
    head = torch.arange(H, device="cuda")
    at = {n: head // (H // wide[n].shape[2]) for n in ("q", "k", "v")}
    scale = 1.0 / math.sqrt(K)
    length = s["lengths"] if s["lengths"] is not None else torch.full((B,), T, device="cuda")
    live = torch.arange(T, device="cuda")[:, None] < length[None, :]                      # [T, B]
    decay = wide["log_decay"].exp().expand(B, T, H)
    S = s["h0"].detach().double() if s["h0"] is not None else torch.zeros(B, H, K, V, device="cuda", dtype=torch.float64)
    S = S.clone()
    o = torch.zeros(B, T, H, V, device="cuda", dtype=torch.float64)
    grads = [t.double() for t in s["grads"]] if case["grad"] else None
    dq = torch.zeros(B, T, H, K, device="cuda", dtype=torch.float64) if grads else None
    for t in range(T):
        m = live[t][:, None, None, None]
        a = torch.where(m, decay[:, t, :, None, None], 1.0)
        S.mul_(a)
        kt, vt = wide["k"][:, t, at["k"]], torch.where(m[..., 0], wide["v"][:, t, at["v"]], 0.0)
        S.addcmul_(kt[..., :, None], vt[..., None, :])
        o[:, t] = torch.where(m[..., 0], scale * (wide["q"][:, t, at["q"], None, :] @ S)[..., 0, :], 0.0)
        if grads:
            dq[:, t] = torch.where(m[..., 0], scale * (S @ grads[0][:, t, :, :, None])[..., 0], 0.0)
    out = [o, S] if case["state"] else [o]
    if not grads:
        return out
    R = grads[1].clone() if case["state"] else torch.zeros_like(S)
    flow = (R * S).sum((-1, -2))                      # <state, its gradient> behind the token
    dk, dv = torch.zeros_like(dq), torch.zeros_like(o)
    dg = torch.zeros(B, T, H, device="cuda", dtype=torch.float64)
    for t in range(T - 1, -1, -1):
        m = live[t][:, None, None, None]
        qt, kt, vt = (wide[n][:, t, at[n]] for n in ("q", "k", "v"))
        R.addcmul_(torch.where(m[..., 0], scale * qt, 0.0)[..., :, None], grads[0][:, t][..., None, :])
        dk[:, t] = torch.where(m[..., 0], (R @ vt[..., None])[..., 0], 0.0)
        dv[:, t] = torch.where(m[..., 0], (kt[..., None, :] @ R)[..., 0, :], 0.0)
        flow = flow + (qt * dq[:, t]).sum(-1) - (kt * dk[:, t]).sum(-1)
        flow = torch.where(m[..., 0, 0] & (decay[:, t] == 0), 0.0, flow)
        dg[:, t] = torch.where(m[..., 0, 0], flow, 0.0)
        R.mul_(torch.where(m, decay[:, t, :, None, None], 1.0))

    def shared(d, n):      # heads of a group sum up
        return d.unflatten(2, (wide[n].shape[2], -1)).sum(3)

    out += [shared(dq, "q"), shared(dk, "k"), shared(dv, "v")]
    if case["decay"] != "fixed":
        out.append(dg if case["decay"] == "gated" else dg.sum((0, 1)))
    return out + [R] if case["state"] else out


def _exact_step(s):
    case, state = s["case"], s["state"].double()
    group = {n: case["heads"] // s[n].shape[1] for n in ("q", "k", "v")}
    o = torch.zeros(case["batch"], case["heads"], case["value_dim"], device="cuda", dtype=torch.float64)
    decay = torch.exp(s["log_decay"].double()).expand(case["batch"], case["heads"])
    for h in range(case["heads"]):
        q, k, v = (s[n][:, h // group[n]].double() for n in ("q", "k", "v"))
        rows = s["slots"].long() if s["slots"] is not None else slice(None)
        new = torch.einsum("b,bkv->bkv", decay[:, h], state[rows, h]) + torch.einsum("bk,bv->bkv", k, v)
        state[rows, h] = new
        o[:, h] = torch.einsum("bk,bkv->bv", q, new) / math.sqrt(case["key_dim"])
    return [o, state]


def _exact_rotate(s):
    case = s["case"]
    r = case["rotary_dim"]
    frequency = torch.exp(torch.arange(r // 2, device="cuda", dtype=torch.float64) * (-2.0 / r * math.log(10000.0)))
    z = torch.polar(torch.ones((), device="cuda", dtype=torch.float64), s["positions"].double()[..., None, None] * frequency)

    def turn(x, z):
        x = x.detach().double().clone()
        first = slice(0, r, 2) if case["layout"] == "interleaved" else slice(0, r // 2)
        second = slice(1, r, 2) if case["layout"] == "interleaved" else slice(r // 2, r)
        w = torch.complex(x[..., first], x[..., second]) * z
        x[..., first], x[..., second] = w.real, w.imag
        return x

    out = [turn(s["q"], z), turn(s["k"], z)]
    return out + [turn(g, z.conj()) for g in s["grads"]] if case["grad"] else out


def _exact_norm(s):
    case = s["case"]
    x, w = s["x"].detach(), s["weight"].detach().double()
    total = x
    if case["residual"]:      # the stored sum is what is normalised
        total = (x.double() + s["residual"].detach().double()).to(x.dtype)
    f = total.double()
    r = 1.0 / torch.sqrt(torch.mean(torch.square(f), -1, keepdim=True) + EPS)
    y = f * r * w
    if case["quant"] == "none":
        out = [y]
    elif case["quant"] == "row":
        out = [None, y.abs().max(-1).values / 448.0]
    else:
        out = [None, y.abs().unflatten(-1, (-1, GROUP)).max(-1).values / 448.0]
    if case["residual"]:
        out.append(f)
    if not case["grad"]:
        return out
    dy = s["grads"][0].double() * w
    dx = r * dy - f * r**3 * torch.mean(dy * f, -1, keepdim=True)
    if case["residual"]:
        dx = dx + s["grads"][1].double()
    out += [dx, (s["grads"][0].double() * f * r).sum((0, 1))]
    return out + [dx] if case["residual"] else out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"attend": _exact_attend, "step": _exact_step, "rotate": _exact_rotate, "norm": _exact_norm}[case["op"]](s)
