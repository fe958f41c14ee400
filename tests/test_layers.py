"""CPU tests of the matrix-state operators: the turns of rotary positions, refusals that need no device, the C entries' checks."""
import ctypes
import math
import re
from pathlib import Path

import pytest
import torch

ROOT = Path(__file__).resolve().parent.parent


def pkg():
    import fast_sequential_scan_b200 as p
    return p


def words(turns):
    return [int(w) % 2 ** 64 for w in turns]


@pytest.mark.parametrize("r,base", [(2, 10000.0), (64, 10000.0), (128, 500000.0), (1024, 10000.0)])
def test_turns(r, base):
    turns, magnitude = pkg().rotary_turns(r, base=base)
    assert turns.dtype == torch.int64 and turns.shape == (r // 2,) and magnitude == 1.0
    for j, w in enumerate(words(turns)):
        # one rounding to 53 bits for the power, the division and the scaling each, and the one to a whole number
        assert w == pytest.approx(base ** (-2 * j / r) / (2 * math.pi) * 2.0 ** 64, rel=1e-14, abs=0.5)


def test_turns_above_half_a_turn_wrap():
    turns, _ = pkg().rotary_turns(2, scaling={"type": "linear", "factor": 1 / 5.0})      # 5 radians a position
    assert turns[0] < 0
    assert words(turns)[0] / 2.0 ** 64 == pytest.approx(5.0 / (2 * math.pi), rel=1e-12)


def test_scaled_turns():
    plain = words(pkg().rotary_turns(64)[0])
    linear = words(pkg().rotary_turns(64, scaling={"type": "linear", "factor": 4})[0])
    assert all(a == pytest.approx(b / 4, rel=1e-9) for a, b in zip(linear, plain))
    base = words(pkg().rotary_turns(64, scaling={"type": "base", "factor": 4})[0])
    assert base[0] == plain[0] and base[-1] == pytest.approx(plain[-1] / 4, rel=1e-9)
    parts, magnitude = pkg().rotary_turns(64, scaling={"type": "parts", "factor": 4, "length": 4096})
    ratio = [b / a for a, b in zip(words(parts), plain)]
    assert ratio[0] == pytest.approx(1.0) and ratio[-1] == pytest.approx(4.0) and all(x <= y * (1 + 1e-9) for x, y in zip(ratio, ratio[1:]))
    rounds = [4096 * w / 2.0 ** 64 for w in plain]      # turns in the training length
    assert all(r == pytest.approx(1.0) for r, n in zip(ratio, rounds) if n > 40) and all(r == pytest.approx(4.0) for r, n in zip(ratio, rounds) if n < 0.8)
    assert magnitude == pytest.approx(0.1 * math.log(4) + 1)
    assert pkg().rotary_turns(64, scaling={"type": "parts", "factor": 4, "length": 4096, "magnitude": 1.0})[1] == 1.0


@pytest.mark.parametrize("args,kw", [((3,), {}), ((0,), {}), ((2048,), {}), ((64,), {"base": 0.0}), ((64,), {"scaling": {"type": "other", "factor": 2}}),
                                     ((64,), {"scaling": {"type": "linear"}}), ((64,), {"scaling": {"type": "linear", "factor": -1}})])
def test_turns_refusals(args, kw):
    with pytest.raises(ValueError):
        pkg().rotary_turns(*args, **kw)


def test_host_tensors_are_refused():
    x = torch.zeros(1, 2, 4, 8)
    p = pkg()
    for call in (lambda: p.linear_attention(x, x, x, torch.zeros(4)), lambda: p.linear_attention_step(x[0], x[0], x[0], torch.zeros(4), x),
                 lambda: p.rotary(x, None, torch.arange(2), torch.zeros(2, dtype=torch.int64)), lambda: p.rms_norm(x, torch.zeros(8)),
                 lambda: p.rms_norm_quantized(x, torch.zeros(8))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(TypeError):
        p.linear_attention(1, x, x, torch.zeros(4))


def test_struct_layouts_match_the_header():
    """Field names and order, read from the header text."""
    from fast_sequential_scan_b200 import _lib
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "fss_b200.h").read_text(), flags=re.S)
    for c_name, struct, size in (("fss_heads", _lib.Heads, 48), ("fss_linear_attention", _lib.LinearAttention, 232), ("fss_norm_weight", _lib.NormWeight, 16),
                                 ("fss_norm_output", _lib.NormOutput, 56), ("fss_rotary", _lib.Rotary, 56)):
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (c_name, c_name), text, flags=re.S).group(1)
        fields = [re.sub(r"[^A-Za-z0-9_]", "", part.split()[-1]) for decl in body.split(";") if decl.strip() for part in decl.split(",")]
        assert fields == [name for name, _ in struct._fields_]
        assert ctypes.sizeof(struct) == size


def _call():
    from fast_sequential_scan_b200 import _lib
    buf = (ctypes.c_float * 4096)()
    at = ctypes.addressof(buf)
    ctx = _lib.ScanCtx(ctypes.sizeof(_lib.ScanCtx), -1, None, None, 0, None, 0, 0)
    heads = lambda h=2, d=16, ptr=at: _lib.Heads(ptr, 4 * h * d, h * d, d, h, d)
    return _lib, _lib.lib(), buf, at, ctx, heads


def test_attention_entry_checks_its_arguments():
    _lib, L, buf, at, ctx, heads = _call()
    make = lambda **kw: _lib.LinearAttention(**dict(dict(struct_bytes=ctypes.sizeof(_lib.LinearAttention), dtype=0, B=2, T=4, H=2, q=heads(), k=heads(1),
                                                         v=heads(2, 8), log_decay=at, decay_stride_h=1, scale=1.0), **kw))
    o = heads(2, 8)
    run = lambda p, out=o, c=ctx: L.fss_linear_attention_forward(ctypes.byref(c), ctypes.byref(p), ctypes.byref(out), None)
    assert run(make(struct_bytes=8)) == -10
    assert run(make(dtype=7)) == -3
    assert run(make(B=-1)) == -2 and run(make(H=0)) == -2 and run(make(H=3)) == -2
    assert run(make(q=heads(2, 300), k=heads(2, 300))) == -11 and run(make(v=heads(2, 257))) == -11
    assert run(make(k=heads(1, 8))) == -2
    assert run(make(q=heads(ptr=0))) == -1 and run(make(log_decay=None)) == -1
    assert run(make(), heads(1, 8)) == -2                                          # outputs have a head for each state
    assert run(make(), _lib.Heads(at, 64, 8, 8, 2, 8)) == -2                       # rows that overlap
    assert run(make(B=0)) == 0 and run(make(T=0)) == 0
    assert run(make(T=1 << 33)) == -2
    bad = _lib.ScanCtx(8, -1, None, None, 0, None, 0, 0)
    assert run(make(), c=bad) == -10
    # one sequence and head, many tokens: segments, which need scratch
    long = make(B=1, T=8192, H=1, q=heads(1), k=heads(1), v=heads(1, 8))
    assert L.fss_linear_attention_workspace_bytes(ctypes.byref(long), 0) > 0
    assert run(long, _lib.Heads(at, 8192 * 8, 8, 8, 1, 8)) == -4
    step = lambda p, pool=2, stride=2 * 16 * 8: L.fss_linear_attention_step(ctypes.byref(ctx), ctypes.byref(p), ctypes.byref(o), at, stride, pool, None)
    assert step(make()) == -10 and step(make(T=1, lengths=at)) == -10
    assert step(make(T=1), pool=1) == -2 and step(make(T=1), stride=8) == -2 and step(make(T=1, B=0)) == 0
    back = lambda p, **kw: L.fss_linear_attention_backward(ctypes.byref(ctx), ctypes.byref(p), ctypes.byref(o), None, kw.get("last"), kw.get("dq"), None, None,
                                                           kw.get("dg"), 0, None)
    assert back(make(), dg=at) == -1                                               # the decays' gradients need those of q and k
    assert back(make(), dg=at, last=at) == -1


def test_norm_and_rotary_entries_check_their_arguments():
    _lib, L, buf, at, ctx, heads = _call()
    view = _lib.View(at, 64, 16)
    w, out = _lib.NormWeight(at, 1), _lib.NormOutput(view, None, None, None, 0)
    run = lambda dt=1, B=2, T=4, D=16, x=view, res=None, weight=w, s=None, o=out: L.fss_rms_norm_forward(
        ctypes.byref(ctx), dt, B, T, D, ctypes.byref(x), ctypes.byref(res) if res else None, ctypes.byref(weight), 1e-6, s, ctypes.byref(o))
    assert run(dt=5) == -3 and run(D=0) == -2 and run(B=-1) == -2 and run(B=1 << 20, T=1 << 20) == -2
    assert run(weight=_lib.NormWeight(None, 1)) == -1 and run(weight=_lib.NormWeight(at, 0)) == -3
    assert run(res=view) == -1 and run(o=_lib.NormOutput(_lib.View(), None, None, None, 0)) == -1
    assert run(o=_lib.NormOutput(view, at, at, None, 0)) == -10 and run(o=_lib.NormOutput(_lib.View(), at, at, None, 48)) == -10
    assert run(o=_lib.NormOutput(_lib.View(), at, at, None, 32)) == -10            # 16 channels
    assert run(x=_lib.View(at, 64, 8)) == -2 and run(B=0) == 0
    back = lambda dw=None, r=at: L.fss_rms_norm_backward(ctypes.byref(ctx), 1, 2, 4, 16, ctypes.byref(view), ctypes.byref(w), r, ctypes.byref(view), None,
                                                         ctypes.byref(view), dw)
    assert back(r=None) == -1 and back(dw=at) == -4
    rot = lambda q=heads(), B=2, **kw: L.fss_rotary_apply(ctypes.byref(ctx), 0, B, 4, ctypes.byref(q), None, at, None, ctypes.byref(_lib.Rotary(
        **dict(dict(struct_bytes=ctypes.sizeof(_lib.Rotary), magnitude=1.0, rotary_dim=16, positions=at, position_stride_t=1, turns=at), **kw))))
    assert rot(struct_bytes=4) == -10 and rot(rotary_dim=3) == -2 and rot(rotary_dim=32) == -2 and rot(positions=None) == -1
    assert rot(q=heads(2, 4096), rotary_dim=2048) == -11 and rot(B=0) == 0


def test_segments_of_a_pass_do_not_depend_on_the_device():
    """Workspaces are asked for before a launch, on a machine without a device too."""
    _lib, L, buf, at, ctx, heads = _call()
    p = lambda T, H: _lib.LinearAttention(struct_bytes=ctypes.sizeof(_lib.LinearAttention), dtype=0, B=1, T=T, H=H, q=heads(H, 128), k=heads(H, 128),
                                          v=heads(H, 128), log_decay=at, decay_stride_h=1, scale=1.0)
    size = lambda T, H, back=0: L.fss_linear_attention_workspace_bytes(ctypes.byref(p(T, H)), back)
    assert size(64, 1) == 0 and size(65536, 512) == 0                              # one chunk; states enough for the device
    assert size(65536, 32) % 256 == 0 and size(65536, 32) >= 2 * 32 * 128 * 128 * 4
    assert size(65536, 32, 2) > size(65536, 32, 1) >= size(65536, 32)
