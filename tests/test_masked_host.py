"""The host side of rope_axes, masked attention and the distillation head on the CPU: pairs and sections, refusals of
the launchers and of the C entry points (nothing is launched), layouts, second derivatives."""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import ops as ref
from rus_amd import _lib, kernels as K, ops

HALF = dict(dtype=torch.float16)
CU = torch.tensor([0, 4], dtype=torch.int32)


# ---- pairs and sections --------------------------------------------------------------------------


def test_sections_of_pairs():
    a = K.RopeAxes.sections((2, 3, 1), 100.0, 16, "cpu")
    assert a.axis.tolist() == [0, 0, 1, 1, 1, 2] and a.pairs == 6 and a.n_axes == 3
    want = [100.0 ** (-i / 6) / (2 * math.pi) for i in range(6)]
    assert a.turns.tolist() == want
    a = K.RopeAxes.sections((2, 3, 1), 100.0, 16, "cpu", order="cycle", restart=True)
    assert a.axis.tolist() == [0, 1, 2, 0, 1, 1]
    want = [1.0, 1.0, 1.0, 100.0**-0.5, 100.0 ** (-1 / 3), 100.0 ** (-2 / 3)]
    assert a.turns.tolist() == [w / (2 * math.pi) for w in want]
    assert K.RopeAxes.sections((0, 2), 10.0, 4, "cpu").axis.tolist() == [1, 1]


@pytest.mark.parametrize("kw,msg", [
    (dict(axis=[0, 1], freq=[1.0], head_dim=8), "2 axes for 1 frequencies"),
    (dict(axis=[], freq=[], head_dim=8), "0 axes"),
    (dict(axis=[0] * 5, freq=[1.0] * 5, head_dim=8), "5 pairs in heads of 8"),
    (dict(axis=[-1], freq=[1.0], head_dim=8), "numbered"),
    (dict(axis=[0], freq=[math.inf], head_dim=8), "finite"),
    (dict(axis=[0] * 513, freq=[1.0] * 513, head_dim=2000), "513 pairs"),
])
def test_pairs_are_checked(kw, msg):
    with pytest.raises(ValueError, match=msg):
        K.RopeAxes(device="cpu", **kw)


@pytest.mark.parametrize("args,msg", [(((), 10.0, 8), "sections"), (((2, -1), 10.0, 8), "sections"),
                                      (((0, 0), 10.0, 8), "sections"), (((2, 2), 0.0, 8), "theta")])
def test_sections_are_checked(args, msg):
    with pytest.raises(ValueError, match=msg):
        K.RopeAxes.sections(*args, "cpu")
    with pytest.raises(ValueError, match="order"):
        K.RopeAxes.sections((2,), 10.0, 8, "cpu", order="blocked")


# ---- refusals of the launchers -------------------------------------------------------------------


def _axes():
    return K.RopeAxes.sections((2, 2), 10.0, 8, "cpu")


@pytest.mark.parametrize("q,k,pos,err,msg", [
    (torch.zeros(4, 2, 16, **HALF), None, torch.zeros(2, 4, dtype=torch.int64), ValueError, r"q must be \[N, heads, 8\]"),
    (torch.zeros(4, 8, **HALF), None, torch.zeros(2, 4, dtype=torch.int64), ValueError, "q must be"),
    (torch.zeros(4, 2, 8, dtype=torch.float64), None, torch.zeros(2, 4, dtype=torch.int64), TypeError, "float64"),
    (torch.zeros(4, 2, 8, **HALF), torch.zeros(4, 2, 8), torch.zeros(2, 4, dtype=torch.int64), ValueError, "k must be"),
    (torch.zeros(4, 2, 8, **HALF), torch.zeros(5, 2, 8, **HALF), torch.zeros(2, 4, dtype=torch.int64), ValueError, "k must be"),
    (torch.zeros(4, 2, 8, **HALF), None, torch.zeros(2, 4, dtype=torch.int16), TypeError, "positions"),
    (torch.zeros(4, 2, 8, **HALF), None, torch.zeros(4, dtype=torch.int64), ValueError, "positions"),
    (torch.zeros(4, 2, 8, **HALF), None, torch.zeros(1, 4, dtype=torch.int64), ValueError, "positions"),
    (torch.zeros(4, 2, 8, **HALF), None, torch.zeros(2, 5, dtype=torch.int64), ValueError, "positions"),
    (torch.zeros(4, 2, 8, **HALF), None, torch.zeros(2, 4, dtype=torch.int64), RuntimeError, "HIP device"),
])
def test_rope_axes_refuses(q, k, pos, err, msg):
    for fn in (K.rope_axes_fwd, K.rope_axes_bwd):
        with pytest.raises(err, match=msg):
            fn(q, k, pos, _axes())


def test_rope_axes_forms_no_gradient_of_positions():
    with pytest.raises(RuntimeError, match="positions is frozen"):
        ops.rope_axes(torch.zeros(4, 2, 8, **HALF), None, torch.zeros(2, 4, requires_grad=True), _axes())


def _attn(**kw):
    args = dict(q=torch.zeros(4, 4, 64, **HALF), k=torch.zeros(4, 2, 64, **HALF), v=torch.zeros(4, 2, 64, **HALF), cu_q=CU)
    args.update(kw)
    return K.attn_masked_fwd(**args)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(q=torch.zeros(4, 4, 96, **HALF)), ValueError, "64 or 128"),
    (dict(q=torch.zeros(4, 4, 64)), TypeError, "fp16 or bf16"),
    (dict(k=torch.zeros(4, 2, 64, dtype=torch.bfloat16)), TypeError, "k must be"),
    (dict(v=torch.zeros(4, 1, 64, **HALF)), ValueError, "differ"),
    (dict(k=torch.zeros(4, 3, 64, **HALF), v=torch.zeros(4, 3, 64, **HALF)), ValueError, "multiple of h_kv"),
    (dict(k=torch.zeros(5, 2, 64, **HALF), v=torch.zeros(5, 2, 64, **HALF)), ValueError, "cu_k of their own"),
    (dict(cu_q=CU.long()), ValueError, "cu_q must be"),
    (dict(cu_q=CU[:1]), ValueError, "start and an end"),
    (dict(cu_k=torch.zeros(3, dtype=torch.int32)), ValueError, "cu_k must be"),
    (dict(prefix=torch.zeros(2, dtype=torch.int32)), ValueError, "prefix must be"),
    (dict(slopes=torch.zeros(2)), ValueError, "slopes must be"),
    (dict(slopes=torch.zeros(4, **HALF)), ValueError, "slopes must be"),
    (dict(softcap=-1.0), ValueError, "softcap"), (dict(softcap=math.nan), ValueError, "softcap"),
    (dict(scale=0.0), ValueError, "scale"), (dict(scale=math.inf), ValueError, "scale"),
    (dict(max_q=-1), ValueError, "max_q"),
    (dict(), RuntimeError, "HIP device"),
])
def test_masked_attention_refuses(kw, err, msg):
    with pytest.raises(err, match=msg):
        _attn(**kw)


@pytest.mark.parametrize("kw,msg", [
    (dict(dout=torch.zeros(4, 4, 32, **HALF)), "dout and out"), (dict(out=torch.zeros(3, 4, 64, **HALF)), "dout and out"),
    (dict(out=torch.zeros(4, 8, 64, **HALF)[:, ::2]), "out must be contiguous"),
    (dict(lse=torch.zeros(4, 4, **HALF)), "lse must be"), (dict(lse=torch.zeros(4, 5)), "lse must be"),
])
def test_masked_attention_backward_refuses(kw, msg, monkeypatch):
    monkeypatch.setattr(K, "_same_device", lambda *a: None)
    args = dict(dout=torch.zeros(4, 4, 64, **HALF), q=torch.zeros(4, 4, 64, **HALF), k=torch.zeros(4, 2, 64, **HALF),
                v=torch.zeros(4, 2, 64, **HALF), out=torch.zeros(4, 4, 64, **HALF), lse=torch.zeros(4, 4), cu_q=CU)
    args.update(kw)
    with pytest.raises(ValueError, match=msg):
        K.attn_masked_bwd(**args)


IDS, LOGITS = torch.zeros(4, 3, dtype=torch.int64), torch.zeros(4, 3)


@pytest.mark.parametrize("kw,err,msg", [
    (dict(temperature=0.0), ValueError, "temperature"), (dict(temperature=math.nan), ValueError, "temperature"),
    (dict(hidden=torch.zeros(4, 2, 64, **HALF)), ValueError, "hidden"),
    (dict(weight=torch.zeros(100, 32, **HALF)), ValueError, "hidden"),
    (dict(weight=torch.zeros(0, 64, **HALF)), ValueError, "weight"),
    (dict(hidden=torch.zeros(4, 96, **HALF), weight=torch.zeros(9, 96, **HALF)), ValueError, "multiple of 64"),
    (dict(ids=IDS.short()), TypeError, "ids"), (dict(logits=LOGITS.double()), TypeError, "logits"),
    (dict(ids=IDS[:, :2]), ValueError, "must both"), (dict(ids=IDS[:3], logits=LOGITS[:3]), ValueError, "must both"),
    (dict(ids=IDS[:, :0], logits=LOGITS[:, :0]), ValueError, "0 teacher entries"),
    (dict(ids=torch.zeros(4, 1025, dtype=torch.int64), logits=torch.zeros(4, 1025)), ValueError, "1025 teacher entries"),
    (dict(hidden=torch.zeros(4, 64)), TypeError, "hidden must be fp16"),
    (dict(weight=torch.zeros(100, 64, dtype=torch.bfloat16)), TypeError, "weight must be fp16"),
    (dict(), RuntimeError, "HIP device"),
])
def test_distillation_refuses(kw, err, msg):
    args = dict(hidden=torch.zeros(4, 64, **HALF), weight=torch.zeros(100, 64, **HALF), ids=IDS, logits=LOGITS)
    args.update(kw)
    with pytest.raises(err, match=msg):
        K.lm_head_distill(args.pop("hidden"), args.pop("weight"), args.pop("ids"), args.pop("logits"), **args)


# ---- refusals of the C entry points (pointers are never followed) --------------------------------

ROPE = [16, 16, 8, 2, 16, 16, 16, 8, 1, 16, 4, 8, 4, 0, 16, 0, 4, 2, 16, 16, 0, 0, None]


@pytest.mark.parametrize("at,value,msg", [
    (10, -1, "bad sizes"), (3, 70000, "bad sizes"), (11, 0, "bad sizes"), (12, 5, "bad sizes"), (12, 0, "bad sizes"),
    (17, 0, "bad sizes"), (21, 7, "unknown dtype"), (15, 9, "unknown position type"), (0, None, "null or misaligned"),
    (0, 17, "null or misaligned"), (14, 20, "null or misaligned"), (18, None, "null or misaligned"),
    (19, 20, "null or misaligned"), (16, -4, "negative ld_pos"),
])
def test_rope_axes_entry_refuses(at, value, msg):
    args = list(ROPE)
    args[at] = value
    with pytest.raises(RuntimeError, match=msg):
        _lib.call("rus_rope_axes", *args)


def test_rope_axes_entry_refuses_what_it_cannot_count():
    args = list(ROPE)
    args[3], args[11], args[12] = 60000, 60000, 4
    with pytest.raises(RuntimeError, match="2\\^28 elements"):
        _lib.call("rus_rope_axes", *args)
    args[3], args[11], args[12] = 1, 60000, 513
    with pytest.raises(RuntimeError, match="at most 512"):
        _lib.call("rus_rope_axes", *args)


QKV = [16, 256, 64] * 3
FWD = QKV + [16, 16, 1, 4, 4, 4, 4, 4, 2, 64, 0.125, 1, None, 0.0, None, 0, 16, 16, None, 0, None]


def _masked(at, value, base=FWD, name="rus_attn_masked_fwd"):
    args = list(base)
    args[at] = value
    _lib.call(name, *args)


@pytest.mark.parametrize("at,value,msg", [
    (0, None, "q must be 16-byte"), (3, 24, "k must be 16-byte"), (7, 100, "v must be 16-byte"), (4, 1 << 26, "2\\^26"),
    (9, None, "null cu"), (11, 0, "n_seq"), (11, 1 << 23, "n_seq"), (12, -1, "n_q"), (13, 1 << 31, "n_k"),
    (14, -1, "max_q"), (16, 5, "multiple of h_kv"), (16, 0, "multiple of h_kv"), (18, 96, "head_dim 96"),
    (19, 0.0, "scale"), (19, math.inf, "scale"), (22, -2.0, "softcap"), (22, math.inf, "softcap"),
    (24, 1, "fp16 or bf16"), (25, None, "output"), (26, None, "output"), (25, 8, "output"),
])
def test_masked_attention_entry_refuses(at, value, msg):
    with pytest.raises(RuntimeError, match=msg):
        _masked(at, value)


BWD = [16, 256, 64] + QKV + [16, 16, 16, 16, 1, 4, 4, 4, 4, 4, 2, 64, 0.125, 1, None, 0.0, None, 0, 16, 16, 16, None, 0,
                             None]


@pytest.mark.parametrize("at,value,msg", [
    (0, None, "dout must be 16-byte"), (12, None, "misaligned argument"), (13, None, "misaligned argument"),
    (30, None, "misaligned argument"), (31, 8, "misaligned argument"), (33, None, "workspace of 0 floats, 2064 needed"),
    (24, 0.0, "scale"), (29, 5, "fp16 or bf16"),
])
def test_masked_attention_backward_entry_refuses(at, value, msg):
    with pytest.raises(RuntimeError, match=msg):
        _masked(at, value, BWD, "rus_attn_masked_bwd")


def test_masked_attention_refuses_what_a_dispatch_cannot_hold():
    args = list(FWD)
    args[12], args[13], args[14], args[15], args[16], args[17] = (1 << 31) - 300, 4, (1 << 31) - 300, 4, 64, 1
    with pytest.raises(RuntimeError, match="beyond one dispatch"):
        _lib.call("rus_attn_masked_fwd", *args)


def _plan(n_seq, n_q, n_k, max_q, max_k, hq, hkv, d):
    got = (ctypes.c_int32 * 3)()
    _lib.call("rus_attn_masked_plan", n_seq, n_q, n_k, max_q, max_k, hq, hkv, d, got)
    floats = ctypes.c_int64()
    _lib.call("rus_attn_masked_workspace", n_seq, n_q, n_k, max_q, max_k, hq, hkv, d, 0, ctypes.byref(floats))
    assert floats.value == (got[0] * n_q * hq * (d + 4) if got[0] > 1 else 0)
    _lib.call("rus_attn_masked_workspace", n_seq, n_q, n_k, max_q, max_k, hq, hkv, d, 1, ctypes.byref(floats))
    assert floats.value == (2 * hq * n_k * d if hq > hkv else 0) + hq * n_q  # the heads' parts, D
    return tuple(got)


def test_layouts_by_sizes():
    assert _plan(1, 1, 131071, 1, 131071, 12, 2, 128)[0] > 64  # one token over a long cache: many parts
    parts, tiles, block = _plan(8, 8, 15000, 1, 8191, 12, 2, 128)
    assert 1 < parts <= 64 and parts * tiles >= 256 and block == 32
    assert _plan(1, 707, 707, 707, 707, 12, 2, 128) == (1, 23, 32)
    assert _plan(10, 2560, 2560, 256, 256, 12, 2, 128) == (0, 0, 128)
    assert _plan(1, 1, 4096, 1, 4096, 40, 1, 128)[0] == 0  # more heads to a group than a block has columns
    with pytest.raises(RuntimeError, match="null result"):
        _lib.call("rus_attn_masked_plan", 1, 1, 1, 1, 1, 1, 1, 64, None)
    with pytest.raises(RuntimeError, match="head_dim"):
        _plan(1, 1, 1, 1, 1, 1, 1, 32)


CHUNK = [16, 64, 16, 64, 16, 128, 16, 64, 4, 64, 100, 0, 100, 100, 16, 0, 16, 1, 3, 1.0, 1, 16, 1 << 30, None]
FINISH = [16, 64, 4, 64, 100, 100, 16, 0, 16, 1, 3, 1.0, 1, None, 16, 16, 16, 16, 16, 1 << 30, None]


@pytest.mark.parametrize("at,value,msg", [
    (9, 96, "multiple of 64"), (8, 0, "bad sizes"), (8, 1 << 22, "bad sizes"), (13, 50, "bad sizes"), (20, 65, "bad sizes"),
    (11, 50, "no chunk"), (10, 90, "no chunk"), (10, 0, "no chunk"), (18, 0, "0 entries"), (18, 1025, "1025 entries"),
    (14, None, "entries"), (14, 20, "entries"), (16, None, "entries"), (17, 5, "unknown dtype 5"), (19, 0.0, "temperature"),
    (19, math.inf, "temperature"), (1, 32, "row strides"), (7, 32, "row strides"), (0, None, "hidden"), (2, 24, "weight_rows"),
    (6, None, "weight is null"), (22, 10, "workspace of 10 floats"), (21, None, "workspace"),
])
def test_distillation_chunk_refuses(at, value, msg):
    args = list(CHUNK)
    args[at] = value
    with pytest.raises(RuntimeError, match=msg):
        _lib.call("rus_lmhead_distill_chunk", *args)


@pytest.mark.parametrize("at,value,msg", [
    (3, 32, "multiple of 64"), (1, 32, "row strides"), (0, None, "weight is null"), (11, -1.0, "temperature"),
    (14, None, "output"), (15, None, "output"), (17, None, "output"), (17, 8, "output"), (19, 10, "workspace of 10"),
])
def test_distillation_finish_refuses(at, value, msg):
    args = list(FINISH)
    args[at] = value
    with pytest.raises(RuntimeError, match=msg):
        _lib.call("rus_lmhead_distill_finish", *args)


def test_distillation_workspace():
    def floats(*sizes):
        got = ctypes.c_int64()
        _lib.call("rus_lmhead_distill_workspace", *sizes, ctypes.byref(got))
        return got.value

    small, full = floats(100, 64, 1000, 1000, 8, 0), floats(100, 64, 1000, 512, 8, 3)
    assert small == 2 * 4 * 100 + 2 * 100 + 800
    assert full == small + 700 + 4 * 100 + 3 * 100 * 64 + 100 * 512 // 2
    with pytest.raises(RuntimeError, match="null result"):
        _lib.call("rus_lmhead_distill_workspace", 1, 64, 10, 10, 1, 0, None)
    with pytest.raises(RuntimeError, match="bad sizes"):
        floats(100, 64, 1000, 300, 8, 3)


# ---- second derivatives --------------------------------------------------------------------------


def test_gradients_of_gradients_are_refused(monkeypatch):
    monkeypatch.setattr(K, "attn_masked_fwd", lambda q, *a, **k: (torch.zeros_like(q), torch.zeros(4, 4)))
    monkeypatch.setattr(K, "attn_masked_bwd", lambda do, q, k, v, *a, **kw: tuple(map(torch.zeros_like, (q, k, v))))
    q = torch.zeros(4, 4, 64, requires_grad=True)
    out = ops.masked_attention(q, torch.zeros(4, 2, 64), torch.zeros(4, 2, 64), CU)
    (dq,) = torch.autograd.grad(out, q, torch.ones_like(out), create_graph=True)
    with pytest.raises(RuntimeError, match="masked_attention: no second derivative"):
        dq.sum().backward()
    with pytest.raises(RuntimeError, match="slopes is frozen"):
        ops.masked_attention(q, q, q, CU, slopes=torch.zeros(4, requires_grad=True))
    monkeypatch.setattr(K, "lm_head_distill", lambda h, *a: (torch.zeros(1), torch.zeros(4), torch.ones(1), torch.zeros(4, 64)))
    monkeypatch.setattr(K, "lm_head_dh_reduce", lambda x, *a, **k: torch.zeros(4, 64))
    h = torch.zeros(4, 64, requires_grad=True)
    loss, kl = ops.chunked_distill_head(h, IDS, LOGITS, torch.zeros(100, 64))
    assert not kl.requires_grad
    (dh,) = torch.autograd.grad(loss, h, create_graph=True)
    with pytest.raises(RuntimeError, match="chunked_distill_head: no second derivative"):
        dh.sum().backward()
    for kw in (dict(w=torch.zeros(100, 64, requires_grad=True)), dict(t=torch.zeros(4, 3, requires_grad=True))):
        with pytest.raises(RuntimeError, match="is frozen"):
            ops.chunked_distill_head(h, IDS, kw.get("t", LOGITS), kw.get("w", torch.zeros(100, 64)))


def test_rotation_is_differentiated_as_often_as_asked(monkeypatch):
    axes, pos = _axes(), torch.tensor([[0, 1, 5, 9], [3, 3, 2, 0]])
    freq = (axes.turns * 2 * math.pi).tolist()
    turn = lambda x, inv: None if x is None else ref.rope_axes(x, pos, axes.axis.tolist(), freq, inverse=inv).to(x.dtype)
    monkeypatch.setattr(K, "rope_axes_fwd", lambda q, k, p, a: (turn(q, False), turn(k, False)))
    monkeypatch.setattr(K, "rope_axes_bwd", lambda q, k, p, a: (turn(q, True), turn(k, True)))
    g = torch.Generator().manual_seed(0)
    q, k = (torch.randn(4, 2, 8, generator=g, dtype=torch.float64, requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(lambda a, b: ops.rope_axes(a, b, pos, axes), (q, k))
    assert torch.autograd.gradgradcheck(lambda a, b: ops.rope_axes(a, b, pos, axes), (q, k))
    assert torch.autograd.gradcheck(lambda a: ops.rope_axes(a, None, pos, axes), (q,))
