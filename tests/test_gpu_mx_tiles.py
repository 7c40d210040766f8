"""The microscaled kernels beyond one dispatch, and each tile of the products in its steady state: ragged sizes,
contractions of many stages, blocks that are not finite. Data whose sums are exact in fp32 shows an element
dropped, doubled or scaled by a neighbour's scale."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import ops as ref
from rus_amd import _lib, kernels as K, ops
from test_gpu_mx_sizes import FORMATS, bits, exact

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64


# ---- frozen parameters ---------------------------------------------------------------------------


def test_parameters_without_gradients_recorded():
    x = torch.randn(5, 64, device=DEV).half()
    w = K.mx_quantize(torch.randn(32, 64, device=DEV).half(), "fp4")
    down = K.mx_quantize(torch.randn(64, 16, device=DEV).half(), "fp4")
    bias = torch.nn.Parameter(torch.randn(32, device=DEV).half())
    weight = torch.nn.Parameter(torch.ones(64, device=DEV).half())
    with torch.no_grad():
        y, z = ops.mx_linear(x, w, bias), ops.mx_norm_mlp(x, weight, w, down)
    assert torch.equal(y, ops.mx_linear(x, w, bias.detach())) and not y.requires_grad
    assert torch.equal(z, ops.mx_norm_mlp(x, weight.detach(), w, down))


def test_gradients_under_create_graph():
    """The same bits, and a gradient of them raises."""
    x = torch.randn(70, 64, device=DEV).half().requires_grad_()
    w = K.mx_quantize(torch.randn(32, 64, device=DEV).half() * 0.1, "fp4")
    down = K.mx_quantize(torch.randn(64, 16, device=DEV).half() * 0.1, "fp4")
    weight = torch.ones(64, device=DEV).half()
    for call in (lambda: ops.mx_linear(x, w), lambda: ops.mx_mlp_glu(x, w),
                 lambda: ops.mx_norm_mlp(x, weight, w, down), lambda: ops.mx_norm_mlp(x, weight, w, down, residual=x)[0]):
        y = call()
        dy = torch.ones_like(y, requires_grad=True)
        (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
        assert torch.equal(dx, torch.autograd.grad(call(), x, dy.detach())[0])
        with pytest.raises(RuntimeError, match="no second derivative"):
            dx.sum().backward()


# ---- more rows than one dispatch holds -----------------------------------------------------------


def slices(rows, step):
    """Ranges that cover all rows, none ending where a launch's slice of 2^n rows does."""
    at = [0, *range(step - 3, rows, step), rows]
    return list(zip(at, at[1:]))


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_quantize_more_rows_than_a_dispatch(fmt):
    rows = (1 << 28) + 5 if fmt == "fp4" else (1 << 27) + 5  # 16 threads a row: more than 2^32, than 2^31
    x = torch.randn(rows, 1, generator=torch.Generator(device=DEV).manual_seed(1), device=DEV, dtype=F16)
    t = K.mx_quantize(x, fmt)
    back = K.mx_dequantize(t, F16)
    for a, b in slices(rows, 1 << 25):
        part = K.mx_quantize(x[a:b], fmt)
        assert torch.equal(t.codes[a:b], part.codes) and torch.equal(t.scales[a:b], part.scales), (a, b)
        assert torch.equal(back[a:b], K.mx_dequantize(part, F16)), (a, b)
    # one element with its own scale lies in [4, 8) or [256, 512) of it: saturating at 6 or 448 costs most
    assert ((back.float() - x.float()).abs() <= x.float().abs() * (2.0**-2 if fmt == "fp4" else 2.0**-3)).all()


def test_dequantize_more_rows_than_a_dispatch():
    rows, cols = (1 << 27) + 5, 128  # 16 threads a row
    g = torch.Generator(device=DEV).manual_seed(2)
    t = K.MXTensor(torch.randint(0, 256, (rows, 64), generator=g, device=DEV, dtype=torch.uint8),
                   torch.randint(120, 130, (rows, 4), generator=g, device=DEV, dtype=torch.uint8), (rows, cols), "fp4")
    out = K.mx_dequantize(t, F16)
    for a, b in slices(rows, 1 << 24):
        part = K.MXTensor(t.codes[a:b], t.scales[a:b], (b - a, cols), "fp4")
        assert torch.equal(out[a:b], K.mx_dequantize(part, F16)), (a, b)


@pytest.mark.parametrize("residual", [False, True])
def test_norm_more_rows_than_a_dispatch(residual):
    rows, cols = (1 << 26) + 5, 8  # 64 threads a row
    g = torch.Generator(device=DEV).manual_seed(3)
    x = torch.randn(rows, cols, generator=g, device=DEV, dtype=F16)
    res = torch.randn(rows, cols, generator=g, device=DEV, dtype=F16) if residual else None
    w = torch.randn(cols, generator=g, device=DEV, dtype=F16)
    q, h, rstd = K.rms_norm_mx_fwd(x, w, residual=res)
    for a, b in slices(rows, 1 << 23):
        p, ph, pr = K.rms_norm_mx_fwd(x[a:b], w, residual=None if res is None else res[a:b])
        assert torch.equal(q.codes[a:b], p.codes) and torch.equal(q.scales[a:b], p.scales), (a, b)
        assert torch.equal(h[a:b], ph) and torch.equal(rstd[a:b], pr), (a, b)


@pytest.mark.parametrize("glu", [False, True])
def test_few_tokens_with_more_features_than_a_dispatch(glu):
    """The few-token kernel takes 32 threads a feature here: from 2^27 features on another one has to."""
    n, k = (1 << 27) + 40, 32
    rows = 2 * n if glu else n
    g = torch.Generator(device=DEV).manual_seed(4)
    codes = torch.zeros(rows, 64, device=DEV, dtype=torch.uint8)
    codes[:, :16] = torch.randint(0, 256, (rows, 16), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.zeros(rows, 4, device=DEV, dtype=torch.uint8)
    scales[:, 0] = 125
    w = K.MXTensor(codes, scales, (rows, k), "fp4")
    x = torch.randint(-3, 4, (1, k), generator=g, device=DEV).to(BF16)
    got = K.mx_mlp_glu_fwd(x, w) if glu else K.mx_gemm(x, w)
    step = 1 << 23
    for a in range(0, n, step):
        b = min(a + step, n)
        part = [K.mx_dequantize(K.MXTensor(codes[o + a: o + b], scales[o + a: o + b], (b - a, k), "fp4"), F32)
                for o in ((0, n) if glu else (0,))]
        y = [torch.matmul(p, x[0].float()) for p in part]  # multiples of 1/8 below 2^8: exact
        if not glu:
            assert torch.equal(got[0, a:b], y[0].to(BF16)), a
            continue
        gate, up = y[0].double(), y[1].double()
        want = gate / (1 + torch.exp(-gate)) * up
        # the sigmoid's error in units of 2^-23 and the result's rounding
        tol = ((10 + gate.abs()) * 2.0**-23 + 2.0**-8) * want.abs() + 2.0**-130
        assert ((got[0, a:b].double() - want).abs() <= tol).all(), a


# ---- every tile over many stages -----------------------------------------------------------------
#
# Sizes that the plan sends to the named tile (asserted: a change of its costs may not leave one untested),
# ragged in tokens and features, contractions of even and odd numbers of 128s, past two quads of scales.


def plan(m, n, k, fx, fw, glu=0):
    got = (ctypes.c_int32 * 3)()
    _lib.call("rus_mx_gemm_plan", m, n, k, _lib.MX_FP8 if fx == "fp8" else _lib.MX_FP4,
              _lib.MX_FP8 if fw == "fp8" else _lib.MX_FP4, glu, got)
    return got[0], got[1], got[2] > 1


PLAIN = [  # rows of W x tokens of a tile, whether the contraction is split, formats, sizes
    (256, 128, False, "fp8", "fp4", 1100, 9000, 1200), (256, 128, False, "fp8", "fp4", 2100, 9001, 1100),
    (256, 128, False, "fp8", "fp4", 521, 7285, 660), (256, 128, False, "fp8", "fp4", 1993, 2058, 633),
    (256, 128, True, "fp8", "fp4", 38, 12346, 13154), (256, 128, True, "fp8", "fp4", 8, 12303, 6120),
    (256, 256, False, "fp4", "fp4", 2100, 4500, 1536), (256, 256, False, "fp4", "fp4", 1100, 9000, 1200),
    (256, 256, False, "fp4", "fp4", 1211, 7069, 637), (256, 256, False, "fp4", "fp4", 666, 11028, 2100),
    (256, 256, True, "fp4", "fp4", 270, 14218, 9674), (256, 256, True, "fp4", "fp4", 386, 8337, 9226),
]
for _fx, _fw in FORMATS:
    PLAIN += [(128, 128, False, _fx, _fw, 4420, 398, 691), (128, 128, False, _fx, _fw, 195, 9917, 633),
              (128, 128, True, _fx, _fw, 3664, 33, 5689), (128, 128, True, _fx, _fw, 3359, 32, 5794),
              (128, 64, False, _fx, _fw, 1345, 120, 1240), (128, 64, False, _fx, _fw, 777, 240, 1074),
              (128, 64, False, _fx, _fw, 707, 2048, 1536),
              (128, 64, True, _fx, _fw, 9, 3449, 6585), (128, 64, True, _fx, _fw, 8, 2061, 12304)]


@pytest.mark.parametrize("bf,bt,split,fx,fw,m,n,k", PLAIN)
def test_product_in_each_tile(bf, bt, split, fx, fw, m, n, k):
    assert plan(m, n, k, fx, fw) == (bf, bt, split)
    w, wb = exact(n, k, fw, n + 1)
    x, xb = exact(m, k, fx, m + 1)
    want = x @ w.T
    assert float(want.abs().max()) < 2.0**15
    bits(K.mx_gemm(xb, wb, dtype=BF16), want)
    bias = torch.arange(n, device=DEV).remainder(7) - 3.0
    bits(K.mx_gemm(xb, wb, bias=bias.to(F16)), want + bias.double())
    odd = torch.full((m, n + 3), 7.0, dtype=F16, device=DEV)  # rows at any alignment, neighbours left alone
    K.mx_gemm(xb, wb, out=odd[:, 1: n + 1])
    bits(odd[:, 1: n + 1], want)
    odd[:, 1: n + 1] = 7.0
    assert (odd == 7.0).all()


GATED = [(256, 128, "fp8", "fp4", 2100, 4501, 1100), (256, 128, "fp8", "fp4", 1290, 5001, 1100),
         (256, 128, "fp8", "fp4", 707, 8960, 1536), (256, 128, "fp8", "fp4", 332, 5657, 645),
         (256, 256, "fp4", "fp4", 1290, 5001, 1100), (256, 256, "fp4", "fp4", 707, 8960, 1536),
         (256, 256, "fp4", "fp4", 302, 13408, 650), (128, 128, "fp4", "fp4", 2100, 4501, 1100),
         (128, 128, "fp8", "fp8", 2100, 2301, 1100), (128, 128, "fp4", "fp8", 1290, 1157, 1200),
         (128, 64, "fp8", "fp4", 687, 304, 959), (128, 64, "fp8", "fp8", 3245, 34, 1817),
         (128, 64, "fp4", "fp4", 596, 77, 4364), (128, 64, "fp4", "fp8", 23, 9081, 958)]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("bf,bt,fx,fw,m,n,k", GATED)
def test_gated_in_each_tile(bf, bt, fx, fw, m, n, k, dtype):
    assert plan(m, n, k, fx, fw, 1) == plan(m, n, k, fx, fw, 2) == (bf, bt, False)
    w, wb = exact(2 * n, k, fw, n, low=119)  # so that g and u stay near one
    x, xb = exact(m, k, fx, m)
    y = x @ w.T
    g, u = y[:, :n], y[:, n:]
    s = 1 / (1 + torch.exp(-g))
    half, least = (2.0**-11, 2.0**-25) if dtype == F16 else (2.0**-8, 2.0**-134)
    tol = (20 + 2 * g.abs()) * 2.0**-23  # the sigmoid's exponential and reciprocal, four products

    def near(got, want, err):
        return bool(((got.double() - want).abs() <= err + half * (want.abs() + err) + least).all())

    want = g * s * u
    assert near(K.mx_mlp_glu_fwd(xb, wb, dtype=dtype), want, tol * want.abs())
    dh = (torch.arange(m * n, device=DEV).remainder(11) - 5.0).view(m, n).to(dtype)
    d = dh.double()
    got = K.mx_mlp_glu_bwd(dh, xb, wb)
    # the two terms of silu' may cancel: each has its own rounding
    assert near(got[:, :n], d * u * (s + g * s * (1 - s)), tol * (d * u).abs() * (s + g.abs() * s))
    assert near(got[:, n:], d * g * s, tol * (d * g * s).abs())
    wide = torch.full((m, 3 * n + 3), 7.0, dtype=dtype, device=DEV)  # dh and the result in one odd matrix
    wide[:, 1: n + 1] = dh
    K.mx_mlp_glu_bwd(wide[:, 1: n + 1], xb, wb, out=wide[:, n + 2: 3 * n + 2])
    assert torch.equal(wide[:, n + 2: 3 * n + 2], got) and torch.equal(wide[:, 1: n + 1], dh)
    assert (wide[:, [0, n + 1, 3 * n + 2]] == 7.0).all()


GRADIENT = [(256, True, 2100, 5000, 1537), (256, False, 4100, 700, 2310), (256, True, 132, 2790, 10810),
            (256, False, 772, 259, 9627), (128, True, 137, 4114, 1799), (128, False, 399, 267, 9259),
            (64, True, 37, 2823, 5470), (64, False, 1763, 258, 1042), (32, True, 8, 3175, 4885),
            (32, False, 86, 383, 1864)]


@pytest.mark.parametrize("fw", ["fp4", "fp8"])
@pytest.mark.parametrize("tm,split,m,n,k", GRADIENT)
def test_gradient_in_each_tile(tm, split, m, n, k, fw):
    got = (ctypes.c_int32 * 2)()
    _lib.call("rus_mx_gemm_t_plan", m, n, k, got)
    assert (got[0], got[1] > 1) == (tm, split)
    w, wb = exact(n, k, fw, 1)
    g = torch.Generator(device=DEV).manual_seed(m)
    dy = torch.randint(-3, 4, (m, n), generator=g, device=DEV).double()
    want = dy @ w
    for dtype in (F16, BF16):
        bits(K.mx_gemm(dy.to(dtype), wb, trans=True), want)
        wide = torch.full((m, n + 2), float("nan"), dtype=dtype, device=DEV)  # rows at any alignment
        wide[:, 1: n + 1] = dy.to(dtype)
        out = torch.full((m, k + 2), 7.0, dtype=dtype, device=DEV)
        K.mx_gemm(wide[:, 1: n + 1], wb, trans=True, out=out[:, 1: k + 1])
        bits(out[:, 1: k + 1], want)
        assert (out[:, [0, k + 1]] == 7.0).all()


# ---- blocks that are not finite, in each tile ----------------------------------------------------

SPECIAL = [(256, 128, False, "fp8", "fp4", 1993, 2058, 633), (256, 256, False, "fp4", "fp4", 2100, 4500, 1100),
           (128, 128, False, "fp8", "fp8", 2100, 2301, 1100), (128, 128, False, "fp4", "fp8", 2100, 2301, 1100),
           (128, 64, False, "fp8", "fp4", 707, 2048, 1536), (128, 64, False, "fp4", "fp4", 777, 240, 1074),
           (32, 32, False, "fp8", "fp4", 40, 700, 640), (128, 64, True, "fp8", "fp8", 9, 3449, 6585),
           (256, 128, True, "fp8", "fp4", 38, 12346, 13154), (256, 256, True, "fp4", "fp4", 270, 14218, 9674)]


def not_finite(m, n, k):
    """x [m, k] and w [n, k] of ones with single infinities and NaNs, and the results they reach: the rows of x
    and of w that hold one. A row of zeros in x is no shield: 0 NaN is NaN."""
    x, w = torch.ones(m, k, device=DEV), torch.ones(n, k, device=DEV)
    x[2] = 0.0
    bad_x, bad_w = [1, m // 2, m - 2], [0, n // 3, n - 1]
    for row, col, v in zip(bad_x, (k - 1, k // 2, 0), ("nan", "inf", "-inf")):
        x[row, col] = float(v)
    for row, col, v in zip(bad_w, (0, k - 1, k // 2), ("-inf", "nan", "inf")):
        w[row, col] = float(v)
    bad = torch.zeros(m, n, dtype=torch.bool, device=DEV)
    bad[bad_x], bad[:, bad_w] = True, True
    return x, w, bad


@pytest.mark.parametrize("bf,bt,split,fx,fw,m,n,k", SPECIAL)
def test_product_of_blocks_that_are_not_finite(bf, bt, split, fx, fw, m, n, k):
    assert plan(m, n, k, fx, fw) == (bf, bt, split)
    x, w, bad = not_finite(m, n, k)
    y = K.mx_gemm(K.mx_quantize(x, fx), K.mx_quantize(w, fw), dtype=F16)
    want = torch.full((m, n), float(k), dtype=F16, device=DEV)
    want[2] = 0.0
    assert torch.equal(torch.isnan(y), bad) and torch.equal(y[~bad], want[~bad])


@pytest.mark.parametrize("bf,bt,fx,fw,m,n,k", [
    (256, 128, "fp8", "fp4", 1290, 5001, 1100), (256, 256, "fp4", "fp4", 1290, 5001, 1100),
    (128, 128, "fp8", "fp8", 2100, 2301, 1100), (128, 64, "fp8", "fp4", 687, 304, 959),
    (32, 32, "fp8", "fp4", 40, 70, 640)])
def test_gated_blocks_that_are_not_finite(bf, bt, fx, fw, m, n, k):
    """A NaN in a gate's or an up row reaches that feature; in x, its token; in dh, its one result of each."""
    assert plan(m, n, k, fx, fw, 1) == plan(m, n, k, fx, fw, 2) == (bf, bt, False)
    x, w, both = not_finite(m, 2 * n, k)
    bad = both[:, :n] | both[:, n:]
    xb, wb = K.mx_quantize(x, fx), K.mx_quantize(w * 2.0**-9, fw)
    clean = K.mx_mlp_glu_fwd(K.mx_quantize(torch.ones(3, k, device=DEV), fx),
                             K.mx_quantize(torch.full((64, k), 2.0**-9, device=DEV), fw), dtype=F16)[0, 0]
    h = K.mx_mlp_glu_fwd(xb, wb, dtype=F16)
    want = clean.expand(m, n).clone()
    want[2] = 0.0
    assert torch.equal(torch.isnan(h), bad)
    # (another kernel, the same exact projections: a step of fp16 at most)
    assert ((h - want)[~bad].abs() <= 2.0**-10 * clean).all()
    dh = torch.ones(m, n, dtype=F16, device=DEV)
    dh[m - 1, 3], dh[0, 5] = float("nan"), float("inf")
    d = K.mx_mlp_glu_bwd(dh, xb, wb)
    # d_up = dh silu(g) needs the gate only, d_gate = dh u silu'(g) both
    bad_up = both[:, :n].clone()
    for b in (bad, bad_up):
        b[m - 1, 3] = True
    assert torch.equal(torch.isnan(d[:, :n]), bad) and torch.equal(torch.isnan(d[:, n:]), bad_up)
    assert torch.isinf(d[0, [5, n + 5]]).all()
    finite = torch.isfinite(d)
    finite[0, [5, n + 5]] = True
    assert torch.equal(finite, ~torch.cat([bad, bad_up], dim=1))


@pytest.mark.parametrize("fw", ["fp4", "fp8"])
@pytest.mark.parametrize("tm,split,m,n,k", [r for r in GRADIENT if r[2:] != (4100, 700, 2310)])
def test_gradient_of_blocks_that_are_not_finite(tm, split, m, n, k, fw):
    """A block of W reaches its 32 columns of every row, a NaN or an infinity of dy its own row."""
    w = torch.ones(n, k, device=DEV)
    w[0, 40], w[n // 2, k - 1], w[n - 1, 0] = float("nan"), float("inf"), float("-inf")
    dy = torch.ones(m, n, dtype=BF16, device=DEV)
    dy[2] = 0.0
    dy[1, n - 1], dy[m // 2, 0], dy[m - 2, n // 2] = float("nan"), float("inf"), float("-inf")
    dx = K.mx_gemm(dy, K.mx_quantize(w, fw), trans=True)
    nan = torch.zeros(m, k, dtype=torch.bool, device=DEV)
    nan[1] = True
    nan[:, :64] = nan[:, (k - 1) // 32 * 32:] = True
    want = torch.full((m, k), float(n), device=DEV).to(BF16)
    want[2] = 0.0
    want[m // 2], want[m - 2] = float("inf"), float("-inf")
    assert torch.equal(torch.isnan(dx), nan) and torch.equal(dx[~nan], want[~nan])


# ---- the layers on inputs of other forms ---------------------------------------------------------


def layers():
    """(name, f of one input) over weights of ragged sizes."""
    d, inner = 200, 150
    g = torch.Generator(device=DEV).manual_seed(5)
    rnd = lambda *s: torch.randn(*s, generator=g, device=DEV, dtype=F16)
    wg, wd = K.mx_quantize(rnd(2 * inner, d) * 0.1, "fp4"), K.mx_quantize(rnd(d, inner) * 0.1, "fp4")
    nw, bias, res = rnd(d) * 0.1 + 1, rnd(2 * inner), rnd(d)
    return d, {"linear": lambda x: ops.mx_linear(x, wg, bias), "glu": lambda x: ops.mx_mlp_glu(x, wg),
               "norm_mlp": lambda x: ops.mx_norm_mlp(x, nw, wg, wd),
               "residual": lambda x: sum(ops.mx_norm_mlp(x, nw, wg, wd, residual=res.expand_as(x).contiguous())),
               "same": lambda x: sum(ops.mx_norm_mlp(x, nw, wg, wd, residual=x))}


@pytest.mark.parametrize("layer", ["linear", "glu", "norm_mlp", "residual", "same"])
def test_layers_on_inputs_of_any_form(layer):
    """Zero tokens, a single vector, transposed, sliced and broadcast inputs, broadcast gradients: what the
    same rows give when contiguous."""
    d, f = layers()
    f = f[layer]
    for shape in ((0, d), (2, 0, d), (1, 0, 3, d)):
        x = torch.zeros(shape, dtype=F16, device=DEV, requires_grad=True)
        y = f(x)
        assert y.shape[:-1] == x.shape[:-1]
        y.sum().backward()
        assert x.grad.shape == x.shape
    base = torch.randn(6, 7, d + 5, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV, dtype=F16)
    views = [base[0, 0, :d], base[:, :, 3: d + 3], base.transpose(0, 1)[..., :d], base[::2, 1:, 5:],
             base[0, :1, :d].expand(9, d), base[:1, :, :d].expand(4, 7, d)]
    for v in views:
        x, c = v.detach().requires_grad_(), v.detach().contiguous().requires_grad_()
        y, want = f(x), f(c)
        assert torch.equal(y, want)
        for dy in (torch.ones((), dtype=F16, device=DEV).expand(y.shape), torch.randn_like(y),
                   torch.randn(y.shape[-1:] + y.shape[:-1], device=DEV, dtype=F16).movedim(0, -1)):
            dx = torch.autograd.grad(y, x, dy, retain_graph=True)[0]
            assert torch.equal(dx, torch.autograd.grad(want, c, dy.contiguous(), retain_graph=True)[0])


# ---- every code at every scale -------------------------------------------------------------------


def every_value(fmt):
    """One row with all codes of a format at all finite scales: (their values in float64, codes, scales)."""
    n = 16 if fmt == "fp4" else 256
    codes = np.tile(np.arange(n, dtype=np.uint8), 255 * max(1, 32 // n))
    scales = np.repeat(np.arange(255, dtype=np.uint8), max(1, n // 32))
    codes = np.pad(codes, (0, -len(codes) % 128))
    scales = np.pad(scales, (0, -len(scales) % 4))
    return ref.mx_values(ref.mx_pack(codes[None], fmt), scales[None], len(codes), fmt)[0], codes, scales


def same(a, b):
    return bool(((a == b) | (torch.isnan(a) & torch.isnan(b))).all())


@pytest.mark.parametrize("m", [1, 40, 100, 300])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("fw", ["fp4", "fp8"])
def test_gradient_decodes_every_value(fw, dtype, m):
    """One weight row times one: the values rounded once to dy's type, subnormal and infinite ones too."""
    v, codes, scales = every_value(fw)
    w = K.MXTensor(torch.from_numpy(ref.mx_pack(codes[None], fw)).to(DEV), torch.from_numpy(scales[None]).to(DEV),
                   (1, len(v)), fw)
    want = torch.from_numpy(v).to(dtype).to(DEV)
    assert same(K.mx_gemm(torch.ones(m, 1, dtype=dtype, device=DEV), w, trans=True), want.expand(m, -1))
    assert same(K.mx_dequantize(w, dtype)[0], want)


@pytest.mark.parametrize("exponent", [-100, 0, 100])
@pytest.mark.parametrize("m", [1, 5, 40, 300])
@pytest.mark.parametrize("fx,fw", FORMATS)
def test_product_of_every_value(fx, fw, m, exponent):
    """One weight a row times a power of two: fp32 products rounded once, at scales whose own product leaves
    fp32."""
    v, codes, scales = every_value(fw)
    code, scale = np.zeros((len(v), 128), np.uint8), np.zeros((len(v), 4), np.uint8)
    code[:, 0], scale[:, 0] = codes, np.repeat(scales, 32)
    w = K.MXTensor(torch.from_numpy(ref.mx_pack(code, fw)).to(DEV), torch.from_numpy(scale).to(DEV), (len(v), 1), fw)
    x = torch.full((m, 1), 2.0**exponent, device=DEV)
    want = torch.from_numpy(v * 2.0**exponent).float().to(BF16).to(DEV)
    assert same(K.mx_gemm(K.mx_quantize(x, fx), w, dtype=BF16), want.expand(m, -1))
