"""The microscaled kernels beyond one dispatch, and each tile of the products in its steady state: ragged sizes,
contractions of many stages, blocks that are not finite. Data whose sums are exact in fp32 shows an element
dropped, doubled or scaled by a neighbour's scale."""

from __future__ import annotations

import pytest
import torch

from rus_amd import kernels as K, ops

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
