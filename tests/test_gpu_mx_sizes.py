"""The microscaled products where their kernels change: one to five tokens, tiles of every height, split
contractions, ragged edges, offsets past 32 bits; on data whose sums are exact, so that an element
dropped, doubled or scaled by a neighbour's scale shows. The definitions are 64-bit ones on the device."""

from __future__ import annotations

import numpy as np
import pytest
import torch

from oracle import ops as ref
from rus_amd import _lib, kernels as K, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
F16, BF16, F32, F64 = torch.float16, torch.bfloat16, torch.float32, torch.float64
FORMATS = [("fp8", "fp4"), ("fp4", "fp4"), ("fp8", "fp8"), ("fp4", "fp8")]
VALUES = [-3.0, -2.0, -1.0, -0.5, 0.0, 0.0, 0.5, 1.0, 1.5, 2.0]


def exact(rows, k, fmt, seed, low=126):
    """Blocks of the values above with scales 2^(low - 127) and the next: (float64 values, MXTensor),
    both on the device. Products of two are multiples of 2^-4 below 144."""
    g = torch.Generator(device=DEV).manual_seed(seed)
    nb = ref.mx_blocks(k)
    pick = torch.randint(len(VALUES), (rows, nb * 32), generator=g, device=DEV)
    pick[:, k:] = 4
    scale = torch.randint(low, low + 2, (rows, nb), generator=g, device=DEV)
    scale[:, (k + 31) // 32:] = 0
    grid = ref.MX_GRID[fmt]
    code = [int(np.searchsorted(grid, abs(v))) + ((8 if fmt == "fp4" else 128) if v < 0 else 0) for v in VALUES]
    codes = torch.tensor(code, dtype=torch.uint8, device=DEV)[pick]
    if fmt == "fp4":
        codes = codes[:, 0::2] | codes[:, 1::2] << 4
    values = torch.tensor(VALUES, dtype=F64, device=DEV)[pick]
    values *= torch.exp2(scale.double() - 127).repeat_interleave(32, dim=1)
    t = K.MXTensor(codes.contiguous(), scale.to(torch.uint8), (rows, k), fmt)
    return values[:, :k].contiguous(), t


def bits(got, want):
    """got is want (float64, exact in fp32) rounded once."""
    assert got.shape == want.shape
    assert torch.equal(got, want.to(got.dtype)), (got.double() - want).abs().max()


# ---- few tokens ----------------------------------------------------------------------------------


@pytest.mark.parametrize("fx,fw", FORMATS)
@pytest.mark.parametrize("n,k", [(1, 1), (7, 31), (8, 32), (9, 33), (100, 257), (515, 1000), (4104, 300), (40, 8960),
                                 (24, 11680), (24, 11700), (17, 23296), (17, 23400)])
def test_few_tokens_exact(n, k, fx, fw):
    """(n, k) on either side of what the few-token kernel takes: 4 and 2 tokens, x in and out of LDS."""
    w, wb = exact(n, k, fw, n + k)
    bias = torch.arange(n, device=DEV).remainder(7) - 3.0
    for m in (1, 2, 3, 4, 5):
        x, xb = exact(m, k, fx, m)
        want = x @ w.T  # multiples of 2^-4 below 2^22: exact in fp32 up to 2^20 of them
        assert float(want.abs().max()) < 2.0**19
        bits(K.mx_gemm(xb, wb, dtype=BF16), want)
        bits(K.mx_gemm(xb, wb, bias=bias.to(BF16), dtype=BF16), want + bias.double())
        bits(K.mx_gemm(xb, wb), want)


@pytest.mark.parametrize("act", ["fp8", "fp4"])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("m,n,k", [(1, 40, 1000), (2, 33, 129), (3, 64, 511), (4, 2048, 1536), (1, 5000, 1536)])
def test_few_tokens_round_as_quantize(m, n, k, dtype, act):
    """Rounded inside the product or before it: the same blocks, so the same bits; rows anywhere."""
    w, wb = exact(n, k, "fp4", 5)
    g = torch.Generator().manual_seed(m + k)
    x = torch.randn(m, k, generator=g) * torch.exp2(torch.arange(k) // 40 % 9 - 4.0)
    for lo, width in ((0, k), (1, k + 3), (8, k + 8)):
        wide = torch.full((m, width + lo), float("nan"), dtype=dtype, device=DEV)
        wide[:, lo: lo + k] = x.to(dtype)
        view = wide[:, lo: lo + k]
        blocks = K.mx_quantize(view, act)
        assert torch.equal(K.mx_gemm(view, wb, act=act), K.mx_gemm(blocks, wb, dtype=dtype))
        if n % 2 == 0:
            assert torch.equal(K.mx_mlp_glu_fwd(view, wb, act=act), K.mx_mlp_glu_fwd(blocks, wb, dtype=dtype))
        # against the formula: exact products, k / 16 + 16 roundings of the fp32 sums
        v = K.mx_dequantize(blocks, F32).double()
        want, mag = v @ w.T, v.abs() @ w.abs().T
        half = 2.0**-11 if dtype == F16 else 2.0**-8
        err = (k / 16 + 16) * 2.0**-24 * mag
        assert ((K.mx_gemm(view, wb, act=act).double() - want).abs() <= err + half * (want.abs() + err) + 2.0**-25).all()


def test_few_tokens_special_values():
    """NaN and infinite blocks reach exactly what they enter; scales whose product leaves fp32 do not."""
    for m in (1, 2, 4):
        x = torch.ones(m, 700, dtype=BF16, device=DEV)
        w = torch.ones(24, 700, device=DEV)
        w[5, 3], w[9, 699] = float("inf"), float("nan")
        x[m - 1, 400] = float("-inf")
        for act in ("fp8", "fp4"):
            for fmt in ("fp8", "fp4"):
                y = K.mx_gemm(x, K.mx_quantize(w, fmt), act=act)
                bad = torch.zeros(m, 24, dtype=torch.bool, device=DEV)
                bad[m - 1], bad[:, 5], bad[:, 9] = True, True, True
                assert torch.equal(torch.isnan(y), bad) and (y[~bad] == 700).all()
        x = torch.full((m, 64), 2.0**120, dtype=BF16, device=DEV)
        w = torch.full((8, 64), 2.0**-118, device=DEV)
        assert (K.mx_gemm(x, K.mx_quantize(w, "fp4")) == 256).all()
        x, w = x.fill_(2.0**126), w.fill_(2.0**100)  # and one that is beyond the result's type
        assert torch.isinf(K.mx_gemm(x, K.mx_quantize(w, "fp4"))).all()
        assert (K.mx_gemm(x.fill_(2.0**-100), K.mx_quantize(w.fill_(2.0**-100), "fp8")) == 0).all()


@pytest.mark.parametrize("m", [1, 2, 3, 4])
def test_few_tokens_write_their_own(m):
    w, wb = exact(50, 96, "fp4", 1)
    x, xb = exact(m, 96, "fp8", 2)
    for lo in (0, 1, 8):
        wide = torch.full((m + 2, 80), 7.0, dtype=F16, device=DEV)
        K.mx_gemm(xb, wb, out=wide[:m, lo: lo + 50])
        bits(wide[:m, lo: lo + 50], x @ w.T)
        wide[:m, lo: lo + 50] = 7.0
        assert (wide == 7.0).all()
        h = K.mx_mlp_glu_fwd(xb, wb)
        K.mx_mlp_glu_fwd(xb, wb, out=wide[:m, lo: lo + 25])
        assert torch.equal(wide[:m, lo: lo + 25], h)
        wide[:m, lo: lo + 25] = 7.0
        assert (wide == 7.0).all()


@pytest.mark.parametrize("fx,fw", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 9, 33), (2, 100, 1536), (3, 515, 300), (4, 40, 8960), (4, 5000, 100)])
def test_few_tokens_glu(m, n, k, fx, fw):
    """silu(g) u of exact g and u: the sigmoid is good to (8 + |g|) 2^-23, the products to 2^-23."""
    w, wb = exact(2 * n, k, fw, 3, low=118)
    x, xb = exact(m, k, fx, 4)
    y = x @ w.T
    g, u = y[:, :n], y[:, n:]
    want = g / (1 + torch.exp(-g)) * u
    got = K.mx_mlp_glu_fwd(xb, wb, dtype=BF16).double()
    assert ((got - want).abs() <= ((10 + g.abs()) * 2.0**-23 + 2.0**-8) * want.abs() + 2.0**-130).all()


# ---- tiles of every height -----------------------------------------------------------------------


@pytest.mark.parametrize("fx,fw", FORMATS)
@pytest.mark.parametrize("m,n,k", [(2100, 4500, 100), (2100, 4500, 300), (2100, 4500, 600), (1290, 2313, 1200),
                                   (8200, 1030, 384), (200, 9000, 1000), (513, 1000, 513)])
def test_tiles_exact(m, n, k, fx, fw):
    """Many tiles in both directions, none a whole one at the edges; contractions of one group of four
    blocks, of fewer than four groups, of an odd number of them."""
    w, wb = exact(n, k, fw, n)
    x, xb = exact(m, k, fx, m)
    want = x @ w.T
    assert float(want.abs().max()) < 2.0**19
    bits(K.mx_gemm(xb, wb, dtype=BF16), want)
    bias = torch.arange(n, device=DEV).remainder(7) - 3.0
    bits(K.mx_gemm(xb, wb, bias=bias.to(F16)), want + bias.double())


@pytest.mark.parametrize("fx,fw", [("fp8", "fp4"), ("fp4", "fp4"), ("fp8", "fp8")])
@pytest.mark.parametrize("m,n,k", [(2100, 2300, 100), (2100, 2300, 600), (1290, 1157, 1200), (300, 4500, 384)])
def test_glu_tiles(m, n, k, fx, fw):
    w, wb = exact(2 * n, k, fw, n, low=119)
    x, xb = exact(m, k, fx, m)
    y = x @ w.T
    g, u = y[:, :n], y[:, n:]
    s = 1 / (1 + torch.exp(-g))
    tol = (20 + 2 * g.abs()) * 2.0**-23
    got = K.mx_mlp_glu_fwd(xb, wb, dtype=BF16).double()
    want = g * s * u
    assert ((got - want).abs() <= (tol + 2.0**-8) * want.abs() + 2.0**-130).all()
    dh = (torch.arange(m * n, device=DEV).remainder(11) - 5.0).view(m, n).to(BF16)
    got = K.mx_mlp_glu_bwd(dh, xb, wb).double()
    d = dh.double()
    gate, up = d * u * (s + g * s * (1 - s)), d * g * s
    # the two terms of silu' may cancel: each has its own rounding
    assert ((got[:, :n] - gate).abs() <= tol * (d * u).abs() * (s + g.abs() * s) + 2.0**-8 * gate.abs() + 2.0**-130).all()
    assert ((got[:, n:] - up).abs() <= (tol + 2.0**-8) * up.abs() + 2.0**-130).all()


@pytest.mark.parametrize("fx,fw", FORMATS)
@pytest.mark.parametrize("m,n,k", [(40, 64, 20000), (9, 65, 8960), (150, 130, 9100), (33, 2051, 4096)])
def test_split_contraction_exact(m, n, k, fx, fw):
    w, wb = exact(n, k, fw, 1)
    x, xb = exact(m, k, fx, 2)
    bias = torch.arange(n, device=DEV).remainder(7) - 3.0
    want = x @ w.T
    bits(K.mx_gemm(xb, wb, dtype=BF16), want)
    bits(K.mx_gemm(xb, wb, bias=bias.to(BF16), dtype=BF16), want + bias.double())


# ---- the gradient product ------------------------------------------------------------------------


@pytest.mark.parametrize("fw", ["fp4", "fp8"])
@pytest.mark.parametrize("m,n,k", [(2100, 600, 1000), (700, 3000, 300), (16, 20000, 65), (1, 9000, 640),
                                   (300, 5000, 258), (4100, 70, 2310), (64, 1000, 4000)])
def test_gradient_tiles_exact(m, n, k, fw):
    w, wb = exact(n, k, fw, 1)
    g = torch.Generator(device=DEV).manual_seed(m)
    dy = torch.randint(-3, 4, (m, n), generator=g, device=DEV).double()
    want = dy @ w
    for dtype in (F16, BF16):
        bits(K.mx_gemm(dy.to(dtype), wb, trans=True), want)


@pytest.mark.parametrize("fw", ["fp4", "fp8"])
@pytest.mark.parametrize("m,n", [(3, 40), (40, 2000), (300, 700)])
def test_gradient_special_values(m, n, fw):
    """A NaN block of W reaches its 32 columns of every row, an infinity or a NaN of dy its own row."""
    k = 200
    w = torch.ones(n, k, device=DEV)
    w[n - 3, 70] = float("nan")
    w[1, 199] = float("inf")
    dy = torch.ones(m, n, dtype=BF16, device=DEV)
    dy[m - 1, 4] = float("nan")
    dy[0, 5] = float("inf")
    dx = K.mx_gemm(dy, K.mx_quantize(w, fw), trans=True)
    nan = torch.zeros(m, k, dtype=torch.bool, device=DEV)
    nan[m - 1] = True
    nan[:, 64:96] = nan[:, 192:] = True
    assert torch.equal(torch.isnan(dx), nan)
    assert torch.isinf(dx[0][~nan[0]]).all()
    assert (dx[1: m - 1][~nan[1: m - 1]] == float(torch.tensor(float(n)).to(BF16))).all()


# ---- the norm --------------------------------------------------------------------------------------


@pytest.mark.parametrize("scale,weight", [(1.0, 1.0), (1e-3, 1.0), (1e18, 1e-9), (1e-18, 1e9), (1.0, 2.0**60),
                                          (1.0, 2.0**-90), (2.0**-120, 1.0), (2.0**110, 2.0**50)])
def test_norm_fp32_and_fp64_products_agree(scale, weight):
    """A million elements: those whose code fp32 cannot settle, and scales it cannot hold, are as in
    float64."""
    g = torch.Generator().manual_seed(3)
    x = (torch.randn(700, 1537, generator=g) * scale).float()
    w = (torch.randn(1537, generator=g) * weight).float()
    q, h, rstd = K.rms_norm_mx_fwd(x.to(DEV), w.to(DEV), eps=0.0)
    d = x.double().numpy()
    r = 1 / np.sqrt((d * d).mean(axis=1, keepdims=True))
    code, byte = ref.mx_quantize(d * r * w.double().numpy(), "fp8")
    assert np.array_equal(q.scales.cpu().numpy(), byte)
    assert np.array_equal(q.codes.cpu().numpy(), ref.mx_pack(code, "fp8"))


def test_norm_rows_with_a_few_values():
    """Blocks of zeros inside a row, a row with one value, weights of zero."""
    x = torch.zeros(5, 1000)
    x[1, 999], x[2, 3], x[3, 64:96], x[4] = 4.0, 1e-30, 2.5, 1.25
    w = torch.ones(1000)
    w[0::3] = 0.0
    w[128:160] = 0.0
    q, _, _ = K.rms_norm_mx_fwd(x.to(DEV), w.to(DEV), eps=1e-5)
    d = x.double().numpy()
    r = 1 / np.sqrt((d * d).mean(axis=1, keepdims=True) + np.float64(np.float32(1e-5)))
    code, byte = ref.mx_quantize(d * r * w.double().numpy(), "fp8")
    assert np.array_equal(q.scales.cpu().numpy(), byte)
    assert np.array_equal(q.codes.cpu().numpy(), ref.mx_pack(code, "fp8"))


# ---- offsets past 32 bits --------------------------------------------------------------------------


def test_blocks_past_32_bits():
    rows, cols = (1 << 22) + 3, 1024
    x = torch.zeros(rows, cols, dtype=F16, device=DEV)
    tail = torch.randn(5, cols, generator=torch.Generator().manual_seed(1)).half().to(DEV)
    x[-5:] = tail
    for fmt in ("fp4", "fp8"):
        t, want = K.mx_quantize(x, fmt), K.mx_quantize(tail, fmt)
        assert torch.equal(t.codes[-5:], want.codes) and torch.equal(t.scales[-5:], want.scales)
        assert not t.codes[-1000:-5].any()
        back = K.mx_dequantize(t, F16, out=x)
        assert torch.equal(back[-5:], K.mx_dequantize(want, F16))
        x[-5:] = tail


def test_products_past_32_bits():
    """Results, operands and gradients of more than 2^31 elements; the last rows and columns."""
    m, n, k = 70000, 32776, 96
    x, xb = exact(m, k, "fp8", 1)
    w, wb = exact(n, k, "fp4", 2)
    y = K.mx_gemm(xb, wb)
    bits(y[-300:], x[-300:] @ w.T)
    bits(y[::4999, -77:], x[::4999] @ w[-77:].T)
    dy = y.fill_(0.0)
    d = torch.randint(-3, 4, (5, n), device=DEV).double()
    dy[-5:] = d.half()
    dx = K.mx_gemm(dy, wb, trans=True)
    bits(dx[-5:], d @ w)
    assert not dx[:-5].any()
    del y, dy, dx
    a = torch.randint(-3, 4, (m, 8), device=DEV).double()  # and of that many results of the gradient
    v, vb = exact(8, n, "fp4", 3)
    dx = K.mx_gemm(a.half(), vb, trans=True)
    bits(dx[-200:], a[-200:] @ v)


def test_weights_past_32_bits():
    n, k = (1 << 21) + 24, 2048
    nb = ref.mx_blocks(k)
    tail, tb = exact(40, k, "fp8", 1)
    codes = torch.zeros(n, nb * 32, dtype=torch.uint8, device=DEV)
    scales = torch.full((n, nb), 127, dtype=torch.uint8, device=DEV)
    codes[-40:], scales[-40:] = tb.codes, tb.scales
    wb = K.MXTensor(codes, scales, (n, k), "fp8")
    for m in (1, 70):
        x, xb = exact(m, k, "fp8", m)
        y = K.mx_gemm(xb, wb)
        bits(y[:, -40:], x @ tail.T)
        assert not y[:, :-40].any()
        if m == 1:
            h = K.mx_mlp_glu_fwd(xb, wb)
            assert not h.any()  # silu(0) u
    dy = torch.zeros(2, n, dtype=F16, device=DEV)
    dy[:, -40:] = torch.randint(-3, 4, (2, 40), device=DEV).half()
    bits(K.mx_gemm(dy, wb, trans=True), dy[:, -40:].double() @ tail)


# ---- streams, graphs, timers -----------------------------------------------------------------------


@pytest.mark.parametrize("m", [1, 3, 9, 40])
def test_two_graphs_and_two_streams_share_nothing(m):
    """Split contractions keep their sums in scratch of their own: two captured graphs and eager calls on
    two streams at once give each the eager result, replay after replay."""
    n, k = 520, 9000
    w, wb = exact(n, k, "fp4", 1)
    v, vb = exact(k, n, "fp8", 2)
    xs = [exact(m, k, "fp8", s)[0].half() for s in (3, 4)]
    run = lambda x: (K.mx_gemm(x, wb, dtype=F16), K.mx_gemm(x, vb, trans=True))
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    graphs, outs = [], []
    for x, s in zip(xs, side):
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            run(x)
        torch.cuda.current_stream().wait_stream(s)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(x))
        graphs.append(g)
    for seed in (5, 6, 7):
        for i, x in enumerate(xs):
            x.copy_(exact(m, k, "fp8", 10 * seed + i)[0])
        want = [run(x) for x in xs]
        for x, (y, dx) in zip(xs, want):
            bits(dx, x.double() @ v)
        torch.cuda.synchronize()
        for s, g in zip(side, graphs):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
        eager = []
        for s, x in zip(side, xs):
            with torch.cuda.stream(s):
                eager.append(run(x))
        torch.cuda.synchronize()
        for a, b in zip(eager, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_capture_beside_an_eager_graph_is_refused():
    """While an eager graph of the same leaf lives: refused when the forward is recorded. (Nothing of the
    backward is: autograd would make the capture wait for the eager graph's stream.)"""
    w = K.mx_quantize(torch.randn(128, 128, device=DEV) * 0.1, "fp4")
    wd = K.mx_quantize(torch.randn(128, 64, device=DEV) * 0.1, "fp4")
    nw = torch.ones(128, dtype=F16, device=DEV)
    x = torch.randn(70, 128, dtype=F16, device=DEV, requires_grad=True)
    for call in (lambda: ops.mx_linear(x, w), lambda: ops.mx_mlp_glu(x, w), lambda: ops.mx_norm_mlp(x, nw, w, wd)):
        alive = call()
        with pytest.raises(RuntimeError, match="still holds"):
            with torch.cuda.graph(torch.cuda.CUDAGraph()):
                call()
        torch.cuda.synchronize()
        assert torch.equal(call(), alive)
        del alive


@pytest.mark.parametrize("tokens", [1, 70])
def test_forward_and_backward_captured(tokens):
    """A whole block with its gradient under capture, warmed up on a side stream, replayed on new inputs."""
    d, inner = 128, 192
    nw = torch.ones(d, dtype=F16, device=DEV)
    wg = K.mx_quantize(torch.randn(2 * inner, d, generator=torch.Generator().manual_seed(1)).to(DEV) * 0.1, "fp4")
    wd = K.mx_quantize(torch.randn(d, inner, generator=torch.Generator().manual_seed(2)).to(DEV) * 0.1, "fp4")
    x = torch.zeros(tokens, d, dtype=F16, device=DEV, requires_grad=True)
    dy = torch.zeros(tokens, d, dtype=F16, device=DEV)

    def step(x):
        y = ops.mx_norm_mlp(x, nw, wg, wd)
        z = ops.mx_linear(ops.mx_mlp_glu(y, wg), wd)
        return z.detach(), torch.autograd.grad(z, x, dy)[0]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(x)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step(x)
    for seed in (3, 4, 5):
        g = torch.Generator().manual_seed(seed)
        with torch.no_grad():
            x.copy_(torch.randn(tokens, d, generator=g))
            dy.copy_(torch.randn(tokens, d, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        want = step(x.detach().clone().requires_grad_())
        assert all(torch.equal(a, b) for a, b in zip(outs, want))


def test_every_launch_is_timed():
    x = torch.randn(3, 256, dtype=F16, device=DEV)
    w = K.mx_quantize(torch.randn(64, 256, device=DEV), "fp4")
    with K.KernelTimer() as t:
        q = K.mx_quantize(x, "fp8")
        K.mx_dequantize(q)
        K.rms_norm_mx_fwd(x, torch.ones(256, dtype=F16, device=DEV))
        y = K.mx_gemm(x, w)
        K.mx_gemm(y, w, trans=True)
        K.mx_mlp_glu_bwd(K.mx_mlp_glu_fwd(x, w), x, w, act="fp8")
    names = [r[0] for r in t.records]
    assert names == ["mx_quantize", "mx_dequantize", "rmsnorm_mx_fwd", "mx_gemm", "mx_gemm_t", "mx_glu_fwd",
                     "mx_quantize", "mx_glu_bwd"]
    assert all(r[3] > 0 for r in t.records)


def test_results_over_operands_are_refused():
    w = K.mx_quantize(torch.ones(64, 64, device=DEV), "fp4")
    for m in (1, 3, 50):
        wide = torch.ones(m, 200, dtype=F16, device=DEV)
        x, dh = wide[:, :64], wide[:, :32]
        for call in (lambda o: K.mx_gemm(x, w, out=o), lambda o: K.mx_gemm(x, w, trans=True, out=o),
                     lambda o: K.mx_mlp_glu_bwd(dh, w2, w, out=o)):
            w2 = K.mx_quantize(x, "fp8")
            with pytest.raises(ValueError, match="shares memory"):
                call(wide[:, 20:84])
            call(wide[:, 64:128])  # beside it
        assert (wide[:, :64] == 1).all() and (wide[:, 128:] == 1).all()
        with pytest.raises(ValueError, match="shares memory"):
            K.mx_mlp_glu_fwd(x, w, out=wide[:, 63:95])
        K.mx_mlp_glu_fwd(x, w, out=wide[:, 64:96])
        with pytest.raises(ValueError, match="the bias"):
            K.mx_gemm(x, w, bias=wide[m - 1, 130:194], out=wide[:, 136:200])


def test_refusals_leave_nothing_behind():
    """A refused call, then a good one."""
    w = K.mx_quantize(torch.ones(64, 256, device=DEV), "fp4")
    x = torch.ones(2, 256, dtype=F16, device=DEV)
    with pytest.raises(RuntimeError, match="stride_x"):
        _lib.call("rus_mx_gemm_rows", x.data_ptr(), 255, 1, w.codes.data_ptr(), w.scales.data_ptr(), 0, 2, 64, 256, None,
                  x.data_ptr(), 256, 0, None, 0, None)
    assert (K.mx_gemm(x, w) == 256).all()
