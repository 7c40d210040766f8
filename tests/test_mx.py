"""Microscaled operators on the CPU: the float64 definitions against known answers and against
differences, and every refusal of the host layer and the C entry points."""

from __future__ import annotations

import ctypes

import numpy as np
import pytest
import torch

from oracle import ops as ref
from rus_amd import _lib, kernels as K, ops


# ---- the definitions -----------------------------------------------------------------------


def test_grids_hold_the_formats_values():
    assert len(ref.MX_GRID["fp4"]) == 8 and len(ref.MX_GRID["fp8"]) == 127
    codes = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().numpy()
    assert np.array_equal(ref.MX_GRID["fp8"], codes)


def test_quantize_known_answers():
    x = np.zeros((1, 32))
    x[0, :9] = [6.0, -5.0, 5.0, 3.5, 2.5, 0.25, -0.75, 0.2, 7.9]  # scale 1: ties to even codes
    code, scale = ref.mx_quantize(x, "fp4")
    assert scale[0].tolist() == [127, 0, 0, 0]
    assert code[0, :9].tolist() == [7, 14, 6, 6, 4, 0, 10, 0, 7]
    x[0, 8] = 8.0  # a power of two raises the scale
    assert ref.mx_quantize(x, "fp4")[1][0, 0] == 128
    x[0, 3] = np.inf
    code, scale = ref.mx_quantize(x, "fp8")
    assert scale[0, 0] == 255 and (code[0, :32] == 127).all()
    assert np.isnan(ref.mx_values(code, scale, 32, "fp8")).all()


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
def test_rounding_is_to_the_nearest(fmt):
    """An element is off by at most half the distance of its neighbours, or saturated."""
    g = np.random.default_rng(0)
    x = g.standard_normal((7, 300)) * np.exp2(g.integers(-30, 30, (7, 300)))
    code, scale = ref.mx_quantize(x, fmt)
    v = ref.mx_values(ref.mx_pack(code, fmt), scale, 300, fmt)
    s = np.exp2(np.repeat(scale.astype(float) - 127, 32, axis=1)[:, :300])
    grid = np.concatenate([-ref.MX_GRID[fmt][:0:-1], ref.MX_GRID[fmt]])
    best = np.abs((x / s)[:, :, None] - grid).min(axis=2)
    assert np.array_equal(np.abs(x / s - v / s), best)


def test_glu_gradient_against_differences():
    g = np.random.default_rng(1)
    gate, up, dh = (g.standard_normal((5, 9)) * 3 for _ in range(3))
    d = ref.mx_glu_bwd(dh, gate, up)
    eps = 1e-5  # central differences: error eps^2 / 6 |f'''| + 1e-16 / eps, well below 1e-8
    dg = dh * (ref.mx_glu(gate + eps, up) - ref.mx_glu(gate - eps, up)) / (2 * eps)
    du = dh * (ref.mx_glu(gate, up + eps) - ref.mx_glu(gate, up - eps)) / (2 * eps)
    assert np.abs(d - np.concatenate([dg, du], axis=1)).max() < 1e-8


# ---- the host layer --------------------------------------------------------------------------


def _mx(rows, cols, fmt="fp4", device="cpu"):
    nb = ref.mx_blocks(cols)
    return K.MXTensor(torch.zeros(rows, nb * (16 if fmt == "fp4" else 32), dtype=torch.uint8, device=device),
                      torch.zeros(rows, nb, dtype=torch.uint8, device=device), (rows, cols), fmt)


@pytest.mark.parametrize("change,err", [
    (dict(fmt="fp6"), "format"),
    (dict(shape=(4, 0)), "bad shape"),
    (dict(codes=torch.zeros(4, 64)), "uint8"),
    (dict(codes=torch.zeros(4, 48, dtype=torch.uint8)), "are codes"),
    (dict(scales=torch.zeros(4, 8, dtype=torch.uint8)), "are codes"),
    (dict(codes=torch.zeros(4, 128, dtype=torch.uint8)[:, ::2]), "contiguous"),
])
def test_mxtensor_refuses(change, err):
    args = dict(codes=torch.zeros(4, 64, dtype=torch.uint8), scales=torch.zeros(4, 4, dtype=torch.uint8),
                shape=(4, 100), fmt="fp4")
    K.MXTensor(**args)
    with pytest.raises((ValueError, TypeError), match=err):
        K.MXTensor(**{**args, **change})


@pytest.mark.parametrize("fmt", ["fp4", "fp8"])
@pytest.mark.parametrize("cols", [1, 31, 32, 33, 127, 129])
def test_from_blocks_pads_and_clears(fmt, cols):
    g = torch.Generator().manual_seed(cols)
    n, w = -(-cols // 32), 16 if fmt == "fp4" else 32
    codes = torch.randint(0, 120, (3, n * w), generator=g, dtype=torch.uint8)
    scales = torch.randint(100, 140, (3, n), generator=g, dtype=torch.uint8)
    t = K.MXTensor.from_blocks(codes, scales, (3, cols), fmt)
    nb = ref.mx_blocks(cols)
    assert t.scales.shape == (3, nb) and not t.scales[:, n:].any()
    full = ref.mx_values(t.codes.numpy(), t.scales.numpy(), nb * 32, fmt)
    assert not full[:, cols:].any()
    own = np.zeros((3, nb * w), dtype=np.uint8)
    own[:, : n * w] = codes.numpy()
    ext = np.zeros((3, nb), dtype=np.uint8)
    ext[:, :n] = scales.numpy()
    assert np.array_equal(full[:, :cols], ref.mx_values(own, ext, cols, fmt))
    with pytest.raises(ValueError, match="are codes"):
        K.MXTensor.from_blocks(codes[:, :-1], scales, (3, cols), fmt)


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 64, dtype=torch.float16), _mx(8, 64)
    for call in (lambda: K.mx_quantize(x), lambda: K.mx_dequantize(w), lambda: K.mx_gemm(x, w),
                 lambda: K.mx_gemm(torch.zeros(2, 8), w, trans=True), lambda: K.mx_mlp_glu_fwd(x, w),
                 lambda: K.mx_mlp_glu_bwd(torch.zeros(2, 4), x, w),
                 lambda: K.rms_norm_mx_fwd(x, torch.ones(64, dtype=torch.float16)),
                 lambda: ops.mx_linear(x, w), lambda: ops.mx_mlp_glu(x, w)):
        with pytest.raises(RuntimeError, match="HIP device tensors"):
            call()


def test_results_apart_from_operands():
    """Rows that share bytes against rows that only share a matrix."""
    flat = torch.zeros(6, 40, dtype=torch.float16)
    whole, left, right = flat, flat[:, :20], flat[:, 20:]
    assert K._apart(left, right) and K._apart(right, left) and K._apart(flat[:3], flat[3:])
    assert K._apart(flat[:, :10], flat[:, 10:12]) and K._apart(flat[1:, :10], flat[:, 30:])
    assert K._apart(left, torch.zeros(6, 40)) and K._apart(whole[:0], whole)
    for a, b in ((whole, whole), (left, whole), (flat[:4], flat[3:]), (flat[:, :21], right), (flat[:, 19:], left),
                 (flat[1:, :21], right), (flat.view(12, 20), left), (flat.view(-1)[7:127].view(3, 40), left),
                 (flat[2:3, 5:], flat[:, :6])):
        assert not K._apart(a, b) and not K._apart(b, a)
    assert K._apart(flat[2:3, 6:], flat[:2]) and K._apart(flat[2:3, 20:], flat[3:])


def test_wrong_operands_are_refused():
    x, w = torch.zeros(2, 64, dtype=torch.float16), _mx(8, 64)
    for call, err in (
            (lambda: K.mx_quantize(x, "int4"), "format"),
            (lambda: K.mx_dequantize(x), "MXTensor"),
            (lambda: K.mx_gemm(x, x), "MXTensor"),
            (lambda: K.mx_gemm(w, w, trans=True), "not blocks"),
            (lambda: K.mx_gemm(x, w, trans=True, bias=x), "bias"),
            (lambda: K.mx_gemm(x, w, trans=True, dtype=torch.bfloat16), "dtype"),
            (lambda: K.mx_mlp_glu_fwd(x, _mx(7, 64)), "even"),
            (lambda: K.mx_mlp_glu_fwd(x, x), "MXTensor"),
            (lambda: K.mx_mlp_glu_bwd(x, x, _mx(7, 64)), "even"),
            (lambda: ops.mx_linear(x, w, bias=torch.zeros(8, requires_grad=True)), "frozen"),
            (lambda: ops.mx_norm_mlp(x, torch.ones(64, requires_grad=True), w, w), "frozen"),
            (lambda: ops.mx_norm_mlp(x.float(), torch.ones(64), w, w), "fp16")):
        with pytest.raises((ValueError, TypeError, RuntimeError), match=err):
            call()


# ---- the C entry points (refused before anything touches a GPU) ------------------------------

F16, F32, BF16, FP4, FP8 = 0, 1, 2, 0, 1


@pytest.mark.parametrize("name,args,msg", [
    ("rus_mx_quantize", (16, F16, -1, 64, 64, FP4, 16, 16, None), "bad sizes"),
    ("rus_mx_quantize", (16, F16, 4, 0, 64, FP4, 16, 16, None), "bad sizes"),
    ("rus_mx_quantize", (16, F16, 4, 64, 63, FP4, 16, 16, None), "stride_row"),
    ("rus_mx_quantize", (16, 3, 4, 64, 64, FP4, 16, 16, None), "dtype"),
    ("rus_mx_quantize", (16, F16, 4, 64, 64, 2, 16, 16, None), "format"),
    ("rus_mx_quantize", (16, F16, 4, 64, 64, FP4, 8, 16, None), "misaligned"),
    ("rus_mx_quantize", (None, F16, 4, 64, 64, FP4, 16, 16, None), "null"),
    ("rus_mx_quantize", (17, F16, 4, 64, 64, FP4, 16, 16, None), "misaligned"),
    ("rus_mx_quantize", (16, F16, 1 << 40, 64, 64, FP4, 16, 16, None), "2\\^36"),
    ("rus_mx_dequantize", (16, 16, 5, 4, 64, 16, F16, 64, None), "format"),
    ("rus_mx_dequantize", (16, 16, FP8, 4, 64, 17, F16, 64, None), "misaligned"),
    ("rus_mx_dequantize", (16, 16, FP8, 4, 64, 16, F16, 32, None), "stride_row"),
    ("rus_mx_dequantize", (16, 16, FP8, 4, 64, 16, 9, 64, None), "dtype"),
    ("rus_rmsnorm_mx_fwd", (16, None, 16, F16, None, 16, 16, 16, 4, 0, 64, 1e-6, F16, None), "bad sizes"),
    ("rus_rmsnorm_mx_fwd", (16, None, 16, F16, None, 16, 16, 16, 4, 64, 60, 1e-6, F16, None), "stride_row"),
    ("rus_rmsnorm_mx_fwd", (16, 16, 16, F16, None, 16, 16, 16, 4, 64, 64, 1e-6, F16, None), "together"),
    ("rus_rmsnorm_mx_fwd", (16, None, 16, F16, None, 16, 16, 16, 4, 64, 64, 1e-6, BF16, None), "fp16 or fp32"),
    ("rus_rmsnorm_mx_fwd", (16, None, None, F16, None, 16, 16, 16, 4, 64, 64, 1e-6, F16, None), "null"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP4, 4, 0, 64, None, 16, 64, F16, None, 0, None), "bad sizes"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP4, 4, 64, 64, None, 16, 63, F16, None, 0, None), "stride"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP4, 4, 64, 64, None, 16, 64, F32, None, 0, None), "fp16 or bf16"),
    ("rus_mx_gemm", (16, 16, 7, 16, 16, FP4, 4, 64, 64, None, 16, 64, F16, None, 0, None), "x has unknown"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 18, FP4, 4, 64, 64, None, 16, 64, F16, None, 0, None), "w codes"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP4, 4, 64, 64, None, None, 64, F16, None, 0, None), "output"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP4, 4, 64, 64, 17, 16, 64, F16, None, 0, None), "bias"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP4, 5, 1536, 8960, None, 16, 1536, F16, 16, 8, None), "workspace holds"),
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP4, 1, 64, 1 << 23, None, 16, 64, F16, None, 0, None), "bad sizes"),
    ("rus_mx_gemm_workspace", (1, 64, 0, FP8, FP4, None), "null result"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 16, FP4, 5, 64, 64, None, 16, 64, F16, 16, 8, None), "scratch holds"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 16, FP4, 5, 64, 64, None, 16, 64, F16, None, 1 << 20, None), "scratch holds"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 16, FP4, 4, 0, 64, None, 16, 64, F16, 16, 1 << 20, None), "bad sizes"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 18, FP4, 4, 64, 64, None, 16, 64, F16, 16, 1 << 20, None), "w codes"),
    ("rus_mx_gemm_rows", (16, 63, FP8, 16, 16, FP4, 5, 64, 64, None, 16, 64, F16, 16, 1 << 20, None), "stride_row"),
    ("rus_mx_gemm_rows", (16, 64, 9, 16, 16, FP4, 4, 64, 64, None, 16, 64, F16, 16, 1 << 20, None), "format"),
    ("rus_mx_glu_fwd_rows", (16, 64, FP8, 16, 16, FP4, 5, 64, 64, 16, 64, F16, 16, 8, None), "scratch holds"),
    ("rus_mx_glu_fwd_rows", (16, 64, FP8, 16, 16, 5, 4, 64, 64, 16, 64, F16, 16, 1 << 20, None), "w has unknown"),
    # a few tokens: no scratch, the same refusals
    ("rus_mx_gemm_rows", (16, 63, FP8, 16, 16, FP4, 2, 64, 64, None, 16, 64, F16, None, 0, None), "stride_x"),
    ("rus_mx_gemm_rows", (None, 64, FP8, 16, 16, FP4, 2, 64, 64, None, 16, 64, F16, None, 0, None), "x is null"),
    ("rus_mx_gemm_rows", (17, 64, FP8, 16, 16, FP4, 2, 64, 64, None, 16, 64, F16, None, 0, None), "misaligned"),
    ("rus_mx_gemm_rows", (16, 64, 9, 16, 16, FP4, 2, 64, 64, None, 16, 64, F16, None, 0, None), "format"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 16, FP4, 2, 64, 64, 17, 16, 64, F16, None, 0, None), "bias"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 8, 16, FP4, 2, 64, 64, None, 16, 64, F16, None, 0, None), "w codes"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 16, FP4, 2, 64, 64, None, 16, 63, F16, None, 0, None), "stride"),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 16, FP4, 2, 64, 64, None, 16, 64, F32, None, 0, None), "fp16 or bf16"),
    ("rus_mx_gemm", (None, 16, FP8, 16, 16, FP4, 2, 64, 64, None, 16, 64, F16, None, 0, None), "x codes"),
    ("rus_mx_glu_fwd_rows", (None, 64, FP8, 16, 16, FP4, 2, 64, 64, 16, 64, F16, None, 0, None), "x is null"),
    ("rus_mx_glu_fwd_rows", (16, 64, FP8, 16, 16, FP4, 2, 64, 64, None, 64, F16, None, 0, None), "output"),
    ("rus_mx_rows_scratch", (1, 64, 64, FP8, FP4, 0, None), "null result"),
    ("rus_mx_glu_fwd", (16, 16, FP8, 16, 16, FP4, 4, 64, 64, 16, 63, F16, None), "stride"),
    ("rus_mx_glu_bwd", (16, 64, 16, 16, FP8, 16, 16, FP4, 4, 64, 64, 16, 127, F16, None), "stride"),
    ("rus_mx_glu_bwd", (16, 63, 16, 16, FP8, 16, 16, FP4, 4, 64, 64, 16, 128, F16, None), "stride_dh"),
    ("rus_mx_glu_bwd", (None, 64, 16, 16, FP8, 16, 16, FP4, 4, 64, 64, 16, 128, F16, None), "dh is null"),
    ("rus_mx_gemm_t", (16, 63, F16, 16, 16, FP4, 4, 64, 64, 16, 64, None, 0, None), "strides"),
    ("rus_mx_gemm_t", (16, 64, F32, 16, 16, FP4, 4, 64, 64, 16, 64, None, 0, None), "fp16 or bf16"),
    ("rus_mx_gemm_t", (16, 64, F16, 16, 16, 3, 4, 64, 64, 16, 64, None, 0, None), "format"),
    ("rus_mx_gemm_t", (16, 64, F16, 16, 16, FP4, 4, 64, 64, None, 64, None, 0, None), "null"),
    ("rus_mx_gemm_t", (16, 17920, F16, 16, 16, FP4, 4, 17920, 1536, 16, 1536, 16, 8, None), "workspace holds"),
    ("rus_mx_gemm_t_workspace", (4, 0, 64, None), "null result"),
])
def test_entry_points_refuse(name, args, msg):
    with pytest.raises(RuntimeError, match=msg):
        _lib.call(name, *args)


def test_empty_batches_launch_nothing():
    _lib.call("rus_mx_quantize", None, F16, 0, 64, 64, FP4, None, None, None)
    _lib.call("rus_mx_gemm", None, None, FP8, None, None, FP4, 0, 64, 64, None, None, 64, F16, None, 0, None)
    _lib.call("rus_mx_gemm_t", None, 64, F16, None, None, FP4, 0, 64, 64, None, 64, None, 0, None)


def test_scratch_sizes():
    """A few tokens take none, as long as they fit; others the codes, the scales and the sums of a split
    contraction."""
    def scratch(m, n, k, glu=0):
        got = ctypes.c_int64()
        _lib.call("rus_mx_rows_scratch", m, n, k, FP8, FP4, glu, ctypes.byref(got))
        return got.value
    assert scratch(0, 64, 64) == scratch(1, 1536, 8960) == scratch(2, 17920, 1536) == scratch(4, 2048, 1536) == 0
    assert scratch(2, 8960, 1536, 1) == 0
    assert scratch(5, 64, 64) >= 5 * 4 * 33 and scratch(3, 17920, 1536) >= 3 * 48 * 33
    assert scratch(1, 64, 1 << 20) >= (1 << 15) * 33
    got = ctypes.c_int64()
    _lib.call("rus_mx_gemm_workspace", 1, 1536, 8960, FP8, FP4, ctypes.byref(got))
    assert got.value == 0
    _lib.call("rus_mx_gemm_workspace", 8, 1536, 8960, FP8, FP4, ctypes.byref(got))
    assert got.value > 0 and got.value % (8 * 1536) == 0


def test_capture_beside_a_living_graph_is_refused():
    """The stream of a leaf's first graph is known while some graph over the leaf lives, and no longer."""
    x = torch.zeros(3, requires_grad=True)

    def record(stream, capturing):
        kept = ops._note_stream("op", x, stream, capturing)
        y = x.exp()
        del kept
        return y

    alive = record(1, False)
    record(2, False)  # another stream, not capturing: autograd's own synchronisation
    record(1, True)
    with pytest.raises(RuntimeError, match="op: a graph recorded on another stream"):
        record(2, True)
    del alive
    captured = record(2, True)
    record(1, False)
    record(2, True)
    with pytest.raises(RuntimeError, match="still holds"):
        record(3, True)
    del captured
    record(3, True)
