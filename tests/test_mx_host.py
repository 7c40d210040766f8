"""The host side of the microscaled operators on the CPU: frozen parameters under ``no_grad``, second
derivatives, size queries of unknown formats, results that one dispatch cannot hold, plans."""

from __future__ import annotations

import ctypes
import threading

import pytest
import torch

from rus_amd import _lib, kernels as K, ops


def _mx(rows, cols, fmt="fp4"):
    nb = 4 * -(-cols // 128)
    return K.MXTensor(torch.zeros(rows, nb * (16 if fmt == "fp4" else 32), dtype=torch.uint8),
                      torch.zeros(rows, nb, dtype=torch.uint8), (rows, cols), fmt)


# ---- frozen parameters ---------------------------------------------------------------------------


def test_parameters_are_taken_where_no_gradient_is_recorded():
    """A module's bias and norm weight require gradients by default: refused only while autograd records.
    (On the CPU a call that is not refused for them ends at the check of its device.)"""
    x, w = torch.zeros(2, 64, dtype=torch.float16), _mx(8, 64)
    weight = torch.nn.Parameter(torch.ones(64, dtype=torch.float16))
    bias = torch.nn.Parameter(torch.zeros(8, dtype=torch.float16))
    calls = (lambda: ops.mx_linear(x, w, bias), lambda: ops.mx_norm_mlp(x, weight, w, w))
    for call in calls:
        with pytest.raises(RuntimeError, match="frozen"):
            call()
        for off in (torch.no_grad, torch.inference_mode):
            with off(), pytest.raises(RuntimeError, match="HIP device tensors"):
                call()


# ---- second derivatives --------------------------------------------------------------------------


@pytest.fixture
def plain_kernels(monkeypatch):
    """Stand-ins of the launchers that return zeros of the right shape on the CPU."""
    zeros = lambda m, n: torch.zeros(m, n, dtype=torch.float16)
    monkeypatch.setattr(K, "mx_quantize", lambda x, fmt="fp4": _mx(*x.shape, fmt))
    monkeypatch.setattr(K, "mx_gemm", lambda x, w, trans=False, **_: zeros(x.shape[0], w.shape[1 if trans else 0]))
    monkeypatch.setattr(K, "mx_mlp_glu_fwd", lambda x, w, **_: zeros(x.shape[0], w.shape[0] // 2))
    monkeypatch.setattr(K, "mx_mlp_glu_bwd", lambda dh, x, w, **_: zeros(dh.shape[0], w.shape[0]))
    monkeypatch.setattr(K, "rms_norm_mx_fwd", lambda x, w, eps, residual: (
        _mx(x.numel() // x.shape[-1], x.shape[-1], "fp8"), x if residual is None else x + residual, torch.zeros(2)))
    monkeypatch.setattr(K, "rms_norm_bwd", lambda dy, h, w, rstd, dresidual=None: torch.zeros_like(dy))


@pytest.mark.parametrize("layer", ["linear", "glu", "norm_mlp", "norm_mlp_residual"])
def test_gradients_of_gradients_are_refused(layer, plain_kernels):
    """The backward runs kernels that autograd does not see: what it returns may not pass for a constant."""
    x = torch.ones(2, 64, dtype=torch.float16, requires_grad=True)
    w, down, norm = _mx(16, 64), _mx(64, 8), torch.ones(64, dtype=torch.float16)
    res = torch.ones_like(x, requires_grad=True)
    y = {"linear": lambda: ops.mx_linear(x, w),
         "glu": lambda: ops.mx_mlp_glu(x, w),
         "norm_mlp": lambda: ops.mx_norm_mlp(x, norm, w, down),
         "norm_mlp_residual": lambda: ops.mx_norm_mlp(x, norm, w, down, residual=res)[0]}[layer]()
    for dy in (torch.ones_like(y), torch.ones_like(y, requires_grad=True)):
        (dx,) = torch.autograd.grad(y, x, dy, create_graph=True)
        if layer == "linear" and not dy.requires_grad:
            assert not dx.requires_grad  # dy W is one
            continue
        with pytest.raises(RuntimeError, match="no second derivative"):
            (dx.sum() + x.sum()).backward()
    assert not torch.autograd.grad(y, x, torch.ones_like(y))[0].requires_grad


def test_first_derivatives_under_create_graph(plain_kernels):
    """A graph of the gradient that nothing differentiates costs nothing."""
    x = torch.ones(2, 64, dtype=torch.float16, requires_grad=True)
    z = ops.mx_mlp_glu(x, _mx(16, 64)).sum() + (x * x).sum()
    (dx,) = torch.autograd.grad(z, x, create_graph=True)
    assert torch.equal(dx, 2 * x)
    (dx,) = torch.autograd.grad(ops.mx_mlp_glu(x, _mx(16, 64)).sum(), x, create_graph=True)
    dx.mul_(2.0)  # a gradient is the caller's to change


# ---- formats that do not exist -------------------------------------------------------------------

F16, FP4, FP8 = 0, 0, 1


def _query(name, *sizes):
    got = ctypes.c_int64()
    _lib.call(name, *sizes, ctypes.byref(got))
    return got.value


@pytest.mark.parametrize("x_fmt,w_fmt,which", [(2, FP4, "x"), (-1, FP8, "x"), (FP8, 2, "w"), (FP8, -2, "w"),
                                               (FP4, 2, "w")])
def test_size_queries_refuse_unknown_formats(x_fmt, w_fmt, which):
    for call in (lambda: _query("rus_mx_gemm_workspace", 64, 2048, 8960, x_fmt, w_fmt),
                 lambda: _query("rus_mx_rows_scratch", 64, 2048, 8960, x_fmt, w_fmt, 0),
                 lambda: _query("rus_mx_rows_scratch", 64, 2048, 8960, x_fmt, w_fmt, 1)):
        with pytest.raises(RuntimeError, match=f"{which} has unknown format"):
            call()


def test_a_refused_format_leaves_other_plans_alone():
    """Sizes are planned once per thread and remembered: a thread whose first calls name formats that do not
    exist sees the sizes that every thread sees."""
    bad = [(x_fmt, w_fmt) for x_fmt in (-1, 0, 1, 2) for w_fmt in (-2, 0, 1, 2, 4) if not {x_fmt, w_fmt} <= {0, 1}]

    def refused(m, n, k, x_fmt, w_fmt):
        rows = (16, k, x_fmt, 16, 16, w_fmt, m, n, k)
        return (lambda: _query("rus_mx_gemm_workspace", m, n, k, x_fmt, w_fmt),
                lambda: _query("rus_mx_rows_scratch", m, n, k, x_fmt, w_fmt, 0),
                # (no scratch: refused before anything is launched)
                lambda: _lib.call("rus_mx_gemm_rows", *rows, None, 16, n, F16, None, 0, None),
                lambda: _lib.call("rus_mx_glu_fwd_rows", *rows, 16, n, F16, None, 0, None))

    def ask(before):
        got = []
        for size in [(64, 512, 20000), (64, 2048, 8960), (100, 4096, 4096)]:
            for good in [(FP4, FP4), (FP8, FP4), (FP4, FP8), (FP8, FP8)]:
                for i in range(4 * len(bad)):
                    _query("rus_mx_gemm_workspace", *size, FP8 - good[0], good[1])  # (takes the other's place)
                    if before:
                        try:
                            refused(*size, *bad[i // 4])[i % 4]()
                        except RuntimeError:
                            pass
                    got.append(_query("rus_mx_gemm_workspace", *size, *good))
        return got

    got = []
    for before in (False, True):
        t = threading.Thread(target=lambda: got.append(ask(before)))
        t.start()
        t.join()
    assert len(got) == 2 and got[0] == got[1]


# ---- results that one dispatch cannot hold -------------------------------------------------------


@pytest.mark.parametrize("name,args", [
    ("rus_mx_gemm", (16, 16, FP8, 16, 16, FP8, 1 << 19, 1 << 20, 64, None, 16, 1 << 20, F16, None, 0, None)),
    ("rus_mx_gemm_rows", (16, 64, FP8, 16, 16, FP8, 1 << 19, 1 << 20, 64, None, 16, 1 << 20, F16, 16, 1 << 60, None)),
    ("rus_mx_glu_fwd", (16, 16, FP8, 16, 16, FP8, 1 << 19, 1 << 19, 64, 16, 1 << 19, F16, None)),
    ("rus_mx_glu_fwd_rows", (16, 64, FP8, 16, 16, FP8, 1 << 19, 1 << 19, 64, 16, 1 << 19, F16, 16, 1 << 60, None)),
    ("rus_mx_glu_bwd", (16, 1 << 19, 16, 16, FP8, 16, 16, FP8, 1 << 19, 1 << 19, 64, 16, 1 << 20, F16, None)),
    ("rus_mx_gemm_t", (16, 64, F16, 16, 16, FP4, 1 << 20, 64, 1 << 20, 16, 1 << 20, None, 0, None)),
])
def test_results_beyond_a_dispatch_are_refused(name, args):
    """2^39 values, a terabyte: refused by name, with nothing launched."""
    with pytest.raises(RuntimeError, match=f"{name}: .* beyond one dispatch"):
        _lib.call(name, *args)


# ---- the plans -----------------------------------------------------------------------------------


def test_plans_agree_with_the_sizes_they_need():
    p, t = (ctypes.c_int32 * 3)(), (ctypes.c_int32 * 2)()
    for m, n, k in [(1, 1536, 8960), (3, 2048, 1536), (8, 1536, 8960), (33, 2051, 4096), (707, 2048, 1536),
                    (270, 14218, 9674), (2100, 9001, 1100), (4100, 700, 2310)]:
        for x_fmt in (FP4, FP8):
            for w_fmt in (FP4, FP8):
                _lib.call("rus_mx_gemm_plan", m, n, k, x_fmt, w_fmt, 0, p)
                assert _query("rus_mx_gemm_workspace", m, n, k, x_fmt, w_fmt) == (p[2] * m * n if p[2] > 1 else 0)
                scratch = _query("rus_mx_rows_scratch", m, n, k, x_fmt, w_fmt, 0)
                assert (scratch == 0) == ((p[0], p[1]) == (8, m))  # few tokens: a feature's row to 8 lanes
                _lib.call("rus_mx_gemm_plan", m, n, k, x_fmt, w_fmt, 2, p)
                assert p[0] >= 32 and p[2] == 1
        _lib.call("rus_mx_gemm_t_plan", m, n, k, t)
        assert _query("rus_mx_gemm_t_workspace", m, n, k) == (t[1] * m * k if t[1] > 1 else 0)


@pytest.mark.parametrize("name,args,msg", [
    ("rus_mx_gemm_plan", (4, 64, 64, FP8, FP4, 0, None), "null result"),
    ("rus_mx_gemm_plan", (4, 0, 64, FP8, FP4, 0, (ctypes.c_int32 * 3)()), "bad sizes"),
    ("rus_mx_gemm_plan", (4, 64, 64, 2, FP4, 0, (ctypes.c_int32 * 3)()), "x has unknown format"),
    ("rus_mx_gemm_plan", (4, 64, 64, FP8, -1, 0, (ctypes.c_int32 * 3)()), "w has unknown format"),
    ("rus_mx_gemm_t_plan", (4, 64, 64, None), "null result"),
    ("rus_mx_gemm_t_plan", (4, 64, 0, (ctypes.c_int32 * 2)()), "bad sizes"),
])
def test_plan_queries_refuse(name, args, msg):
    with pytest.raises(RuntimeError, match=msg):
        _lib.call(name, *args)
