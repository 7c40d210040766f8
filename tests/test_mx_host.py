"""The host side of the microscaled operators where a first reading of it went wrong: frozen parameters under
``no_grad``, second derivatives, size queries of unknown formats, launches that one dispatch cannot hold."""

from __future__ import annotations

import pytest
import torch

from rus_amd import kernels as K, ops


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
