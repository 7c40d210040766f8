"""GPU tests of rotary positions with several axes against the definition in float64.

Bounds: the angle in turns is a product in 64 bits, pos * f / 2 pi (2^-52 relative, twice), of which an eighth of a turn
at most goes to 32 bits; sine and cosine are then good to 2^-23, and two products and a sum in 32 bits add 3 x 2^-24 of
|x1| + |x2|. One rounding to the type: half a step (fp16 2^-11, bf16 2^-8, fp32 2^-24), below fp16's normal range 2^-25.
"""

from __future__ import annotations

import copy
import math
import pickle

import pytest
import torch

from oracle import ops as ref
from rus_amd import kernels as K
from rus_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8, torch.float32: 2.0**-24}


def _check(got, x, pos, axis, freq, adjacent, inverse=False):
    want = ref.rope_axes(x, pos, axis, freq, adjacent, inverse)
    p = len(axis)
    assert torch.equal(got.cpu()[..., 2 * p:], x[..., 2 * p:])
    i, j = (slice(0, 2 * p, 2), slice(1, 2 * p, 2)) if adjacent else (slice(0, p), slice(p, 2 * p))
    size = torch.zeros_like(want)
    size[..., i] = size[..., j] = x.double()[..., i].abs() + x.double()[..., j].abs()
    angle = pos.double()[torch.tensor(axis)].t().abs() * torch.tensor(freq, dtype=torch.float64)
    e = torch.zeros(x.shape[0], 1, x.shape[2], dtype=torch.float64)
    e[:, 0, i] = e[:, 0, j] = 2.0**-23 + 3 * 2.0**-24 + 2.0**-50 * angle
    tol = e * size + U[x.dtype] * want.abs() * (1 + 2.0**-7) + (2.0**-25 if x.dtype == torch.float16 else 1e-38)
    err = (got.double().cpu() - want).abs()
    assert bool((err <= tol).all()), float((err / tol).max())


def _case(n, hq, hk, d, sections, dtype, adjacent=False, restart=False, order="blocks", seed=0, far=5000):
    g = torch.Generator().manual_seed(seed)
    axes = K.RopeAxes.sections(sections, 1e6, d, DEV, order=order, restart=restart, adjacent=adjacent)
    q = torch.randn(n, hq, d, generator=g).to(dtype)
    k = torch.randn(n, hk, d, generator=g).to(dtype)
    pos = torch.randint(0, far, (len(sections), n), generator=g)
    axis = axes.axis.cpu().tolist()
    freq = (axes.turns.cpu() * (2 * math.pi)).tolist()
    return axes, q, k, pos, axis, freq


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32], ids=["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("adjacent", [False, True], ids=["halves", "adjacent"])
@pytest.mark.parametrize("n,d,sections", [(1, 128, (16, 24, 24)), (70, 128, (16, 24, 24)), (33, 80, (9, 11)),
                                          (2, 80, (20, 20)), (5, 96, (7, 13, 17)), (129, 64, (32,)), (3, 256, (40, 1, 23)),
                                          (2050, 64, (8, 4, 4)), (4, 6, (1, 1))])
def test_against_float64(dtype, adjacent, n, d, sections):
    for restart in (False, True):
        axes, q, k, pos, axis, freq = _case(n, 3, 1, d, sections, dtype, adjacent, restart, seed=n + d)
        dev = (q.to(DEV), k.to(DEV), pos.to(DEV), axes)
        got = K.rope_axes_fwd(*dev)
        back = K.rope_axes_bwd(*dev)
        for i, x in enumerate((q, k)):
            _check(got[i], x, pos, axis, freq, adjacent)
            _check(back[i], x, pos, axis, freq, adjacent, inverse=True)


def test_sections_in_turn_and_own_pairs():
    axes = K.RopeAxes.sections((4, 2, 3), 100.0, 32, "cpu", order="cycle")
    assert axes.axis.tolist() == [0, 1, 2, 0, 1, 2, 0, 2, 0] and axes.n_axes == 3
    own = K.RopeAxes([0, 2, 2], [1.0, 0.5, 0.0], 8, device=DEV)
    g = torch.Generator().manual_seed(1)
    x = torch.randn(5, 2, 8, generator=g)
    pos = torch.randint(-50, 50, (3, 5), generator=g)
    q, k = K.rope_axes_fwd(x.to(DEV), None, pos.to(DEV), own)
    assert k is None
    _check(q, x, pos, [0, 2, 2], [1.0, 0.5, 0.0], False)


@pytest.mark.parametrize("pos", [torch.int64, torch.int32, torch.float32])
def test_positions_far_negative_and_between(pos):
    axes, q, k, p, axis, freq = _case(64, 2, 2, 128, (16, 24, 24), torch.float32, far=1 << 30)
    p[:, ::3] = -p[:, ::3]
    p = p.to(pos)
    if pos == torch.float32:
        p = p / 4096 + 0.25
    p[:, 0] = 0
    got = K.rope_axes_fwd(q.to(DEV), k.to(DEV), p.to(DEV), axes)
    _check(got[0], q, p, axis, freq, False)
    _check(got[1], k, p, axis, freq, False)


@pytest.mark.parametrize("offset", [0, 1, 2, 4])
def test_views_at_any_stride_and_alignment(offset):
    axes, q, k, pos, axis, freq = _case(21, 4, 2, 64, (12, 20), torch.bfloat16)
    rows = torch.empty(21, 6 * 64 + 2 * offset, dtype=torch.bfloat16, device=DEV)
    body = rows[:, offset:offset + 384].view(21, 6, 64) if offset == 0 else rows[:, offset:offset + 384].unflatten(1, (6, 64))
    body[:, :4], body[:, 4:] = q.to(DEV), k.to(DEV)
    before = rows.clone()
    wide = torch.zeros(2, 50, dtype=torch.int64, device=DEV)
    wide[:, 7:28] = pos.to(DEV)
    got = K.rope_axes_fwd(body[:, :4], body[:, 4:], wide[:, 7:28], axes)
    _check(got[0], q, pos, axis, freq, False)
    _check(got[1], k, pos, axis, freq, False)
    assert torch.equal(rows.view(torch.int16), before.view(torch.int16))
    # tokens and heads the other way round, every second element
    t = q.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(K.rope_axes_fwd(t, None, pos.to(DEV), axes)[0], got[0])
    s = torch.zeros(21, 4, 128, dtype=torch.bfloat16, device=DEV)
    s[..., ::2] = q.to(DEV)
    assert torch.equal(K.rope_axes_fwd(s[..., ::2], None, pos.to(DEV), axes)[0], got[0])


def test_gradients_of_every_order():
    """The rotation is linear: its gradient is the inverse rotation, whose gradient is the rotation again."""
    axes, q, k, pos, axis, freq = _case(9, 2, 1, 16, (3, 5), torch.float32, seed=4)
    a, b = q.to(DEV).requires_grad_(), k.to(DEV).requires_grad_()
    g = torch.Generator().manual_seed(5)
    dq, dk = torch.randn(q.shape, generator=g).to(DEV).requires_grad_(), torch.randn(k.shape, generator=g).to(DEV)
    y, z = ops.rope_axes(a, b, pos.to(DEV), axes)
    ga, gb = torch.autograd.grad((y, z), (a, b), (dq, dk), create_graph=True)
    want = K.rope_axes_bwd(dq.detach(), dk, pos.to(DEV), axes)
    assert torch.equal(ga, want[0]) and torch.equal(gb, want[1])
    (gg,) = torch.autograd.grad(ga, dq, q.to(DEV))
    assert torch.equal(gg, K.rope_axes_fwd(q.to(DEV), None, pos.to(DEV), axes)[0])
    e = torch.randn(q.shape, generator=g).double()  # against differences: the map is linear
    up = ref.rope_axes(q.double() + e, pos, axis, freq) - ref.rope_axes(q.double() - e, pos, axis, freq)
    slope = (up / 2 * dq.detach().cpu().double()).sum()
    assert abs(float((ga.detach().cpu().double() * e).sum() - slope)) <= 2.0**-20 * float((e.abs().sum() + 1) * 8)
    (only,) = torch.autograd.grad(ops.rope_axes(a, None, pos.to(DEV), axes), a, dq)
    assert torch.equal(only, want[0])
    (unused,) = torch.autograd.grad(ops.rope_axes(a, b, pos.to(DEV), axes)[0], b, dq)
    assert not bool(unused.any())


def test_no_tokens():
    axes, q, k, pos, *_ = _case(1, 2, 1, 16, (3, 5), torch.float16)
    a, b = K.rope_axes_fwd(q[:0].to(DEV), k[:0].to(DEV), pos[:, :0].to(DEV), axes)
    assert a.shape == (0, 2, 16) and b.shape == (0, 1, 16)


def test_a_copied_handle_reads_its_own_tables():
    """A model that is deep-copied or pickled takes its handle along; the first one's memory may be gone."""
    axes = K.RopeAxes.sections((5, 7, 4), 1e4, 32, DEV)
    q = torch.randn(9, 2, 32, device=DEV)
    pos = torch.arange(27, device=DEV).view(3, 9)
    want, _ = K.rope_axes_fwd(q, None, pos, axes)
    for twin in (copy.deepcopy(axes), pickle.loads(pickle.dumps(axes))):
        assert twin.axis.data_ptr() != axes.axis.data_ptr()
        axes.turns.zero_()  # (the first handle's memory in other hands)
        got, _ = K.rope_axes_fwd(q, None, pos, twin)
        axes.turns.copy_(twin.turns)
        assert torch.equal(got, want)
