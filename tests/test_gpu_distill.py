"""GPU tests of the distillation loss over the lm_head against the definition in float64.

Bounds: logits are products of d terms summed in 32 bits (2^-24 a step: 2^-19 of the sum of absolute products covers
d <= 2048 and their conversions), delta; kl and lse move by 2 delta plus 2^-21 of their size. P is rounded to fp16 once
(2^-11 of it; 2^-25 of the token's reference below fp16's normal range, at most 2^-25 e^15 / e^7 of the largest P),
the teacher's entries are not; dH is in fp32.
"""

from __future__ import annotations

import math

import pytest
import torch

from oracle import ops as ref
from rus_amd import kernels as K
from rus_amd import ops
from rus_amd.hostload import HostHead

pytestmark = pytest.mark.gpu
DEV = "cuda"


def _inputs(n, d, v, k, seed=0, h_scale=3.0, missing=0.2, w_scale=0.05):
    g = torch.Generator().manual_seed(seed)
    h = (torch.randn(n, d, generator=g) * h_scale).half()
    w = (torch.randn(v, d, generator=g) * w_scale).half()
    ids = torch.stack([torch.randperm(v, generator=g)[:k] for _ in range(n)])
    logits = 10.0 - torch.cumsum(torch.rand(n, k, generator=g) * 2, 1)
    ids[torch.rand(n, k, generator=g) < missing] = -1
    if n > 2:
        ids[1] = -100  # a token without a teacher
    return h, w, ids, logits


def _bounds(h, w, ids, logits, t, want, num=None):
    """(bound of kl per token, bound of dh [n, d]) beside the definition's values."""
    h64, w64 = h.double(), w.double()
    z = h64 @ w64.t() / t
    raw = (h64.abs() @ w64.abs().t()) / t
    delta = 2.0**-19 * raw.amax(1)  # of any logit of the token
    p = torch.softmax(z, 1)
    log_p = torch.log_softmax(z, 1)
    valid = (ids >= 0) & (ids < w.shape[0]) & (logits != -math.inf)
    taught = valid.any(1)
    s = (logits.double() / t).masked_fill(~valid, -math.inf)
    q = torch.nan_to_num(torch.softmax(s, 1))
    log_q = torch.log(q.clamp(min=1e-300))
    size = (q * (log_q.abs() + log_p.gather(1, ids.clamp(0, w.shape[0] - 1)).abs())).sum(1)
    b_kl = 2 * delta + 2.0**-20 * (size + 1)
    denom = max(float(taught.sum() if num is None else num), 1.0)
    # P in fp16 away from the entries, everything's delta, the entries' p and q in fp32
    floor = 2.0**-24 * p.amax(1, keepdim=True) * 2.0  # the reference is within 2^8 of the largest, P at least 1 there
    err_p = (2.0**-11 + 2 * delta[:, None] + 2.0**-20) * p + floor
    b = (err_p @ w64.abs())
    b += (2.0**-20 * q)[..., None].mul(w64[ids.clamp(0, w.shape[0] - 1)].abs()).sum(1)
    b += 2.0**-20 * ((p @ w64.abs()) + 0)  # sums of fp32 products
    return b_kl, (t / denom) * b * taught[:, None]


def _check(got, h, w, ids, logits, t, num=None):
    loss, kl, dh = got
    want = ref.distill_head(h, w, ids, logits, t, num)
    b_kl, b_dh = _bounds(h, w, ids, logits, t, want, num)
    err = (kl.double().cpu() - want["kl"]).abs()
    assert bool((err <= b_kl).all()), ("kl", float((err / b_kl).max()))
    valid = ((ids >= 0) & (ids < w.shape[0]) & (logits != -math.inf)).any(1)
    assert not bool(kl.cpu()[~valid].any())
    denom = max(float(valid.sum() if num is None else num), 1.0)
    assert abs(float(loss) - float(want["loss"])) <= t * t * float(b_kl[valid].sum()) / denom + 2.0**-22 * abs(float(want["loss"]))
    if dh is not None:
        e = (dh.double().cpu() * 2.0**-16 - want["dh"]).abs()
        tol = b_dh + 2.0**-22 * want["dh"].abs() + 1e-30
        assert bool((e <= tol).all()), ("dh", float((e / tol).max()))
        assert not bool(dh.cpu()[~valid].any())


def _run(h, w, ids, logits, t=1.0, **kw):
    loss, kl, denom, dh = K.lm_head_distill(h.to(DEV), w.to(DEV), ids.to(DEV), logits.to(DEV), temperature=t, **kw)
    torch.cuda.synchronize()
    return loss, kl, dh


@pytest.mark.parametrize("n,d,v,k,t", [(1, 64, 1000, 1, 1.0), (5, 128, 257, 8, 2.0), (33, 192, 700, 16, 0.5),
                                       (70, 256, 3001, 33, 3.0), (300, 64, 513, 5, 1.0), (2, 1536, 1999, 128, 1.5),
                                       (9, 64, 64, 64, 1.0), (3, 128, 1, 1, 1.0), (4, 64, 2050, 1024, 1.0)])
def test_against_float64(n, d, v, k, t):
    h, w, ids, logits = _inputs(n, d, v, k, seed=n + v)
    _check(_run(h, w, ids, logits, t), h, w, ids, logits, t)


@pytest.mark.parametrize("chunk", [256, 512, 1024, 4096])
def test_chunks_of_the_vocabulary(chunk):
    """References that move from chunk to chunk: logits that grow and shrink along the vocabulary."""
    h, w, ids, logits = _inputs(40, 128, 2100, 12, seed=3)
    w = (w.float() * torch.linspace(0.1, 4.0, 2100)[:, None]).half()
    for weight in (w, w.flip(0)):
        _check(_run(h, weight, ids, logits, 1.0, v_chunk=chunk), h, weight, ids, logits, 1.0)


@pytest.mark.parametrize("logits_dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ids_dtype", [torch.int64, torch.int32])
def test_types_of_the_teacher(logits_dtype, ids_dtype):
    h, w, ids, logits = _inputs(20, 64, 900, 7, seed=5)
    x = logits.to(logits_dtype)
    _check(_run(h, w, ids.to(ids_dtype), x, 1.7), h, w, ids, x.float(), 1.7)


def test_entries_that_are_none_and_entries_that_come_twice():
    h, w, ids, logits = _inputs(6, 64, 500, 9, seed=6, missing=0.0)
    ids[0] = torch.tensor([3, 3, 7, 3, 7, 499, 0, 0, 12])
    ids[2, 4], ids[2, 5], ids[2, 6] = 500, 1 << 40, -(1 << 40)
    logits[3, 2], logits[3, 3] = -math.inf, -math.inf
    logits[4] = -math.inf
    ids[3, 4] = ids[3, 2]  # once without weight, once with
    _check(_run(h, w, ids, logits, 1.0), h, w, ids, logits, 1.0)


def test_a_student_that_has_learnt_its_teacher():
    """The teacher's logits are the student's own largest: the entries cancel but for the rest of the vocabulary."""
    n, d, v = 24, 128, 3000
    h, w, ids, _ = _inputs(n, d, v, 4, seed=7, h_scale=6.0, missing=0.0)
    z = h.double() @ w.double().t()
    logits, ids = z.topk(64, dim=1)
    logits = logits.float()
    _check(_run(h, w, ids, logits, 1.0), h, w, ids, logits, 1.0)


def test_num_items_evaluation_and_no_gradient():
    h, w, ids, logits = _inputs(50, 128, 1500, 6, seed=8)
    for num in (7, 123.0, torch.tensor(77)):
        _check(_run(h, w, ids, logits, 2.0, num_items_in_batch=num), h, w, ids, logits, 2.0, num=float(num))
    loss, kl, dh = _run(h, w, ids, logits, 2.0, need_grad=False)
    assert dh is None
    _check((loss, kl, None), h, w, ids, logits, 2.0)
    nothing = torch.full_like(ids, -1)
    loss, kl, dh = _run(h, w, nothing, logits)
    assert float(loss) == 0.0 and not bool(kl.any()) and not bool(dh.any())


@pytest.mark.parametrize("resident", [True, False])
def test_loss_over_a_host_head_and_its_gradient(resident):
    h, w, ids, logits = _inputs(60, 128, 1300, 10, seed=9)
    head = HostHead(w, DEV, v_chunk=512, resident=resident)
    x = h.to(DEV).view(3, 20, 128).requires_grad_()
    loss, kl = ops.chunked_distill_head(x, ids.to(DEV).view(3, 20, 10), logits.to(DEV).view(3, 20, 10), head, 2.0)
    (loss * 512.0).backward()
    want = ref.distill_head(h, w, ids, logits, 2.0)
    _, b = _bounds(h, w, ids, logits, 2.0, want)
    assert not kl.requires_grad
    err = (x.grad.double().cpu().view(60, 128) - 512.0 * want["dh"]).abs()
    tol = 512.0 * b + 2.0**-11 * 512.0 * want["dh"].abs() * 1.01 + 2.0**-25
    assert bool((err <= tol).all()), float((err / tol).max())
    with torch.no_grad():
        loss2, _ = ops.chunked_distill_head(x, ids.to(DEV), logits.to(DEV), head, 2.0)
    assert abs(float(loss2) - float(loss.detach())) <= 1e-5 * abs(float(loss.detach()))


@pytest.mark.parametrize("resident", [True, False])
@pytest.mark.parametrize("num", [None, 0, 7])
def test_no_tokens_and_no_teacher(resident, num):
    h, w, ids, logits = _inputs(9, 64, 700, 3, seed=14)
    ids[:] = -100
    head = HostHead(w, DEV, v_chunk=256, resident=resident)
    for n in (0, 9):
        x = h[:n].to(DEV).requires_grad_()
        loss, kl = ops.chunked_distill_head(x, ids[:n].to(DEV), logits[:n].to(DEV), head, 2.0, num)
        loss.backward()
        assert float(loss.detach()) == 0.0 and kl.shape == (n,) and not bool(kl.any())
        assert x.grad.shape == (n, 64) and not bool(x.grad.any())


def test_rows_of_wider_buffers_and_rows_that_are_not_addressable():
    h, w, ids, logits = _inputs(21, 128, 800, 6, seed=15)
    loss, kl, dh = _run(h, w, ids, logits, 1.5)
    for cols, first in ((160, 16), (131, 2)):
        hb, wb = (torch.full((x.shape[0], cols), math.nan, dtype=torch.float16) for x in (h, w))
        hb[:, first:first + 128], wb[:, first:first + 128] = h, w
        ib = torch.full((21, 11), -1)
        ib[:, 3:9] = ids
        got = K.lm_head_distill(hb.to(DEV)[:, first:first + 128], wb.to(DEV)[:, first:first + 128], ib.to(DEV)[:, 3:9],
                                logits.t().contiguous().to(DEV).t(), temperature=1.5)
        assert torch.equal(got[0], loss) and torch.equal(got[1], kl) and torch.equal(got[3], dh)


def test_gradient_against_differences():
    h, w, ids, logits = _inputs(7, 64, 400, 6, seed=10)
    _, _, dh = _run(h, w, ids, logits, 1.3)
    g = torch.Generator().manual_seed(11)
    e = torch.randn(7, 64, generator=g, dtype=torch.float64)
    f = lambda x: float(ref.distill_head(x, w, ids, logits, 1.3)["loss"])
    slope = (f(h.double() + 1e-5 * e) - f(h.double() - 1e-5 * e)) / 2e-5
    want = ref.distill_head(h, w, ids, logits, 1.3)
    _, b = _bounds(h, w, ids, logits, 1.3, want)
    tol = float((b * e.abs()).sum()) + 1e-6
    assert abs(float((dh.double().cpu() * 2.0**-16 * e).sum()) - slope) <= tol


def test_tokens_that_are_not_finite_stay_their_own():
    h, w, ids, logits = _inputs(40, 64, 700, 5, seed=12)
    clean = _run(h, w, ids, logits)
    bad = h.clone()
    bad[3, 2], bad[17, 1], bad[1, 0] = math.nan, math.inf, math.nan  # token 1 has no teacher
    loss, kl, dh = _run(bad, w, ids, logits)
    keep = torch.ones(40, dtype=torch.bool)
    keep[[3, 17]] = False
    assert torch.equal(kl.cpu()[keep], clean[1].cpu()[keep])
    assert torch.equal(dh.cpu()[keep], clean[2].cpu()[keep])
    assert bool(torch.isnan(kl.cpu()[~keep]).all()) and math.isnan(float(loss))


def test_refusals_of_the_device():
    h, w, ids, logits = (t.to(DEV) for t in _inputs(4, 64, 100, 3))
    with pytest.raises(RuntimeError, match="teacher_logits is frozen"):
        ops.chunked_distill_head(h, ids, logits.requires_grad_(), w)
    logits = logits.detach()
    with pytest.raises(RuntimeError, match="weight is frozen"):
        ops.chunked_distill_head(h, ids, logits, torch.nn.Parameter(w))
    x = h.clone().requires_grad_()
    loss, _ = ops.chunked_distill_head(x, ids, logits, w)
    (g,) = torch.autograd.grad(loss, x, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        g.sum().backward()
