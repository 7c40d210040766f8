"""A student's training step as its operators are used together: q, k and v of one projection, rotary positions of
three axes, attention over packed rows that begin with an image, the output projection, and the distillation loss over
the lm_head; gradients of every weight against float64 autograd of the definitions.

Bounds: each 16-bit tensor on the way is rounded once (2^-11 relative to its rows), some eight of them between a weight
and the loss and as many back; errors of different roundings add at most linearly, so the 2-norm of a gradient is within
32 x 2^-11 = 1.6% of its own. The loss is a mean of differences of fp32 logits: 16 x 2^-11 of the logits' spread.
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
HQ, HKV, D, HID, V = 6, 2, 64, 256, 900
ROWS, PREFIX = [61, 20, 40], [25, 0, 9]
N = sum(ROWS)


def _data(seed=0):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, scale=1.0: (torch.randn(*s, generator=g) * scale).half()
    x = r(N, HID)
    w_qkv, w_o = r((HQ + 2 * HKV) * D, HID, scale=HID**-0.5), r(HID, HQ * D, scale=2 * (HQ * D) ** -0.5)
    head = r(V, HID, scale=0.1)
    pos = torch.stack([torch.randint(0, n, (N,), generator=g) for n in (40, 16, 16)])
    ids = torch.stack([torch.randperm(V, generator=g)[:8] for _ in range(N)])
    ids[:30] = -1  # the image and the prompt have no teacher
    logits = 8.0 - torch.cumsum(torch.rand(N, 8, generator=g) * 2, 1)
    return x, w_qkv, w_o, head, pos, ids, logits


def _cu():
    cu = [0]
    for n in ROWS:
        cu.append(cu[-1] + n)
    return cu


def _definition(x, w_qkv, w_o, head, pos, ids, logits, axes):
    a, b = w_qkv.double().requires_grad_(), w_o.double().requires_grad_()
    freq = (axes.turns.cpu() * (2 * math.pi)).tolist()
    qkv = (x.double() @ a.t()).view(N, HQ + 2 * HKV, D)
    p = len(freq)
    ang = pos.double()[axes.axis.cpu().long()].t() * torch.tensor(freq, dtype=torch.float64)
    c, s = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    turn = lambda t: torch.cat([t[..., :p] * c - t[..., p:2 * p] * s, t[..., p:2 * p] * c + t[..., :p] * s, t[..., 2 * p:]], -1)
    q, k, v = turn(qkv[:, :HQ]), turn(qkv[:, HQ:HQ + HKV]), qkv[:, HQ + HKV:]
    out = []
    cu = _cu()
    for i, n in enumerate(ROWS):
        rows = slice(cu[i], cu[i + 1])
        heads = []
        for h in range(HQ):
            z = 20.0 * torch.tanh(q[rows, h] @ k[rows, h // 3].t() * D**-0.5 / 20.0)
            j = torch.arange(n)
            seen = (j[None] <= j[:, None]) | (j[None] < PREFIX[i])
            heads.append(torch.softmax(z.masked_fill(~seen, -math.inf), -1) @ v[rows, h // 3])
        out.append(torch.stack(heads, 1))
    h = torch.cat(out).reshape(N, HQ * D) @ b.t() + x.double()
    t = 2.0
    log_p = torch.log_softmax(h @ head.double().t() / t, 1)
    on = (ids >= 0).any(1)
    q_t = torch.softmax(logits.double() / t, 1)
    kl = (q_t * (torch.log(q_t) - log_p.gather(1, ids.clamp(min=0)))).sum(1)[on]
    loss = t * t * kl.mean()
    return loss.detach(), *torch.autograd.grad(loss, (a, b))


def _step(x, w_qkv, w_o, head, pos, ids, logits, axes, cu, prefix):
    qkv = (x @ w_qkv.t()).view(N, HQ + 2 * HKV, D)
    q, k = ops.rope_axes(qkv[:, :HQ], qkv[:, HQ:HQ + HKV], pos, axes)
    out = ops.masked_attention(q, k, qkv[:, HQ + HKV:], cu, prefix=prefix, softcap=20.0, max_q=61, max_k=61)
    h = out.reshape(N, HQ * D) @ w_o.t() + x
    return ops.chunked_distill_head(h, ids, logits, head, 2.0)


def _setup(seed=0):
    data = _data(seed)
    axes = K.RopeAxes.sections((8, 12, 10), 1e4, D, DEV)
    dev = [t.to(DEV) for t in data]
    head = HostHead(data[3], DEV)
    cu = torch.tensor(_cu(), dtype=torch.int32, device=DEV)
    prefix = torch.tensor(PREFIX, dtype=torch.int32, device=DEV)
    return data, axes, dev, head, cu, prefix


def test_step_against_float64():
    data, axes, dev, head, cu, prefix = _setup()
    x, w_qkv, w_o, _, pos, ids, logits = dev
    w_qkv.requires_grad_(), w_o.requires_grad_()
    loss, kl = _step(x, w_qkv, w_o, head, pos, ids, logits, axes, cu, prefix)
    (loss * 256.0).backward()
    want, dw_qkv, dw_o = _definition(*data, axes)
    assert kl.shape == (N,) and not bool(kl[:30].any())
    assert abs(float(loss.detach()) - float(want)) <= 16 * 2.0**-11 * max(1.0, float(want))
    for got, exact in ((w_qkv.grad, dw_qkv), (w_o.grad, dw_o)):
        rel = float((got.double().cpu() / 256.0 - exact).norm() / exact.norm())
        assert rel <= 32 * 2.0**-11, rel


def test_step_with_its_backward_in_a_graph():
    """The whole step captured once and replayed on other data between eager steps: the eager step's bits."""
    _, axes, dev, head, cu, prefix = _setup()
    sets = [[t.to(DEV) for t in _data(s)] for s in range(3)]
    static = [t.clone() for t in dev]

    def step(t):
        x, w_qkv, w_o, _, pos, ids, logits = t
        w_qkv, w_o = w_qkv.detach().requires_grad_(), w_o.detach().requires_grad_()
        loss, kl = _step(x, w_qkv, w_o, head, pos, ids, logits, axes, cu, prefix)
        return loss.detach(), kl, *torch.autograd.grad(loss * 256.0, (w_qkv, w_o))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step(static)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(static)
    for rep in range(6):
        data = sets[rep % 3]
        want = step(data)
        for i in (0, 1, 2, 4, 5, 6):
            static[i].copy_(data[i])
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b), rep


@pytest.mark.parametrize("which", ["rope", "attention", "distill"])
def test_capture_beside_an_eager_graph_is_refused(which):
    """An eager graph of the same leaf, recorded on another stream and still alive: capturing would end the process."""
    _, axes, dev, head, cu, prefix = _setup()
    g = torch.Generator(device=DEV).manual_seed(1)
    leaf = torch.randn(N, HQ, D, generator=g, device=DEV).half().requires_grad_()
    kv = torch.randn(N, HKV, D, generator=g, device=DEV).half()
    hid = torch.randn(N, HID, generator=g, device=DEV).half().requires_grad_()
    call = {"rope": lambda: ops.rope_axes(leaf, None, dev[4], axes),
            "attention": lambda: ops.masked_attention(leaf, kv, kv, cu),
            "distill": lambda: ops.chunked_distill_head(hid, dev[5], dev[6], head)}[which]
    alive = call()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="drop that graph's outputs before capturing"):
        with torch.cuda.graph(graph):
            call()
    del alive, graph
    torch.cuda.synchronize()
    call()


def test_single_tokens_continue_a_row():
    """A row's last tokens one at a time over its cache: what the whole row gives there."""
    _, axes, dev, *_ = _setup()
    g = torch.Generator(device=DEV).manual_seed(2)
    qkv = torch.randn(70, HQ + 2 * HKV, D, generator=g, device=DEV).half()
    pos = torch.arange(70, device=DEV).expand(3, 70).contiguous()
    q, k = K.rope_axes_fwd(qkv[:, :HQ], qkv[:, HQ:HQ + HKV], pos, axes)
    v = qkv[:, HQ + HKV:]
    cu = torch.tensor([0, 70], dtype=torch.int32, device=DEV)
    whole, _ = K.attn_masked_fwd(q, k, v, cu, softcap=20.0)
    cache_k, cache_v = torch.zeros(70, HKV, D, dtype=torch.float16, device=DEV), torch.zeros(70, HKV, D, dtype=torch.float16, device=DEV)
    cache_k[:64], cache_v[:64] = k[:64], v[:64]
    one = torch.tensor([0, 1], dtype=torch.int32, device=DEV)
    for t in range(64, 70):
        qt, kt = K.rope_axes_fwd(qkv[t:t + 1, :HQ], qkv[t:t + 1, HQ:HQ + HKV], pos[:, t:t + 1], axes)
        assert torch.equal(qt[0], q[t]) and torch.equal(kt[0], k[t])
        cache_k[t], cache_v[t] = kt[0], v[t]
        # rows of the cache behind the sequence are not read
        out, _ = K.attn_masked_fwd(qt, cache_k, cache_v, one, torch.tensor([0, t + 1], dtype=torch.int32, device=DEV),
                                   softcap=20.0, max_q=1, max_k=t + 1)
        # P is rounded once against another reference: 2 x 2^-11 of sum P |v|, and the result's rounding
        tol = 3 * 2.0**-11 * float(v[:t + 1].abs().max())
        assert float((out[0].float() - whole[t].float()).abs().max()) <= tol
