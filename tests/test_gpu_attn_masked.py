"""GPU tests of attention with capped scores, a bias by distance, a prefix and rows of fewer queries than keys,
against the definition in float64 on the same inputs.

Bounds, per element, with u half a step of the type (fp16 2^-11, bf16 2^-8): P and dS are rounded once for their
products, P's sum is of the rounded values (u each), O is rounded once and read rounded by D = dO.O. Scores are sums
of d products in 32 bits (2^-24 a step; 2^-20 of the sum of absolute products covers d of them) and the cap's tanh is
good to 2^-22 of the largest score; such an error delta is a relative one of P. fp16 values below 2^-14 have an
absolute step of 2^-24.
"""

from __future__ import annotations

import ctypes
import math

import pytest
import torch

from oracle import ops as ref
from rus_amd import _lib
from rus_amd import kernels as K
from rus_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
U = {torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
TINY = {torch.float16: 2.0**-25, torch.bfloat16: 0.0}


def _cu(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def _inputs(ql, kl, hq, hkv, d, dtype, seed, q_scale=2.0, extra=0):
    g = torch.Generator().manual_seed(seed)
    nq, nk = sum(ql) + extra, sum(kl) + extra
    q = (torch.randn(nq, hq, d, generator=g) * q_scale).to(dtype)
    k, v = (torch.randn(nk, hkv, d, generator=g).to(dtype) for _ in range(2))
    return q, k, v, torch.randn(nq, hq, d, generator=g).to(dtype)


def _definition(q, k, v, dout, ql, kl, prefix=None, causal=True, softcap=0.0, slopes=None, scale=None):
    """float64 results and their bounds: {name: (value, bound)}."""
    u, tiny = U[q.dtype], TINY[q.dtype]
    hq, d = q.shape[1:]
    hkv = k.shape[1]
    grp, sc = hq // hkv, d**-0.5 if scale is None else scale
    z64 = lambda t: torch.zeros(t.shape, dtype=torch.float64)
    out, dq, dk, dv = z64(q), z64(q), z64(k), z64(v)
    bo, bq, bk, bv = z64(q), z64(q), z64(k), z64(v)
    lse = torch.full((hq, q.shape[0]), -math.inf, dtype=torch.float64)
    bl = torch.zeros(hq, q.shape[0], dtype=torch.float64)
    cq, ck = _cu(ql), _cu(kl)
    for s, (lq, lk) in enumerate(zip(ql, kl)):
        if lq == 0 or lk == 0:
            continue
        rq, rk = slice(cq[s], cq[s + 1]), slice(ck[s], ck[s + 1])
        for g in range(hkv):
            hs = slice(g * grp, (g + 1) * grp)
            qh, go = (t[rq, hs].transpose(0, 1).double() for t in (q, dout))
            kd, vd = k[rk, g].double(), v[rk, g].double()
            z, seen, f = ref.masked_scores(qh, kd, lq, lk, causal, 0 if prefix is None else prefix[s], softcap,
                                           None if slopes is None else slopes[hs], scale)
            any_seen = seen.any(1)
            z = z.masked_fill(~seen, -math.inf)
            lse[hs, rq] = torch.logsumexp(z, 2)
            p = torch.exp(z - torch.where(any_seen, lse[hs, rq], torch.zeros(()).double())[..., None])
            o = p @ vd
            dp = go @ vd.t()
            dsum = (go * o).sum(-1, keepdim=True)
            ds = p * (dp - dsum) * f
            out[rq, hs] = o.transpose(0, 1)
            dq[rq, hs] = sc * (ds @ kd).transpose(0, 1)
            dk[rk, g] = sc * (ds.transpose(1, 2) @ qh).sum(0)
            dv[rk, g] = (p.transpose(1, 2) @ go).sum(0)
            raw = sc * (qh.abs() @ kd.abs().t())
            delta = 2.0**-20 * raw + 2.0**-21 * z.masked_fill(~seen, 0.0).abs()
            delta = delta.masked_fill(~seen, 0.0)
            delta = 2.0 * delta.amax(-1, keepdim=True) + 2.0**-20  # numerator, and the sum below it
            bp = p * (2.0 * u + delta) + tiny * seen
            bo[rq, hs] = (bp @ vd.abs()).transpose(0, 1)
            bl[hs, rq] = (delta[..., 0] + 2.0**-22 * torch.where(any_seen, lse[hs, rq], torch.zeros(()).double()).abs())
            e_d = u * (go.abs() * o.abs()).sum(-1, keepdim=True) + (go.abs() * (bp @ vd.abs())).sum(-1, keepdim=True)
            e_p = 2.0**-20 * (go.abs() @ vd.abs().t())
            # the factor's own error: 1 - t^2 from t good to 2^-22
            eds = u * ds.abs() + p * f * (e_d + e_p) + delta * p * (dp.abs() + dsum.abs()) * (f + 2.0**-20) + tiny * seen
            bq[rq, hs] = sc * (eds @ kd.abs()).transpose(0, 1)
            bk[rk, g] = sc * (eds.transpose(1, 2) @ qh.abs()).sum(0)
            bv[rk, g] = (bp.transpose(1, 2) @ go.abs()).sum(0)
    return {"out": (out, bo), "lse": (lse, bl), "dq": (dq, bq), "dk": (dk, bk), "dv": (dv, bv)}


def _check(got, want, dtype):
    for name, x in got.items():
        value, bound = want[name]
        x = x.double().cpu()
        same = (x == value)  # infinities among them
        tol = bound * 1.01 + 1e-30
        if name != "lse":
            tol = tol + U[dtype] * (value.abs() + bound) + TINY[dtype]
        bad = ~(same | ((x - value).abs() <= tol))
        worst = ((x - value).abs() / tol).masked_fill(same, 0.0)
        assert not bool(bad.any()), (name, int(bad.sum()), float(worst.max()), bad.nonzero()[0].tolist())


def _ints(x):
    return None if x is None else torch.tensor(x, dtype=torch.int32, device=DEV)


def _run(q, k, v, dout, ql, kl, prefix=None, slopes=None, **kw):
    d = [t.to(DEV) for t in (q, k, v, dout)]
    args = dict(cu_k=_ints(_cu(kl)), prefix=_ints(prefix), slopes=None if slopes is None else slopes.to(DEV),
                max_q=max(max(ql), 0), max_k=max(kl), **kw)
    out, lse = K.attn_masked_fwd(*d[:3], _ints(_cu(ql)), **args)
    dq, dk, dv = K.attn_masked_bwd(d[3], *d[:3], out, lse, _ints(_cu(ql)), **args)
    torch.cuda.synchronize()
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _slopes(hq):
    return torch.exp2(-8.0 * (torch.arange(hq, dtype=torch.float32) + 1) / hq)


ROWS = {
    "one": ([1], [1]),
    "packed": ([33, 1, 64, 95, 7], [33, 1, 64, 95, 7]),
    "odd": ([129, 31, 200], [129, 31, 200]),
    "cache": ([1, 3, 1, 9], [300, 3, 1, 131]),
    "cache_long": ([1, 2], [1500, 777]),
    "suffix": ([40, 130], [170, 131]),
    "empty": ([0, 5, 12, 3, 0], [4, 0, 5, 3, 0]),  # rows without queries, without keys, with more queries than keys
    "few_keys": ([140, 33], [2, 1]),
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("rows", list(ROWS))
@pytest.mark.parametrize("form", ["causal", "prefix_cap", "bias", "full_cap_bias"])
def test_against_float64(dtype, d, rows, form):
    ql, kl = ROWS[rows]
    hq, hkv = (6, 1) if d == 128 else (4, 4)
    q, k, v, dout = _inputs(ql, kl, hq, hkv, d, dtype, seed=len(rows) + d)
    kw = {"causal": {}, "prefix_cap": dict(softcap=5.0, prefix=[(40 * s + 3) % 70 for s in range(len(ql))]),
          "bias": dict(slopes=_slopes(hq)), "full_cap_bias": dict(causal=False, softcap=30.0, slopes=-0.01 * _slopes(hq))}
    kw = kw[form]
    want = _definition(q, k, v, dout, ql, kl, **kw)
    _check(_run(q, k, v, dout, ql, kl, **kw), want, dtype)


@pytest.mark.parametrize("heads", [(1, 1), (12, 2), (14, 2), (8, 1), (3, 3), (20, 1)])
def test_head_layouts(heads):
    ql, kl = [70, 37, 1], [70, 40, 90]
    q, k, v, dout = _inputs(ql, kl, *heads, 128, torch.float16, seed=heads[0])
    want = _definition(q, k, v, dout, ql, kl, softcap=20.0)
    _check(_run(q, k, v, dout, ql, kl, softcap=20.0), want, torch.float16)


@pytest.mark.parametrize("softcap", [1e-2, 0.7, 1e4, 1e30])
@pytest.mark.parametrize("scale", [1e-3, 1.0])
def test_caps_far_from_the_scores(softcap, scale):
    """A cap far above the scores changes nothing and costs no accuracy; one far below flattens them."""
    ql = kl = [65, 20]
    q, k, v, dout = _inputs(ql, kl, 2, 1, 64, torch.float16, seed=3)
    kw = dict(softcap=softcap, scale=scale)
    _check(_run(q, k, v, dout, ql, kl, **kw), _definition(q, k, v, dout, ql, kl, **kw), torch.float16)


@pytest.mark.parametrize("prefix", [[-5, 1000], [0, 0], [200, 1], [64, 33]])
def test_prefixes_are_clamped(prefix):
    ql = kl = [200, 33]
    q, k, v, dout = _inputs(ql, kl, 2, 2, 64, torch.bfloat16, seed=5)
    got = _run(q, k, v, dout, ql, kl, prefix=prefix)
    want = _definition(q, k, v, dout, ql, kl, prefix=[min(max(p, 0), n) for p, n in zip(prefix, kl)])
    _check(got, want, torch.bfloat16)


def test_tokens_behind_the_rows_get_zeros():
    ql = kl = [33, 20]
    q, k, v, dout = _inputs(ql, kl, 4, 2, 128, torch.float16, seed=6, extra=150)
    q[53:], k[53:], v[53:], dout[53:] = math.nan, math.nan, math.nan, math.nan  # what padding may hold
    got = _run(q, k, v, dout, ql, kl)
    for name in ("out", "dq", "dk", "dv"):
        assert not bool(got[name][53:].any()), name
    assert bool((got["lse"][:, 53:] == -math.inf).all())
    cut = {n: (t[:, :53] if n == "lse" else t[:53]) for n, t in got.items()}
    _check(cut, _definition(q[:53], k[:53], v[:53], dout[:53], ql, kl), torch.float16)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("rows", [([100, 40], [100, 40]), ([1, 3], [300, 61])])
def test_hidden_elements_do_not_get_through(bad, where, rows):
    """Token 70 of the first row (or its last query) and the last token of the second are not finite: who does not see
    them (or is not seen) has the results that it has without them."""
    ql, kl = rows
    t = dict(zip(("q", "k", "v", "dout"), _inputs(ql, kl, 4, 2, 64, torch.float16, seed=8)))
    clean = _run(*t.values(), ql, kl, softcap=10.0)
    x = t[where].clone()
    queries = where in ("q", "dout")
    spots = [min(70, (ql if queries else kl)[0] - 1), len(x) - 1]
    for s in spots:
        x[s, :, 5] = bad
    t[where] = x
    got = _run(*t.values(), ql, kl, softcap=10.0)
    cq, ck = _cu(ql), _cu(kl)
    touched_q, touched_k = torch.zeros(cq[-1], dtype=torch.bool), torch.zeros(ck[-1], dtype=torch.bool)
    for s, (lq, lk) in enumerate(zip(ql, kl)):
        vis = torch.arange(lk)[None, :] <= torch.arange(lk - lq, lk)[:, None]
        if queries:
            hit = torch.tensor([cq[s] + i in spots for i in range(lq)])
            touched_q[cq[s]:cq[s + 1]] |= hit
            touched_k[ck[s]:ck[s + 1]] |= (vis & hit[:, None]).any(0)
        else:
            hit = torch.tensor([ck[s] + i in spots for i in range(lk)])
            saw = (vis & hit[None, :]).any(1)
            touched_q[cq[s]:cq[s + 1]] |= saw
            touched_k[ck[s]:ck[s + 1]] |= (vis & saw[:, None]).any(0)
    for name in ("out", "dq"):
        if where == "dout" and name == "out":
            touched = torch.zeros_like(touched_q)
        else:
            touched = touched_q
        a, b = got[name].cpu()[~touched], clean[name].cpu()[~touched]
        assert torch.isfinite(a).all() and torch.allclose(a.float(), b.float(), rtol=2e-3, atol=2e-3), name
    for name in ("dk", "dv"):
        a, b = got[name].cpu()[~touched_k], clean[name].cpu()[~touched_k]
        assert torch.isfinite(a).all() and torch.allclose(a.float(), b.float(), rtol=4e-3, atol=4e-3), name
    if where == "v":  # and who sees them is told
        assert bool(torch.isnan(got["out"].cpu()[touched_q]).any() | torch.isinf(got["out"].cpu()[touched_q]).any())


def test_views_of_a_fused_projection_and_expanded_gradients():
    ql = kl = [100, 29]
    g = torch.Generator().manual_seed(9)
    fused = torch.randn(129, 12 + 4, 128, generator=g).half()
    q, k, v = fused[:, :12], fused[:, 12:14], fused[:, 14:]
    dout = torch.randn(1, 1, 128, generator=g).half().expand(129, 12, 128)
    f = fused.to(DEV)
    args = dict(max_q=100, max_k=100, softcap=15.0)
    cu = _ints(_cu(ql))
    views = f[:, :12], f[:, 12:14], f[:, 14:]
    out, lse = K.attn_masked_fwd(*views, cu, **args)
    grads = K.attn_masked_bwd(dout[:1, :1].to(DEV).expand(129, 12, 128), *views, out, lse, cu, **args)
    got = dict(zip(("out", "lse", "dq", "dk", "dv"), (out, lse, *grads)))
    _check(got, _definition(q, k, v, dout, ql, kl, softcap=15.0), torch.float16)
    # strides that the kernels do not address are laid out first
    odd = [torch.empty(t.shape[0], t.shape[1], 131, dtype=t.dtype, device=DEV)[..., 1:129].copy_(t.to(DEV)) for t in (q, k, v)]
    out2, lse2 = K.attn_masked_fwd(*odd, cu, **args)
    assert torch.equal(out, out2) and torch.equal(lse, lse2)


def test_operands_that_look_contiguous_but_are_not_addressable():
    """One token whose token stride is odd, and tensors that start 2 bytes behind an aligned address."""
    q, k, v, dout = (x.to(DEV) for x in _inputs([1], [1], 4, 2, 64, torch.bfloat16, seed=31))
    cu = _ints([0, 1])

    def odd(x):
        rows = torch.empty(3, x.shape[1] * 64 + 3, dtype=x.dtype, device=DEV)
        view = rows[1:2, : x.shape[1] * 64].unflatten(1, x.shape[1:])
        return view.copy_(x)

    def shifted(x):
        return torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)[1:].view(x.shape).copy_(x)

    out, lse = K.attn_masked_fwd(q, k, v, cu)
    grads = K.attn_masked_bwd(dout, q, k, v, out, lse, cu)
    for f in (odd, shifted):
        assert f(q).is_contiguous()
        got, _ = K.attn_masked_fwd(f(q), f(k), f(v), cu)
        assert torch.equal(got, out), f.__name__
        for a, b in zip(K.attn_masked_bwd(f(dout), f(q), f(k), f(v), out, lse, cu), grads):
            assert torch.equal(a, b), f.__name__


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("ql", [[1], [1, 1, 40, 1], [1] * 70 + [700] * 12], ids=["one", "few", "blocks_of_128"])
def test_a_single_key_has_no_score_gradient(dtype, ql):
    """The P of a query that sees one key is 1 whatever the score: its dq, and what it adds to dk, are 0."""
    q, k, v, dout = _inputs(ql, ql, 8, 4, 64, dtype, seed=33)
    for kw in ({}, dict(softcap=5.0, slopes=_slopes(8))):
        got = _run(q, k, v, dout, ql, ql, **kw)
        starts = torch.tensor(_cu(ql)[:-1])
        alone = starts[torch.tensor(ql) == 1]
        assert not bool(got["dq"].cpu()[starts].any())
        assert not bool(got["dk"].cpu()[alone].any())


def test_gradients_against_differences():
    """(f(x + h e) - f(x - h e)) / 2 h of the definition in float64 along random directions, with the operator's
    gradients from the same inputs."""
    ql, kl = [37, 5], [37, 20]
    q, k, v, dout = _inputs(ql, kl, 4, 2, 64, torch.float16, seed=11)
    kw = dict(softcap=6.0, prefix=[9, 0], slopes=_slopes(4))
    got = _run(q, k, v, dout, ql, kl, **kw)
    want = _definition(q, k, v, dout, ql, kl, **kw)
    g = torch.Generator().manual_seed(12)

    def loss(q, k, v):
        total = 0.0
        cq, ck = _cu(ql), _cu(kl)
        for s, (lq, lk) in enumerate(zip(ql, kl)):
            for h in range(4):
                z, seen, _ = ref.masked_scores(q[cq[s]:cq[s + 1], h][None], k[ck[s]:ck[s + 1], h // 2], lq, lk, True,
                                               kw["prefix"][s], 6.0, kw["slopes"][h:h + 1])
                p = torch.softmax(z.masked_fill(~seen, -math.inf), -1)
                total = total + (p[0] @ v[ck[s]:ck[s + 1], h // 2] * dout[cq[s]:cq[s + 1], h].double()).sum()
        return total

    base = [t.double() for t in (q, k, v)]
    for i, name in enumerate(("dq", "dk", "dv")):
        e = torch.randn(base[i].shape, generator=g, dtype=torch.float64)
        up, down = list(base), list(base)
        up[i], down[i] = base[i] + 1e-4 * e, base[i] - 1e-4 * e
        slope = (loss(*up) - loss(*down)) / 2e-4
        # the bound of each element carried through the direction, and the difference's own 1e-8 x third derivative
        tol = float(((want[name][1] + U[torch.float16] * want[name][0].abs()) * e.abs()).sum()) + 1e-4
        assert abs(float((got[name].double().cpu() * e).sum()) - float(slope)) <= tol, name


def test_autograd_and_refusals():
    ql = [20, 13]
    q, k, v, dout = (t.to(DEV) for t in _inputs(ql, ql, 4, 2, 64, torch.bfloat16, seed=13))
    cu = _ints(_cu(ql))
    leaves = [t.clone().requires_grad_() for t in (q, k, v)]
    out = ops.masked_attention(*leaves, cu, softcap=9.0)
    out.backward(dout, retain_graph=True)
    o, lse = K.attn_masked_fwd(q, k, v, cu, softcap=9.0)
    want = K.attn_masked_bwd(dout, q, k, v, o, lse, cu, softcap=9.0)
    assert torch.equal(out, o)
    for leaf, w in zip(leaves, want):
        assert torch.equal(leaf.grad, w)
    grads = torch.autograd.grad(out, leaves, dout, create_graph=True)
    with pytest.raises(RuntimeError, match="no second derivative"):
        grads[0].sum().backward()
    with pytest.raises(RuntimeError, match="slopes is frozen"):
        ops.masked_attention(*leaves, cu, slopes=torch.ones(4, device=DEV, requires_grad=True))


def test_long_cache_offsets_past_32_bits():
    """Keys whose bytes lie beyond 2^32 (and elements beyond 2^31): the last rows of a large cache."""
    n, d = (1 << 24) + 77, 128  # 2^31 + elements, 4 GiB a tensor
    g = torch.Generator(device=DEV).manual_seed(14)
    k, v = (torch.zeros(n, 1, d, dtype=torch.float16, device=DEV) for _ in range(2))
    lk = 333
    k[n - lk:] = torch.randn(lk, 1, d, generator=g, device=DEV).half()
    v[n - lk:] = torch.randn(lk, 1, d, generator=g, device=DEV).half()
    q = torch.randn(4, 6, d, generator=g, device=DEV).half()
    dout = torch.randn(4, 6, d, generator=g, device=DEV).half()
    cu_q, cu_k = _ints([0, 0, 4]), _ints([0, n - lk, n])
    out, lse = K.attn_masked_fwd(q, k, v, cu_q, cu_k, max_q=4, max_k=n - lk)
    torch.cuda.synchronize()
    want = _definition(q.cpu(), k[n - lk:].cpu(), v[n - lk:].cpu(), dout.cpu(), [4], [lk])
    _check({"out": out, "lse": lse}, want, torch.float16)


def _plan(ql, kl, hq, hkv, d):
    got = (ctypes.c_int32 * 3)()
    _lib.call("rus_attn_masked_plan", len(ql), sum(ql), sum(kl), max(ql), max(kl), hq, hkv, d, got)
    return tuple(got)


_LONG = [33, 255, 64, 200, 190, 129, 256, 90, 255, 161, 128, 97, 200]
_ODD = [161] * 3 + [255, 97, 3, 128, 127, 200, 90, 1]
# (rows of queries, of keys, heads, plan: parts (0: blocks of 128 queries), backward block)
LAYOUTS = {
    "blocks_of_128": (_LONG, _LONG, 24, 4, 0, 128),
    "blocks_of_128_few_queries": ([20, 1, 64, 131, 7, 129, 100, 90, 255, 161, 128, 97, 200], _LONG, 24, 4, 0, 128),
    "blocks_of_128_odd_ends": (_ODD, _ODD, 28, 2, 0, 128),
    "few_queries_one_part": ([300, 150], [300, 150], 6, 2, 1, 32),
    "few_queries_many_parts": ([1, 2, 3], [900, 1500, 64], 6, 2, None, 32),
    "one_head_per_kv": ([257, 64, 130], [257, 64, 130], 8, 8, 1, 32),
    "many_rows": ([3] * 90 + [40], [3] * 45 + [70] * 45 + [40], 4, 2, None, 128),  # more rows than a wave has lanes
}


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16], ids=["fp16", "bf16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("layout", list(LAYOUTS))
@pytest.mark.parametrize("form", ["causal", "prefix_cap", "prefix_bias", "full_cap_bias"])
def test_layouts_against_float64(dtype, d, layout, form):
    ql, kl, hq, hkv, parts, block = LAYOUTS[layout]
    got_plan = _plan(ql, kl, hq, hkv, d)
    assert (got_plan[0] > 1 if layout == "few_queries_many_parts" else parts is None or got_plan[0] == parts), got_plan
    assert got_plan[2] == block, got_plan
    q, k, v, dout = _inputs(ql, kl, hq, hkv, d, dtype, seed=d + len(layout))
    prefix = [(50 * s + 3) % 150 for s in range(len(ql))]
    kw = {"causal": {}, "prefix_cap": dict(softcap=5.0, prefix=prefix), "prefix_bias": dict(slopes=_slopes(hq), prefix=prefix),
          "full_cap_bias": dict(causal=False, softcap=30.0, slopes=-0.01 * _slopes(hq))}[form]
    _check(_run(q, k, v, dout, ql, kl, **kw), _definition(q, k, v, dout, ql, kl, **kw), dtype)


@pytest.mark.parametrize("where", ["q", "k", "v", "dout"])
@pytest.mark.parametrize("layout", ["blocks_of_128", "few_queries_many_parts", "one_head_per_kv"])
def test_hidden_elements_in_every_layout(where, layout):
    """The last token of each row is not finite: of it, every other query (and what only those see) knows nothing."""
    ql, kl, hq, hkv, *_ = LAYOUTS[layout]
    t = dict(zip(("q", "k", "v", "dout"), _inputs(ql, kl, hq, hkv, 128, torch.float16, seed=21)))
    kw = dict(slopes=_slopes(hq))
    clean = _run(*t.values(), ql, kl, **kw)
    cq, ck = _cu(ql), _cu(kl)
    x = t[where].clone()
    for e in (cq if where in ("q", "dout") else ck)[1:]:
        x[e - 1, :, 7] = math.nan
    t[where] = x
    got = _run(*t.values(), ql, kl, **kw)
    last_q = torch.tensor([e - 1 for e in cq[1:]])
    keep = torch.ones(cq[-1], dtype=torch.bool)
    keep[last_q] = False
    for name in ("out", "dq"):
        a, b = got[name].cpu()[keep], clean[name].cpu()[keep]
        assert torch.isfinite(a).all() and torch.allclose(a.float(), b.float(), rtol=4e-3, atol=4e-3), name
        if name == "dq" or where != "dout":
            assert torch.isnan(got[name].cpu()[last_q]).flatten(1).any(1).all(), name
    if where != "dout":  # every key of a row is seen by its last query, whose P is no number (v: dS is not, P is)
        assert torch.isnan(got["dk"].cpu()).any()
    else:
        seen = got["dv"].cpu()[..., 7]
        assert torch.isnan(seen).all() and torch.isfinite(got["dv"].cpu()[..., :7]).all()


def test_a_captured_step_beside_eager_work():
    """Forward and backward in one graph, replayed with other inputs, eager calls and another stream's between: every
    replay has the eager call's bits."""
    ql, kl = [70, 33], [90, 33]
    cu_q, cu_k = _ints(_cu(ql)), _ints(_cu(kl))
    args = dict(cu_k=cu_k, max_q=70, max_k=90, softcap=9.0)
    sets = [[t.to(DEV) for t in _inputs(ql, kl, 6, 2, 128, torch.float16, seed=s)] for s in range(4)]
    static = [t.clone() for t in sets[0]]

    def step(q, k, v, do):
        out, lse = K.attn_masked_fwd(q, k, v, cu_q, **args)
        return out, lse, *K.attn_masked_bwd(do, q, k, v, out, lse, cu_q, **args)

    step(*static)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step(*static)
    other = torch.cuda.Stream()
    for rep in range(6):
        data = sets[rep % 4]
        want = step(*data)
        for s, t in zip(static, data):
            s.copy_(t)
        graph.replay()
        other.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(other):
            beside = step(*sets[(rep + 1) % 4])
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), rep
        assert all(torch.equal(a, b) for a, b in zip(beside, step(*sets[(rep + 1) % 4]))), rep


def test_parts_are_joined_alike_on_two_streams_at_once():
    q, k, v, _ = (t.to(DEV) for t in _inputs([1] * 4, [5000, 70, 3000, 1], 12, 2, 128, torch.bfloat16, seed=30))
    cu_q, cu_k = _ints(range(5)), _ints(_cu([5000, 70, 3000, 1]))
    call = lambda: K.attn_masked_fwd(q, k, v, cu_q, cu_k, max_q=1, max_k=5000)
    want = call()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for _ in range(5):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(call())
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for g in got for a, b in zip(g, want))


def test_malformed_rows_stay_inside_the_arrays():
    """Starts out of order or range are clamped: nothing is read or written outside (results of such rows say nothing)."""
    q, k, v, dout = (t.to(DEV) for t in _inputs([64], [64], 4, 2, 64, torch.float16, seed=31))
    for cu in ([0, 100, 64], [-5, 30, 64], [60, 10, 64], [64, 64, 0], [2**31 - 1, -(2**31), 7]):
        cu = _ints(cu)
        out, lse = K.attn_masked_fwd(q, k, v, cu, softcap=3.0)
        K.attn_masked_bwd(dout, q, k, v, out, lse, cu, softcap=3.0)
        torch.cuda.synchronize()


def test_other_longest_rows_cost_time_only():
    ql, kl = [5, 40], [700, 40]
    q, k, v, dout = _inputs(ql, kl, 4, 2, 64, torch.float16, seed=32)
    want = _definition(q, k, v, dout, ql, kl)
    d = [t.to(DEV) for t in (q, k, v)]
    for max_q, max_k in ((0, 0), (1, 1), (45, 740), (10000, 1 << 30), (None, None)):
        out, lse = K.attn_masked_fwd(*d, _ints(_cu(ql)), _ints(_cu(kl)), max_q=max_q, max_k=max_k)
        _check({"out": out, "lse": lse}, want, torch.float16)


def test_no_queries_or_no_keys():
    z = lambda n, h: torch.zeros(n, h, 64, dtype=torch.float16, device=DEV)
    cu0, cu4 = _ints([0, 0]), _ints([0, 4])
    out, lse = K.attn_masked_fwd(z(0, 4), z(4, 2), z(4, 2), cu0, cu4)
    assert out.shape == (0, 4, 64)
    dq, dk, dv = K.attn_masked_bwd(out, z(0, 4), z(4, 2), z(4, 2), out, lse, cu0, cu4)
    assert not bool(dk.any()) and not bool(dv.any())
    q = z(4, 4) + 1
    out, lse = K.attn_masked_fwd(q, z(0, 2), z(0, 2), cu4, cu0)
    assert not bool(out.any()) and bool((lse == -math.inf).all())
    dq, dk, dv = K.attn_masked_bwd(q, q, z(0, 2), z(0, 2), out, lse, cu4, cu0)
    assert not bool(dq.any()) and dk.shape == (0, 2, 64)
