"""Performance cases of the operators for rows that begin with image or video tokens and for a teacher's logits.

Widths are those of the repository's training configuration (hidden 1536, 12 query and 2 key/value heads of 128,
vocabulary 151936); token counts run from a decoding step (one token) to long packed batches, odd sizes between.

Kinds of case:
  rope     rotary positions with several axes: q and k rotated, in training their gradients rotated back
           (``kernels.rope_axes_fwd``, ``rope_axes_bwd``)
  attn     attention over packed rows with a tanh cap on the scores, a bias by distance, a prefix that every
           query of the row sees, and fewer queries than keys where a cache is read
           (``kernels.attn_masked_fwd``, ``attn_masked_bwd``)
  distill  KL divergence from a teacher's top logits over the lm_head, with the hidden gradient
           (``kernels.lm_head_distill``)
"""

import math

import torch

own = False

HIDDEN, VOCAB, THETA = 1536, 151936, 1e6
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
GRAD_SCALE = 1024.0  # the loss scale an fp16 gradient of a mean over tokens needs


def listed():
    return [
        # eight sequences decode one token each
        {"name": "rope_8", "kind": "rope", "n": 8, "hq": 12, "hk": 2, "d": 128, "sections": "16,24,24",
         "restart": False, "adjacent": False, "far": 32768, "dtype": "float16", "train": False},
        # the default batch in training, time / height / width sections
        {"name": "rope_707", "kind": "rope", "n": 707, "hq": 12, "hk": 2, "d": 128, "sections": "16,24,24",
         "restart": False, "adjacent": False, "far": 2048, "dtype": "bfloat16", "train": True},
        # a vision tower's patches: rows and columns, each axis with frequencies of its own, pairs side by side
        {"name": "rope_patches_4097", "kind": "rope", "n": 4097, "hq": 16, "hk": 16, "d": 64, "sections": "16,16",
         "restart": True, "adjacent": True, "far": 64, "dtype": "float32", "train": True},
        # a batch of long rows at far positions: bandwidth
        {"name": "rope_16381", "kind": "rope", "n": 16381, "hq": 12, "hk": 2, "d": 128, "sections": "16,24,24",
         "restart": False, "adjacent": False, "far": 1000000, "dtype": "float16", "train": True},
        # one new token for each of eight sequences, ragged caches, capped scores
        {"name": "attn_tokens_8", "kind": "attn", "q": "1,1,1,1,1,1,1,1", "k": "8191,4096,2048,707,129,64,17,1",
         "hq": 12, "hkv": 2, "d": 128, "causal": True, "prefix": 0, "cap": 50.0, "bias": False,
         "dtype": "float16", "train": False},
        # one new token over a very long cache: the cache's bytes
        {"name": "attn_token_long", "kind": "attn", "q": "1", "k": "131071", "hq": 12, "hkv": 2, "d": 128,
         "causal": True, "prefix": 0, "cap": 0.0, "bias": True, "dtype": "bfloat16", "train": False},
        # the default batch in training: rows that begin with an image, capped scores
        {"name": "attn_707", "kind": "attn", "q": "377,207,64,42,16,1", "k": "377,207,64,42,16,1", "hq": 12, "hkv": 2,
         "d": 128, "causal": True, "prefix": 64, "cap": 50.0, "bias": False, "dtype": "float16", "train": True},
        # long rows in training: an image prefix and a bias by distance
        {"name": "attn_8161", "kind": "attn", "q": "4096,2048,1024,993", "k": "4096,2048,1024,993", "hq": 12,
         "hkv": 2, "d": 128, "causal": True, "prefix": 257, "cap": 0.0, "bias": True, "dtype": "bfloat16",
         "train": True},
        # a vision tower: every patch of an image sees every other, heads of 64, a cap
        {"name": "attn_patches_1923", "kind": "attn", "q": "1025,577,257,64", "k": "1025,577,257,64", "hq": 16,
         "hkv": 16, "d": 64, "causal": False, "prefix": 0, "cap": 30.0, "bias": False, "dtype": "float16",
         "train": True},
        # a short batch with few teacher logits
        {"name": "distill_64", "kind": "distill", "n": 64, "d": HIDDEN, "v": VOCAB, "k": 8, "t": 1.0,
         "masked": 0.0, "ragged": False},
        # the default batch: prompt tokens without a teacher, entries missing here and there
        {"name": "distill_707", "kind": "distill", "n": 707, "d": HIDDEN, "v": VOCAB, "k": 32, "t": 2.0,
         "masked": 0.3, "ragged": True},
        # the rotary table's length, a broad teacher
        {"name": "distill_2048", "kind": "distill", "n": 2048, "d": HIDDEN, "v": VOCAB, "k": 64, "t": 1.0,
         "masked": 0.0, "ragged": False},
    ]


def _cost(case):
    w = work(case)
    return w["bytes"] / 5e12 + w["flops"] / 1e15


def _lens(text):
    return [int(x) for x in text.split(",")]


def draw(rng):
    def spread(lo, hi):  # over the logarithm of the range, odd values among them
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(("rope", "attn", "attn", "attn", "distill"))
    case = {"kind": kind}
    largest = max(_cost(c) for c in listed() if c["kind"] == kind)
    if kind == "rope":
        d = rng.choice((64, 80, 128, 256))
        pairs = d // 2 if rng.random() < 0.7 else d // 4
        first = rng.randint(1, pairs - 2)
        if rng.random() < 0.6:
            second = rng.randint(1, pairs - first - 1)
            sections = (first, second, pairs - first - second)
        else:
            sections = (first, pairs - first)
        hk = rng.choice((1, 2, 4, 8))
        case.update(n=spread(1, 16381), hq=hk * rng.choice((1, 2, 6)), hk=hk, d=d,
                    sections=",".join(map(str, sections)), restart=rng.random() < 0.4,
                    adjacent=rng.random() < 0.4, far=spread(64, 1000000),
                    dtype=rng.choice(("float16", "bfloat16", "float32")), train=rng.random() < 0.7)
        while _cost(case) > largest:
            case["n"] = max(1, case["n"] // 2)
        return case
    if kind == "distill":
        case.update(n=spread(1, 2048), d=64 * rng.randint(2, 32), v=spread(1000, VOCAB), k=spread(1, 128),
                    t=round(rng.uniform(0.5, 4.0), 2), masked=rng.choice((0.0, 0.3)), ragged=rng.random() < 0.5)
        while _cost(case) > largest:
            case["n"] = max(1, case["n"] // 2)
        return case
    hkv = rng.choice((1, 2, 4, 8))
    case.update(hq=hkv * rng.choice((1, 2, 6, 7)), hkv=hkv, d=rng.choice((64, 128, 128)))
    tokens = rng.random() < 0.35  # few queries over longer caches
    rows = spread(1, 16)
    if tokens:
        top = spread(64, 65536 // rows)
        q = [rng.choice((1, 1, 1, rng.randint(1, 9))) for _ in range(rows)]
        k = [spread(n, max(n, top)) for n in q]
    else:
        q = [spread(1, 4096) for _ in range(rows)]
        k = list(q)
    case.update(q=",".join(map(str, q)), k=",".join(map(str, k)), causal=rng.random() < 0.8,
                prefix=rng.choice((0, 0, spread(1, 512))), cap=rng.choice((0.0, 30.0, 50.0)),
                bias=rng.random() < 0.4, dtype=rng.choice(("float16", "bfloat16")),
                train=not tokens and rng.random() < 0.8)
    while _cost(case) > largest:
        q, k = [max(1, n // 2) for n in q], [max(1, n // 2) for n in k]
        k = [max(a, b) for a, b in zip(q, k)]
        case.update(q=",".join(map(str, q)), k=",".join(map(str, k)))
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------


def _offsets(lens):
    cu = [0]
    for n in lens:
        cu.append(cu[-1] + n)
    return cu


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2 + 1)

    def normal(*shape, scale=1.0, dtype=torch.float32):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    def whole(lo, hi, *shape):
        return torch.randint(lo, hi, shape, generator=gen, device="cuda")

    state = {"case": case}
    if case["kind"] == "rope":
        dt, n, d = DTYPES[case["dtype"]], case["n"], case["d"]
        # q, k and v come out of one projection: q and k are views of its rows
        fused = normal(n, case["hq"] + 2 * case["hk"], d, dtype=dt)
        state["q"], state["k"] = fused[:, : case["hq"]], fused[:, case["hq"] : case["hq"] + case["hk"]]
        axes = len(_lens(case["sections"]))
        state["pos"] = whole(0, case["far"], axes, n)
        if case["train"]:
            state["dq"] = normal(n, case["hq"], d, dtype=dt)
            state["dk"] = normal(n, case["hk"], d, dtype=dt)
        state["axis"], state["freq"] = _pairs(case)
        if own:  # the handle a model keeps: the pairs' axes and frequencies on the device
            from rus_amd import kernels as K

            state["axes"] = K.RopeAxes(state["axis"], state["freq"], d, adjacent=case["adjacent"], device="cuda")
        return state
    if case["kind"] == "attn":
        dt, d, hq, hkv = DTYPES[case["dtype"]], case["d"], case["hq"], case["hkv"]
        ql, kl = _lens(case["q"]), _lens(case["k"])
        nq, nk = sum(ql), sum(kl)
        state["q"] = normal(nq, hq, d, scale=3.0, dtype=dt)
        state["k"] = normal(nk, hkv, d, dtype=dt)
        if case["train"]:  # v as the projection left it, beside q and k
            state["v"] = normal(nk, hq + 2 * hkv, d, dtype=dt)[:, hq + hkv :]
            state["dout"] = normal(nq, hq, d, dtype=dt)
        else:
            state["v"] = normal(nk, hkv, d, dtype=dt)
        as_int = dict(dtype=torch.int32, device="cuda")
        state["cu_q"] = torch.tensor(_offsets(ql), **as_int)
        state["cu_k"] = torch.tensor(_offsets(kl), **as_int)
        state["max_q"], state["max_k"] = max(ql), max(kl)
        state["prefix"] = None
        if case["prefix"]:  # every second row begins with an image
            state["prefix"] = torch.tensor([min(case["prefix"], n) * (i % 2 == 0) for i, n in enumerate(kl)], **as_int)
        state["slopes"] = None
        if case["bias"]:
            state["slopes"] = torch.exp2(-8.0 * (torch.arange(hq, device="cuda", dtype=torch.float32) + 1) / hq)
        return state
    n, d, v, k = case["n"], case["d"], case["v"], case["k"]
    w = normal(v, d, scale=0.02, dtype=torch.float16)
    # the teacher's entries: k distinct vocabulary rows per token; the student leans to the first few of them
    start, step = whole(0, v, n, 1), whole(1, max(2, v // (k + 1)), n, 1)
    ids = (start + step * torch.arange(k, device="cuda")) % v
    h = normal(n, d, scale=3.0)
    for j in range(min(k, 3)):
        h += w[ids[:, j]].float() * normal(n, 1, scale=4.0).abs() * math.sqrt(HIDDEN / d)
    state["h"] = h.to(torch.float16)
    state["w"] = w
    state["w_t"] = torch.zeros(d, -(-v // 64) * 64, dtype=torch.float16, device="cuda")
    state["w_t"][:, :v] = w.t()
    state["logits"] = 12.0 - torch.cumsum(normal(n, k, scale=0.7).abs(), dim=1)
    keep = torch.rand(n, k, generator=gen, device="cuda") > (0.1 if case["ragged"] else -1.0)
    keep &= torch.rand(n, 1, generator=gen, device="cuda") >= case["masked"]
    state["ids"] = torch.where(keep, ids, torch.full_like(ids, -1))
    state["grad"] = torch.full((1,), GRAD_SCALE, device="cuda")
    return state


def _pairs(case):
    """(axis, frequency) of each rotated pair, from the sections."""
    sections = _lens(case["sections"])
    total = sum(sections)
    axis = [a for a, s in enumerate(sections) for _ in range(s)]
    if case["restart"]:
        freq = [THETA ** (-j / s) for s in sections for j in range(s)]
    else:
        freq = [THETA ** (-i / total) for i in range(total)]
    return axis, freq


def _visible_pairs(case):
    """Query-key pairs with a score, over all rows (per head)."""
    total = 0
    for i, (lq, lk) in enumerate(zip(_lens(case["q"]), _lens(case["k"]))):
        if not case["causal"]:
            total += lq * lk
            continue
        prefix = min(case["prefix"], lk) * (i % 2 == 0)
        first = lk - lq + 1  # keys the first query sees by the causal rule
        # sum over queries of max(first + i, prefix)
        below = max(0, min(lq, prefix - first))
        rest = lq - below
        total += below * prefix + rest * (first + below) + rest * (rest - 1) // 2
    return total


def work(case):
    if case["kind"] == "rope":
        w = 4 if case["dtype"] == "float32" else 2
        heads, axes = case["hq"] + case["hk"], len(_lens(case["sections"]))
        passes = 2 if case["train"] else 1
        pairs = sum(_lens(case["sections"]))
        return {"bytes": passes * 2 * case["n"] * heads * case["d"] * w + 8 * axes * case["n"],
                "flops": passes * 6 * case["n"] * heads * pairs}
    if case["kind"] == "attn":
        nq, nk, d = sum(_lens(case["q"])), sum(_lens(case["k"])), case["d"]
        q, kv = nq * case["hq"] * d * 2, nk * case["hkv"] * d * 2
        flops = 4 * d * case["hq"] * _visible_pairs(case)
        if not case["train"]:
            return {"bytes": 2 * q + 2 * kv + 4 * nq * case["hq"], "flops": flops}
        return {"bytes": 4 * q + 4 * kv + 4 * nq * case["hq"], "flops": flops * 7 // 2}
    n, d, v, k = case["n"], case["d"], case["v"], case["k"]
    return {"bytes": 2 * v * d + 4 * n * d + 12 * n * k + 4 * n, "flops": 4 * n * v * d}


# ---- one pass -------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from rus_amd import kernels as K

    case = state["case"]
    if case["kind"] == "rope":
        q, k = K.rope_axes_fwd(state["q"], state["k"], state["pos"], state["axes"])
        if not case["train"]:
            return {"q": q, "k": k}
        dq, dk = K.rope_axes_bwd(state["dq"], state["dk"], state["pos"], state["axes"])
        return {"q": q, "k": k, "dq": dq, "dk": dk}
    if case["kind"] == "attn":
        rows = dict(cu_k=state["cu_k"], max_q=state["max_q"], max_k=state["max_k"], causal=case["causal"],
                    prefix=state["prefix"], softcap=case["cap"], slopes=state["slopes"])
        out, lse = K.attn_masked_fwd(state["q"], state["k"], state["v"], state["cu_q"], **rows)
        if not case["train"]:
            return {"out": out, "lse": lse}
        dq, dk, dv = K.attn_masked_bwd(state["dout"], state["q"], state["k"], state["v"], out, lse, state["cu_q"],
                                       **rows)
        return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}
    loss, kl, _, dh = K.lm_head_distill(state["h"], state["w"], state["ids"], state["logits"],
                                        temperature=case["t"], weight_t=state["w_t"])
    # the hidden gradient comes times 2^16; the incoming gradient of the loss joins here
    dh = K.lm_head_dh_reduce(dh.unsqueeze(0), 2.0**-16, torch.float16, scale_dev=state["grad"])
    return {"loss": loss, "kl": kl, "dh": dh}


def _run_plain(state):
    return {"rope": _plain_rope, "attn": _plain_attn, "distill": _plain_distill}[state["case"]["kind"]](state)


def _plain_rope(state):
    case = state["case"]
    p = sum(_lens(case["sections"]))
    # angles of far positions: 64 bits
    freq = torch.tensor(state["freq"], dtype=torch.float64, device="cuda")
    angle = state["pos"][torch.tensor(state["axis"], device="cuda")].t().double() * freq
    cos, sin = torch.cos(angle).float()[:, None], torch.sin(angle).float()[:, None]

    def rotate(x, sin):
        y = x.float()
        if case["adjacent"]:
            a, b = y[..., 0 : 2 * p : 2], y[..., 1 : 2 * p : 2]
            turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
        else:
            a, b = y[..., :p], y[..., p : 2 * p]
            turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
        return torch.cat([turned, y[..., 2 * p :]], dim=-1).to(x.dtype)

    out = {"q": rotate(state["q"], sin), "k": rotate(state["k"], sin)}
    if case["train"]:
        out.update(dq=rotate(state["dq"], -sin), dk=rotate(state["dk"], -sin))
    return out


def _plain_attn(state):
    case = state["case"]
    q, k, v = state["q"], state["k"], state["v"]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    grp, dt, scale, cap = hq // hkv, q.dtype, 1.0 / math.sqrt(d), case["cap"]
    out = torch.empty(q.shape, dtype=dt, device="cuda")
    lse = torch.empty(hq, q.shape[0], dtype=torch.float32, device="cuda")
    dq, dk, dv = (torch.empty(t.shape, dtype=dt, device="cuda") for t in (q, k, v))
    cq, ck = _offsets(_lens(case["q"])), _offsets(_lens(case["k"]))
    for i in range(len(cq) - 1):
        lq, lk = cq[i + 1] - cq[i], ck[i + 1] - ck[i]
        rows, keys = slice(cq[i], cq[i + 1]), slice(ck[i], ck[i + 1])

        def grouped(x):  # [lq, hq, d] -> [hkv, grp * lq, d]
            return x[rows].float().transpose(0, 1).reshape(hkv, grp * lq, d)

        qf = grouped(q)
        kf, vf = (x[keys].float().transpose(0, 1).contiguous() for x in (k, v))
        z = torch.matmul(qf, kf.transpose(1, 2).contiguous()) * scale
        t = None
        if cap:
            t = torch.tanh(z / cap)
            z = t * cap
        z = z.view(hkv, grp, lq, lk)
        at = torch.arange(lq, device="cuda")[:, None] + (lk - lq)
        j = torch.arange(lk, device="cuda")[None, :]
        if state["slopes"] is not None:
            z = z - state["slopes"].view(hkv, grp, 1, 1) * (at - j).abs().float()
        if case["causal"]:
            seen = j <= at
            if state["prefix"] is not None:
                seen = seen | (j < state["prefix"][i])
            z = z.masked_fill(~seen, float("-inf"))
        top = z.amax(dim=3, keepdim=True)
        p = torch.exp(z - top)
        total = p.sum(dim=3, keepdim=True)
        p = (p / total).view(hkv, grp * lq, lk)
        lse[:, rows] = (top + torch.log(total)).view(hq, lq)
        o = torch.matmul(p, vf)
        out[rows] = o.view(hq, lq, d).transpose(0, 1).to(dt)
        if not case["train"]:
            continue
        do = grouped(state["dout"])
        dv[keys] = torch.matmul(p.transpose(1, 2).contiguous(), do).transpose(0, 1).to(dt)
        dz = torch.matmul(do, vf.transpose(1, 2).contiguous())
        dz = p * (dz - (do * o).sum(dim=2, keepdim=True)) * scale
        if cap:
            dz = dz * (1.0 - t * t)
        dq[rows] = torch.matmul(dz, kf).view(hq, lq, d).transpose(0, 1).to(dt)
        dk[keys] = torch.matmul(dz.transpose(1, 2).contiguous(), qf).transpose(0, 1).to(dt)
    if not case["train"]:
        return {"out": out, "lse": lse}
    return {"out": out, "lse": lse, "dq": dq, "dk": dk, "dv": dv}


def _plain_distill(state):
    case = state["case"]
    t, ids = case["t"], state["ids"]
    valid = ids >= 0
    taught = valid.any(dim=1)
    safe = ids.clamp(min=0)
    # the teacher's probabilities over its valid entries
    s = (state["logits"] / t).masked_fill(~valid, float("-inf"))
    s = s - s.amax(dim=1, keepdim=True).where(taught[:, None], torch.zeros_like(s[:, :1]))
    e = torch.exp(s)
    q = e / e.sum(dim=1, keepdim=True).clamp(min=1e-30)
    log_q = torch.where(valid, s - torch.log(e.sum(dim=1, keepdim=True).clamp(min=1e-30)), torch.zeros_like(s))
    w = state["w"].float()
    z = torch.matmul(state["h"].float(), w.t()) / t
    top = z.amax(dim=1, keepdim=True)
    p = torch.exp(z - top)
    total = p.sum(dim=1, keepdim=True)
    log_p = torch.gather(z, 1, safe) - top - torch.log(total)
    kl = (q * (log_q - log_p)).masked_fill(~valid, 0.0).sum(dim=1)
    denom = taught.sum().clamp(min=1).float()
    loss = kl.sum() * (t * t) / denom
    g = p.div_(total)
    g.scatter_add_(1, safe, -q)
    g *= taught[:, None]
    dh = torch.matmul(g, w) * (t / denom) * state["grad"]
    return {"loss": loss.view(1), "kl": kl, "dh": dh.to(torch.float16)}


# ---- the definition in 64 bits, apart from the plain form -----------------------------------------------------


def exact(case, seed):
    state = prepare(case, seed)
    return {"rope": _exact_rope, "attn": _exact_attn, "distill": _exact_distill}[case["kind"]](case, state)


def _exact_rope(case, state):
    """Pairs as complex numbers, turned by e^(i a)."""
    p = sum(_lens(case["sections"]))
    angle = torch.stack([state["pos"][a].double() * f for a, f in zip(state["axis"], state["freq"])], dim=1)
    turn = torch.polar(torch.ones_like(angle), angle)[:, None]

    def rotate(x, turn):
        y = x.double().clone()
        even = slice(0, 2 * p, 2) if case["adjacent"] else slice(0, p)
        odd = slice(1, 2 * p, 2) if case["adjacent"] else slice(p, 2 * p)
        c = torch.complex(y[..., even], y[..., odd]) * turn
        y[..., even], y[..., odd] = c.real, c.imag
        return y

    out = {"q": rotate(state["q"], turn), "k": rotate(state["k"], turn)}
    if case["train"]:
        out.update(dq=rotate(state["dq"], turn.conj()), dk=rotate(state["dk"], turn.conj()))
    return out


def _exact_attn(case, state):
    """Head by head, the gradients by autograd."""
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    ql, kl = _lens(case["q"]), _lens(case["k"])
    nq, nk = sum(ql), sum(kl)
    zeros = dict(dtype=torch.float64, device="cuda")
    got = {"out": torch.zeros(nq, hq, d, **zeros), "lse": torch.zeros(hq, nq, **zeros)}
    if case["train"]:
        got.update(dq=torch.zeros(nq, hq, d, **zeros), dk=torch.zeros(nk, hkv, d, **zeros),
                   dv=torch.zeros(nk, hkv, d, **zeros))
    a = b = 0
    for i, (lq, lk) in enumerate(zip(ql, kl)):
        dist = (torch.arange(lk - lq, lk, device="cuda")[:, None] - torch.arange(lk, device="cuda")).double()
        hidden = dist < 0 if case["causal"] else torch.zeros_like(dist, dtype=torch.bool)
        if state["prefix"] is not None:
            hidden[:, : int(state["prefix"][i])] = False
        for h in range(hq):
            g = h // (hq // hkv)
            x, y, w = (t.double().detach().requires_grad_(case["train"])
                       for t in (state["q"][a : a + lq, h], state["k"][b : b + lk, g], state["v"][b : b + lk, g]))
            s = (x @ y.t()) / math.sqrt(d)
            if case["cap"]:
                s = torch.tanh(s / case["cap"]) * case["cap"]
            if state["slopes"] is not None:
                s = s - state["slopes"][h].double() * dist.abs()
            s = s.masked_fill(hidden, float("-inf"))
            o = torch.softmax(s, dim=1) @ w
            got["out"][a : a + lq, h] = o.detach()
            got["lse"][h, a : a + lq] = torch.logsumexp(s.detach(), dim=1)
            if case["train"]:
                gx, gy, gw = torch.autograd.grad(o, (x, y, w), state["dout"][a : a + lq, h].double())
                got["dq"][a : a + lq, h] = gx
                got["dk"][b : b + lk, g] += gy
                got["dv"][b : b + lk, g] += gw
        a, b = a + lq, b + lk
    return got


def _exact_distill(case, state):
    """Token block by token block."""
    n, t = case["n"], case["t"]
    w = state["w"].double()
    kl = torch.zeros(n, dtype=torch.float64, device="cuda")
    dh = torch.zeros(n, case["d"], dtype=torch.float64, device="cuda")
    taught = (state["ids"] >= 0).any(dim=1)
    denom = max(1, int(taught.sum()))
    for a in range(0, n, 256):
        rows = slice(a, min(n, a + 256))
        ids, on = state["ids"][rows], taught[rows]
        teacher = torch.zeros(ids.shape[0], case["v"], dtype=torch.float64, device="cuda")
        weights = torch.softmax((state["logits"][rows].double() / t).masked_fill(ids < 0, float("-inf")), dim=1)
        weights = torch.nan_to_num(weights)  # tokens without a teacher
        teacher.scatter_add_(1, ids.clamp(min=0), weights)
        log_p = torch.log_softmax(state["h"][rows].double() @ w.t() / t, dim=1)
        kl[rows] = (torch.xlogy(teacher, teacher).sum(1) - (teacher * log_p).sum(1)) * on
        dh[rows] = ((log_p.exp() - teacher) * on[:, None]) @ w
    return {"loss": (kl.sum() * t * t / denom).view(1), "kl": kl, "dh": dh * (t / denom) * GRAD_SCALE}
