"""Performance cases of the microscaled operators: 4- and 8-bit blocks that the matrix cores read directly.

A microscaled row holds blocks of 32 elements, each element in 4 bits (e2m1, "fp4") or 8 (e4m3, "fp8"), with one
power-of-two scale (E8M0) per block. Widths are those of the repository's training configuration (hidden 1536,
intermediate 8960, fused q|k|v 2048 rows, fused gate|up 17920 rows), token counts those of a decoding step (one
token) up to long packed batches, and odd sizes between.

Kinds of case:
  quantize  rows to blocks and back to the source's type (``kernels.mx_quantize``, ``mx_dequantize``)
  norm      RMSNorm of the residual sum, written as fp8 blocks (``kernels.rms_norm_mx_fwd``)
  product   x W^T (+ bias) with W in blocks and x quantised in the call (``kernels.mx_gemm``)
  gradient  dy W, the product's gradient, W decoded to dy's type (``kernels.mx_gemm(..., trans=True)``)
  glu       silu(x Wg^T) * (x Wu^T) in one kernel: forward, or forward, gradient of [gate|up] and of x
            (``kernels.mx_mlp_glu_fwd``, ``mx_mlp_glu_bwd``, ``mx_gemm``)
"""

import math

import torch

own = False

HIDDEN, INTER, QKV, EPS = 1536, 8960, 2048, 1e-6
BLOCK, PAD = 32, 4  # elements per block; a stored row is padded to whole groups of 4 blocks
DTYPES = {"float16": torch.float16, "bfloat16": torch.bfloat16, "float32": torch.float32}
# element format: exponent of the largest binade, of the smallest normal, mantissa bits, largest value
FORMATS = {"fp4": (2, 0, 1, 6.0), "fp8": (8, -6, 3, 448.0)}


def listed():
    return [
        # the fused gate|up weight of a layer, quantised when a model is loaded
        {"name": "quantize_gate_up", "kind": "quantize", "m": 2 * INTER, "k": HIDDEN, "fmt": "fp4", "dtype": "float16"},
        # activations of the default batch, one column wider than the hidden size: no row is aligned
        {"name": "quantize_odd", "kind": "quantize", "m": 707, "k": HIDDEN + 1, "fmt": "fp8", "dtype": "bfloat16"},
        # the attention norm of the default batch, with the residual sum
        {"name": "norm_707", "kind": "norm", "m": 707, "k": HIDDEN, "dtype": "float16", "residual": True},
        # the same for a batch of long rows: bandwidth
        {"name": "norm_16381", "kind": "norm", "m": 16381, "k": HIDDEN, "dtype": "float16", "residual": True},
        # the down projection of one decoded token: latency and the weight's bytes
        {"name": "product_1", "kind": "product", "m": 1, "k": INTER, "n": HIDDEN, "act": "fp8", "fmt": "fp4",
         "dtype": "float16", "bias": False},
        # q|k|v of the default batch, with the bias Qwen2 has there
        {"name": "product_707", "kind": "product", "m": 707, "k": HIDDEN, "n": QKV, "act": "fp8", "fmt": "fp4",
         "dtype": "float16", "bias": True},
        # gate|up of a batch of long rows, both sides in 4 bits: the matrix cores' highest rate
        {"name": "product_8161", "kind": "product", "m": 8161, "k": HIDDEN, "n": 2 * INTER, "act": "fp4",
         "fmt": "fp4", "dtype": "bfloat16", "bias": False},
        # the input gradient of q|k|v for one short row
        {"name": "gradient_16", "kind": "gradient", "m": 16, "k": HIDDEN, "n": QKV, "fmt": "fp4", "dtype": "float16"},
        # the input gradient of gate|up at the rotary table's length
        {"name": "gradient_2048", "kind": "gradient", "m": 2048, "k": HIDDEN, "n": 2 * INTER, "fmt": "fp4",
         "dtype": "bfloat16"},
        # the feed-forward gate of one decoded token
        {"name": "glu_1", "kind": "glu", "m": 1, "k": HIDDEN, "n": INTER, "act": "fp8", "fmt": "fp4",
         "dtype": "float16", "train": False},
        # the same in training, default batch
        {"name": "glu_707", "kind": "glu", "m": 707, "k": HIDDEN, "n": INTER, "act": "fp8", "fmt": "fp4",
         "dtype": "float16", "train": True},
        # and a batch of long rows
        {"name": "glu_4096", "kind": "glu", "m": 4096, "k": HIDDEN, "n": INTER, "act": "fp8", "fmt": "fp4",
         "dtype": "float16", "train": True},
    ]


def draw(rng):
    def spread(lo, hi):  # over the logarithm of the range, odd values among them
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    kind = rng.choice(("quantize", "norm", "product", "product", "gradient", "glu", "glu"))
    case = {"kind": kind, "m": spread(1, 8161), "dtype": rng.choice(("float16", "bfloat16"))}
    if kind == "quantize":
        case.update(m=spread(1, 17920), k=spread(32, 8960), fmt=rng.choice(("fp4", "fp8")),
                    dtype=rng.choice(("float16", "bfloat16", "float32")))
        return case
    if kind == "norm":
        case.update(m=spread(1, 16381), k=spread(64, 8192), dtype=rng.choice(("float16", "float32")),
                    residual=rng.random() < 0.7)
        while case["m"] * case["k"] > 16381 * HIDDEN:
            case["m"] = max(1, case["m"] // 2)
        return case
    case.update(k=spread(64, INTER), n=spread(16, 2 * INTER), fmt=rng.choice(("fp4", "fp4", "fp4", "fp8")))
    if kind == "product":
        case.update(act=rng.choice(("fp8", "fp8", "fp4")), bias=rng.random() < 0.5)
    if kind == "glu":
        case.update(n=spread(16, INTER), act="fp8", train=rng.random() < 0.7)
    while case["m"] * case["k"] * case["n"] > 4096 * HIDDEN * INTER:
        case["m"] = max(1, case["m"] // 2)
    return case


# ---- inputs ---------------------------------------------------------------------------------------------------


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed * 2 + 1)

    def normal(*shape, scale=1.0, dtype=DTYPES[case["dtype"]]):
        return (torch.randn(*shape, generator=gen, device="cuda") * scale).to(dtype)

    m, k = case["m"], case["k"]
    state = {"case": case}
    if case["kind"] == "quantize":
        state["x"] = normal(m, k, scale=0.02 if case["fmt"] == "fp4" else 1.0)
        return state
    if case["kind"] == "norm":
        state["x"] = normal(m, k)
        state["residual"] = normal(m, k, scale=2.0) if case["residual"] else None
        state["weight"] = (1 + normal(k, scale=0.05, dtype=torch.float32)).to(DTYPES[case["dtype"]])
        return state
    n = case["n"]
    rows = 2 * n if case["kind"] == "glu" else n
    # a weight of N(0, 0.02) in blocks: what a model's loading step leaves
    codes, scales = _to_blocks(normal(rows, k, scale=0.02, dtype=torch.float32), case["fmt"])
    state["w_codes"], state["w_scales"] = codes, scales
    if case["kind"] == "gradient":
        state["dy"] = normal(m, n, scale=0.05)
        return state
    x = normal(m, k, dtype=torch.float32)
    x[:, :: max(1, k // 5)] *= 8.0  # activations meet a few channels of large values
    state["x"] = x.to(DTYPES[case["dtype"]])
    if case["kind"] == "product":
        state["bias"] = normal(n) if case["bias"] else None
    if case["kind"] == "glu" and case["train"]:
        state["dh"] = normal(m, n, scale=0.05)
    return state


def work(case):
    m, k, w = case["m"], case["k"], 4 if case["dtype"] == "float32" else 2
    nb = -(-k // BLOCK)
    if case["kind"] == "quantize":  # the rows, the values that come back and the scales
        return {"bytes": 2 * m * k * w + m * nb, "flops": 4 * m * k}
    if case["kind"] == "norm":
        streams = 3 if case["residual"] else 1  # x, the residual, their sum
        return {"bytes": streams * m * k * w + m * k + m * nb + k * w + 4 * m, "flops": 8 * m * k}
    n = case["n"]
    per = nb * (16 if case["fmt"] == "fp4" else 32) + nb  # bytes of one row of W
    if case["kind"] == "product":
        return {"bytes": m * k * w + n * per + m * n * w + (n * w if case["bias"] else 0), "flops": 2 * m * n * k}
    if case["kind"] == "gradient":
        return {"bytes": m * n * w + n * per + m * k * w, "flops": 2 * m * n * k}
    if not case["train"]:
        return {"bytes": m * k * w + 2 * n * per + m * n * w, "flops": 4 * m * n * k}
    return {"bytes": 2 * m * k * w + 2 * n * per + 4 * m * n * w, "flops": 8 * m * n * k}


# ---- one pass -------------------------------------------------------------------------------------------------


def run(state):
    return (_run_own if own else _run_plain)(state)


def _run_own(state):
    from rus_amd import kernels as K

    case = state["case"]
    if case["kind"] == "quantize":
        q = K.mx_quantize(state["x"], case["fmt"])
        return {"values": K.mx_dequantize(q, state["x"].dtype), "scales": q.scales}
    if case["kind"] == "norm":
        q, h, rstd = K.rms_norm_mx_fwd(state["x"], state["weight"], eps=EPS, residual=state["residual"])
        return {"codes": q.codes.view(torch.float8_e4m3fn), "scales": q.scales, "sum": h, "rstd": rstd}
    rows = case["n"] * (2 if case["kind"] == "glu" else 1)
    w = K.MXTensor(state["w_codes"], state["w_scales"], (rows, case["k"]), case["fmt"])
    if case["kind"] == "product":
        return K.mx_gemm(state["x"], w, bias=state["bias"], act=case["act"])
    if case["kind"] == "gradient":
        return K.mx_gemm(state["dy"], w, trans=True)
    if not case["train"]:
        return K.mx_mlp_glu_fwd(state["x"], w, act=case["act"])
    x = K.mx_quantize(state["x"], case["act"])
    h = K.mx_mlp_glu_fwd(x, w, dtype=state["x"].dtype)
    d_gu = K.mx_mlp_glu_bwd(state["dh"], x, w)
    return {"h": h, "d_gate_up": d_gu, "dx": K.mx_gemm(d_gu, w, trans=True)}


def _run_plain(state):
    case = state["case"]
    if case["kind"] == "quantize":
        values, scales = _rounded(state["x"].float(), case["fmt"])
        return {"values": values[:, : case["k"]].to(state["x"].dtype), "scales": scales}
    if case["kind"] == "norm":
        h = state["x"]
        if state["residual"] is not None:
            h = (h.float() + state["residual"].float()).to(h.dtype)
        # 64 bits: a value next to a border between two codes has to fall on its side of it
        h64 = h.double()
        rstd = 1.0 / torch.sqrt(h64.square().mean(dim=1, keepdim=True) + EPS)
        values, scales = _rounded(h64 * rstd * state["weight"].double(), "fp8")
        elements = values / torch.exp2(scales.to(values.dtype) - 127.0).repeat_interleave(BLOCK, dim=1)
        return {"codes": elements.to(torch.float8_e4m3fn), "scales": scales, "sum": h, "rstd": rstd[:, 0].float()}
    w = _values(state["w_codes"], state["w_scales"], case["fmt"])[:, : case["k"]]
    if case["kind"] == "gradient":
        return torch.matmul(state["dy"].float(), w).to(state["dy"].dtype)
    x = _rounded(state["x"].float(), case["act"])[0][:, : case["k"]]
    dtype = state["x"].dtype
    y = torch.matmul(x, w.t())
    if case["kind"] == "product":
        return (y if state["bias"] is None else y + state["bias"].float()).to(dtype)
    gate, up = y[:, : case["n"]], y[:, case["n"] :]
    sig = 1.0 / (1.0 + torch.exp(-gate))
    h = (gate * sig * up).to(dtype)
    if not case["train"]:
        return h
    dh = state["dh"].float()
    d_gate = dh * up * (sig + gate * sig * (1.0 - sig))
    d_gu = torch.cat([d_gate, dh * gate * sig], dim=1).to(dtype)
    return {"h": h, "d_gate_up": d_gu, "dx": torch.matmul(d_gu.float(), w).to(dtype)}


# ---- blocks in elementary torch operations ---------------------------------------------------------------------


def _split(x):
    """[rows, k] -> [rows, blocks, 32], zeros behind the row's end up to a whole group of blocks."""
    rows, k = x.shape
    wide = -(-k // (BLOCK * PAD)) * BLOCK * PAD
    if wide != k:
        x = torch.cat([x, x.new_zeros(rows, wide - k)], dim=1)
    return x.view(rows, wide // BLOCK, BLOCK)


def _rounded(x, fmt):
    """The values that x's blocks stand for, in x's type, and the scales' exponent bytes."""
    emax, emin, bits, top = FORMATS[fmt]
    blocks = _split(x)
    amax = blocks.abs().amax(dim=2)
    exponent = torch.frexp(amax)[1] - 1 - emax  # floor(log2 amax) - emax
    exponent = torch.where(amax > 0, exponent, torch.full_like(exponent, -127)).clamp(-127, 127)
    scale = torch.exp2(exponent.to(x.dtype)).unsqueeze(2)
    v = (blocks / scale).clamp(-top, top)
    step = torch.exp2((torch.frexp(v)[1] - 1).clamp(min=emin).to(x.dtype) - bits)
    values = torch.round(v / step) * step * scale  # ties to even
    return values.reshape(x.shape[0], -1), (exponent + 127).to(torch.uint8)


def _to_blocks(x, fmt):
    """Codes and scales as they are stored: fp4 two to a byte, the even element in the low half."""
    values, scales = _rounded(x, fmt)
    elements = _split(values) / torch.exp2(scales.float() - 127.0).unsqueeze(2)
    if fmt == "fp8":
        return elements.to(torch.float8_e4m3fn).view(torch.uint8).reshape(x.shape[0], -1), scales
    a = elements.abs()
    code = (2 * a).where(a < 2, (a + 2).where(a < 4, a / 2 + 4)).to(torch.uint8)  # 0 .5 1 1.5 2 3 4 6
    code = (code + 8 * torch.signbit(elements).to(torch.uint8)).reshape(x.shape[0], -1)
    return code[:, 0::2] + 16 * code[:, 1::2], scales


def _values(codes, scales, fmt):
    """What stored blocks stand for, in 32 bits."""
    if fmt == "fp8":
        elements = codes.view(torch.float8_e4m3fn).float()
    else:
        table = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], device=codes.device)
        table = torch.cat([table, -table])
        elements = torch.stack([table[(codes & 15).long()], table[(codes >> 4).long()]], dim=2)
    elements = elements.reshape(codes.shape[0], scales.shape[1], BLOCK)
    return (elements * torch.exp2(scales.float() - 127.0).unsqueeze(2)).reshape(codes.shape[0], -1)


# ---- the definition in 64 bits, apart from the plain form -----------------------------------------------------


def _grid(fmt):
    """All values >= 0 of an element format in the order of their codes."""
    if fmt == "fp4":
        got = [m * 0.5 for m in range(2)] + [2.0 ** (e - 1) * (1 + m / 2) for e in range(1, 4) for m in range(2)]
    else:
        got = [m * 2.0**-9 for m in range(8)]
        got += [2.0 ** (e - 7) * (1 + m / 8) for e in range(1, 16) for m in range(8) if (e, m) != (15, 7)]
    return torch.tensor(got, dtype=torch.float64, device="cuda")


def _exact_blocks(x, fmt):
    """(elements, scales) of x's blocks in 64 bits: the nearest of the format's values, found in their list."""
    grid = _grid(fmt)
    rows, k = x.shape
    nb = -(-k // (BLOCK * PAD)) * PAD
    full = torch.zeros(rows, nb * BLOCK, dtype=torch.float64, device=x.device)
    full[:, :k] = x.double()
    full = full.view(rows, nb, BLOCK)
    top = full.abs().max(dim=2).values
    log = torch.floor(torch.log2(top.clamp(min=2.0**-200)))
    log = torch.where(torch.exp2(log) > top, log - 1, torch.where(torch.exp2(log + 1) <= top, log + 1, log))
    log = (log - math.floor(math.log2(float(grid[-1])))).clamp(-127, 127)
    scale = torch.exp2(log).unsqueeze(2)
    v = full / scale
    a = v.abs().clamp(max=float(grid[-1])).contiguous()
    hi = torch.searchsorted(grid, a).clamp(1, grid.numel() - 1)
    below, above = a - grid[hi - 1], grid[hi] - a
    hi = torch.where((below < above) | ((below == above) & (hi % 2 == 1)), hi - 1, hi)
    return torch.copysign(grid[hi], v), scale


def exact(case, seed):
    state = prepare(case, seed)
    if case["kind"] == "quantize":
        e, s = _exact_blocks(state["x"], case["fmt"])
        return {"values": (e * s).reshape(case["m"], -1)[:, : case["k"]], "scales": None}
    if case["kind"] == "norm":
        h = state["x"].double()
        if state["residual"] is not None:
            h = (h + state["residual"].double()).to(state["x"].dtype).double()
        r = (h.square().sum(1) / case["k"] + EPS) ** -0.5
        e, _ = _exact_blocks(h * r[:, None] * state["weight"].double(), "fp8")
        return {"codes": e.reshape(case["m"], -1), "scales": None, "sum": h, "rstd": r}
    codes, scales = state["w_codes"], state["w_scales"]
    if case["fmt"] == "fp8":
        c = codes.long()
        e = _grid("fp8")[c & 127] * torch.where(c > 127, -1.0, 1.0).double()
    else:
        c = torch.stack([codes % 16, codes // 16], dim=2).reshape(codes.shape[0], -1).long()
        e = _grid("fp4")[c & 7] * torch.where(c > 7, -1.0, 1.0).double()
    e = e.view(codes.shape[0], -1, BLOCK) * (2.0 ** (scales.double() - 127)).unsqueeze(2)
    w = e.reshape(codes.shape[0], -1)[:, : case["k"]]
    if case["kind"] == "gradient":
        return state["dy"].double() @ w
    e, s = _exact_blocks(state["x"], case["act"])
    x = (e * s).reshape(case["m"], -1)[:, : case["k"]]
    if case["kind"] == "product":
        y = x @ w.t()
        return y if state["bias"] is None else y + state["bias"].double()
    n = case["n"]
    g, u = x @ w[:n].t(), x @ w[n:].t()
    sig = torch.sigmoid(g)
    h = g * sig * u
    if not case["train"]:
        return h
    dh = state["dh"].double()
    d_gu = torch.cat([dh * u * sig * (1 + g * (1 - sig)), dh * g * sig], 1)
    return {"h": h, "d_gate_up": d_gu, "dx": d_gu @ w}
