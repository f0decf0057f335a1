"""What this package's operators of 8-bit linear layers are measured by: the root
mean square norm that feeds them and its gradients, quantisation to 8-bit
floating point in blocks of 128, products of such operands, and the norm of a
model's gradients with clipping, over the range of sizes and types that
training and serving use them with.

Kinds of case ("op"):
  rms_fwd   y and rstd of a [R, D] matrix's rows, with a residual's addition
            where "residual" names its type; y in 8 bits with scales where "out"
            is e4m3 or e5m2.
  rms_bwd   dx and dweight; "dh" adds the gradient that the sum's other reader
            gives.
  quant     a [R, C] matrix in 8 bits and back: rows in groups of 128 or
            128 x 128 tiles; "transposed": of the matrix's transpose.
  linear    x @ W.T of 8-bit operands, x [M, K] scaled by groups of its rows,
            W [N, K] by tiles or by groups of its rows.
  grad_norm the norm of a stack of layers' gradients and the factor that clips
            it; "clip": the gradients multiplied by it.

With `own` false, run() computes the operators in elementary torch operations
in 32 bits; with `own` true it calls the package.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn, "e5m2": torch.float8_e5m2}
LARGEST = {"e4m3": 448.0, "e5m2": 57344.0}
SMALLEST = 2.0 ** -100  # a block's largest magnitude counts as at least this
GROUP = 128
EPS = 1e-5
CLIP_EPS = 1e-6


def _rms(name, op, dtype, R, D, residual="", out="", dh=False):
    c = {"name": name, "op": op, "dtype": dtype, "R": R, "D": D}
    return {**c, "residual": residual, "out": out or dtype} if op == "rms_fwd" else {**c, "dh": dh}


def _quant(name, dtype, R, C, block, transposed, to):
    return {"name": name, "op": "quant", "dtype": dtype, "R": R, "C": C, "block": block, "transposed": transposed,
            "to": to}


def _linear(name, M, N, K, x, w, tiles, out):
    return {"name": name, "op": "linear", "M": M, "N": N, "K": K, "x": x, "w": w, "tiles": tiles, "out": out}


def _grads(name, dtype, layers, width, hidden, clip):
    return {"name": name, "op": "grad_norm", "dtype": dtype, "layers": layers, "width": width, "hidden": hidden,
            "clip": clip}


def listed():
    return [
        # One token's activations beside the residual stream: all latency.
        _rms("rms_token", "rms_fwd", "bf16", 1, 4096, "bf16"),
        # A ragged fp32 batch: rows that are not whole 16-byte groups.
        _rms("rms_ragged", "rms_fwd", "f32", 4099, 3001),
        # A batch of 16384 tokens, normalised into an 8-bit product's operand.
        _rms("rms_8bit", "rms_fwd", "bf16", 16384, 4096, "bf16", "e4m3"),
        # The backward pass of a small fp32 layer of odd width.
        _rms("rms_grad_ragged", "rms_bwd", "f32", 1000, 1009),
        # The backward pass over the batch, joined with the stream's gradient.
        _rms("rms_grad_batch", "rms_bwd", "bf16", 16384, 4096, dh=True),
        # A weight matrix, quantised once a step.
        _quant("quant_weight", "bf16", 8192, 4096, 128, False, "e4m3"),
        # A gradient's transpose, as the weight gradient's product reads it.
        _quant("quant_transposed", "f32", 4099, 3001, 1, True, "e5m2"),
        # One token against one weight matrix: bound by reading it.
        _linear("linear_token", 1, 4096, 4096, "e4m3", "e4m3", True, "bf16"),
        # A weight's gradient: both operands scaled by row groups, all ragged.
        _linear("linear_ragged", 1000, 3001, 4097, "e5m2", "e4m3", False, "f32"),
        # The largest: a training batch through a wide layer.
        _linear("linear_batch", 8192, 8192, 8192, "e4m3", "e4m3", True, "bf16"),
        # A small model's gradients (12 layers of width 64): launches and host work.
        _grads("norm_small", "f32", 12, 64, 256, False),
        # A stack's bf16 gradients, clipped in place.
        _grads("clip_stack", "bf16", 8, 2048, 8192, True),
    ]


# Limits of a drawn case, all at or below the largest listed one's cost.
MAX_RMS = 1 << 26
MAX_QUANT = 1 << 26
MAX_LINEAR_FLOPS = 2 * 8192 ** 3
MAX_OPERAND = 1 << 27
MAX_GRADS = 1 << 28


def _size(rng, lo, hi):
    """A size log-uniform in [lo, hi]; half of those above 64 are multiples of
    64, as model widths are, the rest any whole number."""
    v = max(lo, min(hi, round(2 ** rng.uniform(math.log2(lo), math.log2(hi)))))
    return v // 64 * 64 if v > 64 and rng.random() < 0.5 else v


def draw(rng):
    while True:
        dtype = rng.choice(("f32", "bf16"))
        bits8 = rng.choice(("e4m3", "e5m2"))
        kind = rng.random()
        if kind < 0.35:
            c = {"op": rng.choice(("rms_fwd", "rms_bwd")), "dtype": dtype, "R": _size(rng, 1, 32768),
                 "D": _size(rng, 16, 20000)}
            if c["op"] == "rms_fwd":
                c["residual"] = rng.choice(("", "f32", "bf16"))
                c["out"] = rng.choice(("f32", "bf16", bits8))
            else:
                c["dh"] = rng.random() < 0.5
            if c["R"] * c["D"] <= MAX_RMS:
                return c
        elif kind < 0.5:
            c = {"op": "quant", "dtype": dtype, "R": _size(rng, 1, 32768), "C": _size(rng, 16, 20000),
                 "block": rng.choice((1, 128)), "transposed": rng.random() < 0.5, "to": bits8}
            if c["R"] * c["C"] <= MAX_QUANT:
                return c
        elif kind < 0.8:
            c = {"op": "linear", "M": _size(rng, 1, 16384), "N": _size(rng, 16, 16384), "K": _size(rng, 16, 16384),
                 "x": bits8, "w": rng.choice(("e4m3", "e5m2")), "tiles": rng.random() < 0.6, "out": dtype}
            if (2 * c["M"] * c["N"] * c["K"] <= MAX_LINEAR_FLOPS
                    and max(c["M"] * c["N"], c["M"] * c["K"], c["N"] * c["K"]) <= MAX_OPERAND):
                return c
        else:
            width = _size(rng, 24, 4096)
            c = {"op": "grad_norm", "dtype": dtype, "layers": rng.randint(1, 24), "width": width,
                 "hidden": _size(rng, width, 4 * width), "clip": rng.random() < 0.5}
            if sum(math.prod(s) for s in shapes(c)) <= MAX_GRADS:
                return c


def shapes(case):
    """The tensors of `layers` layers: a square and two feed-forward matrices,
    a bias and two norm vectors each."""
    d, f = case["width"], case["hidden"]
    return [(d, d), (f, d), (d, f), (f,), (d,), (d,)] * case["layers"]


# ---------------------------------------------------------------------------
# Inputs
# ---------------------------------------------------------------------------

def _normal(gen, shape, std=1.0, mean=0.0):
    return torch.randn(shape, generator=gen, device="cuda").mul_(std).add_(mean)


def _codes(gen, rows, cols, to, block):
    """8-bit codes [rows, cols], rows at multiples of 16 bytes, and float32
    scales of blocks of `block` x 128: normal values, spread differently from
    block to block, that use the whole range of the codes."""
    room = -(-cols // 16) * 16
    top = LARGEST[to]
    codes = _normal(gen, (rows, room), top / 4).clamp_(-top, top).to(DTYPES[to])[:, :cols]
    scales = torch.exp2(_normal(gen, (-(-rows // block), -(-cols // GROUP)))).mul_(4 / top)
    return codes, scales


def _views(flat, sizes, align):
    """Views of `flat` with the given sizes, each starting at a multiple of
    `align` elements, as an allocator places them."""
    at, out = 0, []
    for n in sizes:
        out.append(flat[at:at + n])
        at += -(-n // align) * align
    return out


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    op = case["op"]
    if op.startswith("rms"):
        # Activations with a mean of their own, as a residual stream has.
        dt, R, D = DTYPES[case["dtype"]], case["R"], case["D"]
        s["x"] = _normal(gen, (R, D), 1.5, 0.25).to(dt)
        s["w"] = _normal(gen, (D,), 0.2, 1.0).to(dt)
        if op == "rms_fwd":
            s["residual"] = _normal(gen, (R, D), 2.0).to(DTYPES[case["residual"]]) if case["residual"] else None
        else:
            s["dy"] = _normal(gen, (R, D)).to(dt)
            s["dh"] = _normal(gen, (R, D)).to(dt) if case["dh"] else None
            s["rstd"] = 1 / torch.sqrt(s["x"].float().square().mean(dim=1) + EPS)
    elif op == "quant":
        # Rows of different sizes, and a few large columns, as activations have.
        dt, R, C = DTYPES[case["dtype"]], case["R"], case["C"]
        x = _normal(gen, (R, C)).mul_(torch.exp2(_normal(gen, (R, 1))))
        s["x"] = x.mul_(torch.exp2(_normal(gen, (1, C)))).to(dt)
    elif op == "linear":
        s["x"] = _codes(gen, case["M"], case["K"], case["x"], 1)
        s["w"] = _codes(gen, case["N"], case["K"], case["w"], 128 if case["tiles"] else 1)
    else:
        n = [math.prod(x) for x in shapes(case)]
        room = sum(-(-k // 64) * 64 for k in n)
        s["flat"] = _normal(gen, (room,), 1e-3).to(DTYPES[case["dtype"]])
        s["grads"] = _views(s["flat"], n, 64)
        # A third of the norm to be expected: the gradients are clipped.
        s["max_norm"] = 1e-3 / 3 * math.sqrt(sum(n))
    return s


# ---------------------------------------------------------------------------
# The plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------

def _blocks(x, block):
    """x [R, C] with zeros up to whole blocks, as [R', block, C', 128]."""
    R, C = x.shape
    x = torch.nn.functional.pad(x, (0, -C % GROUP, 0, -R % block))
    return x.view(x.shape[0] // block, block, x.shape[1] // GROUP, GROUP)


def _plain_quantize(x, block, to):
    """(values, scales): x rounded to 8 bits in blocks of `block` x 128."""
    R, C = x.shape
    b = _blocks(x, block)
    top = b.abs().amax(dim=(1, 3), keepdim=True).clamp(min=SMALLEST)
    largest = torch.full_like(top, LARGEST[to])
    scale = top / largest
    values = (b * (largest / top)).to(DTYPES[to]).float() * scale
    return values.reshape(values.shape[0] * block, -1)[:R, :C], scale[:, 0, :, 0]


def _plain_values(codes, scales, block):
    R, C = codes.shape
    return (_blocks(codes.float(), block) * scales[:, None, :, None]).view(-1, scales.shape[1] * GROUP)[:R, :C]


def _plain_rms_fwd(s):
    case, h = s["case"], s["x"]
    out = {}
    if s["residual"] is not None:
        h = out["h"] = (h.float() + s["residual"].float()).to(s["residual"].dtype)
    x = h.float()
    rstd = out["rstd"] = 1 / torch.sqrt((x * x).sum(dim=1) / x.shape[1] + EPS)
    y = x * rstd[:, None] * s["w"].float()
    if case["out"] in LARGEST:
        y, out["scales"] = _plain_quantize(y, 1, case["out"])
        return {**out, "y": y.to(torch.bfloat16)}
    return {**out, "y": y.to(DTYPES[case["out"]])}


def _plain_rms_bwd(s):
    x, dy, rstd = s["x"].float(), s["dy"].float(), s["rstd"][:, None]
    xhat = x * rstd
    wdy = dy * s["w"].float()
    c = (wdy * xhat).sum(dim=1, keepdim=True) / x.shape[1]
    dx = rstd * (wdy - xhat * c)
    if s["dh"] is not None:
        dx = dx + s["dh"].float()
    return {"dx": dx.to(s["dy"].dtype), "dw": (dy * xhat).sum(dim=0)}


def _plain_quant(s):
    case = s["case"]
    x = s["x"].float()
    values, scales = _plain_quantize(x.t().contiguous() if case["transposed"] else x, case["block"], case["to"])
    return {"values": values.to(s["x"].dtype), "scales": scales}


def _plain_linear(s):
    x = _plain_values(*s["x"], 1)
    w = _plain_values(*s["w"], 128 if s["case"]["tiles"] else 1)
    return {"out": torch.mm(x, w.t()).to(DTYPES[s["case"]["out"]])}


def _plain_grad_norm(s):
    flat = torch.cat(s["grads"]).float()
    norm = torch.sqrt((flat * flat).sum())
    scale = torch.clamp(s["max_norm"] / (norm + CLIP_EPS), max=1.0)
    if not s["case"]["clip"]:
        return {"norm": norm, "scale": scale}
    torch._foreach_copy_(s["grads"], list((flat * scale).split([g.numel() for g in s["grads"]])))
    return {"norm": norm, "grads": s["flat"]}


def _own(s):
    import tilec
    case, op = s["case"], s["case"]["op"]
    if op == "rms_fwd":
        y, h, rstd = tilec.ext.rms_norm(s["x"], s["w"], s["residual"], eps=EPS, dtype=DTYPES[case["out"]])
        out = {"rstd": rstd} if s["residual"] is None else {"h": h, "rstd": rstd}
        if case["out"] in LARGEST:  # the values that the codes stand for
            out["scales"] = y[1]
            y = tilec.ext.dequantize_fp8(y, dtype=torch.bfloat16)
        return {**out, "y": y}
    if op == "rms_bwd":
        dx, dw = tilec.ext.rms_norm_backward(s["dy"], s["x"], s["rstd"], s["w"], dh=s["dh"])
        return {"dx": dx, "dw": dw}
    if op == "quant":
        x = s["x"].t() if case["transposed"] else s["x"]
        q = tilec.ext.quantize_fp8(x, block=(case["block"], GROUP), dtype=DTYPES[case["to"]])
        return {"values": tilec.ext.dequantize_fp8(q, dtype=s["x"].dtype), "scales": q[1]}
    if op == "linear":
        return {"out": tilec.ext.linear_fp8(s["x"], s["w"], dtype=DTYPES[case["out"]])}
    if case["clip"]:
        return {"norm": tilec.ext.clip_grads(s["grads"], s["max_norm"]), "grads": s["flat"]}
    norm, scale = tilec.ext.grad_norm(s["grads"], s["max_norm"])
    return {"norm": norm, "scale": scale}


def run(state):
    if own:
        return _own(state)
    op = state["case"]["op"]
    if op == "rms_fwd":
        return _plain_rms_fwd(state)
    if op == "rms_bwd":
        return _plain_rms_bwd(state)
    if op == "quant":
        return _plain_quant(state)
    return _plain_linear(state) if op == "linear" else _plain_grad_norm(state)


# ---------------------------------------------------------------------------
# 64-bit values, from the definitions
# ---------------------------------------------------------------------------

def _spread(scales, block, rows, cols):
    """A value for every element, of its block's scale."""
    s = scales.double()
    return s.repeat_interleave(block, dim=0)[:rows].repeat_interleave(GROUP, dim=1)[:, :cols]


def _exact_quantize(x, block, to):
    R, C = x.shape
    rows, cols = -(-R // block), -(-C // GROUP)
    full = torch.zeros(rows * block, cols * GROUP, dtype=torch.float64, device=x.device)
    full[:R, :C] = x.abs()
    scales = full.view(rows, block, cols, GROUP).amax(dim=3).amax(dim=1).clamp_(min=SMALLEST).div_(LARGEST[to])
    each = _spread(scales, block, R, C)
    return (x / each).to(DTYPES[to]).double() * each, scales


def _exact_rms_fwd(s):
    case, h, out = s["case"], s["x"].double(), {}
    if s["residual"] is not None:
        h = out["h"] = (h + s["residual"].double()).to(s["residual"].dtype).double()
    rstd = out["rstd"] = (h.square().mean(dim=1) + EPS).rsqrt()
    y = torch.einsum("rd,r,d->rd", h, rstd, s["w"].double())
    if case["out"] in LARGEST:
        y, out["scales"] = _exact_quantize(y, 1, case["out"])
    return {**out, "y": y}


def _exact_rms_bwd(s):
    # dx = rstd J wdy with J = I - xhat xhat' / D, and what the sum's other reader gives.
    dy, rstd = s["dy"].double(), s["rstd"].double()[:, None]
    xhat = s["x"].double() * rstd
    wdy = dy * s["w"].double()
    dx = rstd * (wdy - xhat * (wdy * xhat).mean(dim=1, keepdim=True))
    if s["dh"] is not None:
        dx += s["dh"].double()
    return {"dx": dx, "dw": torch.einsum("rd,rd->d", dy, xhat)}


def _exact_linear(s):
    case = s["case"]
    x = s["x"][0].double() * _spread(s["x"][1], 1, case["M"], case["K"])
    w = s["w"][0].double() * _spread(s["w"][1], 128 if case["tiles"] else 1, case["N"], case["K"])
    return {"out": torch.mm(x, w.t().contiguous())}


def _exact_grad_norm(s):
    norm = math.sqrt(math.fsum(float(g.double().square().sum()) for g in s["grads"]))
    scale = min(1.0, s["max_norm"] / (norm + CLIP_EPS))
    if not s["case"]["clip"]:
        return {"norm": norm, "scale": scale}
    flat, at = s["flat"].double(), 0
    for g in s["grads"]:  # what lies between the tensors stays
        flat[at:at + g.numel()] *= scale
        at += -(-g.numel() // 64) * 64
    return {"norm": norm, "grads": flat}


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "rms_fwd":
        return _exact_rms_fwd(s)
    if case["op"] == "rms_bwd":
        return _exact_rms_bwd(s)
    if case["op"] == "quant":
        x = s["x"].double()
        values, scales = _exact_quantize(x.t().contiguous() if case["transposed"] else x, case["block"], case["to"])
        return {"values": values, "scales": scales}
    return _exact_linear(s) if case["op"] == "linear" else _exact_grad_norm(s)


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------

def _bytes(dtype):
    return {"f32": 4, "bf16": 2, "e4m3": 1, "e5m2": 1}[dtype]


def work(case):
    op = case["op"]
    if op.startswith("rms"):
        R, D, esz = case["R"], case["D"], _bytes(case["dtype"])
        if op == "rms_bwd":
            return {"bytes": (4 if case["dh"] else 3) * R * D * esz + D * esz + 4 * D + 4 * R, "flops": 10 * R * D}
        per = esz + (2 * _bytes(case["residual"]) if case["residual"] else 0)
        bits8 = case["out"] in LARGEST
        # In 8 bits: the codes and scales, written and read back, and the values that they stand for.
        per += 1 + 1 + 2 if bits8 else _bytes(case["out"])
        scales = 8 * R * -(-D // GROUP) if bits8 else 0
        return {"bytes": R * D * per + scales + D * esz + 4 * R, "flops": (9 if bits8 else 5) * R * D}
    if op == "quant":
        rows, cols = (case["C"], case["R"]) if case["transposed"] else (case["R"], case["C"])
        scales = -(-rows // case["block"]) * -(-cols // GROUP)
        return {"bytes": rows * cols * (2 * _bytes(case["dtype"]) + 2) + 8 * scales, "flops": 4 * rows * cols}
    if op == "linear":
        M, N, K = case["M"], case["N"], case["K"]
        groups = -(-K // GROUP)
        scales = M * groups + (-(-N // 128) if case["tiles"] else N) * groups
        return {"bytes": M * K + N * K + 4 * scales + M * N * _bytes(case["out"]), "flops": 2 * M * N * K}
    n, esz = sum(math.prod(x) for x in shapes(case)), _bytes(case["dtype"])
    # Clipping reads every gradient again and writes it.
    return {"bytes": n * esz * (3 if case["clip"] else 1) + 8, "flops": (3 if case["clip"] else 2) * n}
