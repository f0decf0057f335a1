"""What the training operators of this package are measured by: layer norm and
its gradients, the cross entropy of a linear layer's outputs and its gradients,
and an AdamW step over many tensors, over the range of sizes and types that a
training step uses them with.

Kinds of case ("op"):
  ln_fwd    y, mean, rstd of a [R, D] matrix's rows.
  ln_bwd    dx and the column reductions dweight, dbias.
  ce_loss   per-row losses of logits = x @ W.T, x [N, H], W [V, H] (evaluation).
  ce_grad   the mean loss with dx and dW, as a training step has them.
  adamw     one step over every tensor of a stack of layers, states in 32 or 8
            bits.

With `own` false, run() computes the operators in elementary torch operations
in 32 bits; with `own` true it calls the package.
"""

import math

import torch

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16}
EPS = 1e-5
IGNORE = -100
BLOCK = 256  # values per scale of an 8-bit state
ADAMW = {"lr": 1e-3, "betas": (0.9, 0.999), "eps": 1e-8, "weight_decay": 0.01}


def _ln(name, op, dtype, R, D):
    return {"name": name, "op": op, "dtype": dtype, "R": R, "D": D}


def _ce(name, op, dtype, N, H, V, ignored):
    return {"name": name, "op": op, "dtype": dtype, "N": N, "H": H, "V": V, "ignored": ignored}


def _adamw(name, bits, grad, layers, width, hidden, copies):
    return {"name": name, "op": "adamw", "bits": bits, "grad": grad, "layers": layers, "width": width,
            "hidden": hidden, "copies": copies}


def listed():
    return [
        # One token's activations: all latency.
        _ln("ln_token", "ln_fwd", "bf16", 1, 4096),
        # A ragged fp32 batch: rows that are not whole 16-byte groups.
        _ln("ln_ragged", "ln_fwd", "f32", 4099, 3001),
        # The backward pass of a small fp32 layer of odd width.
        _ln("ln_grad_ragged", "ln_bwd", "f32", 1000, 1009),
        # The backward pass over a training batch of 16384 tokens.
        _ln("ln_grad_batch", "ln_bwd", "bf16", 16384, 4096),
        # Losses of an evaluation batch, one per token, nothing kept.
        _ce("ce_eval", "ce_loss", "bf16", 2048, 2048, 65536, 0.0),
        # A few tokens' training step: bound by reading W and writing dW.
        _ce("ce_grad_few", "ce_grad", "bf16", 7, 1024, 32768, 0.0),
        # Ragged rows, hidden width and vocabulary; a third of the targets ignored.
        _ce("ce_grad_ragged", "ce_grad", "bf16", 1000, 1000, 50021, 0.33),
        # An fp32 classifier or small language model.
        _ce("ce_grad_f32", "ce_grad", "f32", 512, 1024, 16384, 0.1),
        # The largest: a training batch against a large vocabulary.
        _ce("ce_grad_batch", "ce_grad", "bf16", 4096, 4096, 131072, 0.1),
        # A small model's tensors (12 layers of width 64): launches and host work.
        _adamw("adamw_small", 32, "f32", 12, 64, 256, False),
        # Mixed precision: fp32 weights and states, bf16 gradients, and the bf16
        # copies of the weights that the next forward pass reads.
        _adamw("adamw_mixed", 32, "bf16", 8, 2048, 8192, True),
        # The same stack's states held in 8 bits.
        _adamw("adamw_8bit", 8, "bf16", 4, 2048, 8192, True),
    ]


# Limits of a drawn case, all at or below the largest listed one's cost.
MAX_LN = 1 << 26
MAX_CE_FLOPS = {"f32": 1 << 39, "bf16": 6 * 4096 * 4096 * 131072}
MAX_CE_LOGITS = 1 << 28
MAX_WEIGHT = 1 << 28
MAX_ADAMW = 1 << 27


def _size(rng, lo, hi):
    """A size log-uniform in [lo, hi]; half of those above 64 are multiples of
    64, as model widths are, the rest any whole number."""
    v = max(lo, min(hi, round(2 ** rng.uniform(math.log2(lo), math.log2(hi)))))
    v = v // 64 * 64 if v > 64 and rng.random() < 0.5 else v
    return v + 64 if v == 3072 else v


def draw(rng):
    while True:
        dtype = rng.choice(("f32", "bf16"))
        kind = rng.random()
        if kind < 0.33:
            c = {"op": rng.choice(("ln_fwd", "ln_bwd")), "dtype": dtype, "R": _size(rng, 1, 32768),
                 "D": _size(rng, 16, 20000)}
            if c["R"] * c["D"] <= MAX_LN:
                return c
        elif kind < 0.72:
            c = {"op": rng.choice(("ce_loss", "ce_grad", "ce_grad")), "dtype": dtype, "N": _size(rng, 1, 8192),
                 "H": _size(rng, 64, 4096), "V": _size(rng, 500, 131072),
                 "ignored": rng.choice((0.0, 0.1, 0.5))}
            if (6 * c["N"] * c["H"] * c["V"] <= MAX_CE_FLOPS[dtype] and c["N"] * c["V"] <= MAX_CE_LOGITS
                    and c["H"] * c["V"] <= MAX_WEIGHT):
                return c
        else:
            width = _size(rng, 24, 4096)
            bits = rng.choice((32, 8))
            c = {"op": "adamw", "bits": bits, "grad": rng.choice(("f32", "bf16")),
                 "layers": rng.randint(1, 24 if bits == 32 else 5), "width": width,
                 "hidden": _size(rng, width, 4 * width), "copies": rng.random() < 0.5}
            if sum(math.prod(s) for s in shapes(c)) <= MAX_ADAMW:
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


def _views(flat, sizes, align):
    """Views of `flat` with the given sizes, each starting at a multiple of
    `align` elements, as an allocator places them."""
    at = 0
    out = []
    for n in sizes:
        out.append(flat[at:at + n])
        at += -(-n // align) * align
    return out


def _room(sizes, align):
    return sum(-(-n // align) * align for n in sizes)


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    s = {"case": case}
    if case["op"].startswith("ln"):
        # Activations with a mean of their own, as a residual stream has.
        dt, R, D = DTYPES[case["dtype"]], case["R"], case["D"]
        s["x"] = _normal(gen, (R, D), 1.5, 0.25).to(dt)
        s["w"] = _normal(gen, (D,), 0.2, 1.0).to(dt)
        s["b"] = _normal(gen, (D,), 0.1).to(dt)
        if case["op"] == "ln_bwd":
            s["dy"] = _normal(gen, (R, D)).to(dt)
            xf = s["x"].float()
            s["mean"] = xf.mean(dim=1)
            s["rstd"] = 1 / torch.sqrt((xf - s["mean"][:, None]).square().mean(dim=1) + EPS)
    elif case["op"].startswith("ce"):
        # Normalised hidden states; logits of standard deviation 2, and the
        # targets' own logits raised, as in a model that has learned something.
        dt, N, H, V = DTYPES[case["dtype"]], case["N"], case["H"], case["V"]
        w = _normal(gen, (V, H), 2 / math.sqrt(H))
        t = torch.randint(V, (N,), generator=gen, device="cuda")
        s["x"] = _normal(gen, (N, H)).add_(w[t], alpha=0.7).to(dt)
        s["w"] = w.to(dt)
        if case["ignored"]:
            t[torch.rand(N, generator=gen, device="cuda") < case["ignored"]] = IGNORE
        s["target"] = t
    else:
        sh = shapes(case)
        n = [math.prod(x) for x in sh]
        room = _room(n, 64)
        s["step"] = 100
        s["p_flat"] = _normal(gen, (room,), 0.02)
        s["params"] = _views(s["p_flat"], n, 64)
        g = _normal(gen, (room,), 1e-3).to(DTYPES[case["grad"]])
        s["grads"] = _views(g, n, 64)
        s["c_flat"] = torch.zeros(room, dtype=torch.bfloat16, device="cuda") if case["copies"] else None
        s["copies"] = _views(s["c_flat"], n, 64) if case["copies"] else None
        if case["bits"] == 32:
            s["m_flat"] = _normal(gen, (room,), 3e-4)
            s["v_flat"] = _normal(gen, (room,), 1e-3).square_().mul_(0.1)
            s["m"], s["v"] = _views(s["m_flat"], n, 64), _views(s["v_flat"], n, 64)
        else:
            blocks = [-(-k // BLOCK) for k in n]
            mc = torch.randint(-127, 128, (room,), generator=gen, device="cuda").to(torch.int8)
            vc = torch.randint(1, 256, (room,), generator=gen, device="cuda").to(torch.uint8)
            ms = _normal(gen, (_room(blocks, 16),), 1e-4, 1e-3).abs_()
            vs = _normal(gen, (_room(blocks, 16),), 1e-7, 1e-6).abs_()
            s["m"] = list(zip(_views(mc, n, 64), _views(ms, blocks, 16)))
            s["v"] = list(zip(_views(vc, n, 64), _views(vs, blocks, 16)))
    return s


# ---------------------------------------------------------------------------
# The plain forms: elementary operations in 32 bits
# ---------------------------------------------------------------------------

def _plain_ln_fwd(s):
    x = s["x"].float()
    mean = x.sum(dim=1) / x.shape[1]
    dev = x - mean[:, None]
    rstd = 1 / torch.sqrt((dev * dev).sum(dim=1) / x.shape[1] + EPS)
    y = dev * rstd[:, None] * s["w"].float() + s["b"].float()
    return {"y": y.to(s["x"].dtype), "mean": mean, "rstd": rstd}


def _plain_ln_bwd(s):
    x, dy, D = s["x"].float(), s["dy"].float(), s["x"].shape[1]
    xhat = (x - s["mean"][:, None]) * s["rstd"][:, None]
    wdy = dy * s["w"].float()
    c1 = wdy.sum(dim=1, keepdim=True) / D
    c2 = (wdy * xhat).sum(dim=1, keepdim=True) / D
    dx = s["rstd"][:, None] * (wdy - c1 - xhat * c2)
    return {"dx": dx.to(s["x"].dtype), "dw": (dy * xhat).sum(dim=0), "db": dy.sum(dim=0)}


def _plain_ce(s, grad):
    x, w, t = s["x"].float(), s["w"].float(), s["target"]
    valid = t != IGNORE
    at = torch.where(valid, t, 0)[:, None]
    logits = torch.mm(x, w.t())
    top = logits.amax(dim=1, keepdim=True)
    e = torch.exp(logits - top)
    total = e.sum(dim=1, keepdim=True)
    loss = (torch.log(total) + top - logits.gather(1, at))[:, 0]
    loss = torch.where(valid, loss, 0.0)
    if not grad:
        return {"loss": loss}
    p = e.div_(total)
    p.scatter_add_(1, at, torch.full_like(at, -1, dtype=torch.float32))
    count = valid.sum().clamp(min=1).float()
    p.mul_((valid.float() / count)[:, None])
    dt = s["x"].dtype
    return {"loss": loss.sum() / count, "dx": torch.mm(p, w).to(dt), "dw": torch.mm(p.t(), x).to(dt)}


def _blocked(tensors):
    """The tensors' values as rows of BLOCK, each tensor from a row of its own."""
    return torch.cat([torch.nn.functional.pad(t, (0, -t.numel() % BLOCK)) for t in tensors]).view(-1, BLOCK)


def _unblocked(rows, tensors):
    parts = rows.view(-1).split([-(-t.numel() // BLOCK) * BLOCK for t in tensors])
    return [p[:t.numel()] for p, t in zip(parts, tensors)]


def _plain_update(p, g, m, v, step):
    b1, b2 = ADAMW["betas"]
    lr = ADAMW["lr"]
    p = p * (1 - lr * ADAMW["weight_decay"])
    m = m * b1 + g * (1 - b1)
    v = v * b2 + g * (1 - b2) * g
    denom = torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + ADAMW["eps"]
    return p - m / denom * (lr / (1 - b1 ** step)), m, v


def _write(to, flat_parts):
    torch._foreach_copy_(to, flat_parts)


def _plain_adamw(s):
    P, G, copies = s["params"], s["grads"], s["copies"]
    sizes = [t.numel() for t in P]
    if s["case"]["bits"] == 32:
        p, m, v = _plain_update(torch.cat(P), torch.cat(G).float(), torch.cat(s["m"]), torch.cat(s["v"]), s["step"])
        _write(s["m"], list(m.split(sizes)))
        _write(s["v"], list(v.split(sizes)))
        p = list(p.split(sizes))
        out = {"m": s["m_flat"], "v": s["v_flat"]}
    else:
        mc, vc = [c for c, _ in s["m"]], [c for c, _ in s["v"]]
        t = _blocked(mc).float() * (1 / 127)
        m = t * t.abs() * torch.cat([a for _, a in s["m"]])[:, None]
        t = _blocked(vc).float() * (1 / 255)
        t = t * t
        v = t * t * torch.cat([a for _, a in s["v"]])[:, None]
        p, m, v = _plain_update(_blocked(P), _blocked(G).float(), m, v, s["step"])
        ms, vs = m.abs().amax(dim=1), v.amax(dim=1)
        some_m, some_v = torch.where(ms > 0, ms, 1.0)[:, None], torch.where(vs > 0, vs, 1.0)[:, None]
        cm = torch.sign(m) * torch.round(torch.sqrt(m.abs() / some_m) * 127)
        cv = torch.round(torch.sqrt(torch.sqrt(v / some_v)) * 255)
        cv = torch.where((v > 0) & (cv < 1), 1.0, cv)
        counts = [a.numel() for _, a in s["m"]]
        _write([a for _, a in s["m"]], list(ms.split(counts)))
        _write([a for _, a in s["v"]], list(vs.split(counts)))
        _write(mc, _unblocked(cm.to(torch.int8), mc))
        _write(vc, _unblocked(cv.to(torch.uint8), vc))
        t = cm * (1 / 127)
        u = cv * (1 / 255)
        u = u * u
        out = {"m": _unblocked(t * t.abs() * ms[:, None], P), "v": _unblocked(u * u * vs[:, None], P)}
        p = _unblocked(p, P)
    _write(P, p)
    if copies is not None:
        _write(copies, p)
        out["c"] = s["c_flat"]
    return {**out, "p": s["p_flat"]}


def _own(s):
    import tilec
    op = s["case"]["op"]
    if op == "ln_fwd":
        y, mean, rstd = tilec.ext.layer_norm(s["x"], s["w"], s["b"], eps=EPS)
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "ln_bwd":
        dx, dw, db = tilec.ext.layer_norm_backward(s["dy"], s["x"], s["mean"], s["rstd"], s["w"])
        return {"dx": dx, "dw": dw, "db": db}
    if op == "ce_loss":
        return {"loss": tilec.ext.linear_cross_entropy(s["x"], s["w"], s["target"], reduction="none",
                                                       ignore_index=IGNORE)}
    if op == "ce_grad":
        loss, dx, dw = tilec.ext.linear_cross_entropy_grad(s["x"], s["w"], s["target"], reduction="mean",
                                                           ignore_index=IGNORE)
        return {"loss": loss, "dx": dx, "dw": dw}
    tilec.ext.adamw_step(s["params"], s["grads"], s["m"], s["v"], step=s["step"], copies=s["copies"], **ADAMW)
    if s["case"]["bits"] == 32:
        out = {"m": s["m_flat"], "v": s["v_flat"]}
    else:  # the values that the 8-bit states stand for
        out = {"m": tilec.ext.adamw_values(s["m"]), "v": tilec.ext.adamw_values(s["v"])}
    if s["copies"] is not None:
        out["c"] = s["c_flat"]
    return {**out, "p": s["p_flat"]}


def run(state):
    op = state["case"]["op"]
    if op == "adamw":
        state["step"] += 1
    if own:
        return _own(state)
    if op == "ln_fwd":
        return _plain_ln_fwd(state)
    if op == "ln_bwd":
        return _plain_ln_bwd(state)
    if op == "adamw":
        return _plain_adamw(state)
    return _plain_ce(state, op == "ce_grad")


# ---------------------------------------------------------------------------
# 64-bit values, from the definitions
# ---------------------------------------------------------------------------

def _exact_ln(s):
    x = s["x"].double()
    if s["case"]["op"] == "ln_fwd":
        var, mean = torch.var_mean(x, dim=1, unbiased=False)
        rstd = (var + EPS).rsqrt()
        return {"y": (x - mean[:, None]) * rstd[:, None] * s["w"].double() + s["b"].double(), "mean": mean,
                "rstd": rstd}
    # dx = rstd J wdy with J the projection off the constant and off xhat.
    dy, rstd = s["dy"].double(), s["rstd"].double()[:, None]
    xhat = (x - s["mean"].double()[:, None]) * rstd
    wdy = dy * s["w"].double()
    dx = rstd * (wdy - wdy.mean(dim=1, keepdim=True) - xhat * (wdy * xhat).mean(dim=1, keepdim=True))
    return {"dx": dx, "dw": torch.einsum("rd,rd->d", dy, xhat), "db": dy.sum(dim=0)}


def _exact_ce(s):
    x, w, t = s["x"].double(), s["w"].double(), s["target"]
    keep = (t != IGNORE).nonzero()[:, 0]
    logits = torch.mm(x[keep], w.t().contiguous())
    rows = torch.arange(len(keep), device=t.device)
    logp = torch.log_softmax(logits, dim=1)
    loss = torch.zeros(len(t), dtype=torch.float64, device=t.device)
    loss[keep] = -logp[rows, t[keep]]
    if s["case"]["op"] == "ce_loss":
        return {"loss": loss}
    count = max(1, len(keep))
    d = logp.exp_()
    d[rows, t[keep]] -= 1
    d /= count
    dx = torch.zeros_like(x)
    dx[keep] = torch.mm(d, w)
    return {"loss": loss.sum() / count, "dx": dx, "dw": torch.mm(d.t().contiguous(), x[keep])}


def _exact_update(p, g, m, v, step):
    b1, b2 = ADAMW["betas"]
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g ** 2
    mhat, vhat = m / (1 - b1 ** step), v / (1 - b2 ** step)
    p = p - ADAMW["lr"] * (ADAMW["weight_decay"] * p + mhat / (vhat.sqrt() + ADAMW["eps"]))
    return p, m, v


def _exact_adamw(s):
    step = s["step"] + 1
    if s["case"]["bits"] == 32:
        # Over the whole storage: what lies between the tensors stays.
        p, m, v = s["p_flat"].double(), s["m_flat"].double(), s["v_flat"].double()
        out = {"p": p, "m": m, "v": v}
        c = s["c_flat"].double() if s["copies"] is not None else None
        at = 0
        for i, t in enumerate(s["params"]):
            n = t.numel()
            i0 = slice(at, at + n)
            p[i0], m[i0], v[i0] = _exact_update(p[i0], s["grads"][i].double(), m[i0], v[i0], step)
            if c is not None:
                c[i0] = p[i0]
            at += -(-n // 64) * 64
        return {**out, "c": c} if c is not None else out
    p_flat = s["p_flat"].double()
    c_flat = s["c_flat"].double() if s["copies"] is not None else None
    ms, vs, at = [], [], 0
    for i, t in enumerate(s["params"]):
        n = t.numel()

        def spread(scales):
            return scales.double().repeat_interleave(BLOCK)[:n]

        def largest(x):
            full = torch.zeros(-(-n // BLOCK) * BLOCK, dtype=torch.float64, device=x.device)
            full[:n] = x
            return spread(full.view(-1, BLOCK).max(dim=1).values)

        cm, cv = s["m"][i][0].double() / 127, s["v"][i][0].double() / 255
        p, m, v = _exact_update(t.double(), s["grads"][i].double(), cm.sign() * cm ** 2 * spread(s["m"][i][1]),
                                cv ** 4 * spread(s["v"][i][1]), step)
        top = largest(m.abs())
        ms.append(m.sign() * ((m.abs() / top).sqrt() * 127).round().div(127) ** 2 * top)
        top = largest(v)
        vs.append(((v / top) ** 0.25 * 255).round().clamp(min=1).div(255) ** 4 * top)
        p_flat[at:at + n] = p
        if c_flat is not None:
            c_flat[at:at + n] = p
        at += -(-n // 64) * 64
    out = {"p": p_flat, "m": ms, "v": vs}
    return {**out, "c": c_flat} if c_flat is not None else out


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"].startswith("ln"):
        return _exact_ln(s)
    return _exact_ce(s) if case["op"].startswith("ce") else _exact_adamw(s)


# ---------------------------------------------------------------------------
# Work
# ---------------------------------------------------------------------------

def work(case):
    if case["op"].startswith("ln"):
        R, D, esz = case["R"], case["D"], 4 if case["dtype"] == "f32" else 2
        if case["op"] == "ln_fwd":
            return {"bytes": 2 * R * D * esz + 2 * D * esz + 8 * R, "flops": 8 * R * D}
        return {"bytes": 3 * R * D * esz + D * esz + 8 * D + 8 * R, "flops": 14 * R * D}
    if case["op"].startswith("ce"):
        N, H, V, esz = case["N"], case["H"], case["V"], 4 if case["dtype"] == "f32" else 2
        inputs = (N * H + V * H) * esz + 8 * N
        if case["op"] == "ce_loss":
            return {"bytes": inputs + 4 * N, "flops": 2 * N * H * V}
        return {"bytes": inputs + (N * H + V * H) * esz + 4, "flops": 6 * N * H * V}
    n = sum(math.prod(x) for x in shapes(case))
    per = 8 + (4 if case["grad"] == "f32" else 2) + (2 if case["copies"] else 0)
    if case["bits"] == 32:
        return {"bytes": n * (per + 16), "flops": 14 * n}
    # Codes and scales read and written, and the states' values written out.
    return {"bytes": n * (per + 4 + 16 / BLOCK + 8), "flops": 30 * n}
