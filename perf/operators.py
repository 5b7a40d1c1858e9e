"""The cell-training operators as measured workloads: group norm with an activation (channels
last), the gated feed-forward block, and distillation from a teacher's top logits.

`listed()` gives the fixed cases and `draw(rng)` more of the same ranges; `prepare(case, seed)`
makes the inputs of one pass on the GPU, and `run(state)` computes it: in elementary torch
operations in 32 bits where `own` is false, through ncas_b200.operators where it is true.
`exact(case, seed)` computes the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
EPS = 1e-5


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one 9x9 board's state between two steps of a normalised cell: the call's own latency
        dict(name="norm board", op="norm", n=1, cells=81, channels=64, groups=8, act="silu",
             dtype="float32", mask=False, train=False),
        # 1000 boards x 8 trials of the 9x9 boards with 64 channels, one training pass
        dict(name="norm boards train", op="norm", n=8000, cells=81, channels=64, groups=8, act="silu",
             dtype="float32", mask=False, train=True),
        # mazes of several sizes padded to 59x59 (cells outside a maze masked), 32 channels
        dict(name="norm padded mazes train", op="norm", n=250, cells=3481, channels=32, groups=4,
             act="relu", dtype="float16", mask=True, train=True),
        # wide feature maps: samples too large for one multiprocessor
        dict(name="norm maps train", op="norm", n=16, cells=16384, channels=512, groups=32, act="silu",
             dtype="bfloat16", mask=False, train=True),
        # one token through a wide block: bound by reading the weights
        dict(name="ffn token", op="ffn", rows=1, d_in=2048, hidden=8192, d_out=2048, act="silu",
             dtype="bfloat16", bias=False, train=False),
        # the cell update of 1000 9x9 boards: perception 4 x 64 -> hidden 256 -> 64 channels
        dict(name="ffn cells train", op="ffn", rows=81000, d_in=256, hidden=256, d_out=64, act="silu",
             dtype="bfloat16", bias=True, train=True),
        # odd sizes everywhere, with biases
        dict(name="ffn odd train", op="ffn", rows=1999, d_in=1001, hidden=2730, d_out=1001, act="gelu",
             dtype="float16", bias=True, train=True),
        # a long batch through a wide block, forward and backward
        dict(name="ffn wide train", op="ffn", rows=8192, d_in=4096, hidden=16384, d_out=4096, act="silu",
             dtype="bfloat16", bias=False, train=True),
        # one 9x9 board's readout of 9 digits against the teacher's top 4
        dict(name="distill board", op="distill", rows=81, classes=9, top=4, temperature=2.0,
             dtype="float32", train=True),
        # a 2-class readout of 1000 30x30 mazes
        dict(name="distill mazes", op="distill", rows=900000, classes=2, top=2, temperature=2.0,
             dtype="bfloat16", train=True),
        # an odd vocabulary: rows that start on no 16-byte boundary
        dict(name="distill odd vocabulary", op="distill", rows=2047, classes=32003, top=20,
             temperature=1.5, dtype="float16", train=True),
        # a long batch over a large vocabulary
        dict(name="distill large vocabulary", op="distill", rows=8192, classes=131072, top=64,
             temperature=1.0, dtype="bfloat16", train=True),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("norm", "ffn", "distill"))
    if op == "norm":
        groups = rng.choice((1, 2, 3, 4, 8, 16, 32))
        per = log_int(rng, 1, max(1, 512 // groups))
        channels = groups * per
        cells = log_int(rng, -(-64 // per), 40401)  # 64 values a group at least
        n = log_int(rng, 1, max(1, min(20000, 2 ** 26 // (cells * channels))))
        return dict(op=op, n=n, cells=cells, channels=channels, groups=groups,
                    act=rng.choice(("none", "relu", "silu", "gelu")), dtype=rng.choice(sorted(DTYPES)),
                    mask=rng.random() < 0.4, train=rng.random() < 0.6)
    if op == "ffn":
        d_in, hidden, d_out = log_int(rng, 16, 4096), log_int(rng, 16, 16384), log_int(rng, 16, 4096)
        if rng.random() < 0.5:  # a multiple of 8, as most programs have
            d_in, hidden, d_out = (8 * max(2, v // 8) for v in (d_in, hidden, d_out))
        rows = log_int(rng, 1, max(1, min(100000, 2 ** 39 // (hidden * (2 * d_in + d_out)))))
        return dict(op=op, rows=rows, d_in=d_in, hidden=hidden, d_out=d_out,
                    act=rng.choice(("relu", "silu", "gelu", "sigmoid")),
                    dtype=rng.choice(("bfloat16", "float16")), bias=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    classes = log_int(rng, 2, 131072)
    rows = log_int(rng, 1, max(1, min(1000000, 2 ** 29 // classes)))
    return dict(op=op, rows=rows, classes=classes, top=log_int(rng, 1, min(classes, 128)),
                temperature=rng.choice((0.5, 1.0, 2.0, 4.0)), dtype=rng.choice(sorted(DTYPES)),
                train=rng.random() < 0.7)


# ----------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return torch.randn(shape, generator=gen, device=DEVICE).mul_(scale).add_(shift).to(to)

    state = {"case": case}
    grads = case["train"] and case["op"] != "distill"
    if case["op"] == "norm":
        n, cells, c = case["n"], case["cells"], case["channels"]
        state["x"] = normal(n, cells, c, scale=1.5, shift=0.25)
        state["weight"] = normal(c, scale=0.2, shift=1.0, to=torch.float32)
        state["bias"] = normal(c, scale=0.2, to=torch.float32)
        state["mask"] = None
        if case["mask"]:  # the first sample is whole, the others keep a prefix of their cells or none
            keep = torch.rand((n, 1), generator=gen, device=DEVICE).mul_(1.1).sub_(0.05)
            keep[0] = 1
            state["mask"] = torch.arange(cells, device=DEVICE)[None] < keep * cells
        state["inputs"] = [state[k] for k in ("x", "weight", "bias")]
        if grads:
            state["dy"] = normal(n, cells, c)
    elif case["op"] == "ffn":
        t, d, f, o = case["rows"], case["d_in"], case["hidden"], case["d_out"]
        state["x"] = normal(t, d)
        state["w_gate"] = normal(f, d, scale=d ** -0.5)
        state["w_up"] = normal(f, d, scale=d ** -0.5)
        state["w_down"] = normal(o, f, scale=f ** -0.5)
        names = ["x", "w_gate", "w_up", "w_down"]
        for name, size in (("b_gate", f), ("b_up", f), ("b_down", o)):
            state[name] = normal(size, scale=0.1) if case["bias"] else None
            names += [name] if case["bias"] else []
        state["inputs"] = [state[k] for k in names]
        if grads:
            state["dy"] = normal(t, o)
    else:
        r, v, k = case["rows"], case["classes"], case["top"]
        logits = torch.randn((r, v), generator=gen, device=DEVICE).mul_(2.0)
        teacher = torch.randn((r, v), generator=gen, device=DEVICE).add_(logits)
        values, index = teacher.topk(k, dim=1)
        del teacher
        # some rows hold fewer entries (the rest are -1), some none; some rows have no weight
        kept = torch.randint(0, k + 1, (r, 1), generator=gen, device=DEVICE)
        short = torch.rand((r, 1), generator=gen, device=DEVICE) < 0.1
        gone = short & (torch.arange(k, device=DEVICE)[None] >= kept)
        state["logits"] = logits.to(dtype)
        state["teacher"] = values.to(dtype)
        state["index"] = index.masked_fill(gone, -1).to(torch.int32)
        weight = torch.rand((r,), generator=gen, device=DEVICE).add_(0.5)
        state["weight"] = torch.where(torch.rand((r,), generator=gen, device=DEVICE) < 0.1,
                                      torch.zeros_like(weight), weight)
        return state
    if grads:
        for t in state["inputs"]:
            t.requires_grad_(True)
    return state


# ------------------------------------------------------------------- the plain forms, in 32 bits
def act_and_slope(z, act):
    """The activation and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp_min(0), (z > 0).to(z.dtype)
    if act == "sigmoid":
        s = 1 / (1 + torch.exp(-z))
        return s, s * (1 - s)
    if act == "silu":
        s = 1 / (1 + torch.exp(-z))
        return z * s, s * (1 + z * (1 - s))
    cdf = 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))
    return z * cdf, cdf + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)


def plain_norm(s):
    case = s["case"]
    n, cells, c = s["x"].shape
    g = case["groups"]
    x = s["x"].float().reshape(n, cells, g, c // g)
    weight, bias = s["weight"].reshape(g, c // g), s["bias"].reshape(g, c // g)
    if s["mask"] is None:
        count = torch.full((n, 1, 1, 1), float(cells * (c // g)), device=x.device)
        on = torch.ones((1, 1, 1, 1), device=x.device)
    else:
        on = s["mask"].float()[:, :, None, None]
        count = (on.sum(1, keepdim=True) * (c // g)).clamp_min(1)
    mean = (x * on).sum((1, 3), keepdim=True) / count
    rstd = torch.rsqrt(((x - mean).square() * on).sum((1, 3), keepdim=True) / count + EPS)
    hat = (x - mean) * rstd
    y, slope = act_and_slope(hat * weight + bias, case["act"])
    out = {"y": (y * on).reshape(n, cells, c).to(s["x"].dtype)}
    if case["train"]:
        dz = s["dy"].float().reshape(x.shape) * slope * on
        out["dweight"] = (dz * hat).sum((0, 1)).reshape(c)
        out["dbias"] = dz.sum((0, 1)).reshape(c)
        dh = dz * weight
        a, b = dh.sum((1, 3), keepdim=True), (dh * hat).sum((1, 3), keepdim=True)
        dx = (dh - (a + hat * b) / count) * rstd * on
        out["dx"] = dx.reshape(n, cells, c).to(s["x"].dtype)
    return out


def plain_ffn(s):
    case, dtype = s["case"], s["x"].dtype
    x, wg, wu, wd = (s[k].float() for k in ("x", "w_gate", "w_up", "w_down"))
    gate, up = x @ wg.t(), x @ wu.t()
    if case["bias"]:
        gate, up = gate + s["b_gate"].float(), up + s["b_up"].float()
    a, slope = act_and_slope(gate, case["act"])
    h = a * up
    y = h @ wd.t()
    if case["bias"]:
        y = y + s["b_down"].float()
    out = {"y": y.to(dtype)}
    if case["train"]:
        dy = s["dy"].float()
        dh = dy @ wd
        out["dw_down"] = (dy.t() @ h).to(dtype)
        dgate, dup = dh * up * slope, dh * a
        out["dx"] = (dgate @ wg + dup @ wu).to(dtype)
        out["dw_gate"], out["dw_up"] = (dgate.t() @ x).to(dtype), (dup.t() @ x).to(dtype)
        if case["bias"]:
            out["db_gate"], out["db_up"] = dgate.sum(0).to(dtype), dup.sum(0).to(dtype)
            out["db_down"] = dy.sum(0).to(dtype)
    return out


def plain_distill(s):
    case, tau = s["case"], s["case"]["temperature"]
    z = s["logits"].float() / tau
    valid = s["index"] >= 0
    at = s["index"].clamp_min(0).long()
    top = z.amax(1, keepdim=True)
    lse = top + torch.exp(z - top).sum(1, keepdim=True).log()
    t = (s["teacher"].float() / tau).masked_fill(~valid, -math.inf)
    some = valid.any(1, keepdim=True) & (s["weight"] != 0)[:, None]
    t = t.masked_fill(~some, 0.0)
    t = t - t.amax(1, keepdim=True)
    logp = t - torch.exp(t).sum(1, keepdim=True).log()
    p = torch.exp(logp) * (valid & some)
    logq = torch.gather(z, 1, at) - lse
    gap = (p * torch.where(p > 0, logp - logq, torch.zeros_like(logp))).sum(1)
    out = {"loss": gap * s["weight"] * tau * tau}
    if case["train"]:
        d = torch.exp(z - lse) * some
        d.scatter_add_(1, at, -p)
        out["dlogits"] = (d * (s["weight"][:, None] * tau)).to(s["logits"].dtype)
    return out


# --------------------------------------------------------------------------- one pass of a case
def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"norm": plain_norm, "ffn": plain_ffn, "distill": plain_distill}[case["op"]](state)
    from ncas_b200 import operators as ops

    if case["op"] == "distill":
        call = ops.distill_loss_and_grad if case["train"] else ops.distill_loss
        got = call(state["logits"], state["teacher"], state["index"], temperature=case["temperature"],
                   weight=state["weight"], reduction="none")
        return {"loss": got[0], "dlogits": got[1]} if case["train"] else {"loss": got}
    if case["op"] == "norm":
        y = ops.group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], eps=EPS,
                               act=case["act"], mask=state["mask"])
        names = ("dx", "dweight", "dbias")
    else:
        y = ops.gated_ffn(state["x"], state["w_gate"], state["w_up"], state["w_down"], state["b_gate"],
                          state["b_up"], state["b_down"], act=case["act"])
        names = ("dx", "dw_gate", "dw_up", "dw_down", "db_gate", "db_up", "db_down")
    out = {"y": y.detach()}
    if case["train"]:
        out.update(zip(names, torch.autograd.grad(y, state["inputs"], state["dy"])))
    return out


def work(case):
    size = torch.tensor([], dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "norm":
        n, cells, c = case["n"], case["cells"], case["channels"]
        # x in, y out; with gradients dy in and dx out too (x is one input, read once)
        data = n * cells * c * size * (4 if case["train"] else 2)
        mask = n * cells if case["mask"] else 0
        return {"bytes": data + mask + 4 * c * (4 if case["train"] else 2),
                "flops": n * cells * c * (30 if case["train"] else 12)}
    if case["op"] == "ffn":
        t, d, f, o = case["rows"], case["d_in"], case["hidden"], case["d_out"]
        weights = 2 * f * d + f * o + (2 * f + o if case["bias"] else 0)
        fwd = 2 * t * f * (2 * d + o)
        if not case["train"]:
            return {"bytes": size * (t * (d + o) + weights), "flops": fwd}
        return {"bytes": 2 * size * (t * (d + o) + weights), "flops": 3 * fwd}
    r, v, k = case["rows"], case["classes"], case["top"]
    return {"bytes": r * v * size * (2 if case["train"] else 1) + r * k * (size + 4) + 8 * r,
            "flops": r * v * (6 if case["train"] else 4)}


# ------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "distill":
        return exact_distill(case, s)
    names = ("x", "weight", "bias") if case["op"] == "norm" else (
        "x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")
    v = {k: s[k].detach().double().requires_grad_(case["train"]) for k in names if s[k] is not None}
    acts = {"none": lambda z: z, "relu": lambda z: torch.where(z > 0, z, 0.0 * z),
            "sigmoid": lambda z: torch.sigmoid(z), "silu": lambda z: z * torch.sigmoid(z),
            "gelu": lambda z: 0.5 * z * torch.erfc(-z / 2 ** 0.5)}
    act = acts[case["act"]]
    if case["op"] == "norm":
        n, cells, c = v["x"].shape
        per = c // case["groups"]
        inside = torch.ones((n, cells), device=DEVICE, dtype=torch.bool) if s["mask"] is None else s["mask"]
        share = inside.double() / (inside.sum(1, keepdim=True).double().clamp_min(1) * per)
        pool = torch.block_diag(*[torch.ones((per, per), dtype=torch.float64, device=DEVICE)] * case["groups"])
        mean = torch.einsum("nl,nlc->nc", share, v["x"]) @ pool
        gap = v["x"] - mean[:, None]
        var = torch.einsum("nl,nlc->nc", share, gap ** 2) @ pool
        y = act(gap / (var[:, None] + EPS).sqrt() * v["weight"] + v["bias"])
        y = torch.where(inside[:, :, None], y, torch.zeros((), dtype=y.dtype, device=DEVICE))
    else:
        lin = torch.nn.functional.linear
        y = lin(act(lin(v["x"], v["w_gate"], v.get("b_gate"))) * lin(v["x"], v["w_up"], v.get("b_up")),
                v["w_down"], v.get("b_down"))
    out = {"y": y.detach()}
    if case["train"]:
        got = torch.autograd.grad(y, list(v.values()), s["dy"].double())
        out.update({"d" + k: g for k, g in zip(v, got)})
    return out


def exact_distill(case, s):
    tau = case["temperature"]
    r, v = s["logits"].shape
    loss = torch.zeros(r, dtype=torch.float64, device=DEVICE)
    grad = torch.zeros((r, v), dtype=torch.float64, device=DEVICE) if case["train"] else None
    step = max(1, 2 ** 27 // v)
    for a in range(0, r, step):
        rows = slice(a, min(r, a + step))
        index, weight = s["index"][rows].long(), s["weight"][rows].double()
        logq = torch.log_softmax(s["logits"][rows].double() / tau, 1)
        t = torch.where(index >= 0, s["teacher"][rows].double() / tau, -torch.inf)
        live = (index >= 0).any(1) & (weight != 0)
        p = torch.where(live[:, None], torch.softmax(t, 1), 0.0).nan_to_num(0.0)
        q = logq.gather(1, index.clamp(min=0))
        loss[rows] = weight * tau ** 2 * (torch.special.xlogy(p, p) - p * q).sum(1)
        if grad is not None:
            full = torch.zeros_like(logq).scatter_add_(1, index.clamp(min=0), p)
            grad[rows] = (logq.exp() * live[:, None] - full) * (weight * tau)[:, None]
    return {"loss": loss, "dlogits": grad} if case["train"] else {"loss": loss}
