"""The student's further operators as measured workloads: a gated scan along the lines of a board or a
long sequence, the orthogonalised update of a matrix (Newton-Schulz products), and sampled answers
(temperature, top-k, top-p, min-p).

`listed()` gives the fixed cases and `draw(rng)` more of the same ranges; `prepare(case, seed)`
makes the inputs of one pass on the GPU, and `run(state)` computes it: in elementary torch
operations where `own` is false, through ncas_b200.operators where it is true.  `exact(case, seed)`
computes the same outputs from the definitions in 64 bits.
"""

import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
COEFFICIENTS = (3.4445, -4.775, 2.0315)
EPS = 1e-7


# ------------------------------------------------------------------------------------ the cases
def listed():
    return [
        # one step of 64 running sequences (the state goes in and comes out): the call's own latency
        dict(name="scan token", op="scan", n=64, m=1, t=1, c=2048, axis=1, dtype="bfloat16", reverse=False,
             mask=False, state=True, train=False),
        # 1000 boards x 8 trials of the 9x9 boards with 64 channels, along the columns, one training pass
        dict(name="scan boards train", op="scan", n=8000, m=9, t=9, c=64, axis=1, dtype="bfloat16", reverse=False,
             mask=False, state=False, train=True),
        # mazes of several sizes padded to 59x59 (cells outside a maze masked), along the rows from their ends
        dict(name="scan padded mazes train", op="scan", n=250, m=59, t=59, c=32, axis=2, dtype="float16", reverse=True,
             mask=True, state=False, train=True),
        # one long sequence: few channels at a time, so the long axis has to be split
        dict(name="scan long train", op="scan", n=1, m=1, t=100001, c=1024, axis=1, dtype="bfloat16", reverse=False,
             mask=False, state=True, train=True),
        # the gate matrix of a cell with 64 channels
        dict(name="orthogonalize cell", op="ortho", batch=1, rows=256, cols=256, dtype="bfloat16", steps=5),
        # the matrices of a dozen layers of one shape in one call
        dict(name="orthogonalize stack", op="ortho", batch=12, rows=1024, cols=1024, dtype="bfloat16", steps=5),
        # odd sizes, taller than wide
        dict(name="orthogonalize odd", op="ortho", batch=1, rows=2730, cols=1001, dtype="float16", steps=5),
        # the gate matrix of a wide block
        dict(name="orthogonalize wide", op="ortho", batch=1, rows=4096, cols=16384, dtype="bfloat16", steps=5),
        # 128 candidate answers of one 9x9 board's readout of 9 digits
        dict(name="sample board", op="sample", rows=81, classes=9, draws=128, temperature=0.7, top_k=0, top_p=0.95,
             min_p=0.0, dtype="float32"),
        # one answer for every cell of 1000 30x30 mazes (2 classes)
        dict(name="sample mazes", op="sample", rows=900000, classes=2, draws=1, temperature=1.0, top_k=0, top_p=1.0,
             min_p=0.05, dtype="bfloat16"),
        # an odd vocabulary (rows that start on no 16-byte boundary), the 50 largest, of which 0.9 of the mass
        dict(name="sample odd vocabulary", op="sample", rows=2047, classes=32003, draws=1, temperature=0.8, top_k=50,
             top_p=0.9, min_p=0.0, dtype="float16"),
        # a batch over a large vocabulary, 0.95 of the whole mass
        dict(name="sample large vocabulary", op="sample", rows=1024, classes=131072, draws=1, temperature=0.7, top_k=0,
             top_p=0.95, min_p=0.0, dtype="bfloat16"),
    ]


def log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("scan", "ortho", "sample"))
    if op == "scan":
        c = log_int(rng, 1, 4096)
        if rng.random() < 0.5:  # a multiple of 8, as most programs have
            c = 8 * max(1, c // 8)
        t = log_int(rng, 1, min(100001, 2 ** 26 // c))
        lines = log_int(rng, 1, max(1, min(100000, 2 ** 26 // (c * t))))
        m = log_int(rng, 1, min(lines, 64))
        return dict(op=op, n=max(1, lines // m), m=m, t=t, c=c, axis=rng.choice((1, 2)), dtype=rng.choice(sorted(DTYPES)),
                    reverse=rng.random() < 0.5, mask=rng.random() < 0.3, state=rng.random() < 0.5,
                    train=rng.random() < 0.6)
    if op == "ortho":
        small = log_int(rng, 8, 3500)
        large = log_int(rng, small, min(16384, 2 ** 26 // small))
        if rng.random() < 0.5:
            small, large = 8 * max(1, small // 8), 8 * max(1, large // 8)
        rows, cols = (small, large) if rng.random() < 0.5 else (large, small)
        batch = log_int(rng, 1, max(1, min(64, 2 ** 24 // (rows * cols))))
        return dict(op=op, batch=batch, rows=rows, cols=cols, dtype=rng.choice(("bfloat16", "float16")),
                    steps=rng.choice((3, 5, 5, 6)))
    classes = log_int(rng, 2, 131072)
    rows = log_int(rng, 1, max(1, min(1000000, 2 ** 27 // classes)))
    draws = log_int(rng, 1, max(1, min(128, 2 ** 20 // rows, 2 ** 24 // classes)))
    return dict(op=op, rows=rows, classes=classes, draws=draws, temperature=rng.choice((0.5, 0.7, 1.0, 1.5)),
                top_k=rng.choice((0, 0, 1, 20, 50, 1000)), top_p=rng.choice((1.0, 1.0, 0.5, 0.9, 0.95)),
                min_p=rng.choice((0.0, 0.0, 0.02, 0.1)), dtype=rng.choice(sorted(DTYPES)))


# ----------------------------------------------------------------------------------- the inputs
def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(seed)
    dtype = DTYPES[case["dtype"]]

    def normal(*shape, scale=1.0, shift=0.0, to=dtype):
        return torch.randn(shape, generator=gen, device=DEVICE).mul_(scale).add_(shift).to(to)

    def uniform(*shape):
        return torch.rand(shape, generator=gen, device=DEVICE)

    state = {"case": case}
    if case["op"] == "scan":
        n, m, t, c, axis = (case[k] for k in ("n", "m", "t", "c", "axis"))
        shape = (n, t, m) if axis == 1 else (n, m, t)  # the line runs along `axis`
        state["x"] = normal(*shape, c)
        # channels forget at different speeds, as trained gates do: half-lives of one cell to hundreds
        gate = torch.randn((*shape, c), generator=gen, device=DEVICE)
        state["gate"] = gate.add_(uniform(c).mul_(6.0)).to(dtype)
        del gate
        state["state"] = normal(n, m, c, to=torch.float32) if case["state"] else None
        state["mask"] = None
        if case["mask"]:  # the first board is whole, the others keep a corner of their own size or nothing
            keep = uniform(n, 2).mul_(1.1).sub_(0.05)
            keep[0] = 1
            rows = torch.arange(shape[1], device=DEVICE)[None] < keep[:, :1] * shape[1]
            cols = torch.arange(shape[2], device=DEVICE)[None] < keep[:, 1:] * shape[2]
            state["mask"] = rows[:, :, None] & cols[:, None]
        state["inputs"] = [state[k] for k in ("x", "gate", "state") if state[k] is not None]
        if case["train"]:
            state["dy"] = normal(*shape, c)
            state["dlast"] = normal(n, m, c, to=torch.float32)
            for v in state["inputs"]:
                v.requires_grad_(True)
    elif case["op"] == "ortho":
        b, m, n = case["batch"], case["rows"], case["cols"]
        # a momentum: few strong directions over noise, of a gradient's size
        rank = max(1, min(m, n) // 16)
        strong = torch.matmul(normal(b, m, rank, to=torch.float32), normal(b, rank, n, to=torch.float32))
        strong.mul_(rank ** -0.5).add_(normal(b, m, n, scale=0.5, to=torch.float32)).mul_(0.01)
        state["matrix"] = (strong[0] if b == 1 else strong).to(dtype)
    else:
        r, v, d = case["rows"], case["classes"], case["draws"]
        # logits of a trained model: a few classes far above a broad rest
        logits = torch.randn((r, v), generator=gen, device=DEVICE).mul_(1.5)
        few = max(1, min(v // 2, 64))
        at = torch.randint(0, v, (r, 1), generator=gen, device=DEVICE)
        at = (at + torch.arange(few, device=DEVICE) * (v // few)) % v  # distinct
        logits.scatter_(1, at, torch.randn((r, few), generator=gen, device=DEVICE).mul_(2.0).add_(4.0 if v > 100 else 0.0))
        # a tenth of the rows may not answer with some classes, the last of several rows with none at all
        some = (uniform(r, 1) < 0.1).float() * 0.3
        logits.masked_fill_(uniform(r, v) < some, -math.inf)
        if r > 8:
            logits[-1] = -math.inf
        state["logits"] = logits.to(dtype)
        state["uniforms"] = uniform(r, d)
    return state


# ------------------------------------------------------------------------------- the plain forms
def doubling(a, b):
    """h_t = a_t h_{t-1} + b_t with h_{-1} = 0 along dim 1, in log2(T) passes over the whole."""
    a, b = a.clone(), b.clone()
    s, t = 1, a.shape[1]
    while s < t:
        b[:, s:] = b[:, s:] + a[:, s:] * b[:, :-s]
        a[:, s:] = a[:, s:] * a[:, :-s]
        s *= 2
    return b


def lines(v, case):
    """(n, ..., c) with the line along `axis`, and from its end, to (n, t, m, c) from the start."""
    if v is None:
        return None
    v = v if case["axis"] == 1 else v.transpose(1, 2)
    return v.flip(1) if case["reverse"] else v


def plain_scan(s):
    case, dtype = s["case"], s["x"].dtype
    x, gate = lines(s["x"], case).float(), lines(s["gate"], case).float()
    a = 1 / (1 + torch.exp(-gate))
    keep = 1 / (1 + torch.exp(gate))  # 1 - a
    on = None if s["mask"] is None else lines(s["mask"], case)[..., None]
    if on is not None:
        a, keep = torch.where(on, a, 1.0), torch.where(on, keep, 0.0)
    h0 = torch.zeros_like(x[:, 0]) if s["state"] is None else s["state"]
    b = keep * x
    b[:, 0] = b[:, 0] + a[:, 0] * h0
    h = doubling(a, b)
    back = lambda v: lines(v, {**case, "axis": 1}) if case["axis"] == 1 else lines(v, {**case, "axis": 1}).transpose(1, 2)  # noqa: E731
    out = {"y": back(h if on is None else h * on).to(dtype).contiguous(), "last": h[:, -1].contiguous()}
    if case["train"]:
        dy = lines(s["dy"], case).float()
        g = dy if on is None else dy * on
        g = g.clone()
        g[:, -1] = g[:, -1] + s["dlast"]
        after = torch.cat([a[:, 1:], torch.zeros_like(a[:, :1])], 1)
        g = doubling(after.flip(1), g.flip(1)).flip(1)
        before = torch.cat([h0[:, None], h[:, :-1]], 1)
        out["dx"] = back(keep * g).to(dtype).contiguous()
        out["dgate"] = back(g * (before - x) * a * keep).to(dtype).contiguous()
        if s["state"] is not None:
            out["dstate"] = (a[:, 0] * g[:, 0]).contiguous()
    return out


def plain_ortho(s):
    a, b, c = COEFFICIENTS
    x = s["matrix"].float()
    tall = x.shape[-2] > x.shape[-1]
    x = x.transpose(-1, -2) if tall else x
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + EPS)
    for _ in range(s["case"]["steps"]):
        p = x @ x.transpose(-1, -2)
        x = a * x + (b * p + c * (p @ p)) @ x
    x = x.transpose(-1, -2) if tall else x
    return {"x": x.to(s["matrix"].dtype).contiguous()}


def plain_sample(s):
    # 64 bits: a draw falls next to the border of two classes now and then
    case, v = s["case"], s["logits"].shape[1]
    z = s["logits"].double()
    top = z.amax(1, keepdim=True)
    w = torch.exp((z - top.clamp_min(-1e300)) / case["temperature"])
    if case["top_k"] or case["top_p"] < 1:
        _, order = torch.sort(z, dim=1, descending=True, stable=True)
        sorted_w = torch.gather(w, 1, order)
        if case["top_k"]:
            sorted_w[:, case["top_k"]:] = 0
        before = sorted_w.cumsum(1) - sorted_w
        keep = sorted_w > 0
        if case["top_p"] < 1:
            keep = keep & (before < case["top_p"] * sorted_w.sum(1, keepdim=True))
        w = torch.zeros_like(w).scatter_(1, order, torch.where(keep, sorted_w, 0.0))
        del order, sorted_w, before, keep
    if case["min_p"] > 0:
        w = torch.where(w >= case["min_p"], w, 0.0)
    c = w.cumsum(1)
    total = c[:, -1:]
    last = v - 1 - (w.flip(1) > 0).to(torch.uint8).argmax(1, keepdim=True)
    u, tokens = s["uniforms"].double() * total, []
    step = max(1, 2 ** 27 // max(1, c.numel()))  # draws at a time
    for i in range(0, u.shape[1], step):
        tokens.append((c[:, None] <= u[:, i:i + step, None]).sum(2))
    tokens = torch.minimum(torch.cat(tokens, 1), last)
    none = total == 0
    probs = torch.gather(w, 1, tokens) / torch.where(none, 1.0, total)
    return {"tokens": torch.where(none, -1, tokens), "probs": probs.float()}


# --------------------------------------------------------------------------- one pass of a case
def run(state):
    case = state["case"]
    if not own:
        with torch.no_grad():
            return {"scan": plain_scan, "ortho": plain_ortho, "sample": plain_sample}[case["op"]](state)
    from ncas_b200 import operators as ops

    if case["op"] == "sample":
        tokens, probs = ops.sample(state["logits"], state["uniforms"], temperature=case["temperature"],
                                   top_k=case["top_k"], top_p=case["top_p"], min_p=case["min_p"])
        return {"tokens": tokens, "probs": probs}
    if case["op"] == "ortho":
        return {"x": ops.orthogonalize(state["matrix"], steps=case["steps"], coefficients=COEFFICIENTS, eps=EPS)}
    y, last = ops.gated_scan(state["x"], state["gate"], state["state"], dim=case["axis"], reverse=case["reverse"],
                             mask=state["mask"])
    out = {"y": y.detach(), "last": last.detach()}
    if case["train"]:
        names = ("dx", "dgate", "dstate")
        out.update(zip(names, torch.autograd.grad([y, last], state["inputs"], [state["dy"], state["dlast"]])))
    return out


def work(case):
    size = torch.tensor([], dtype=DTYPES[case["dtype"]]).element_size()
    if case["op"] == "scan":
        values = case["n"] * case["m"] * case["t"] * case["c"]
        edge = case["n"] * case["m"] * case["c"] * 4
        train = case["train"]
        # x, gate in, y out; with gradients dy in, dx and dgate out too (x and gate are one input each, read once)
        edges = 1 + (1 if case["state"] else 0)
        mask = values // case["c"] if case["mask"] else 0
        return {"bytes": values * size * (6 if train else 3) + edge * edges * (2 if train else 1) + mask,
                "flops": values * (20 if train else 8)}
    if case["op"] == "ortho":
        small, large = sorted((case["rows"], case["cols"]))
        # X X^T and A A are symmetric: half of each is enough
        step = small * small * large + small ** 3 + 2 * small * small * large
        return {"bytes": case["batch"] * small * large * size * 2, "flops": case["batch"] * case["steps"] * step}
    r, v, d = case["rows"], case["classes"], case["draws"]
    return {"bytes": r * v * size + r * d * (4 + 8 + 4), "flops": r * v * 4}


# ------------------------------------------------------------ the definitions, in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"scan": exact_scan, "ortho": exact_ortho, "sample": exact_sample}[case["op"]](case, s)


def exact_scan(case, s):
    # step by step along the line; the parts that do not depend on a step's neighbours for all steps at once
    axis, t = case["axis"], case["t"]
    steps = list(range(t - 1, -1, -1) if case["reverse"] else range(t))
    x, gate = s["x"].detach().double(), s["gate"].detach().double()
    a, keep = torch.sigmoid(gate), torch.sigmoid(-gate)
    off = None if s["mask"] is None else ~s["mask"][..., None]
    if off is not None:
        a.masked_fill_(off, 1.0)
        keep.masked_fill_(off, 0.0)
    del gate
    start = torch.zeros_like(x.select(axis, 0)) if s["state"] is None else s["state"].detach().double()
    h = keep * x
    at, ht = a.unbind(axis), h.unbind(axis)
    prev = start
    for i in steps:
        ht[i].addcmul_(at[i], prev)
        prev = ht[i]
    out = {"y": h if off is None else h.masked_fill(off, 0.0), "last": prev.clone()}
    if case["train"]:
        g = s["dy"].double()
        if off is not None:
            g = g.masked_fill(off, 0.0)
        gt = g.unbind(axis)
        gt[steps[-1]].add_(s["dlast"])
        for i, after in zip(reversed(steps[:-1]), reversed(steps[1:])):
            gt[i].addcmul_(at[after], gt[after])
        out["dx"] = keep * g
        if s["state"] is not None:
            out["dstate"] = at[steps[0]] * gt[steps[0]]
        gap = torch.empty_like(h)  # the state before each step
        gap.select(axis, steps[0]).copy_(start)
        if t > 1:
            if case["reverse"]:
                gap.narrow(axis, 0, t - 1).copy_(h.narrow(axis, 1, t - 1))
            else:
                gap.narrow(axis, 1, t - 1).copy_(h.narrow(axis, 0, t - 1))
        out["dgate"] = gap.sub_(x).mul_(g).mul_(a).mul_(keep)
    return out


def exact_ortho(case, s):
    a, b, c = COEFFICIENTS
    out = []
    for m in s["matrix"].double().reshape(-1, case["rows"], case["cols"]):
        x = m / (torch.linalg.matrix_norm(m) + EPS)
        for _ in range(case["steps"]):
            if case["rows"] <= case["cols"]:
                p = x @ x.T
                x = torch.addmm(x, p, torch.addmm(x, p, x, beta=b, alpha=c), beta=a)
            else:
                p = x.T @ x
                x = torch.addmm(x, torch.addmm(x, x, p, beta=b, alpha=c), p, beta=a)
        out.append(x)
    return {"x": torch.stack(out).reshape(s["matrix"].shape)}


def exact_sample(case, s):
    rows, v = s["logits"].shape
    tokens = torch.full(s["uniforms"].shape, -1, dtype=torch.int64, device=DEVICE)
    probs = torch.zeros(s["uniforms"].shape, dtype=torch.float64, device=DEVICE)
    step = max(1, 2 ** 26 // v)
    for r0 in range(0, rows, step):
        z = s["logits"][r0:r0 + step].double() / case["temperature"]
        u = s["uniforms"][r0:r0 + step].double()
        live = torch.isfinite(z).any(1)
        # ranks by two stable sorts: the place of every class in the order
        order = torch.argsort(-z, dim=1, stable=True)
        rank = torch.empty_like(order).scatter_(1, order, torch.arange(v, device=DEVICE).expand_as(order).contiguous())
        kept = torch.isfinite(z)
        if case["top_k"]:
            kept &= rank < case["top_k"]
        q = torch.softmax(torch.where(kept, z, -torch.inf), 1).nan_to_num(0.0)
        if case["top_p"] < 1:
            in_order = q.gather(1, order)
            mass = torch.cat([torch.zeros_like(in_order[:, :1]), in_order.cumsum(1)[:, :-1]], 1)
            kept &= mass.gather(1, rank) < case["top_p"]
        if case["min_p"] > 0:
            kept &= z - z.amax(1, keepdim=True) >= math.log(case["min_p"])
        q = torch.softmax(torch.where(kept, z, -torch.inf), 1).nan_to_num(0.0)
        c = q.cumsum(1)
        got = torch.searchsorted(c, (u * c[:, -1:]).contiguous(), right=True)
        last = torch.where(kept, torch.arange(v, device=DEVICE), -1).amax(1, keepdim=True)
        got = torch.minimum(got, last).clamp_min(0)
        tokens[r0:r0 + step] = torch.where(live[:, None], got, -1)
        probs[r0:r0 + step] = torch.where(live[:, None], q.gather(1, got), 0.0)
    return {"tokens": tokens, "probs": probs}
