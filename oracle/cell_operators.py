"""The cell-training operators in 64 bits, from their definitions, with explicit gradients.

CPU tensors in, float64 tensors out; nothing of the library is used.  The kernels' tests compare with
these, and these are themselves checked against finite differences.
"""

from __future__ import annotations

import math

import torch


def act(z, name):
    """The activation and its derivative."""
    if name == "none":
        return z, torch.ones_like(z)
    if name == "relu":
        return torch.where(z > 0, z, 0 * z), (z > 0).double()
    if name == "sigmoid":
        s = torch.sigmoid(z)
        return s, s * (1 - s)
    if name == "silu":
        s = torch.sigmoid(z)
        return z * s, s + z * s * (1 - s)
    if name == "gelu":
        cdf = 0.5 * torch.erfc(-z / math.sqrt(2))
        return z * cdf, cdf + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)
    raise ValueError(name)


def group_norm_act(x, groups, weight=None, bias=None, eps=1e-5, name="silu", mask=None, dy=None):
    """y, or with dy (y, dx, dweight, dbias).  A loop over samples; masked cells are left out."""
    n, c = x.shape[0], x.shape[-1]
    xs = x.double().reshape(n, -1, c)
    cells = xs.shape[1]
    w = torch.ones(c, dtype=torch.float64) if weight is None else weight.double()
    b = torch.zeros(c, dtype=torch.float64) if bias is None else bias.double()
    keep = torch.ones(n, cells, dtype=torch.bool) if mask is None else mask.reshape(n, -1) != 0
    y = torch.zeros(n, cells, c, dtype=torch.float64)
    dx, dw, db = torch.zeros_like(y), torch.zeros_like(w), torch.zeros_like(b)
    g = None if dy is None else dy.double().reshape(n, cells, c)
    for i in range(n):
        rows = keep[i].nonzero()[:, 0]
        if len(rows) == 0:
            continue
        v = xs[i, rows].reshape(len(rows), groups, c // groups)
        mean = v.mean((0, 2), keepdim=True)
        rstd = 1 / torch.sqrt(((v - mean) ** 2).mean((0, 2), keepdim=True) + eps)
        h = ((v - mean) * rstd).reshape(len(rows), c)
        out, slope = act(h * w + b, name)
        y[i, rows] = out
        if g is None:
            continue
        dz = g[i, rows] * slope
        dw += (dz * h).sum(0)
        db += dz.sum(0)
        dh = (dz * w).reshape(v.shape)
        hg = h.reshape(v.shape)
        d = rstd * (dh - dh.mean((0, 2), keepdim=True) - hg * (dh * hg).mean((0, 2), keepdim=True))
        dx[i, rows] = d.reshape(len(rows), c)
    if dy is None:
        return y.reshape(x.shape)
    return y.reshape(x.shape), dx.reshape(x.shape), dw, db


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, name="silu", dy=None):
    """y, or with dy a dict of y and every gradient."""
    x, wg, wu, wd = (t.double() for t in (x, w_gate, w_up, w_down))
    zero = torch.zeros((), dtype=torch.float64)
    gate = x @ wg.T + (zero if b_gate is None else b_gate.double())
    up = x @ wu.T + (zero if b_up is None else b_up.double())
    a, slope = act(gate, name)
    h = a * up
    y = h @ wd.T + (zero if b_down is None else b_down.double())
    if dy is None:
        return y
    dy = dy.double()
    dh = dy @ wd
    dg, du = dh * up * slope, dh * a
    return dict(y=y, x=dg @ wg + du @ wu, w_gate=dg.T @ x, w_up=du.T @ x, w_down=dy.T @ h,
                b_gate=dg.sum(0), b_up=du.sum(0), b_down=dy.sum(0))


def distill(logits, teacher, index, temperature=1.0, weight=None):
    """(loss of each row, gradient of their sum by the logits).  A loop over rows and entries."""
    rows, classes = logits.shape
    loss = torch.zeros(rows, dtype=torch.float64)
    grad = torch.zeros(rows, classes, dtype=torch.float64)
    for r in range(rows):
        w = 1.0 if weight is None else float(weight[r])
        at = [(int(i), float(t)) for i, t in zip(index[r], teacher[r]) if 0 <= int(i) < classes]
        at = [(i, t) for i, t in at if t != -math.inf]
        if w == 0 or not at:
            continue
        logq = torch.log_softmax(logits[r].double() / temperature, 0)
        logp = torch.log_softmax(torch.tensor([t for _, t in at], dtype=torch.float64) / temperature, 0)
        target = torch.zeros(classes, dtype=torch.float64)
        for (i, _), lp in zip(at, logp):
            p = math.exp(lp)
            target[i] += p
            loss[r] += w * temperature**2 * p * (lp - logq[i])
        grad[r] = w * temperature * (logq.exp() - target)
    return loss, grad


def gated_scan(x, gate, state=None, dim=-2, reverse=False, mask=None, dy=None, dlast=None):
    """(y, last), or with dy a dict of y, last, x, gate, state.  A loop over the steps of axis `dim`."""
    dim = dim % x.dim()
    x, gate = x.double().movedim(dim, 0), gate.double().movedim(dim, 0)
    steps = list(range(x.shape[0]))[:: -1 if reverse else 1]
    on = torch.ones(x.shape[:-1], dtype=torch.bool) if mask is None else mask.movedim(dim, 0) != 0
    h = torch.zeros(x.shape[1:], dtype=torch.float64) if state is None else state.double()
    before, after, y = {}, {}, torch.zeros_like(x)
    for t in steps:
        a = torch.sigmoid(gate[t])
        before[t] = h
        h = torch.where(on[t][..., None], a * h + torch.sigmoid(-gate[t]) * x[t], h)
        after[t] = h
        y[t] = torch.where(on[t][..., None], h, 0.0)
    if dy is None:
        return y.movedim(0, dim), h
    dy = dy.double().movedim(dim, 0)
    g = torch.zeros_like(h) if dlast is None else dlast.double()
    dx, dgate = torch.zeros_like(x), torch.zeros_like(x)
    for t in reversed(steps):
        live = on[t][..., None]
        a, keep = torch.sigmoid(gate[t]), torch.sigmoid(-gate[t])
        full = dy[t] + g
        dx[t] = torch.where(live, keep * full, 0.0)
        dgate[t] = torch.where(live, full * (before[t] - x[t]) * a * keep, 0.0)
        g = torch.where(live, a * full, g)
    return dict(y=y.movedim(0, dim), last=h, x=dx.movedim(0, dim), gate=dgate.movedim(0, dim), state=g)


def orthogonalize(m, steps=5, coefficients=(3.4445, -4.775, 2.0315), eps=1e-7, rounded=False):
    """Newton-Schulz steps of a stack of matrices.  rounded: with the roundings to fp16 that the library's
    kernels document (operands X 2^12, A 2^10, B 2^10; X itself, and the operands of the last steps, as two fp16 values),
    everything else exact."""
    a, b, c = coefficients
    once = lambda t, s: (t * s).half().double() / s if rounded else t  # noqa: E731
    twice = lambda t, s: once(t, s) + once(t - once(t, s), s) if rounded else t  # noqa: E731
    few = min(m.shape[-2:]) < 64 or (m.dtype == torch.float16 and steps <= 2)
    full = m.dtype == torch.float16 or few
    arrived = max(0.0, steps - 0.5 * math.log(max(1, min(m.shape[-2:]))) / math.log(abs(a))) if abs(a) > 1.05 else steps
    precise = steps if few else min(steps, math.ceil(arrived)) if full else 0 if arrived <= 3 else math.ceil(arrived - 1.2)
    out = []
    for x in m.double().reshape(-1, *m.shape[-2:]):
        x = x / (x.square().sum().sqrt() + eps)
        if x.shape[0] > x.shape[1]:
            x = x.T
        for k in range(steps):
            late = k + precise >= steps
            early = twice if late and full else once
            y, x = early(x, 4096.0), twice(x, 4096.0)
            p = early(y @ y.T, 1024.0)
            q = (twice if late else once)(b * p + c * (p @ p), 1024.0)
            x = a * x + q @ (x if late else y)
        out.append(x.T if m.shape[-2] > m.shape[-1] else x)
    return torch.stack(out).reshape(m.shape)


def sample(logits, uniforms, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(classes, probabilities, nearest) of rows x classes and rows x draws: `nearest` is the least distance of a
    draw, or of the cut by top_p, from a border, as a share of the mass.  A loop over rows."""
    rows, classes = logits.shape
    tokens = torch.full(uniforms.shape, -1, dtype=torch.int64)
    probs = torch.zeros(uniforms.shape, dtype=torch.float64)
    nearest = 1.0
    for r in range(rows):
        z = logits[r].double()
        z = torch.where(z.isnan(), -math.inf, z)
        top = z.max()
        if top == -math.inf:
            continue
        w = torch.where(z == top, 1.0, torch.exp((z - top) / (temperature or 1.0)))
        order = torch.argsort(-z, stable=True)
        kept = order[z[order] > -math.inf]
        if temperature == 0 or top_k:
            kept = kept[: 1 if temperature == 0 else top_k]
        if top_p < 1:
            ends = w[kept].cumsum(0)
            before = ends - w[kept]
            target = top_p * ends[-1]
            nearest = min(nearest, float((before - target).abs().min() / ends[-1]))
            kept = kept[before < target]
        kept = kept[w[kept] >= min_p].sort().values
        c = w[kept].cumsum(0)
        for k, u in enumerate(uniforms[r].double().tolist()):
            t = (u if u > 0 else 0.0) * c[-1]  # NaN: the first
            at = min(int((c <= t).sum()), len(kept) - 1)
            if 0 < u < 1:
                nearest = min(nearest, float((c - t).abs().min() / c[-1]))
            while w[kept[at]] == 0:  # u = 1: the last that can be drawn
                at -= 1
            tokens[r, k], probs[r, k] = kept[at], w[kept[at]] / c[-1]
    return tokens, probs, nearest
