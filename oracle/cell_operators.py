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
