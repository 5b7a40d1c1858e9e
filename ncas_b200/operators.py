"""Operators for training a normalised, gated cell beside the rollout, on hand-written sm_100a kernels.

    group_norm_act          group norm with an activation, channels last
    gated_ffn               gated feed-forward block: (act(x Wg^T + bg) * (x Wu^T + bu)) Wd^T + bd
    gated_scan              gated linear recurrence along the lines of boards or long sequences
    distill_loss            distillation from a teacher's top logits
    distill_loss_and_grad   the same with its gradient in one pass over the logits
    orthogonalize           an optimiser's update with its singular values brought towards 1
    sample                  classes drawn from logits with temperature, top-k, top-p and min-p

The reference's cells have the first two as `norm_groups` and `update="swiglu"`
(src/nca/model.py:48-137, 440-455), which the rollout kernels do not run.  The functions take CUDA
tensors, run on torch's current stream, are differentiable (once, backward) where a gradient is named,
and raise ValueError or TypeError for arguments they do not take.  There is no CPU fallback, no
forward-mode derivative and no form for torch.compile or vmap (a compiled or mapped function has to
leave the calls out).  Results do
not depend on the order in which blocks run.
"""

from __future__ import annotations

import torch

from ._lib import NcaError
from ._ops import ops

_overloads: dict = {}


def _op(name):
    """torch.ops.nca_b200.<name>.default, looked up once."""
    op = _overloads.get(name)
    if op is None:
        op = _overloads[name] = getattr(ops(), name).default
    return op


def group_norm_act(x, groups, weight=None, bias=None, *, eps=1e-5, act="silu", mask=None):
    """act((x - mean) / sqrt(var + eps) * weight + bias) of x (N, ..., C), contiguous.

    Mean and biased variance run over the cells of a sample and the C / groups channels of a group,
    in fp32.  x: float32, bfloat16 or float16, any strides (adjacent channels and evenly spaced
    cells are read in place, others copied).  weight, bias: (C,), float32 or x's type.  act: "none",
    "relu", "silu", "gelu" (erf form) or "sigmoid".  mask: bool or uint8 (N, ...): cells where it is
    zero are not read, count in no statistic, and have y and gradient 0; a sample without cells is 0.
    Differentiable in x, weight and bias.
    """
    return _op("group_norm_act")(x, groups, weight, bias, eps, act, mask)


def gated_ffn(x, w_gate, w_up, w_down, b_gate=None, b_up=None, b_down=None, *, act="silu"):
    """(act(x w_gate^T + b_gate) * (x w_up^T + b_up)) w_down^T + b_down of x (..., d_in).

    x and the weights (out, in): all bfloat16 or all float16; the biases float32 or of that type.  act:
    "relu", "silu", "gelu" (erf form) or "sigmoid".  Products are summed in fp32 on the tensor cores;
    the hidden product and the gradients of its two factors are rounded to the type of x in between.  Matrices whose rows start on 16-byte boundaries are read in place, others are
    copied first.  Differentiable in every tensor.  The first call on a device makes its control words:
    it must precede a stream capture.
    """
    return _op("gated_ffn")(x, w_gate, w_up, w_down, b_gate, b_up, b_down, act)


def distill_loss(logits, teacher_logits, teacher_index, *, temperature=1.0, weight=None, reduction="mean"):
    """weight * T^2 * KL(p || q) of each row, p = softmax(teacher_logits / T) over the row's entries and
    q = softmax(logits / T) over all classes.

    logits (..., classes); teacher_logits (..., top) with the classes they belong to in teacher_index
    (int32 or int64; an index outside [0, classes), such as -1, marks no entry; entries of one class
    add up).  weight: float32 (...).  A row without entries or with weight 0 has loss and gradient 0.
    temperature: 1e-30 to 1e30.  reduction: "none" (float32, (...)), "sum", or "mean" over all rows.  Differentiable in logits.
    The same call gives the same bits; another number of rows, or distill_loss_and_grad, may run another
    kernel, whose sums differ by rounding.
    """
    return _op("distill_loss")(logits, teacher_logits, teacher_index, temperature, weight, reduction)


def distill_loss_and_grad(logits, teacher_logits, teacher_index, *, temperature=1.0, weight=None,
                          reduction="mean"):
    """(distill_loss, gradient of its sum over rows, or of its mean, by the logits) with one read of the
    logits where a row fits on the chip; for training loops that call `logits.backward(grad)`."""
    return _op("distill_loss_and_grad")(logits, teacher_logits, teacher_index, temperature, weight, reduction)


def gated_scan(x, gate, state=None, *, dim=-2, reverse=False, mask=None):
    """(y, last) of the recurrence y_t = a_t y_{t-1} + (1 - a_t) x_t, a = sigmoid(gate), along axis `dim` of x (..., C).

    x, gate: float32, bfloat16 or float16, one type and shape, any strides (adjacent channels with collapsible axes
    on either side of `dim` are read in place, others copied); y is contiguous, of that type, and rounded once: the
    recurrence runs in fp32.  state: the value before the first step, float32, of x's shape without `dim` (absent:
    zeros); last: the value after the last step, likewise, for the next call of a line that goes on.  reverse: from
    the last step to the first.  mask: bool or uint8, x's shape without C: where it is zero the value stays as it
    is, y and the gradients are 0, and what x and gate hold has no effect.  Differentiable in x, gate and state,
    through y and last.
    """
    return _op("gated_scan")(x, gate, state, dim, reverse, mask)


def orthogonalize(matrix, *, steps=5, coefficients=(3.4445, -4.775, 2.0315), eps=1e-7):
    """matrix (..., rows, cols) with its singular values brought towards 1 by Newton-Schulz products: X = M / (|M|_F + eps),
    then `steps` times X = a X + (b A + c A^2) X, A = X X^T, with coefficients (a, b, c).

    bfloat16 or float16, any strides (adjacent columns are read in place, others copied); the result is contiguous and
    of the same type.  Products are summed in fp32 over fp16 operands, X keeps 22 bits between the steps, and the
    result is rounded once: its error is 1.0 to 1.4 times that rounding on average, 1.9 at most (of up to 8 steps).
    Coefficients that let a singular value grow beyond 2 are refused.  A norm below a millionth of eps leaves X, and the
    result (then below 1e-3), fewer bits than its type has.  Not differentiable: for the update of an optimiser.  The first call on a device makes its control words: it must precede a stream capture.
    """
    return _op("orthogonalize")(matrix, steps, coefficients, eps)


def sample(logits, uniforms, *, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(classes, probabilities) drawn from each row of logits (..., classes) with the given uniform numbers of [0, 1):
    uniforms (..., draws), or (...) for one draw; both results have its shape (int64, float32).

    Classes in the order of their logits, the lower index first among equals.  Kept are the first top_k (0: all); of
    those, the ones before which less than top_p of their mass exp(logit / temperature) lies; of those, the ones of at
    least min_p times the largest one's mass.  A draw is the first kept class, by index, at which the sum of the kept
    masses exceeds the uniform number times the whole; its probability is its share of it.  Masses are computed in
    64 bits and added up in fixed point: a border between two classes is off by 5e-13 of the largest mass at most up to 2048
    classes, by 2e-9 at 131072 and 3e-8 at 2^19, and beyond by classes 2^-52 of the whole.  logits: float32, bfloat16 or
    float16, any strides; NaN counts as -inf; +inf beats every finite logit; a row that is -inf alone gives -1 and 0.
    temperature 0: the first of the largest.  Not differentiable.
    """
    return _op("sample")(logits, uniforms, temperature, top_k, top_p, min_p)


def check(device="cuda") -> None:
    """Synchronises the current stream and raises NcaError when a kernel's bounded wait ran out since this
    thread's last call (at first: since it began to use the operators).

    A gated_ffn or orthogonalize whose wait ran out leaves its outputs unfinished; later calls are not affected.  The
    record is the device's: every thread that uses the operators is told once, whichever of them ran
    the call and whichever asks first."""
    status, site = _op("operators_status")(torch.empty(0, device=device))
    if status != 0:
        raise NcaError(status, "cell-training operators", site)
