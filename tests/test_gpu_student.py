"""The cell-training operators together: the student of ncas_b200.student against the same model in plain
64-bit torch, and its training on a rollout."""

import pytest
import torch

import oracle.cell_operators as O
from ncas_b200.student import Student, main, perceive

pytestmark = pytest.mark.gpu

DEV = "cuda"


def plain(student, inputs, values, index, weight, mask, temperature):
    """The student and its loss in float64 with torch's own gradients."""
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in student.named_parameters()}
    x = p["embed"][inputs]
    groups = student.cell.groups
    for _ in range(student.depth):
        z = perceive(x)
        n, h, w, c = z.shape
        v = z.reshape(n, h * w, groups, c // groups)
        on = mask.reshape(n, h * w, 1, 1).double()
        count = on.sum((1, 3), keepdim=True).clamp_min(1) * (c // groups)
        mean = (v * on).sum((1, 3), keepdim=True) / count
        var = ((v - mean) ** 2 * on).sum((1, 3), keepdim=True) / count
        z = ((v - mean) / torch.sqrt(var + 1e-5)).reshape(z.shape) * p["cell.norm_weight"] + p["cell.norm_bias"]
        z = z * torch.sigmoid(z) * mask[..., None]
        gate = z @ p["cell.w_gate"].T + p["cell.b_gate"]
        up = z @ p["cell.w_up"].T + p["cell.b_up"]
        x = x + (gate * torch.sigmoid(gate) * up) @ p["cell.w_down"].T + p["cell.b_down"]
    logits = x @ p["head.weight"].T + p["head.bias"]
    loss, grad = O.distill(logits.detach().reshape(-1, logits.shape[-1]), values.reshape(-1, values.shape[-1]),
                           index.reshape(-1, index.shape[-1]), temperature, weight.reshape(-1))
    got = torch.autograd.grad(logits, list(p.values()), grad.reshape(logits.shape))
    return loss.sum(), dict(zip(p, got))


def test_student_against_plain_torch():
    # bf16 states and weights: each of the 4 steps rounds its state, norm and block once or twice to
    # 2^-9 on average, 2^-8 at most, and a gradient passes them forward and backward: 16 roundings of
    # 2^-8 in a row stay below 2^-4 of a parameter's gradient norm
    torch.manual_seed(0)
    student = Student(10, 32, 64, 9).to(DEV)
    g = torch.Generator().manual_seed(1)
    inputs = torch.randint(0, 10, (3, 9, 9), generator=g)
    mask = torch.ones(3, 9, 9, dtype=torch.bool)
    mask[1, 6:] = False
    mask[2, :, 5:] = False
    values, index = torch.randn((3, 9, 9, 9), generator=g).topk(4)
    weight = torch.rand((3, 9, 9), generator=g) * mask
    from ncas_b200 import operators as ops

    logits = student(inputs.to(DEV), mask.to(DEV))
    loss = ops.distill_loss(logits, values.to(DEV), index.to(DEV), temperature=2.0, weight=weight.to(DEV), reduction="sum")
    loss.backward()
    ops.check()
    want, grads = plain(student, inputs, values, index, weight, mask, 2.0)
    assert abs(loss.item() - want.item()) <= 2**-6 * want.item()
    for k, p in student.named_parameters():
        off = (p.grad.cpu().double() - grads[k]).norm() / grads[k].norm()
        assert off <= 2**-4, (k, float(off))


@pytest.mark.parametrize("task", ["sudoku", "maze"])
def test_training_on_a_rollout(task):
    losses = main(["--task", task, "--boards", "24", "--steps", "40", "--teacher-steps", "24"])
    assert len(losses) == 40 and losses[-1] < 0.7 * losses[0]
