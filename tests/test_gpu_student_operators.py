"""gated_scan, orthogonalize and sample together, as the student uses them: a cell that looks along lines, an optimiser
that orthogonalises its matrices, answers drawn from its readout."""

import pytest
import torch

import oracle.cell_operators as O
from ncas_b200 import operators as ops
from ncas_b200.student import GatedCell, Muon, Student, answers, look_along, main, make_optimizers, perceive

pytestmark = pytest.mark.gpu

DEV = "cuda"


def plain_scan(x, gate, dim, reverse, mask):
    steps = list(range(x.shape[dim]))[:: -1 if reverse else 1]
    h, out = torch.zeros_like(x.select(dim, 0)), [None] * x.shape[dim]
    for t in steps:
        a, on = torch.sigmoid(gate.select(dim, t)), mask.select(dim, t)[..., None]
        h = torch.where(on, a * h + (1 - a) * x.select(dim, t), h)
        out[t] = h * on
    return torch.stack(out, dim)


def plain(student, inputs, mask):
    """The student's logits in float64 with torch's own gradients."""
    p = {k: v.detach().cpu().double().requires_grad_() for k, v in student.named_parameters()}
    x = p["embed"][inputs]
    c, groups = x.shape[-1], student.cell.groups
    for _ in range(student.depth):
        gates = x @ p["cell.w_scan"].T + p["cell.b_scan"]
        seen = [perceive(x)]
        for i, (dim, reverse) in enumerate(((2, False), (2, True), (1, False), (1, True))):
            seen.append(plain_scan(x, gates[..., i * c : (i + 1) * c], dim, reverse, mask))
        z = torch.cat(seen, -1)
        n, h, w, wide = z.shape
        v = z.reshape(n, h * w, groups, wide // groups)
        on = mask.reshape(n, h * w, 1, 1).double()
        count = on.sum((1, 3), keepdim=True).clamp_min(1) * (wide // groups)
        mean = (v * on).sum((1, 3), keepdim=True) / count
        var = ((v - mean) ** 2 * on).sum((1, 3), keepdim=True) / count
        z = ((v - mean) / torch.sqrt(var + 1e-5)).reshape(z.shape) * p["cell.norm_weight"] + p["cell.norm_bias"]
        z = z * torch.sigmoid(z) * mask[..., None]
        gate = z @ p["cell.w_gate"].T + p["cell.b_gate"]
        up = z @ p["cell.w_up"].T + p["cell.b_up"]
        x = x + (gate * torch.sigmoid(gate) * up) @ p["cell.w_down"].T + p["cell.b_down"]
    return p, x @ p["head.weight"].T + p["head.bias"]


def test_student_that_looks_along_lines_against_plain_torch():
    # bf16 states and weights, as in the student without scans: each of the 4 steps rounds its state, gates, scans, norm and
    # block to 2^-8 at most and a gradient passes them forward and backward: 24 roundings of 2^-8 in a row stay below
    # 0.1 of a parameter's gradient norm
    torch.manual_seed(0)
    student = Student(10, 32, 64, 9, scan=True).to(DEV)
    g = torch.Generator().manual_seed(1)
    inputs = torch.randint(0, 10, (3, 9, 9), generator=g)
    mask = torch.ones(3, 9, 9, dtype=torch.bool)
    mask[1, 6:] = False
    mask[2, :, 5:] = False
    mask[2, 3] = False
    values, index = torch.randn((3, 9, 9, 9), generator=g).topk(4)
    weight = torch.rand((3, 9, 9), generator=g) * mask
    logits = student(inputs.to(DEV), mask.to(DEV))
    loss = ops.distill_loss(logits, values.to(DEV), index.to(DEV), temperature=2.0, weight=weight.to(DEV), reduction="sum")
    loss.backward()
    ops.check()
    p, want = plain(student, inputs, mask)
    flat = lambda t: t.reshape(-1, t.shape[-1])  # noqa: E731
    loss64, grad = O.distill(flat(want.detach()), flat(values), flat(index), 2.0, weight.reshape(-1))
    grads = dict(zip(p, torch.autograd.grad(want, list(p.values()), grad.reshape(want.shape))))
    assert abs(loss.item() - loss64.sum().item()) <= 2**-5 * loss64.sum().item()
    for k, v in student.named_parameters():
        off = (v.grad.cpu().double() - grads[k]).norm() / grads[k].norm()
        assert off <= 0.1, (k, float(off))


def test_look_along_sees_a_whole_line():
    # with gates that keep everything the far end of a row is seen at its other end; masked cells are passed by
    x = torch.zeros((1, 5, 7, 4), device=DEV)
    x[0, 2, 0] = 1.0
    gates = torch.zeros((1, 5, 7, 16), device=DEV)
    gates[..., 1:, :] = 30.0
    mask = torch.ones((1, 5, 7), dtype=torch.bool, device=DEV)
    mask[0, 2, 3] = False
    seen = look_along(x, gates, mask)
    assert (seen[0, 2, 1:, :4] > 0.49).sum() == 5 * 4 and (seen[0, 2, 3] == 0).all()
    assert (seen[0, :2, :, :4] == 0).all() and (seen[0, 3:, :, :4] == 0).all()


def test_muon_adds_orthogonalised_momenta():
    torch.manual_seed(1)
    shapes = [(64, 48), (64, 48), (48, 64), (40, 40)]
    params = [torch.nn.Parameter((torch.randn(s, device=DEV) * 0.1).to(torch.bfloat16)) for s in shapes]
    idle = torch.nn.Parameter(torch.zeros(8, 8, device=DEV, dtype=torch.bfloat16))
    before = [p.detach().clone() for p in params]
    opt = Muon([*params, idle], lr=0.5, momentum=0.9)
    momenta = [torch.zeros(s, dtype=torch.float32) for s in shapes]
    for step in range(2):
        grads = [(torch.randn(s, device=DEV) * 0.01).to(torch.bfloat16) for s in shapes]
        for p, g in zip(params, grads):
            p.grad = g
        opt.step()
        for i, g in enumerate(grads):
            momenta[i] = momenta[i] * 0.9 + g.cpu().float()
            update = (g.cpu().float() + 0.9 * momenta[i]).to(torch.bfloat16)
            want = O.orthogonalize(update).to(torch.bfloat16).double()
            rate = 0.5 * max(1.0, shapes[i][0] / shapes[i][1]) ** 0.5
            moved = (before[i].cpu().double() - params[i].detach().cpu().double()) / rate
            # the parameter and the product are rounded to bf16 once more each, the update's own error is below 2^-8 of its norm
            tol = 2.0**-7 * want.norm() + 2.0**-8 * before[i].cpu().double().norm() / rate * 2
            assert (moved - want).norm() <= tol, (step, i)
        before = [p.detach().clone() for p in params]
    assert (idle == 0).all()
    for bad in (torch.zeros(4, device=DEV, dtype=torch.bfloat16), torch.zeros(4, 4, device=DEV)):
        with pytest.raises(ValueError, match="Muon"):
            Muon([torch.nn.Parameter(bad)])


@pytest.mark.parametrize("size,steps", [(3e4, 20), (1e-7, 1)])
def test_muon_of_fp16_matrices_at_the_ends_of_their_range(size, steps):
    # momenta beyond 65504, and updates of one or two steps of fp16: as the same gradients of about 1 move them
    g = torch.Generator(device=DEV).manual_seed(4)
    sign = (torch.rand((48, 64), generator=g, device=DEV) < 0.5).half() * 2 - 1
    params = [torch.nn.Parameter(torch.zeros(48, 64, device=DEV, dtype=torch.float16)) for _ in range(2)]
    opts = [Muon([p], lr=0.5) for p in params]
    for p, opt, scale in zip(params, opts, (size, 1.0)):
        p.grad = sign * scale
        for _ in range(steps):
            p.data.zero_()
            opt.step()
    ops.check()
    assert params[1].abs().max() > 0.01
    # entries of one size: after the scaling both are the same matrix, but for the rounding of 20 sums of fp32
    assert (params[0].double() - params[1].double()).norm() <= 2.0**-10 * params[1].double().norm()


def test_every_parameter_has_an_optimizer():
    student = Student(10, 32, 64, 9, scan=True)
    for name in ("adam", "muon"):
        held = [p for o in make_optimizers(student, name) for g in o.param_groups for p in g["params"]]
        assert sorted(map(id, held)) == sorted(map(id, student.parameters()))
    with pytest.raises(ValueError, match="optimizer"):
        make_optimizers(student, "sgd")
    assert not hasattr(GatedCell(32, 64), "w_scan")


def test_answers_are_scored_by_their_probability():
    g = torch.Generator(device=DEV).manual_seed(2)
    logits = torch.randn((4, 5, 6, 9), generator=g, device=DEV)
    given = torch.rand((4, 5, 6), generator=g, device=DEV) < 0.3
    tokens = torch.randint(0, 9, (4, 5, 6), generator=g, device=DEV)
    classes, scores = answers(logits, 7, given=given, tokens=tokens, generator=torch.Generator(device=DEV).manual_seed(3))
    assert classes.shape == (4, 7, 5, 6) and scores.shape == (4, 7)
    logp = torch.log_softmax(logits.double(), -1)
    for b in range(4):
        for k in range(7):
            assert torch.equal(classes[b, k][given[b]], tokens[b][given[b]])
            picked = logp[b].gather(-1, classes[b, k][..., None])[..., 0][~given[b]]
            assert abs(picked.mean().item() - scores[b, k].item()) <= 1e-5
    again, _ = answers(logits, 7, given=given, tokens=tokens, generator=torch.Generator(device=DEV).manual_seed(3))
    assert torch.equal(again, classes)
    sharp, score = answers(logits, 2, temperature=0.0)
    assert torch.equal(sharp[:, 0], logits.argmax(-1)) and torch.equal(sharp[:, 1], sharp[:, 0]) and (score == 0).all()


@pytest.mark.parametrize("task", ["sudoku", "maze"])
def test_the_command_runs_with_all_of_them(task, capsys):
    losses = main(["--task", task, "--boards", "12", "--steps", "6", "--teacher-steps", "8", "--scan", "--optimizer", "muon",
                   "--trials", "5"])
    assert len(losses) == 6 and all(v == v for v in losses)
    assert "5 answers a board" in capsys.readouterr().out
