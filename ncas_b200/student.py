"""A normalised, gated cell trained on the rollout: the operators of a student as they are used together.

The teacher is a model of the rollout engine: many asynchronous steps of each board.  Its readout of
the final state, the top logits of every cell, is what a rollout would keep for training.  The student
runs few synchronous steps of a cell with group norm and a gated update
(x + gated_ffn(act(group_norm(perceive(x))))) over channels-last states, and learns the teacher's
readout by distillation of those top logits.  Perception (fixed 3x3 taps) and the head (one matrix)
are plain torch.  With `scan`, a cell also sees gated scans along its row and column, from both ends: what a
3x3 stencil would need a step a cell for.  `Muon` orthogonalises the updates of the matrices.  `answers`
draws candidates of every board from the trained readout and scores them by their probability, as the rollout
scores its trials by their confidence.

    python -m ncas_b200.student --task sudoku --boards 64 --steps 100
    python -m ncas_b200.student --task maze --scan --optimizer muon --trials 8
"""

from __future__ import annotations

import argparse

import torch
from torch import nn

from . import operators as ops
from .configs import build, model_config
from .model import FIXED_TAPS
from .tasks import maze_boards, sudoku_boards


def perceive(x: torch.Tensor) -> torch.Tensor:
    """The four fixed 3x3 heads of every channel (zero padding): (N, H, W, C) to (N, H, W, 4C)."""
    n, h, w, c = x.shape
    p = torch.nn.functional.pad(x, (0, 0, 1, 1, 1, 1))
    heads = []
    for taps in FIXED_TAPS:
        out = 0
        for i in range(3):
            for j in range(3):
                if taps[i, j]:
                    out = out + float(taps[i, j]) * p[:, i : i + h, j : j + w]
        heads.append(out)
    return torch.cat(heads, -1)


def look_along(x: torch.Tensor, gates: torch.Tensor, mask: torch.Tensor | None = None) -> torch.Tensor:
    """Gated scans along the rows and columns of boards (N, H, W, C), from both ends: (N, H, W, 4C).  gates (N, H, W, 4C):
    how much of what came before each cell keeps (sigmoid), a direction after the other; masked cells are passed by."""
    heads = []
    for i, (dim, reverse) in enumerate(((2, False), (2, True), (1, False), (1, True))):
        gate = gates[..., i * x.shape[-1] : (i + 1) * x.shape[-1]]
        heads.append(ops.gated_scan(x, gate, dim=dim, reverse=reverse, mask=mask)[0])
    return torch.cat(heads, -1)


class GatedCell(nn.Module):
    """One step of the student: perception, group norm with an activation, gated update, residual.  scan: the cell also
    perceives what look_along gives, with gates from one matrix (the scans remember about 7 cells at first)."""

    def __init__(self, channels: int, hidden: int, groups: int = 4, act: str = "silu", dtype=torch.bfloat16,
                 scan: bool = False):
        super().__init__()
        wide = 8 * channels if scan else 4 * channels
        self.groups, self.act = groups, act
        if scan:
            self.w_scan = nn.Parameter((torch.randn(4 * channels, channels) * 0.1 * channels**-0.5).to(dtype))
            self.b_scan = nn.Parameter(torch.full((4 * channels,), 2.0, dtype=dtype))
        self.norm_weight = nn.Parameter(torch.ones(wide))
        self.norm_bias = nn.Parameter(torch.zeros(wide))
        self.w_gate = nn.Parameter((torch.randn(hidden, wide) * wide**-0.5).to(dtype))
        self.w_up = nn.Parameter((torch.randn(hidden, wide) * wide**-0.5).to(dtype))
        self.w_down = nn.Parameter((torch.randn(channels, hidden) * 0.1 * hidden**-0.5).to(dtype))
        self.b_gate = nn.Parameter(torch.zeros(hidden, dtype=dtype))
        self.b_up = nn.Parameter(torch.zeros(hidden, dtype=dtype))
        self.b_down = nn.Parameter(torch.zeros(channels, dtype=dtype))

    def forward(self, x: torch.Tensor, mask: torch.Tensor | None = None) -> torch.Tensor:
        """x (N, H, W, C); mask (N, H, W): the cells of boards padded to one size."""
        seen = perceive(x)
        if hasattr(self, "w_scan"):
            gates = torch.nn.functional.linear(x, self.w_scan, self.b_scan)
            seen = torch.cat([seen, look_along(x, gates, mask)], -1)
        z = ops.group_norm_act(seen, self.groups, self.norm_weight, self.norm_bias, act=self.act, mask=mask)
        return x + ops.gated_ffn(z, self.w_gate, self.w_up, self.w_down, self.b_gate, self.b_up, self.b_down)


class Student(nn.Module):
    """Token embedding, `depth` steps of one GatedCell, a linear readout of `n_out` classes."""

    def __init__(self, vocab: int, channels: int, hidden: int, n_out: int, depth: int = 4, dtype=torch.bfloat16,
                 scan: bool = False):
        super().__init__()
        self.depth, self.dtype = depth, dtype
        self.embed = nn.Parameter(torch.randn(vocab, channels))
        self.cell = GatedCell(channels, hidden, dtype=dtype, scan=scan)
        self.head = nn.Linear(channels, n_out)

    def forward(self, inputs: torch.Tensor, mask: torch.Tensor | None = None) -> torch.Tensor:
        """Logits (N, H, W, n_out) in fp32 of token boards (N, H, W)."""
        x = self.embed[inputs].to(self.dtype)
        for _ in range(self.depth):
            x = self.cell(x, mask)
        return self.head(x.float())


def teacher_top(engine, inputs, given, top: int, steps: int, p_fire: float = 0.5, seed: int = 0):
    """The teacher's top logits of every cell after `steps` steps: values and indices (N, H, W, top)."""
    n, h, w = inputs.shape
    cfg = engine.cfg
    batch = engine.batch_from_boards(inputs, given, 1)
    state = engine.new_state(n, h * w)
    engine.init_state(state, batch)
    engine.run(state, batch, steps, mode="philox", p_fire=p_fire, seed=seed)
    x = engine.store_nchw(state).reshape(n, -1, h, w)
    engine.check()
    out = x[:, cfg.out_offset : cfg.out_offset + cfg.c_out].permute(0, 2, 3, 1)  # identity head
    values, index = out.topk(min(top, cfg.c_out), dim=-1)
    return values.contiguous(), index.to(torch.int32).contiguous()


def near_one(matrices: torch.Tensor) -> torch.Tensor:
    """float32 matrices (..., rows, cols), each times the power of two that brings its largest entry to [1/2, 1).  What is
    orthogonalised does not depend on its size, but fp16 holds no more than 65504 and little below 6e-8."""
    if matrices.numel() == 0:
        return matrices
    exponent = torch.frexp(matrices.abs().amax((-2, -1), keepdim=True)).exponent
    half = torch.div(exponent, 2, rounding_mode="floor")  # two factors: 2^149 is no float32
    power = lambda n: ((n + 127) << 23).view(torch.float32)  # noqa: E731  exact
    return matrices * power(-half) * power(half - exponent)


class Muon(torch.optim.Optimizer):
    """Momentum whose matrices are orthogonalised before they are added: an update of w (out, in) has all its singular
    values near 1, times lr sqrt(max(1, out / in)).  Matrices of one shape are orthogonalised in one call.  Takes bfloat16 and
    float16 matrices; momenta are float32."""

    def __init__(self, params, lr: float = 0.02, momentum: float = 0.95, nesterov: bool = True, steps: int = 5):
        super().__init__(params, dict(lr=lr, momentum=momentum, nesterov=nesterov, steps=steps))

    def add_param_group(self, param_group):
        super().add_param_group(param_group)
        for p in self.param_groups[-1]["params"]:
            if p.dim() != 2 or p.dtype not in (torch.bfloat16, torch.float16):
                self.param_groups.pop()
                raise ValueError(f"Muon takes bfloat16 and float16 matrices, not {p.dtype} {tuple(p.shape)}")

    def load_state_dict(self, state_dict):
        """Momenta stay float32 (the base class casts them to the type of their matrices), copies of the given ones."""
        super().load_state_dict(state_dict)
        names = [n for group in state_dict["param_groups"] for n in group["params"]]
        for name, p in zip(names, (p for group in self.param_groups for p in group["params"])):
            if "momentum" in state_dict["state"].get(name, {}):
                momentum = state_dict["state"][name]["momentum"]
                self.state[p]["momentum"] = momentum.to(device=p.device, dtype=torch.float32, copy=True)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            shapes: dict = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                state = self.state[p]
                if "momentum" not in state:
                    state["momentum"] = torch.zeros_like(p, dtype=torch.float32)
                m = state["momentum"]
                m.mul_(group["momentum"]).add_(p.grad)
                update = p.grad.float().add(m, alpha=group["momentum"]) if group["nesterov"] else m
                shapes.setdefault((p.shape, p.dtype, p.device), []).append((p, update))
            for (shape, dtype, _), pairs in shapes.items():
                rates = -group["lr"] * max(1.0, shape[0] / max(1, shape[1])) ** 0.5
                updates = near_one(torch.stack([u for _, u in pairs])).to(dtype)
                for (p, _), u in zip(pairs, ops.orthogonalize(updates, steps=group["steps"])):
                    p.add_(u, alpha=rates)
        return loss


def make_optimizers(student: Student, name: str = "adam", lr: float = 3e-3) -> list[torch.optim.Optimizer]:
    """"adam": Adam for all; "muon": Muon for the cell's matrices (with its own lr), Adam for the rest.  lr: Adam's."""
    if name == "adam":
        return [torch.optim.Adam(student.parameters(), lr=lr)]
    if name != "muon":
        raise ValueError(f"optimizer must be 'adam' or 'muon', not {name!r}")
    matrices = [p for p in student.cell.parameters() if p.dim() == 2]
    chosen = {id(p) for p in matrices}
    rest = [p for p in student.parameters() if id(p) not in chosen]
    return [Muon(matrices), torch.optim.Adam(rest, lr=lr)]


@torch.no_grad()
def answers(logits: torch.Tensor, trials: int, *, given=None, tokens=None, temperature: float = 1.0, top_k: int = 0,
            top_p: float = 1.0, min_p: float = 0.0, generator=None):
    """(candidates (N, trials, H, W), scores (N, trials)) of every board, drawn from logits (N, H, W, n_out): a candidate is a
    class for every cell, its score the mean log-probability of its classes over the cells that are not `given` (bool
    (N, H, W)), whose classes are `tokens` in all candidates.  The best of a board: scores.argmax(1)."""
    n, h, w, _ = logits.shape
    u = torch.rand((n, h, w, trials), generator=generator, device=logits.device)
    classes, probs = ops.sample(logits.detach(), u, temperature=temperature, top_k=top_k, top_p=top_p, min_p=min_p)
    score = probs.clamp_min(1e-30).log()
    cells = torch.full((n, 1), h * w, device=logits.device)
    if given is not None:
        score = score.masked_fill(given[..., None], 0.0)
        cells = (~given).sum((1, 2)).clamp_min(1)[:, None]
        if tokens is not None:
            classes = torch.where(given[..., None], tokens[..., None].to(classes.dtype), classes)
    return classes.permute(0, 3, 1, 2).contiguous(), score.sum((1, 2)) / cells


def train(student: Student, inputs, given, values, index, steps: int, lr: float = 3e-3, temperature: float = 2.0,
          optimizer: str = "adam"):
    """Trains on the cells that are not given; returns the loss of every step."""
    free = (~given).float()
    weight = free / free.sum()
    optimizers = make_optimizers(student, optimizer, lr)
    losses = []
    for _ in range(steps):
        loss = ops.distill_loss(student(inputs), values, index, temperature=temperature, weight=weight, reduction="sum")
        for o in optimizers:
            o.zero_grad()
        loss.backward()
        for o in optimizers:
            o.step()
        losses.append(loss.detach())
    ops.check(inputs.device)
    return torch.stack(losses).tolist()


def main(argv=None) -> list[float]:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--task", choices=("sudoku", "maze"), default="sudoku")
    ap.add_argument("--boards", type=int, default=64)
    ap.add_argument("--size", type=int, default=19, help="side of a maze")
    ap.add_argument("--steps", type=int, default=100)
    ap.add_argument("--teacher-steps", type=int, default=64)
    ap.add_argument("--seed", type=int, default=0)
    ap.add_argument("--scan", action="store_true", help="cells also see gated scans along rows and columns")
    ap.add_argument("--optimizer", choices=("adam", "muon"), default="adam")
    ap.add_argument("--trials", type=int, default=0, help="candidate answers to draw of every board after the training")
    a = ap.parse_args(argv)
    device = torch.device("cuda", torch.cuda.current_device())
    torch.manual_seed(a.seed)
    cfg = model_config(a.task)
    boards = sudoku_boards(a.boards, seed=a.seed) if a.task == "sudoku" else maze_boards(a.boards, a.size, seed=a.seed)
    engine = build(a.task, seed=a.seed, device=device).engine()
    values, index = teacher_top(engine, boards.inputs, boards.given, 4, a.teacher_steps, seed=a.seed)
    student = Student(cfg.vocab_size, cfg.channels, 4 * cfg.channels, cfg.c_out, scan=a.scan).to(device)
    inputs = torch.from_numpy(boards.inputs).long().to(device)
    given = torch.from_numpy(boards.given).bool().to(device)
    losses = train(student, inputs, given, values, index, a.steps, optimizer=a.optimizer)
    print(f"distillation loss a free cell: {losses[0]:.4f} at the first step, {losses[-1]:.4f} after {a.steps}")
    if a.trials:
        with torch.no_grad():
            logits = student(inputs)
        classes, scores = answers(logits, a.trials, given=given, top_p=0.95)
        teacher = index[..., 0].long()  # the class of the teacher's largest logit
        agree = ((classes == teacher[:, None]) | given[:, None]).float().mean((2, 3))
        best = agree.gather(1, scores.argmax(1, keepdim=True)).mean()
        print(f"{a.trials} answers a board: {agree.mean():.4f} of the cells as the teacher's, {best:.4f} in the best by score")
    return losses


if __name__ == "__main__":
    main()
