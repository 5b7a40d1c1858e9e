"""A normalised, gated cell trained on the rollout: the cell-training operators as they are used together.

The teacher is a model of the rollout engine: many asynchronous steps of each board.  Its readout of
the final state, the top logits of every cell, is what a rollout would keep for training.  The student
runs few synchronous steps of a cell with group norm and a gated update
(x + gated_ffn(act(group_norm(perceive(x))))) over channels-last states, and learns the teacher's
readout by distillation of those top logits.  Perception (fixed 3x3 taps) and the head (one matrix)
are plain torch.

    python -m ncas_b200.student --task sudoku --boards 64 --steps 100
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


class GatedCell(nn.Module):
    """One step of the student: perception, group norm with an activation, gated update, residual."""

    def __init__(self, channels: int, hidden: int, groups: int = 4, act: str = "silu", dtype=torch.bfloat16):
        super().__init__()
        wide = 4 * channels
        self.groups, self.act = groups, act
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
        z = ops.group_norm_act(perceive(x), self.groups, self.norm_weight, self.norm_bias, act=self.act, mask=mask)
        return x + ops.gated_ffn(z, self.w_gate, self.w_up, self.w_down, self.b_gate, self.b_up, self.b_down)


class Student(nn.Module):
    """Token embedding, `depth` steps of one GatedCell, a linear readout of `n_out` classes."""

    def __init__(self, vocab: int, channels: int, hidden: int, n_out: int, depth: int = 4, dtype=torch.bfloat16):
        super().__init__()
        self.depth, self.dtype = depth, dtype
        self.embed = nn.Parameter(torch.randn(vocab, channels))
        self.cell = GatedCell(channels, hidden, dtype=dtype)
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


def train(student: Student, inputs, given, values, index, steps: int, lr: float = 3e-3, temperature: float = 2.0):
    """Trains on the cells that are not given; returns the loss of every step."""
    free = (~given).float()
    weight = free / free.sum()
    optimizer = torch.optim.Adam(student.parameters(), lr=lr)
    losses = []
    for _ in range(steps):
        loss = ops.distill_loss(student(inputs), values, index, temperature=temperature, weight=weight, reduction="sum")
        optimizer.zero_grad()
        loss.backward()
        optimizer.step()
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
    a = ap.parse_args(argv)
    device = torch.device("cuda", torch.cuda.current_device())
    torch.manual_seed(a.seed)
    cfg = model_config(a.task)
    boards = sudoku_boards(a.boards, seed=a.seed) if a.task == "sudoku" else maze_boards(a.boards, a.size, seed=a.seed)
    engine = build(a.task, seed=a.seed, device=device).engine()
    values, index = teacher_top(engine, boards.inputs, boards.given, 4, a.teacher_steps, seed=a.seed)
    student = Student(cfg.vocab_size, cfg.channels, 4 * cfg.channels, cfg.c_out).to(device)
    inputs = torch.from_numpy(boards.inputs).long().to(device)
    given = torch.from_numpy(boards.given).bool().to(device)
    losses = train(student, inputs, given, values, index, a.steps)
    print(f"distillation loss a free cell: {losses[0]:.4f} at the first step, {losses[-1]:.4f} after {a.steps}")
    return losses


if __name__ == "__main__":
    main()
