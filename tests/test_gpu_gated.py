"""gated_ffn on the GPU against the 64-bit oracle: types, activations, odd and ragged sizes, one row to
thousands, strides, refusals, streams, repeatability.

Tolerances follow the roundings, element by element (u the unit roundoff of the matrix type, e =
2^-23 a step of a sum on the tensor cores, a 2^-20 for the activation's own arithmetic):
  gate, up        e K sum |terms|
  h               their effect (|act'| <= 1.13), 2^-20 and u of itself
  saved           2^-15 of gate and up
  dgate, dup      the same way from dh = dy Wd (|act''| <= 1.6), and u of themselves
  outputs         what their operands carry, e K sum |terms|, and u of themselves."""

import ctypes as C
import os
import subprocess
import sys
from pathlib import Path

import pytest
import torch
import torch.autograd.forward_ad as fwd

import oracle.cell_operators as O
from ncas_b200 import _lib as L
from ncas_b200 import operators as ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11, torch.float32: 2.0**-24}
E = 2.0**-23
NAMES = ("x", "w_gate", "w_up", "w_down", "b_gate", "b_up", "b_down")


def make(t, d, f, o, dtype, bias=True, seed=0, bias_dtype=None):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s, k=1.0: torch.randn(s, generator=g) * k  # noqa: E731
    a = dict(x=r(t, d), w_gate=r(f, d, k=d**-0.5), w_up=r(f, d, k=d**-0.5), w_down=r(o, f, k=f**-0.5))
    a = {k: v.to(DEV, dtype) for k, v in a.items()}
    for k, n in (("b_gate", f), ("b_up", f), ("b_down", o)):
        a[k] = r(n, k=0.3).to(DEV, bias_dtype or dtype) if bias else None
    return a, r(t, o).to(DEV, dtype)


def bounds(a, dy, act):
    """The oracle's values and how far each output may be from them."""
    h64 = {k: None if v is None else v.detach().cpu().double() for k, v in a.items()}
    want = O.gated_ffn(**h64, name=act, dy=dy.detach().cpu())
    u = UNIT[a["x"].dtype]
    x, wg, wu, wd = (h64[k] for k in NAMES[:4])
    z = torch.zeros((), dtype=torch.float64)
    bg, bu, bd = (z if h64[k] is None else h64[k] for k in NAMES[4:])
    T, D = x.shape
    F, Od = wg.shape[0], wd.shape[0]
    gate, up = x @ wg.T + bg, x @ wu.T + bu
    eg = E * (D + 2) * (x.abs() @ wg.abs().T + bg.abs())
    eu = E * (D + 2) * (x.abs() @ wu.abs().T + bu.abs())
    val, slope = O.act(gate, act)
    h = val * up
    ea = 1.13 * eg + 2.0**-20 * (val.abs() + slope.abs())
    eh = ea * up.abs() + val.abs() * eu + ea * eu + u * h.abs() * 1.01 + 2.0**-24 * (u == 2.0**-11)
    tol = {"y": eh @ wd.abs().T + E * (F + 2) * (h.abs() @ wd.abs().T + bd.abs()) + u * want["y"].abs()}
    d = dy.detach().cpu().double()
    dh = d @ wd
    edh = E * (Od + 2) * (d.abs() @ wd.abs())
    eg, eu = eg + 2.0**-15 * gate.abs(), eu + 2.0**-15 * up.abs()
    es = 1.6 * eg + 2.0**-20 * (1 + gate.abs())
    if act == "relu":
        es = (gate.abs() <= eg).double()
    ea = 1.13 * eg + 2.0**-20 * (val.abs() + slope.abs())
    dg, du = dh * up * slope, dh * val
    tiny = 2.0**-24 * (u == 2.0**-11)  # fp16's spacing below 2^-14
    edg = edh * (up * slope).abs() + dh.abs() * (eu * slope.abs() + up.abs() * es + eu * es) + edh * up.abs() * es
    edg = edg + 1.02 * u * dg.abs() + tiny
    edu = edh * val.abs() + dh.abs() * ea + edh * ea + 1.02 * u * du.abs() + tiny
    tol["x"] = edg @ wg.abs() + edu @ wu.abs() + E * 2 * (F + 2) * (dg.abs() @ wg.abs() + du.abs() @ wu.abs())
    for k, e, v in (("w_gate", edg, dg), ("w_up", edu, du)):
        tol[k] = e.T @ x.abs() + E * (T + 2) * (v.abs().T @ x.abs())
        tol["b" + k[1:]] = e.sum(0) + E * (T + 2) * v.abs().sum(0)
    tol["w_down"] = d.abs().T @ eh + E * (T + 2) * (d.abs().T @ h.abs())
    tol["b_down"] = E * (T + 2) * d.abs().sum(0)
    for k in NAMES:
        if a[k] is not None:
            tol[k] = tol[k] + UNIT[a[k].dtype] * want[k].abs() + 2.0**-24
    return want, tol


def compare(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape, what
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {float(((got - want).abs() / tol).max()):.2f}"


def check(a, dy, act="silu"):
    leaves = {k: v.detach().requires_grad_() for k, v in a.items() if v is not None}
    y = ops.gated_ffn(**{k: leaves.get(k) for k in NAMES}, act=act)
    grads = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    with torch.no_grad():
        again = ops.gated_ffn(**a, act=act)
    ops.check()
    want, tol = bounds(a, dy, act)
    assert y.dtype == a["x"].dtype
    compare(y, want["y"], tol["y"], "y")
    compare(again, want["y"], tol["y"], "y of the inference call")
    for k, g in grads.items():
        assert g.dtype == a[k].dtype
        compare(g, want[k], tol[k], "d" + k)
    return y, grads


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,d,f,o", [
    (1, 64, 64, 64), (1, 8, 8, 8), (1, 1, 1, 1), (2, 3, 5, 7), (17, 100, 36, 20), (64, 256, 256, 64), (81, 256, 256, 64),
    (129, 130, 131, 132), (200, 72, 520, 40), (300, 33, 65, 129), (777, 128, 96, 256), (1, 520, 1000, 264),
    (8, 1024, 640, 512), (16, 200, 1030, 17), (31, 264, 2048, 128), (33, 72, 136, 8), (1500, 16, 24, 9),
    (130, 40, 9000, 24), (3, 700, 8200, 41), (70, 4100, 300, 40), (900, 33, 2100, 269),  # long k axes, few tiles
    (16, 640, 256, 4100), (48, 96, 1300, 1000),
])
def test_against_the_oracle(dtype, t, d, f, o):
    check(*make(t, d, f, o, dtype, seed=t + d))


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t", [3, 150])
def test_activations_and_biases(act, dtype, t):
    check(*make(t, 72, 200, 48, dtype, seed=1), act=act)
    check(*make(t, 72, 200, 48, dtype, bias=False, seed=2), act=act)
    check(*make(t, 72, 200, 48, dtype, seed=3, bias_dtype=torch.float32), act=act)
    a, dy = make(t, 72, 200, 48, dtype, seed=4)
    a["b_up"] = None
    check(a, dy, act)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_tiles_on_multiprocessor_pairs(dtype):
    # large enough for the 256 x 256 tiles of two multiprocessors in every product, with ragged edges
    check(*make(2600, 280, 2072, 2064, dtype, seed=5))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,d,f,o", [
    (5216, 2048, 64, 2048),  # y and dx: 21 x 8 tiles of 256 x 256, the last row of tiles with 96 rows
    (72, 2048, 5216, 40),    # dWg, dWu
    (72, 40, 2048, 5216),    # dWd
])
def test_tiles_without_rows_between_tiles_with_rows(dtype, t, d, f, o):
    # several tiles for each pair of multiprocessors and a short k axis: the warps whose 32 rows of a tile
    # lie beyond the matrix go on at once to the next tile while their stores of the tile before are read
    a, dy = make(t, d, f, o, dtype, seed=16)
    y, grads = check(a, dy)
    for _ in range(10):
        leaves = {k: v.detach().requires_grad_() for k, v in a.items()}
        y2 = ops.gated_ffn(**leaves)
        got = torch.autograd.grad(y2, list(leaves.values()), dy)
        assert torch.equal(y2, y)
        for k, g in zip(leaves, got):
            assert torch.equal(g, grads[k]), k


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_first_tiles_of_many_repeat(dtype, act):
    # the saved planes of a block's first tile are there before its accumulators: 12 x 8 tiles of 256 x 256
    # of dh, each block's first piece against the oracle, and bit for bit in ten runs
    a, dy = make(3001, 80, 2000, 208, dtype, seed=18)
    _, grads = check(a, dy, act)
    for _ in range(10):
        leaves = {k: v.detach().requires_grad_() for k, v in a.items()}
        got = torch.autograd.grad(ops.gated_ffn(**leaves, act=act), list(leaves.values()), dy)
        for k, g in zip(leaves, got):
            assert torch.equal(g, grads[k]), k


@pytest.mark.parametrize("dtype,act", [(torch.float16, "sigmoid"), (torch.bfloat16, "sigmoid"), (torch.bfloat16, "silu")])
def test_backward_of_many_pieces_repeats(dtype, act):
    # 294 x 18 tiles of dh, 8 pieces of 32 columns each: a piece's planes are asked for as soon as those
    # before have been read
    g = torch.Generator(device=DEV).manual_seed(19)
    r = lambda *s, k=1.0: torch.randn(s, generator=g, device=DEV).mul_(k).to(dtype)  # noqa: E731
    t, d, f, o = 75243, 56, 4444, 639
    leaves = [v.requires_grad_() for v in (r(t, d), r(f, d, k=d**-0.5), r(f, d, k=d**-0.5), r(o, f, k=f**-0.5),
                                           r(f, k=0.1), r(f, k=0.1), r(o, k=0.1))]
    y, dy = ops.gated_ffn(*leaves, act=act), r(t, o)
    first = torch.autograd.grad(y, leaves, dy, retain_graph=True)
    for _ in range(150):
        got = torch.autograd.grad(y, leaves, dy, retain_graph=True)
        assert all(torch.equal(p, q) for p, q in zip(first, got))


def test_long_row_axis_in_pieces():
    check(*make(20001, 64, 72, 24, torch.bfloat16, seed=6))


@pytest.mark.parametrize("t", [5, 140])
def test_strides(t):
    dtype = torch.bfloat16
    a, dy = make(t, 64, 88, 40, dtype, seed=7)
    y, grads = check(a, dy)

    def same(b, dyb=dy):
        leaves = {k: v.detach().requires_grad_() for k, v in b.items() if v is not None}
        y2 = ops.gated_ffn(**{k: leaves.get(k) for k in NAMES})
        g2 = torch.autograd.grad(y2, list(leaves.values()), dyb)
        assert torch.equal(y2, y) and all(torch.equal(p, q) for p, q in zip(g2, grads.values()))

    fused = torch.cat([a["w_gate"], a["w_up"]])  # one matrix, two halves
    same({**a, "w_gate": fused[:88], "w_up": fused[88:]})
    mixed = torch.stack([a["w_gate"], a["w_up"]], 1)  # rows of the two in turn
    same({**a, "w_gate": mixed[:, 0], "w_up": mixed[:, 1]})
    for k in ("x", "w_gate", "w_up", "w_down"):
        same({**a, k: a[k].t().contiguous().t()})  # transposed
        wide = torch.full((a[k].shape[0], a[k].shape[1] + 24), float("nan"), device=DEV, dtype=dtype)
        for off in (8, 3):  # rows on 16-byte boundaries, and not
            v = wide[:, off : off + a[k].shape[1]]
            v.copy_(a[k])
            same({**a, k: v})
    same(a, dy.t().contiguous().t())
    wide = torch.full((t, 61), float("nan"), device=DEV, dtype=dtype)
    wide[:, 7:47] = dy
    same(a, wide[:, 7:47])
    b = {**a, "b_gate": torch.stack([a["b_gate"]] * 2, 1)[:, 0]}
    same(b)
    # expanded inputs: one row for all, and the gradient of a broadcast dy
    x = a["x"][:1].expand(t, 64)
    check({**a, "x": x}, dy[:1].expand(t, 40))
    check(a, torch.ones((), device=DEV, dtype=dtype).expand(t, 40))


def test_leading_sizes():
    a, dy = make(24, 32, 40, 16, torch.float16, seed=8)
    y, grads = check(a, dy)
    x = a["x"].view(2, 3, 4, 32).requires_grad_()
    y3 = ops.gated_ffn(x, *[a[k] for k in NAMES[1:]])
    assert y3.shape == (2, 3, 4, 16) and torch.equal(y3.view(24, 16), y)
    (gx,) = torch.autograd.grad(y3, x, dy.view(2, 3, 4, 16))
    assert torch.equal(gx.view(24, 32), grads["x"])
    with torch.no_grad():
        one = ops.gated_ffn(a["x"][0], *[a[k] for k in NAMES[1:]])
    assert one.shape == (16,)


def test_empty_rows():
    a, _ = make(0, 32, 40, 16, torch.bfloat16)
    leaves = {k: v.detach().requires_grad_() for k, v in a.items()}
    y = ops.gated_ffn(**leaves)
    assert y.shape == (0, 16)
    for k, g in zip(leaves, torch.autograd.grad(y.sum(), list(leaves.values()))):
        assert g.shape == leaves[k].shape and (g == 0).all()


def test_parts_of_the_gradient():
    a, dy = make(70, 40, 56, 24, torch.bfloat16, seed=9)
    _, grads = check(a, dy)
    for only in [("x",), ("w_gate",), ("w_up",), ("w_down",), ("b_gate",), ("b_up",), ("b_down",), ("x", "w_up")]:
        b = {k: v.detach().requires_grad_(k in only) for k, v in a.items()}
        got = torch.autograd.grad(ops.gated_ffn(**b), [b[k] for k in only], dy)
        # alone, a weight's product may be cut into other pieces: one more rounding of the type
        for k, g in zip(only, got):
            assert ((g - grads[k]).abs() <= 2.0**-7 * grads[k].abs() + 2.0**-14 * grads[k].abs().max()).all(), k
    leaf = a["x"].detach().requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(ops.gated_ffn(leaf, *[a[k] for k in NAMES[1:]]).sum(), leaf, create_graph=True)


def test_gradient_against_differences():
    # the loss of rows that differ in x by +-h v, in fp16 with fp32 sums: h v with h = 2^-4 is exact in
    # the sum x + h v only to 2^-11, so the difference quotient carries 2^-11 * 2^4 |f'| |x| and the
    # curvature h^2 / 6 |f'''|: about 2^-6 of sum |g v| for these well-scaled inputs
    a, dy = make(40, 32, 64, 16, torch.float16, seed=10)
    v = (torch.randint(0, 2, (40, 32), generator=torch.Generator().manual_seed(3)) * 2 - 1).to(DEV, torch.float16)
    f = lambda x: (ops.gated_ffn(**{**a, "x": x}).double() * dy.double()).sum().item()  # noqa: E731
    leaf = a["x"].detach().requires_grad_()
    (g,) = torch.autograd.grad(ops.gated_ffn(**{**a, "x": leaf}), leaf, dy)
    h = 2.0**-4
    plus, minus = a["x"] + h * v, a["x"] - h * v
    slope = f(plus) - f(minus)
    want = float((g.double() * (plus.double() - minus.double())).sum())
    size = float((g.double() * (plus.double() - minus.double())).abs().sum())
    assert abs(slope - want) <= 2.0**-6 * size


def test_large_pre_activations_do_not_overflow_in_fp16():
    # gate and up of 1e5 do not fit fp16; h, which does, and the gradients have to survive
    a, dy = make(9, 64, 32, 16, torch.float16, bias=False, seed=11)
    with torch.no_grad():
        a["w_up"].mul_(4000).clamp_(-60000, 60000)
        a["x"].mul_(20)
        a["w_gate"].mul_(0.0005)
        a["w_down"].mul_(0.01)
        dy = dy * 1e-4
    h = (a["x"].double() @ a["w_up"].double().T).abs().max()
    assert h > 70000
    y = ops.gated_ffn(**a, act="relu")
    assert torch.isfinite(y).all()
    check(a, dy, act="relu")


def test_non_finite_rows_stay_in_their_rows():
    a, _ = make(200, 64, 96, 40, torch.bfloat16, seed=12)
    want = ops.gated_ffn(**a)
    x = a["x"].clone()
    x[7, 3] = float("nan")
    x[150] = float("inf")
    y = ops.gated_ffn(**{**a, "x": x})
    rows = torch.ones(200, dtype=torch.bool, device=DEV)
    rows[7] = rows[150] = False
    assert torch.equal(y[rows], want[rows]) and not torch.isfinite(y[7]).any()


def test_repeatable_and_on_other_streams():
    a, dy = make(3000, 128, 136, 64, torch.bfloat16, seed=13)
    run = lambda: (lambda l: torch.autograd.grad(ops.gated_ffn(**l), list(l.values()), dy))(  # noqa: E731
        {k: v.detach().requires_grad_() for k, v in a.items()})
    first = run()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got.append(run())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    for g in got:
        assert all(torch.equal(p, q) for p, q in zip(first, g))


def test_from_a_thread_without_a_context():
    import threading

    a, dy = make(64, 64, 72, 24, torch.bfloat16, seed=15)
    with torch.no_grad():
        want = ops.gated_ffn(**a)
    torch.cuda.synchronize()
    got = []
    thread = threading.Thread(target=lambda: got.append(ops.gated_ffn(**a)))
    thread.start()
    thread.join()
    torch.cuda.synchronize()
    assert len(got) == 1 and torch.equal(got[0], want)


def test_inside_a_cuda_graph():
    a, _ = make(1, 256, 512, 128, torch.bfloat16, seed=14)
    with torch.no_grad():
        want = ops.gated_ffn(**a)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.gated_ffn(**a)
        y.zero_()
        graph.replay()
        assert torch.equal(y, want)


@pytest.mark.parametrize("saved", [True, False])
def test_a_wait_that_runs_out_is_reported(saved):
    """The C ABI with a limit of 1 ms on products over 2^27 values a row: one tile, or the eighth of it that a
    block of the few-row product takes, is at least 2^18 steps of 0.1 us, and a wait polls 64 times for at
    most 0.5 ms before it looks at its limit.  The call ends with the status set, and the device goes on."""
    lib = L.lib()
    wide, out = 1 << 27, 8
    x, w = (torch.zeros((1, wide), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    down = torch.zeros((out, 1), device=DEV, dtype=torch.bfloat16)
    bias = torch.ones(1, device=DEV)
    y = torch.empty((1, out), device=DEV, dtype=torch.bfloat16)
    ctrl = torch.zeros(4, device=DEV, dtype=torch.int32)
    d = L.NcaGatedDesc(rows=1, d_in=wide, hidden=1, d_out=out, dtype=1, bias_dtype=0, act=2)
    for name, t in (("x_stride", x), ("w_gate_stride", w), ("w_up_stride", w), ("w_down_stride", down)):
        getattr(d, name)[0], getattr(d, name)[1] = t.stride()
    size = C.c_size_t(0)
    assert lib.nca_b200_gated_workspace(C.byref(d), 0, C.byref(size)) == 0
    ws = torch.empty(size.value, device=DEV, dtype=torch.uint8)
    assert lib.nca_b200_gated_saved_bytes(C.byref(d), C.byref(size)) == 0
    kept = torch.empty(size.value, device=DEV, dtype=torch.uint8) if saved else None
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: None if t is None else C.c_void_p(t.data_ptr())  # noqa: E731
    detail = C.c_int32(0)
    late = (104,) if saved else (112, 113)  # the second few-row product waits for the first
    for limit, status, sites in ((1, 4, late), (20000, 0, (0,))):
        st = lib.nca_b200_gated_ffn(C.byref(d), p(x), p(w), p(w), p(down), p(bias), p(bias), None, p(y), p(kept), p(ws),
                                    ws.numel(), p(ctrl), limit, stream)
        assert st == 0
        assert lib.nca_b200_ctrl_status(p(ctrl), C.byref(detail), stream) == status
        assert detail.value in sites
        torch.cuda.synchronize()
    assert (y == 0).all()
    a, dy = make(70, 40, 56, 24, torch.bfloat16, seed=17)
    check(a, dy)


@pytest.mark.parametrize("saved", [True, False])
def test_a_failure_that_nobody_has_read_does_not_end_later_calls(saved):
    """The same products with control words that an earlier call has set: waits long enough to look at them
    still end with the product, and the words stay for whoever asks."""
    lib = L.lib()
    wide, out = 1 << 27, 8
    x, w = (torch.zeros((1, wide), device=DEV, dtype=torch.bfloat16) for _ in range(2))
    down = torch.ones((out, 1), device=DEV, dtype=torch.bfloat16)
    bias = torch.ones(1, device=DEV)
    y = torch.zeros((1, out), device=DEV, dtype=torch.bfloat16)
    ctrl = torch.tensor([4, 77, 0, 1], device=DEV, dtype=torch.int32)
    d = L.NcaGatedDesc(rows=1, d_in=wide, hidden=1, d_out=out, dtype=1, bias_dtype=0, act=1)
    for name, t in (("x_stride", x), ("w_gate_stride", w), ("w_up_stride", w), ("w_down_stride", down)):
        getattr(d, name)[0], getattr(d, name)[1] = t.stride()
    size = C.c_size_t(0)
    assert lib.nca_b200_gated_workspace(C.byref(d), 0, C.byref(size)) == 0
    ws = torch.zeros(size.value, device=DEV, dtype=torch.uint8)
    assert lib.nca_b200_gated_saved_bytes(C.byref(d), C.byref(size)) == 0
    kept = torch.zeros(size.value, device=DEV, dtype=torch.uint8) if saved else None
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: None if t is None else C.c_void_p(t.data_ptr())  # noqa: E731
    st = lib.nca_b200_gated_ffn(C.byref(d), p(x), p(w), p(w), p(down), p(bias), p(bias), None, p(y), p(kept), p(ws),
                                ws.numel(), p(ctrl), 20000, stream)
    assert st == 0
    detail = C.c_int32(0)
    assert lib.nca_b200_ctrl_status(p(ctrl), C.byref(detail), stream) == 4 and detail.value == 77
    assert (y == 1).all()  # relu(1) 1 through weights of 1


THREADS = """
import queue, threading
import torch
from ncas_b200 import operators as ops
from ncas_b200._lib import NcaError

def told():
    try:
        ops.check()
    except NcaError:
        return True
    return False

small = [torch.zeros(s, device="cuda", dtype=torch.bfloat16) for s in ((2, 8), (8, 8), (8, 8), (8, 8))]
ask, answer = queue.Queue(), queue.Queue()
def user():
    torch.cuda.set_device(0)
    ops.gated_ffn(*small)
    answer.put(told())
    while ask.get():
        answer.put(told())
other = threading.Thread(target=user)
other.start()
assert not answer.get() and not told()
x, w = (torch.zeros((1, 1 << 27), device="cuda", dtype=torch.bfloat16) for _ in range(2))
ops.gated_ffn(x, w, w, small[0][:, :1])
assert told() and not told()
for first in (True, False):  # the other thread is told too, once
    ask.put(True)
    assert answer.get() == first
ask.put(False)
other.join()
late = threading.Thread(target=lambda: answer.put(told()))  # began after the failure
late.start()
assert not answer.get()
late.join()
print("told")
"""


def test_every_thread_is_told_of_a_wait_that_ran_out():
    env = {**os.environ, "NCA_B200_TIMEOUT_MS": "1"}
    got = subprocess.run([sys.executable, "-c", THREADS], env=env, cwd=Path(__file__).parent.parent, capture_output=True,
                         text=True, timeout=120)
    assert got.returncode == 0 and got.stdout.split() == ["told"], got.stderr[-2000:]


def test_forward_mode_tangents_are_refused():
    a, dy = make(4, 16, 24, 8, torch.bfloat16)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for k in NAMES:
            with pytest.raises(ValueError, match=f"{k} carries a forward-mode tangent"):
                ops.gated_ffn(**{**a, k: dual(a[k])})
        leaf = a["x"].clone().requires_grad_()
        y = ops.gated_ffn(**{**a, "x": leaf})
        with pytest.raises(ValueError, match="tangent"):
            torch.autograd.grad(y, leaf, dual(dy))


def test_refusals():
    a, _ = make(4, 16, 24, 8, torch.bfloat16)
    for kw, exc, text in [
        (dict(act="none"), ValueError, "act"), (dict(act="tanh"), ValueError, "act"),
        (dict(x=a["x"].float()), TypeError, "bfloat16"), (dict(w_up=a["w_up"].half()), TypeError, "w_up"),
        (dict(w_up=a["w_up"][:-1]), ValueError, "w_up"), (dict(w_gate=a["w_gate"][:, :-1]), ValueError, "w_gate"),
        (dict(w_down=a["w_down"][:, :-1]), ValueError, "w_down"), (dict(w_down=a["w_down"][0]), ValueError, "w_down"),
        (dict(w_down=a["w_down"].cpu()), ValueError, "CUDA"), (dict(b_up=a["b_up"][:-1]), ValueError, "b_up"),
        (dict(b_up=a["b_up"].float()), TypeError, "one type"), (dict(b_up=a["b_up"].double()), TypeError, "b_up"),
        (dict(x=a["x"][:, :0]), ValueError, "d_in"), (dict(w_gate=a["w_gate"][:0]), ValueError, "w_gate"),
    ]:
        with pytest.raises(exc, match=text):
            ops.gated_ffn(**{**a, **kw})
