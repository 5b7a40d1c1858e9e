"""gated_scan and its gradient on the GPU against the 64-bit oracle.

Tolerances follow the recurrence's own rounding errors, element by element (e = 2^-24).  a and 1 - a carry
k = e (|gate| + 8) of themselves: the product gate log2(e), the exponential (2 units), the sum, the reciprocal and
a product.  A step a h + (1 - a) x then adds k of both products, e of the second and e of their sum, and passes on a of the
error before it; G = dy + r adds e, and r = a G k a |G| (two 16-bit channels: G - (1 - a) G, k (1 - a) |G|) and e of itself.
The bounds E below are these sums, run along the line; maps of several steps, composed, round each factor and sum once more, at
most as much again for the warps of a block and once more for the pieces of a line, so four times E holds for every
path.  Outputs add half a step of their type."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

import oracle.cell_operators as O
from ncas_b200 import operators as ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
E = 2.0**-24
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-126, torch.bfloat16: 2.0**-126, torch.float16: 2.0**-25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(shape, dim, dtype, seed=0, state=True, mask=None):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(shape, generator=g).to(dtype)
    gate = (torch.randn(shape, generator=g) + 4 * torch.rand(shape[-1], generator=g)).to(dtype)
    dy = torch.randn(shape, generator=g).to(dtype)
    edge = [s for i, s in enumerate(shape) if i != dim % len(shape)]
    h = torch.randn(edge, generator=g) if state else None
    dlast = torch.randn(edge, generator=g)
    m = None
    if mask is not None:
        m = torch.rand(shape[:-1], generator=g) < mask
        m.movedim(dim, -1).reshape(-1, shape[dim])[0] = False  # a line without any step
    return x, gate, h, m, dy, dlast


def bounds(x, gate, h, dim, reverse, mask, dy, dlast):
    """The oracle's values and the error bounds of y, last, x, gate, state (before the type's rounding)."""
    dim = dim % x.dim()
    want = O.gated_scan(x, gate, h, dim, reverse, mask, dy, dlast)
    mv = lambda t: t.double().movedim(dim, 0)  # noqa: E731
    xs, gs, ds = mv(x), mv(gate), mv(dy)
    steps = list(range(xs.shape[0]))[:: -1 if reverse else 1]
    on = torch.ones(xs.shape[:-1], dtype=torch.bool) if mask is None else mask.movedim(dim, 0) != 0
    state = torch.zeros(xs.shape[1:], dtype=torch.float64) if h is None else h.double()
    a, keep, k = torch.sigmoid(gs), torch.sigmoid(-gs), E * (gs.abs() + 8)
    err, ey, eb, before = torch.zeros_like(state), torch.zeros_like(xs), torch.zeros_like(xs), torch.zeros_like(xs)
    for t in steps:
        live = on[t][..., None]
        eb[t], before[t] = err, state
        state = torch.where(live, a[t] * state + keep[t] * xs[t], state)
        step = a[t] * err + a[t] * k[t] * before[t].abs() + keep[t] * (k[t] + E) * xs[t].abs() + E * state.abs()
        err = torch.where(live, step, err)
        ey[t] = err
    el = err
    r = torch.zeros_like(state) if dlast is None else dlast.double()
    er, ex, eg = torch.zeros_like(r), torch.zeros_like(xs), torch.zeros_like(xs)
    for t in reversed(steps):
        live = on[t][..., None]
        G, q = ds[t] + r, before[t] - xs[t]
        eG = er + E * G.abs()
        ex[t] = keep[t] * eG + (k[t] + 2 * E) * (keep[t] * G).abs()
        eg[t] = (a[t] * keep[t]) * (G.abs() * (eb[t] + E * q.abs()) + q.abs() * eG + (2 * k[t] + 5 * E) * (G * q).abs())
        r = torch.where(live, a[t] * G, r)
        share = a[t] if x.dtype == torch.float32 else torch.maximum(a[t], keep[t])
        er = torch.where(live, a[t] * eG + share * k[t] * G.abs() + E * (a[t] * G).abs(), er)
    back = lambda t: t.movedim(0, dim)  # noqa: E731
    return want, dict(y=back(ey), last=el, x=back(ex), gate=back(eg), state=er)


def close(got, want, bound, name):
    u = 0.0 if name in ("last", "state") else UNIT[got.dtype]
    off = (got.detach().cpu().double() - want).abs()
    tol = 4 * bound + (u + E) * want.abs() + TINY[got.dtype]
    assert (off <= tol).all(), (name, float((off / tol).max()))


def check(x, gate, h=None, mask=None, dy=None, dlast=None, dim=-2, reverse=False, put=lambda t: t.to(DEV)):
    want, bound = bounds(x, gate, h, dim, reverse, mask, dy, dlast)
    leaves = [None if t is None else put(t).requires_grad_() for t in (x, gate, h)]
    m = None if mask is None else put(mask)
    y, last = ops.gated_scan(*leaves, dim=dim, reverse=reverse, mask=m)
    assert y.is_contiguous() and y.dtype == x.dtype and y.shape == x.shape and last.dtype == torch.float32
    close(y, want["y"], bound["y"], "y")
    close(last, want["last"], bound["last"], "last")
    with torch.no_grad():  # without the states that a backward pass needs
        y0, last0 = ops.gated_scan(*leaves, dim=dim, reverse=reverse, mask=m)
        assert torch.equal(y0, y) and torch.equal(last0, last)
    named = [(n, t) for n, t in zip(("x", "gate", "state"), leaves) if t is not None]
    grads = torch.autograd.grad([y, last], [t for _, t in named], [put(dy), put(dlast)])
    for (n, _), g in zip(named, grads):
        close(g, want[n], bound[n], n)
    if mask is not None:
        gone = ~m.bool()
        assert (y[gone] == 0).all() and (grads[0][gone] == 0).all() and (grads[1][gone] == 0).all()
    return y, last, grads


@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,t,c", [
    (1, 1, 1), (3, 1, 64), (2, 2, 7), (5, 9, 64), (4, 16, 10), (4, 17, 10), (3, 59, 32), (2, 100, 33), (1, 257, 8),
    (1, 1000, 5), (2, 1031, 66), (1, 5000, 24), (300, 40, 260)])
def test_against_the_oracle(n, t, c, dtype, reverse):
    x, gate, h, _, dy, dlast = inputs((n, t, c), 1, dtype, seed=t)
    check(x, gate, h, None, dy, dlast, 1, reverse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape,dim", [((6, 9, 9, 16), 1), ((6, 9, 9, 16), 2), ((6, 9, 9, 16), 0), ((3, 30, 31, 5), -2),
                                       ((2, 40, 3, 7), 1), ((700, 3), 0), ((4, 2, 3, 20, 6), 2)])
def test_axes(shape, dim, dtype):
    x, gate, h, m, dy, dlast = inputs(shape, dim % len(shape), dtype, seed=3, mask=0.8)
    check(x, gate, h, m, dy, dlast, dim, False)
    check(x, gate, None, None, dy, dlast, dim, True)


# a few steps, whose rows a thread takes 16 bytes at a time where they lie on such places
@pytest.mark.parametrize("reverse", [False, True])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,t,m,c", [(1, 1, 1, 8), (130, 1, 1, 40), (7, 2, 3, 16), (3, 3, 50, 4), (5, 4, 9, 24), (2, 5, 4, 8), (4, 4, 4, 12)])
def test_a_few_steps(n, t, m, c, dtype, reverse):
    for dim, shape in ((1, (n, t, m, c)), (2, (n, m, t, c))):
        x, gate, h, mask, dy, dlast = inputs(shape, dim, dtype, seed=n + t, mask=0.6)
        check(x, gate, h, mask, dy, dlast, dim, reverse)
        check(x, gate, None, None, dy, dlast, dim, reverse)
        # the state on a 4-byte boundary; rows on 16 bytes in a wider tensor; rows off them
        def padded(k):
            def put(t):
                if t.dim() == 3 and t.dtype == torch.float32:
                    return torch.cat((torch.zeros(1), t.reshape(-1))).to(DEV)[1:].view(t.shape)
                return torch.cat((t, t[..., :1].expand(*t.shape[:-1], k)), -1).to(DEV)[..., : t.shape[-1]] if t.dim() == 4 else t.to(DEV)
            return put

        check(x, gate, h, mask, dy, dlast, dim, reverse, put=padded(8))
        check(x, gate, h, mask, dy, dlast, dim, reverse, put=padded(1))


# many lines of up to 64 steps: a thread a line with several channels, in the backward alone or in both directions
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,t,m,c", [(300, 9, 9, 64), (700, 9, 9, 64), (2500, 5, 2, 64), (1300, 8, 30, 8), (1, 16, 5000, 72),
                                     (90, 64, 7, 512), (5000, 33, 1, 64), (1200, 65, 1, 256)])
def test_many_lines(n, t, m, c, dtype):
    for dim, shape, reverse in ((1, (n, t, m, c), False), (2, (n, m, t, c), True)):
        x, gate, h, mask, dy, dlast = inputs(shape, dim, dtype, seed=t, mask=0.8)
        check(x, gate, None, None, dy, dlast, dim, reverse)
        check(x, gate, h, mask, dy, dlast, dim, reverse)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,t,c", [(5, 9, 32), (300, 3, 16), (2, 300, 16), (1, 3000, 6)])
def test_masked_steps_hold_anything(n, t, c, dtype):
    x, gate, h, m, dy, dlast = inputs((n, t, c), 1, dtype, seed=1, mask=0.6)
    want = check(x, gate, h, m, dy, dlast, 1, True)
    for bad in (float("nan"), float("inf"), -float("inf")):
        xs, gs, ds = (v.masked_fill(~m[..., None], bad).to(DEV) for v in (x, gate, dy))
        leaves = [xs.requires_grad_(), gs.requires_grad_(), h.to(DEV).requires_grad_()]
        y, last = ops.gated_scan(*leaves, dim=1, reverse=True, mask=m.to(DEV).to(torch.uint8))
        grads = torch.autograd.grad([y, last], leaves, [ds, dlast.to(DEV)])
        for a, b in zip((y, last, *grads), (*want[:2], *want[2])):
            assert torch.equal(a, b)


def test_gates_at_their_limits():
    gate = torch.tensor([-float("inf"), -200.0, -20.0, -1.0, 0.0, 1.0, 20.0, 200.0, float("inf"), 60000.0]).repeat(40, 1)[None]
    x = torch.randn((1, 40, 10), generator=torch.Generator().manual_seed(0))
    h = torch.full((1, 10), 3.0)
    y, last = ops.gated_scan(x.to(DEV), gate.to(DEV), h.to(DEV), dim=1)
    want, _ = O.gated_scan(x, gate, h, 1)
    # beyond 87 the gate's smaller share is below 2^-125; sigmoid(20) leaves 2^-29 a step
    assert (y.cpu().double() - want).abs().max() <= 40 * 30 * E
    assert torch.equal(y[0, :, 0].cpu(), x[0, :, 0]) and (y[0, :, 8] == 3.0).all()
    gate[0, 7, 4] = float("nan")
    x[0, 9, 2] = float("inf")
    y, last = ops.gated_scan(x.to(DEV), gate.to(DEV), h.to(DEV), dim=1)
    assert y[0, 7:, 4].isnan().all() and not y[0, :7].isnan().any()
    assert y[0, 9, 2] == float("inf")


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    x, gate, h, m, dy, dlast = inputs((3, 50, 12), 1, dtype, seed=2, mask=0.9)
    views = [
        lambda t: t.to(DEV).transpose(0, -1).contiguous().transpose(0, -1) if t.dim() == 3 else t.to(DEV),  # copied
        lambda t: torch.cat([t, t], -1).to(DEV)[..., : t.shape[-1]] if t.dim() == 3 else t.to(DEV),
        lambda t: torch.cat([t[..., :1], t], -1).to(DEV)[..., 1:] if t.dim() == 3 else t.to(DEV),  # odd starts and rows
        lambda t: t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1),
    ]
    for put in views:
        check(x, gate, h, m, dy, dlast, 1, False, put)


def test_broadcast_inputs_sum_their_gradients():
    x, gate, h, _, dy, dlast = inputs((4, 33, 6), 1, torch.float32, seed=5)
    gate = gate[:1, :1]
    full = gate.expand(4, 33, 6)
    want, bound = bounds(x, full, h, 1, False, None, dy, dlast)
    g = gate.to(DEV).requires_grad_()
    y, last = ops.gated_scan(x.to(DEV), g.expand(4, 33, 6), h.to(DEV), dim=1)
    (got,) = torch.autograd.grad([y, last], [g], [dy.to(DEV), dlast.to(DEV)])
    total = want["gate"].sum((0, 1), keepdim=True)
    tol = (4 * bound["gate"] + 2 * E * want["gate"].abs()).sum((0, 1), keepdim=True) + 140 * E * want["gate"].abs().sum((0, 1), keepdim=True)
    assert ((got.cpu().double() - total).abs() <= tol).all()


@pytest.mark.parametrize("shape", [(0, 5, 4), (3, 0, 4), (3, 5, 0), (2, 0, 3, 4)])
def test_sizes_of_zero(shape):
    x = torch.zeros(shape, device=DEV, requires_grad=True)
    h = torch.randn([shape[0], *shape[2:]], device=DEV, requires_grad=True)
    y, last = ops.gated_scan(x, x, h, dim=1)
    assert y.shape == x.shape and (torch.equal(last, h) or shape[1] != 0)
    gx, gh = torch.autograd.grad([y, last], [x, h], [torch.zeros_like(y), torch.ones_like(last)])
    assert gx.shape == x.shape and (shape[1] != 0 or (gh == 1).all())
    assert ops.gated_scan(x.detach(), x.detach(), dim=1)[1].abs().sum() == 0


def test_a_line_in_parts_is_the_whole_line():
    # single tokens and pieces with the state handed on: the states in between are fp32, so nothing but the order
    # of a few roundings differs
    x, gate, h, _, dy, dlast = inputs((3, 70, 20), 1, torch.float32, seed=7)
    want, bound = bounds(x, gate, h, 1, False, None, dy, dlast)
    state, parts = h.to(DEV), []
    for a, b in [(0, 1), (1, 2), (2, 40), (40, 41), (41, 70)]:
        y, state = ops.gated_scan(x[:, a:b].to(DEV), gate[:, a:b].to(DEV), state, dim=1)
        parts.append(y)
    close(torch.cat(parts, 1), want["y"], bound["y"], "y")
    close(state, want["last"], bound["last"], "last")


@pytest.mark.parametrize("use", ["y", "last"])
def test_one_output_alone(use):
    x, gate, h, _, dy, dlast = inputs((2, 200, 6), 1, torch.float32, seed=8)
    zero = torch.zeros_like
    want, bound = bounds(x, gate, h, 1, False, None, dy if use == "y" else zero(dy), dlast if use == "last" else zero(dlast))
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate, h)]
    y, last = ops.gated_scan(*leaves, dim=1)
    grads = torch.autograd.grad(y if use == "y" else last, leaves, (dy if use == "y" else dlast).to(DEV))
    for n, g in zip(("x", "gate", "state"), grads):
        close(g, want[n], bound[n], n)
    (only,) = torch.autograd.grad(ops.gated_scan(x.to(DEV), leaves[1], h.to(DEV), dim=1)[0], leaves[1], dy.to(DEV))
    if use == "y":
        assert torch.equal(only, grads[1])


def test_gradient_against_differences():
    # central differences of fp32 outputs summed in 64 bits: h^2 of the third derivative and E / h of the outputs
    x, gate, h, _, dy, dlast = inputs((2, 21, 3), 1, torch.float32, seed=9)
    leaves = [t.to(DEV).requires_grad_() for t in (x, gate, h)]
    outs = ops.gated_scan(*leaves, dim=1)
    grads = torch.autograd.grad(outs, leaves, [dy.to(DEV), dlast.to(DEV)])
    step = 2.0**-7
    for i, g in enumerate(grads):
        v = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(i)).to(DEV)

        def value(sign):
            moved = [t.detach() + sign * step * v if j == i else t.detach() for j, t in enumerate(leaves)]
            y, last = ops.gated_scan(*moved, dim=1)
            return (y.double() * dy.to(DEV)).sum() + (last.double() * dlast.to(DEV)).sum()

        slope = float(value(1) - value(-1)) / (2 * step)
        size = float(g.double().norm() * v.double().norm())
        assert abs(slope - float((g.double() * v).sum())) <= 2e-3 * size


def test_pieces_of_a_long_line_repeat_bit_for_bit_on_other_streams():
    x, gate, h, _, dy, dlast = (None if t is None else t.to(DEV) for t in inputs((1, 20011, 40), 1, torch.bfloat16, seed=4))
    leaves = [t.requires_grad_() for t in (x, gate, h)]

    def once():
        y, last = ops.gated_scan(*leaves, dim=1)
        return y, last, *torch.autograd.grad([y, last], leaves, [dy, dlast])

    want = once()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(3)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(once())
    torch.cuda.synchronize()
    for g in got:
        assert all(torch.equal(a, b) for a, b in zip(g, want))


def test_captured_and_replayed():
    x, gate, h, _, dy, dlast = (None if t is None else t.to(DEV) for t in inputs((1, 3000, 24), 1, torch.bfloat16, seed=6))
    want = ops.gated_scan(x, gate, h, dim=1)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, last = ops.gated_scan(x, gate, h, dim=1)
    graph.replay()
    assert torch.equal(y, want[0]) and torch.equal(last, want[1])
    x.neg_()
    h.neg_()
    graph.replay()
    assert torch.equal(y, -want[0]) and torch.equal(last, -want[1])


def test_a_training_pass_captured_and_replayed():
    x, gate, h, m, dy, dlast = inputs((6, 70, 12), 1, torch.bfloat16, seed=10, mask=0.8)
    x, gate, h, m, dy, dlast = (t.to(DEV) for t in (x, gate, h, m, dy, dlast))

    def once():
        leaves = [t.detach().requires_grad_() for t in (x, gate, h)]  # fresh: no graph outlives the pass
        outs = ops.gated_scan(*leaves, dim=1, mask=m)
        return [t.detach() for t in outs] + list(torch.autograd.grad(outs, leaves, [dy, dlast]))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        once()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = once()
    x.mul_(0.5)
    dy.neg_()
    graph.replay()
    for a, b in zip(got, once()):
        assert torch.equal(a, b)


def test_the_same_tensor_twice():
    x = torch.randn((3, 40, 6), generator=torch.Generator().manual_seed(11))
    dy, dlast = torch.randn((3, 40, 6)), torch.zeros((3, 6))
    want, bound = bounds(x, x, None, 1, False, None, dy, dlast)
    leaf = x.to(DEV).requires_grad_()
    y, _ = ops.gated_scan(leaf, leaf, dim=1)
    (g,) = torch.autograd.grad(y, leaf, dy.to(DEV))
    tol = 4 * (bound["x"] + bound["gate"]) + 3 * E * (want["x"].abs() + want["gate"].abs()) + 2.0**-126
    assert ((g.cpu().double() - want["x"] - want["gate"]).abs() <= tol).all()


def test_offsets_beyond_32_bits():
    # rows 2^31 elements and more apart: two lines of 3 steps in a view of a large buffer
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 16 GB")
    big = torch.empty(2**31 + 2**12, dtype=torch.bfloat16, device=DEV)
    x = big.as_strided((2, 3, 8), (2**31, 8, 1))
    v, gate, h, _, dy, dlast = inputs((2, 3, 8), 1, torch.bfloat16)
    x.copy_(v)
    y, last = ops.gated_scan(x, gate.to(DEV), h.to(DEV), dim=1)
    y0, last0 = ops.gated_scan(v.to(DEV), gate.to(DEV), h.to(DEV), dim=1)
    assert torch.equal(y, y0) and torch.equal(last, last0)


def test_refusals():
    x = torch.zeros((2, 3, 4), device=DEV)
    ok = dict(dim=1)
    cases = [
        (ValueError, "dim", (x, x), dict(dim=2)), (ValueError, "dim", (x, x), dict(dim=-1)), (ValueError, "dim", (x, x), dict(dim=3)),
        (ValueError, "gate", (x, x[:1]), ok), (TypeError, "gate", (x, x.half()), ok), (ValueError, "gate", (x, x.cpu()), ok),
        (TypeError, "x must be", (x.double(), x.double()), ok), (ValueError, "state", (x, x, x[:, 0, :3]), ok),
        (TypeError, "state", (x, x, x[:, 0].half()), ok), (ValueError, "x must have", (x[0, 0], x[0, 0]), dict(dim=0)),
        (TypeError, "mask", (x, x), dict(dim=1, mask=torch.ones(2, 3, device=DEV))),
        (ValueError, "mask", (x, x), dict(dim=1, mask=torch.ones(2, 4, device=DEV, dtype=torch.bool))),
        (ValueError, "mask", (x, x), dict(dim=1, mask=torch.ones(2, 3, dtype=torch.bool))),
    ]
    for kind, match, args, kw in cases:
        with pytest.raises(kind, match=match):
            ops.gated_scan(*args, **kw)
    leaf = torch.zeros((2, 3, 4), device=DEV, requires_grad=True)
    y, _ = ops.gated_scan(leaf, leaf, dim=1)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(y.sum(), leaf, create_graph=True)
    with fwd.dual_level(), pytest.raises(ValueError, match="tangent"):
        ops.gated_scan(fwd.make_dual(x, x), x, dim=1)


# a line's warps and pieces, a thread a line, 16 bytes of a row a thread
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,t,c", [(1, 100001, 32), (3, 40, 64), (800, 200, 512), (1200, 60, 512), (7, 3, 64)])
def test_open_gates_hold_the_state(n, t, c, dtype):
    # 1 - sigmoid(gate) below 2^-25: the nearest fp32 of sigmoid(gate) is 1, so that a state without input stays as it is; the
    # formula's own decay, of t (1 - a) of it at most, is all that it is off by.  `want` itself is rounded in 64 bits: an exponential
    # near 1 within 2^-52 and its product with h within 2^-53 of it, below 2^-50
    gate = torch.linspace(17.5, 30.0, c).to(dtype)
    share = torch.sigmoid(-gate.double())
    assert (share < 2.0**-25).all()
    h = torch.randn((n, c), generator=torch.Generator().manual_seed(0))
    x = torch.zeros((1, 1, c), dtype=dtype, device=DEV).expand(n, t, c).contiguous()
    gates = gate.to(DEV).expand(n, t, c).contiguous()
    y, last = ops.gated_scan(x, gates, h.to(DEV), dim=1)
    want = h.double() * torch.exp(t * torch.log1p(-share))
    off = (last.cpu().double() - want).abs()
    tol = (t * share + 2.0**-50) * h.double().abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert torch.equal(y[:, -1], last.to(dtype))


# 16 bytes of a row a thread (once, walking), a thread a line, a line's warps, its pieces
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,t,c", [(5, 4, 64), (600, 9, 512), (300, 40, 260), (40, 16, 10), (2, 100, 32), (1, 3000, 6)])
def test_gradients_through_closed_gates_keep_their_precision(n, t, c, dtype):
    # a gradient from `last` alone passes closed gates, a of 4e-8 to 3e-4: what is left keeps a relative error.  The bounds of
    # fp32 data (r = a G off by k a |G|) for all types
    x, gate, h, _, dy, dlast = inputs((n, t, c), 1, dtype, seed=t)
    g = torch.Generator().manual_seed(t + 1)
    closed = torch.rand((n, t, c), generator=g) < min(0.3, 3 / t)
    shut = (-8 - 9 * torch.rand((n, t, c), generator=g)).to(dtype)
    gate = torch.where(closed, shut, gate)
    dy = torch.zeros_like(dy)
    want, bound = bounds(x.float(), gate.float(), h, 1, False, None, dy.float(), dlast)
    leaves = [v.to(DEV).requires_grad_() for v in (x, gate, h)]
    y, last = ops.gated_scan(*leaves, dim=1)
    grads = torch.autograd.grad([last], leaves, [dlast.to(DEV)])
    for name, got in zip(("x", "gate", "state"), grads):
        close(got, want[name], bound[name], name)


def test_a_gradient_of_last_alone_takes_no_copy():
    # dx, dgate and the states of every 8 steps (held already), no third tensor of x's size
    x = torch.randn((4, 4000, 512), device=DEV, dtype=torch.bfloat16).requires_grad_()
    gate = torch.randn_like(x).requires_grad_()
    last = ops.gated_scan(x, gate, dim=1)[1]
    size = x.numel() * x.element_size()
    torch.cuda.reset_peak_memory_stats()
    held = torch.cuda.memory_allocated()
    grads = torch.autograd.grad(last, [x, gate], torch.ones_like(last))
    assert torch.cuda.max_memory_allocated() - held <= 2.5 * size
    y, last = ops.gated_scan(x, gate, dim=1)
    full = torch.autograd.grad([y, last], [x, gate], [torch.zeros_like(y), torch.ones_like(last)])
    assert all(torch.equal(a, b) for a, b in zip(grads, full))
