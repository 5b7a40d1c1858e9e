"""distill_loss and its gradient on the GPU against the 64-bit oracle.

Tolerances (u the unit roundoff of the gradient's type, e = 2^-24).  exp(d / T) of a difference d of
fp32 values carries e (|d| / T + 4) of itself (the scaling and the exponential), sums of positive
terms at most 64 e more on the longest path of these sizes; with |d| / T <= D of a row:
  gradient  |error| <= u |g| + w T e (D + 80) (q + p)        (q and p below 1)
  loss      |error| <= w T^2 e (D + 80) (1 + sum p |log p - log q|)."""

import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import oracle.cell_operators as O
from ncas_b200 import operators as ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
E = 2.0**-24
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TINY = {torch.float32: 2.0**-149, torch.bfloat16: 2.0**-133, torch.float16: 2.0**-25}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(rows, classes, top, dtype, seed=0, scale=2.0, index=torch.int32):
    g = torch.Generator().manual_seed(seed)
    s = (torch.randn((rows, classes), generator=g) * scale).to(dtype)
    t = (torch.randn((rows, top), generator=g) * scale).to(dtype)
    i = torch.stack([torch.randperm(classes, generator=g)[:top] if top <= classes else
                     torch.randint(0, classes, (top,), generator=g) for _ in range(rows)]) if rows else torch.zeros(0, top)
    w = torch.rand((rows,), generator=g) + 0.5
    return s.to(DEV), t.to(DEV), i.to(index).to(DEV), w.to(DEV)


def check(s, t, i, w, temperature=1.0):
    ls, lg = O.distill(s.detach().cpu(), t.detach().cpu(), i.cpu(), temperature, None if w is None else w.cpu())
    loss, grad = ops.distill_loss_and_grad(s, t, i, temperature=temperature, weight=w, reduction="none")
    assert loss.dtype == torch.float32 and grad.dtype == s.dtype and grad.is_contiguous()
    w64 = torch.ones(s.shape[0], dtype=torch.float64) if w is None else w.cpu().double()
    spread = 0.0
    for x in (s, t):
        f = x.detach().double().cpu()
        f = f[torch.isfinite(f)]
        spread = max(spread, float(f.max() - f.min()) / temperature) if f.numel() else spread
    c = E * (spread + 80)
    tol = w64.abs() * temperature**2 * c * (1 + spread + 20)
    assert ((loss.cpu().double() - ls).abs() <= tol).all(), float((loss.cpu().double() - ls).abs().max())
    u = UNIT[s.dtype]
    gt = u * lg.abs() + (w64.abs() * temperature * c * 2)[:, None] + TINY[s.dtype]
    assert ((grad.cpu().double() - lg).abs() <= gt).all(), float((grad.cpu().double() - lg).abs().max())
    # the differentiable form: the same loss, and the gradient of any weighted sum of the rows
    leaf = s.detach().requires_grad_()
    rows = ops.distill_loss(leaf, t, i, temperature=temperature, weight=w, reduction="none")
    assert torch.equal(rows.detach(), loss)
    with torch.no_grad():
        assert torch.equal(ops.distill_loss(s, t, i, temperature=temperature, weight=w, reduction="none"), loss)
    up = torch.linspace(-1.5, 2.0, s.shape[0], device=DEV)
    (g2,) = torch.autograd.grad(rows, leaf, up)
    want = lg * up.cpu().double()[:, None]
    # the upstream factor is one more fp32 product
    gt2 = u * want.abs() + (up.cpu().double().abs() * w64.abs() * temperature * c * 2)[:, None] + 2 * E * want.abs() + TINY[s.dtype]
    assert ((g2.cpu().double() - want).abs() <= gt2).all()
    return loss, grad


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,top", [
    (1, 1, 1), (5, 2, 2), (300, 3, 1), (33, 4, 4), (81, 9, 4), (7, 17, 17), (20, 64, 8), (9, 65, 3), (6, 300, 40),
    (5, 1000, 33), (4, 1025, 10), (3, 5003, 64), (2, 20001, 7), (1, 70007, 130), (3, 40, 0)])
def test_against_the_oracle(dtype, rows, classes, top):
    check(*inputs(rows, classes, top, dtype, seed=classes), temperature=1.5)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,top,offset", [
    (2600, 1500, 3, 0),    # more rows than blocks that run at once: a block goes through several
    (1000, 7001, 2, 1),    # the same, rows on no 16-byte boundary
    (150, 40003, 5, 3),    # up to a whole multiprocessor for a row
    (2, 300007, 9, 0),     # a row over a cluster of blocks
    (3, 20000, 200, 0),    # more entries than the entry warp holds
])
def test_rows_that_are_held(dtype, rows, classes, top, offset):
    g = torch.Generator().manual_seed(rows)
    wide = (torch.randn((rows, classes + offset), generator=g) * 2).to(DEV, dtype)
    s = wide[:, offset:]  # with an offset, the gradient's rows are aligned unlike the logits'
    _, t, i, w = inputs(rows, classes, top, dtype, seed=classes) if rows < 10 else inputs(rows, 50, top, dtype, seed=classes)
    w[::7] = 0.0
    i[::5, 0] = -1
    i[1::5, :2] = classes - 1  # the last class, twice where top > 1
    loss, grad = check(s, t, i, w, 1.5)
    assert (loss[::7] == 0).all() and (grad[::7] == 0).all()


@pytest.mark.parametrize("dtype,classes,top,offset", [
    (torch.bfloat16, 9001, 3, 0), (torch.float16, 15000, 40, 0), (torch.float16, 22001, 2, 1),
    (torch.bfloat16, 24576, 128, 0), (torch.bfloat16, 40003, 5, 3), (torch.float16, 60008, 4, 0),
    (torch.float32, 5000, 3, 0), (torch.float32, 20011, 7, 2), (torch.float32, 34560, 1, 0)])
def test_many_long_rows(dtype, classes, top, offset):
    """Enough rows that none is shared by blocks; a few of them are compared, with the tolerances of check()."""
    g = torch.Generator().manual_seed(classes)
    wide = (torch.randn((640, classes + offset), generator=g) * 2).to(DEV, dtype)
    s = wide[:, offset:]
    t = (torch.randn((640, top), generator=g) * 2).to(DEV, dtype)
    i = torch.randint(0, classes, (640, top), generator=g).int().to(DEV)
    w = (torch.rand((640,), generator=g) + 0.5).to(DEV)
    w[::9] = 0.0
    i[1::9] = -1
    i[2::9, 0] = classes - 1
    i[3::9, 0] = 0
    s[4::9, 1] = -math.inf
    loss, grad = ops.distill_loss_and_grad(s, t, i, temperature=1.5, weight=w, reduction="none")
    with torch.no_grad():
        alone = ops.distill_loss(s, t, i, temperature=1.5, weight=w, reduction="none")
    leaf = s.detach().requires_grad_()
    (later,) = torch.autograd.grad(ops.distill_loss(leaf, t, i, temperature=1.5, weight=w, reduction="sum"), leaf)
    some = torch.arange(0, 640, 31)
    ls, lg = O.distill(s[some].cpu(), t[some].cpu(), i[some].cpu(), 1.5, w[some].cpu())
    f = torch.cat([s[some].double().flatten(), t[some].double().flatten()]).cpu()
    f = f[torch.isfinite(f)]
    spread = float(f.max() - f.min()) / 1.5
    c = E * (spread + 80)
    w64 = w[some].cpu().double()
    for v in (loss, alone):
        assert (v[:: 9] == 0).all() and (v[1::9] == 0).all()
        fine = torch.isfinite(ls)  # an entry of a class that is ruled out: an infinite loss
        got = v[some].cpu().double()
        assert torch.equal(torch.isfinite(got), fine)
        assert ((got - ls).abs() <= w64 * 1.5**2 * c * (1 + spread + 20))[fine].all()
    for v in (grad, later):
        assert (v[::9] == 0).all() and (v[1::9] == 0).all()
        assert ((v[some].cpu().double() - lg).abs() <= UNIT[dtype] * lg.abs() + (w64 * 1.5 * c * 2)[:, None] + TINY[dtype]).all()


@pytest.mark.parametrize("dtype,classes,top,offset", [
    (torch.bfloat16, 131072, 200, 0), (torch.float16, 100003, 131, 1), (torch.float32, 70001, 300, 2)])
def test_clusters_that_go_through_rows_without_a_weight(dtype, classes, top, offset):
    """More than 128 entries and rows that several blocks share, several rows a cluster, rows of weight 0
    between the others; a few of them are compared, with the tolerances of check()."""
    rows = 1500
    g = torch.Generator(device=DEV).manual_seed(classes)
    s = torch.randn((rows, classes + offset), generator=g, device=DEV).mul_(2).to(dtype)[:, offset:]
    t = torch.randn((rows, top), generator=g, device=DEV).mul_(2).to(dtype)
    i = torch.randint(0, classes, (rows, top), generator=g, device=DEV, dtype=torch.int32)
    w = torch.rand((rows,), generator=g, device=DEV) + 0.5
    w[rows // 2 :][torch.rand((rows - rows // 2,), generator=g, device=DEV) < 0.5] = 0.0
    w[1 : rows // 2 : 2] = 0.0
    loss, grad = ops.distill_loss_and_grad(s, t, i, temperature=1.5, weight=w, reduction="none")
    off = w == 0
    assert (loss[off] == 0).all() and (grad[off] == 0).all()
    some = torch.arange(0, rows, 61)
    ls, lg = O.distill(s[some].cpu(), t[some].cpu(), i[some].cpu(), 1.5, w[some].cpu())
    spread = max(float(s[some].max() - s[some].min()), float(t[some].max() - t[some].min())) / 1.5
    c = E * (spread + 80)
    w64 = w[some].cpu().double()
    assert ((loss[some].cpu().double() - ls).abs() <= w64 * 1.5**2 * c * (1 + spread + 20)).all()
    assert ((grad[some].cpu().double() - lg).abs() <= UNIT[dtype] * lg.abs() + (w64 * 1.5 * c * 2)[:, None] + TINY[dtype]).all()
    for _ in range(5):
        again, again_grad = ops.distill_loss_and_grad(s, t, i, temperature=1.5, weight=w, reduction="none")
        assert torch.equal(again, loss) and torch.equal(again_grad, grad)


@pytest.mark.parametrize("temperature", [0.25, 1.0, 8.0])
@pytest.mark.parametrize("classes", [3, 40, 700, 3001])
def test_temperatures_and_index_types(temperature, classes):
    s, t, i, w = inputs(6, classes, 3, torch.float32, seed=1, index=torch.int64)
    check(s, t, i, w, temperature)
    check(s, t.bfloat16(), i, None, temperature)


@pytest.mark.parametrize("classes", [3, 50, 900, 4099])
def test_entries_that_are_missing_or_repeated(classes):
    s, t, i, w = inputs(8, classes, 12, torch.float32, seed=2)
    i[0] = -1                       # no entry at all
    i[1, 3:] = -1                   # the last ones missing
    i[2, ::2] = -7
    i[3, 4] = classes               # beyond the classes: no entry
    i[3, 5] = 2**31 - 1
    i[4] = i[4, 0]                  # one class, twelve times
    i[5, 1] = i[5, 0]
    t[6, 2] = -math.inf             # no probability
    t[7] = -math.inf                # nothing left
    w[5] = 0.0
    loss, grad = check(s, t, i, w, 2.0)
    for r in (0, 5, 7):
        assert loss[r] == 0 and (grad[r] == 0).all()
    j = i.long()
    j[3, 5] = 2**40 + 1             # must not wrap round to a class
    a, b = ops.distill_loss_and_grad(s, t, j, temperature=2.0, weight=w, reduction="none")
    assert torch.equal(a, loss) and torch.equal(b, grad)


@pytest.mark.parametrize("classes", [4, 40, 900, 4099])
def test_infinite_and_undefined_logits(classes):
    s, t, i, w = inputs(7, classes, 2, torch.float32, seed=3)
    i[:, 0], i[:, 1] = 1, 2
    s[0, 3] = -math.inf             # a class that is ruled out, without an entry: q = 0
    s[1, 1] = -math.inf             # ruled out with an entry: infinite loss, finite gradient
    s[2, 0] = float("nan")
    s[3, 0] = math.inf
    s[4] = -math.inf
    s[5, 0] = float("nan")
    w[5] = 0.0                      # no weight: not looked at
    s[6, 3:] = torch.finfo(torch.float32).min
    loss, grad = ops.distill_loss_and_grad(s, t, i, weight=w, reduction="none")
    ls, lg = O.distill(s.cpu(), t.cpu(), i.cpu(), 1.0, w.cpu())
    assert loss[1] == math.inf and torch.isfinite(grad[1]).all()
    assert grad[0, 3] == 0 and grad[1, 3 % classes].isfinite()
    for r in (2, 3, 4):
        assert loss[r].isnan() and grad[r].isnan().all()
    assert loss[5] == 0 and (grad[5] == 0).all()
    for r in (0, 1, 6):
        assert ((grad[r].cpu().double() - lg[r]).abs() <= 2e-5).all()
    assert abs(float(loss[0]) - float(ls[0])) <= 2e-5 * (1 + abs(float(ls[0])))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_leading_sizes(dtype):
    s, t, i, w = inputs(12, 37, 5, dtype, seed=4)
    loss, grad = check(s, t, i, w)
    wide = torch.zeros(12, 45, device=DEV, dtype=dtype)
    wide[:, 3:40] = s
    wt = torch.zeros(12, 9, device=DEV, dtype=dtype)
    wt[:, 2:7] = t
    wi = torch.zeros(12, 9, device=DEV, dtype=torch.int32)
    wi[:, 1:6] = i
    for a, b, c in [(wide[:, 3:40], wt[:, 2:7], wi[:, 1:6]), (s.t().contiguous().t(), t.t().contiguous().t(), i)]:
        l2, g2 = ops.distill_loss_and_grad(a, b, c, weight=w, reduction="none")
        assert torch.equal(l2, loss) and torch.equal(g2, grad)
    l3, g3 = ops.distill_loss_and_grad(s.view(3, 4, 37), t.view(3, 4, 5), i.view(3, 4, 5), weight=w.view(3, 4),
                                       reduction="none")
    assert l3.shape == (3, 4) and torch.equal(l3.view(-1), loss) and torch.equal(g3.view(12, 37), grad)
    l1, g1 = ops.distill_loss_and_grad(s[0], t[0], i[0], weight=w[0], reduction="none")  # one row, no leading size
    assert l1.shape == () and l1 == loss[0] and torch.equal(g1, grad[0])
    one = s[:1].expand(4, 37)  # one row for all
    l4, _ = ops.distill_loss_and_grad(one, t[:1].expand(4, 5), i[:1].expand(4, 5), reduction="none")
    assert (l4 == l4[0]).all()


def test_reductions():
    s, t, i, w = inputs(1000, 11, 3, torch.float32, seed=5)
    rows, g = ops.distill_loss_and_grad(s, t, i, weight=w, reduction="none")
    total, gs = ops.distill_loss_and_grad(s, t, i, weight=w, reduction="sum")
    mean, gm = ops.distill_loss_and_grad(s, t, i, weight=w)
    exact = rows.double().sum().item()
    # 1000 positive terms added in fp32, any order: at most 1000 e of the sum (and e per division)
    assert abs(total.item() - exact) <= 1000 * E * exact and torch.equal(gs, g)
    assert abs(mean.item() - exact / 1000) <= 1002 * E * exact / 1000
    assert ((gm - g / 1000).abs() <= 8 * E * g.abs() / 1000 + 2.0**-140).all()
    leaf = s.clone().requires_grad_()
    value = ops.distill_loss(leaf, t, i, weight=w)
    assert abs(value.item() - exact / 1000) <= 1002 * E * exact / 1000
    (g1,) = torch.autograd.grad(value, leaf)
    assert ((g1 - g / 1000).abs() <= 8 * E * g.abs() / 1000 + 2.0**-140).all()


def test_gradient_against_differences():
    # central differences of the fp32 loss with h = 2^-7: h^2 / 6 f''' below 2^-14 of the slope's size,
    # and 2^7 e |loss| 80 from rounding
    s, t, i, w = inputs(20, 30, 4, torch.float32, seed=6)
    v = torch.randn((20, 30), generator=torch.Generator().manual_seed(7)).to(DEV)
    f = lambda x: ops.distill_loss(x, t, i, temperature=2.0, weight=w, reduction="none").double().sum().item()  # noqa: E731
    _, g = ops.distill_loss_and_grad(s, t, i, temperature=2.0, weight=w, reduction="sum")
    h = 2.0**-7
    slope = (f(s + h * v) - f(s - h * v)) / (2 * h)
    size = float((g * v).abs().double().sum()) + f(s)
    assert abs(slope - float((g * v).double().sum())) <= size * 2**-10


def test_empty_batches():
    s = torch.zeros(0, 5, device=DEV, requires_grad=True)
    i = torch.zeros(0, 2, device=DEV, dtype=torch.int32)
    rows = ops.distill_loss(s, torch.zeros(0, 2, device=DEV), i, reduction="none")
    assert rows.shape == (0,)
    assert torch.autograd.grad(rows.sum(), s)[0].shape == (0, 5)
    loss, grad = ops.distill_loss_and_grad(s.detach(), torch.zeros(0, 2, device=DEV), i, reduction="sum")
    assert loss == 0 and grad.shape == (0, 5)


def test_repeatable_and_on_other_streams():
    s, t, i, w = inputs(50, 3000, 20, torch.bfloat16, seed=8)
    want = ops.distill_loss_and_grad(s, t, i, weight=w)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = ops.distill_loss_and_grad(s, t, i, weight=w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("classes", [2, 9, 300, 700, 5000])
def test_temperatures_at_the_ends(classes):
    # so small that the largest logit takes all of q, and p sits on another class: loss tau^2 (gap / tau) = tau gap
    s = torch.zeros((3, classes), device=DEV)
    s[:, 1] = 2.0
    t, i = torch.tensor([[1.0, 0.0]] * 3, device=DEV), torch.tensor([[0, 1]] * 3, device=DEV)
    tau = 1e-20
    loss, grad = ops.distill_loss_and_grad(s, t, i, temperature=tau, reduction="none")
    assert ((loss - tau * 2.0).abs() <= 2.0**-20 * tau * 2.0).all()
    want = torch.zeros((3, classes), device=DEV)
    want[:, 0], want[:, 1] = -tau, tau
    assert ((grad - want).abs() <= 2.0**-20 * tau).all()
    for bad in (1e-31, 1e-40, 1e-60, 1e31, 1e60, float("inf"), -1.0):
        with pytest.raises(ValueError, match="temperature"):
            ops.distill_loss(s, t, i, temperature=bad)


def test_forward_mode_tangents_are_refused():
    s, t, i, w = inputs(5, 9, 3, torch.float32)
    with fwd.dual_level():
        dual = lambda v: fwd.make_dual(v, torch.ones_like(v))  # noqa: E731
        for call in (ops.distill_loss, ops.distill_loss_and_grad):
            for name, args, kw in (("logits", (dual(s), t, i), {}), ("teacher_logits", (s, dual(t), i), {}),
                                   ("weight", (s, t, i), dict(weight=dual(w)))):
                with pytest.raises(ValueError, match=f"{name} carries a forward-mode tangent"):
                    call(*args, **kw)
        leaf = s.clone().requires_grad_()
        loss = ops.distill_loss(leaf, t, i, reduction="none")
        with pytest.raises(ValueError, match="tangent"):
            torch.autograd.grad(loss, leaf, dual(torch.ones_like(loss)))


def test_refusals():
    s, t, i, w = inputs(4, 9, 3, torch.float32)
    for kw, exc, text in [
        (dict(temperature=0.0), ValueError, "temperature"), (dict(temperature=float("nan")), ValueError, "temperature"),
        (dict(reduction="max"), ValueError, "reduction"), (dict(weight=w[:3]), ValueError, "weight"),
        (dict(weight=w.double()), TypeError, "weight"), (dict(t=t[:, :2]), ValueError, "teacher_index"),
        (dict(t=t[:3], i=i[:3]), ValueError, "teacher_logits"), (dict(i=i.float()), TypeError, "teacher_index"),
        (dict(i=i.cpu()), ValueError, "CUDA"), (dict(s=s.double()), TypeError, "float32"),
        (dict(s=s[:, :0]), ValueError, "classes"), (dict(t=t.clone().requires_grad_()), ValueError, "teacher_logits"),
        (dict(weight=w.clone().requires_grad_()), ValueError, "weight"),
    ]:
        a = dict(s=s, t=t, i=i)
        a.update({k: v for k, v in kw.items() if k in a})
        rest = {k: v for k, v in kw.items() if k not in a}
        with pytest.raises(exc, match=text):
            ops.distill_loss(a["s"], a["t"], a["i"], **rest)
    leaf = s.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(ops.distill_loss(leaf, t, i), leaf, create_graph=True)
