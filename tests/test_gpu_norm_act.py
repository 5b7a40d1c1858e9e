"""group_norm_act on the GPU against the 64-bit oracle: types, group widths, odd sizes, strides, masks
that leave samples empty, far means, refusals, streams and repeatability.

Tolerances (u the unit roundoff of the output's type, e = 2^-24).  A value passes through one
rounding to its type and about 64 fp32 operations on terms of size `scale`: |error| <= u |y| + 64 e
scale.  h = (x - mean) rstd carries e |x| rstd from the subtraction, so `scale` is the largest term
times (1 + max |x| rstd).  A parameter's gradient adds at most 300 partial sums one after another on
the longest path of these sizes: 300 e sum |terms| (1 + max |x| rstd)."""

import ctypes as C

import pytest
import torch
import torch.autograd.forward_ad as fwd

import oracle.cell_operators as O
from ncas_b200 import _lib as L
from ncas_b200 import operators as ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
E = 2.0**-24
UNIT = {torch.float32: 2.0**-24, torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def normal(*shape, seed=0, scale=1.0, shift=0.0):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g) * scale + shift


def close(got, want, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, worst {float((got - want).abs().max()):.3e}"


def check(x, groups, weight, bias, act="silu", mask=None, eps=1e-5, dy=None):
    """Forward, gradients and every tolerance for one set of CUDA inputs."""
    host = lambda t: None if t is None else t.detach().cpu()  # noqa: E731
    dy = normal(*x.shape, seed=99).to(x) if dy is None else dy
    leaves = [t.detach().requires_grad_() for t in (x, weight, bias) if t is not None]
    it = iter(leaves)
    args = [next(it) if t is not None else None for t in (x, weight, bias)]
    y = ops.group_norm_act(args[0], groups, args[1], args[2], eps=eps, act=act, mask=mask)
    assert y.is_contiguous() and y.dtype == x.dtype
    grads = torch.autograd.grad(y, leaves, dy)
    with torch.no_grad():
        again = ops.group_norm_act(x, groups, weight, bias, eps=eps, act=act, mask=mask)
    assert torch.equal(again, y)  # the inference call is the training call's forward
    wy, wdx, wdw, wdb = O.group_norm_act(host(x), groups, host(weight), host(bias), eps, act, host(mask), host(dy))
    keep = torch.ones(x.shape[:-1], dtype=torch.bool) if mask is None else host(mask) != 0
    xs = host(x).double()[keep]
    u = UNIT[x.dtype]
    n, c = x.shape[0], x.shape[-1]
    rstd = 1.0
    far = 0.0
    for i in range(n):  # largest |x| rstd and rstd of any group
        rows = host(x)[i].double()[keep[i]].reshape(-1, groups, c // groups)
        if len(rows):
            r = 1 / torch.sqrt(rows.var((0, 2), unbiased=False) + eps)
            rstd = max(rstd, float(r.max()))
            far = max(far, float((rows.abs().amax((0, 2)) * r).max()))
    wmax = 1.0 if weight is None else float(weight.abs().max())
    bmax = 0.0 if bias is None else float(bias.abs().max())
    amp = (1 + far) ** 2 if len(xs) else 1.0
    scale = amp * (wmax + bmax + 1)
    close(y, wy, u * wy.abs() + 64 * E * scale, "y")
    g = float(dy.abs().max()) * wmax * rstd * (1 + wmax) * 3
    close(grads[0], wdx, u * wdx.abs() + 64 * E * scale * g, "dx")
    terms = float(host(dy).double()[keep].abs().sum(0).max()) if keep.any() else 0.0
    for got, want, p, name in zip(grads[1:], [w for w, p in ((wdw, weight), (wdb, bias)) if p is not None],
                                  [p for p in (weight, bias) if p is not None], ("dweight", "dbias")):
        assert got.dtype == p.dtype
        close(got, want, UNIT[p.dtype] * want.abs() + 300 * E * terms * 2 * scale * (1 + far), name)
    if mask is not None:
        out = ~keep.to(DEV)
        assert (y.detach()[out] == 0).all() and (grads[0][out] == 0).all()
    return y, grads


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,cells,channels,groups", [
    (1, 1, 64, 1),       # one cell: statistics over the channels alone
    (3, 81, 64, 8),      # 9x9 boards
    (2, 900, 32, 4),     # 30x30 mazes
    (5, 7, 12, 4),       # three channels a group
    (4, 50, 33, 3),      # odd channels: one value a load
    (2, 130, 6, 6),      # one channel a group
    (3, 257, 40, 5),     # cells and vectors that fill no block evenly
    (2, 70, 1030, 2),    # more vectors than threads (two a load)
    (2, 40, 2304, 9),    # more 16-byte vectors than threads
    (1, 6000, 16, 2),    # a long sample, cut into pieces
    (700, 9, 8, 2),      # many small samples
    (3, 100, 80, 8),     # ten channels a group: 16-byte loads that span groups
    (2, 3000, 320, 32),  # the same over several blocks of channels and cells
    (4, 33, 48, 8),      # six channels a group
    (5, 19, 8, 4),       # pairs
    (40, 500, 2, 1),     # two channels: all threads over the cells
    (2, 30000, 64, 1),   # one group too large for a cluster of blocks
    (1, 20000, 96, 32),  # the same with three channels a group
])
def test_against_the_oracle(dtype, n, cells, channels, groups):
    x = normal(n, cells, channels, seed=cells, scale=1.5, shift=0.25).to(DEV, dtype)
    w = normal(channels, seed=1, scale=0.3, shift=1.0).to(DEV)
    b = normal(channels, seed=2, scale=0.3).to(DEV)
    check(x, groups, w, b)


@pytest.mark.parametrize("act", ["none", "relu", "silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dtype", TYPES)
def test_activations(act, dtype):
    x = normal(3, 45, 24, seed=5, scale=2.0).to(DEV, dtype)
    w, b = normal(24, seed=1, shift=1.0).to(DEV), normal(24, seed=2).to(DEV)
    check(x, 3, w, b, act=act)
    check(x, 3, None, None, act=act)
    check(x, 3, w.to(dtype), None, act=act)
    check(x, 3, None, b.to(dtype), act=act)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("kind", [torch.bool, torch.uint8])
def test_masks(dtype, kind):
    n, cells, c = 6, 90, 16
    x = normal(n, cells, c, seed=3, shift=1.0).to(DEV, dtype)
    keep = torch.rand((n, cells), generator=torch.Generator().manual_seed(4)) < 0.5
    keep[1] = False          # no cell
    keep[2] = True
    keep[3] = False
    keep[3, 40] = True       # one cell
    keep[4, :70] = False     # whole pieces without a cell
    mask = (keep * 255).to(kind).to(DEV) if kind == torch.uint8 else keep.to(DEV)
    w, b = normal(c, seed=1, shift=1.0).to(DEV), normal(c, seed=2).to(DEV)
    y, grads = check(x, 4, w, b, mask=mask)
    # what lies in masked places, in x and in dy, is not looked at
    dy = normal(*x.shape, seed=99).to(DEV, dtype)
    xn, dyn = x.clone(), dy.clone()
    for t in (xn, dyn):
        t[~keep] = float("nan")
        t[5, ~keep[5]] = float("inf")
        t[0, ~keep[0]] = torch.finfo(dtype).min
    y2, grads2 = check_same_call(xn, 4, w, b, mask, dyn)
    assert torch.equal(y2, y) and all(torch.equal(p, q) for p, q in zip(grads2, grads))


def check_same_call(x, groups, w, b, mask, dy):
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], act="silu", mask=mask)
    return y, torch.autograd.grad(y, leaves, dy)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,cells,c,groups", [(5, 3481, 32, 4), (4, 500, 40, 4), (2, 20000, 64, 1), (3, 700, 6, 2), (9, 70, 40, 40)])
def test_masks_of_padded_boards(dtype, n, cells, c, groups):
    # a prefix of every sample's cells: whole pieces, and whole samples, without a cell
    x = normal(n, cells, c, seed=6, shift=0.5).to(DEV, dtype)
    keep = torch.arange(cells)[None] < torch.linspace(0, cells, n).round()[:, None]
    check(x, groups, normal(c, seed=1, shift=1.0).to(DEV), normal(c, seed=2).to(DEV), act="relu", mask=keep.to(DEV))


@pytest.mark.parametrize("dtype", TYPES)
def test_strides(dtype):
    n, h, w_, c = 2, 5, 7, 16
    wt, b = normal(c, seed=1, shift=1.0).to(DEV), normal(c, seed=2).to(DEV)
    nchw = normal(n, c, h, w_, seed=3).to(DEV, dtype)
    views = {
        "channels last": nchw.contiguous(memory_format=torch.channels_last).permute(0, 2, 3, 1),
        "planar (copied)": nchw.permute(0, 2, 3, 1),
        "channel slice": normal(n, h, w_, 48, seed=4).to(DEV, dtype)[..., 16:32],
        "odd channel slice": normal(n, h, w_, 35, seed=5).to(DEV, dtype)[..., 3:19],
        "every other sample": normal(2 * n, h, w_, c, seed=6).to(DEV, dtype)[::2],
        "every other column": normal(n, h, 2 * w_, c, seed=7).to(DEV, dtype)[:, :, ::2],
        "crop (copied)": normal(n, h + 2, w_ + 2, c, seed=8).to(DEV, dtype)[:, 1:-1, 1:-1],
        "one sample for all": normal(1, h, w_, c, seed=9).to(DEV, dtype).expand(n, h, w_, c),
        "transposed grid": normal(n, w_, h, c, seed=10).to(DEV, dtype).transpose(1, 2),
    }
    mask = torch.rand((n, w_, h), generator=torch.Generator().manual_seed(1)).transpose(1, 2).to(DEV) < 0.7
    for name, x in views.items():
        check(x, 4, wt, b)
        check(x, 4, wt, b, mask=mask)
    x = views["channels last"]
    check(x, 4, wt, b, dy=normal(1, 1, 1, c, seed=11).to(DEV, dtype).expand(n, h, w_, c))
    check(x, 4, wt, b, dy=normal(n, c, h, w_, seed=12).to(DEV, dtype).permute(0, 2, 3, 1))
    check(x, 4, normal(2 * c, seed=1).to(DEV)[::2], b)
    check(normal(3, 8, seed=13).to(DEV, dtype), 2, None, None)  # (N, C): one cell a sample


@pytest.mark.parametrize("shift", [1e3, 3e5])
def test_far_means_and_outliers(shift):
    # (x - mean) keeps the digits that fp32 values this far from zero have
    x = normal(2, 700, 32, seed=3, shift=shift).to(DEV)
    check(x, 4, None, None, act="none")
    x = normal(2, 700, 32, seed=4).to(DEV)
    x[:, 0] = shift  # the first value of every channel lies far from all others
    check(x, 4, None, None, act="none")


def test_non_finite_values_stay_in_their_group():
    x = normal(3, 50, 16, seed=3).to(DEV)
    x[0, 3, 1] = float("nan")
    x[1, 7, 9] = float("inf")
    y = ops.group_norm_act(x, 4, act="none")
    bad = torch.zeros(3, 50, 4, 4, dtype=torch.bool)
    bad[0, :, 0] = True
    bad[1, :, 2] = True
    assert torch.equal(~torch.isfinite(y).cpu().reshape(3, 50, 4, 4) & bad, bad)
    assert torch.isfinite(y.cpu().reshape(3, 50, 4, 4)[~bad]).all()


def test_empty_batches():
    for shape in [(0, 9, 8), (3, 0, 8), (0, 8)]:
        x = torch.zeros(shape, device=DEV, requires_grad=True)
        w = torch.ones(8, device=DEV, requires_grad=True)
        b = torch.ones(8, device=DEV, requires_grad=True)
        y = ops.group_norm_act(x, 2, w, b)
        assert y.shape == x.shape
        dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
        assert dx.shape == x.shape and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("shape", [(2, 3, 0, 4), (2, 0, 3, 4), (3, 2, 0, 5, 4), (2, 5, 1, 0, 8), (0, 3, 0, 4)])
def test_a_size_of_zero_among_the_cells(shape):
    x = torch.empty(shape, device=DEV, requires_grad=True)
    w = torch.ones(shape[-1], device=DEV, requires_grad=True)
    for mask in (None, torch.ones(shape[:-1], device=DEV, dtype=torch.bool)):
        with torch.no_grad():
            assert ops.group_norm_act(x, 2, w, mask=mask).shape == shape
        y = ops.group_norm_act(x, 2, w, mask=mask)
        gx, gw = torch.autograd.grad(y.sum(), [x, w])
        assert y.shape == shape and gx.shape == shape and (gw == 0).all()
    view = torch.empty((2, 3, 6, 4), device=DEV)[:, :, 3:3]  # at an address, with strides of its own
    assert ops.group_norm_act(view, 2).shape == (2, 3, 0, 4)


def test_gradient_against_differences():
    # f(x + h v) - f(x - h v) over 2 h, in the kernel's own fp32: h = 2^-7 leaves h^2 / 6 f''' (about
    # 2^-16 of |f'|) and 2^-24 |f| 2^7 from rounding; f sums 2 * 20 * 12 terms of size about 1
    x, v = normal(2, 20, 12, seed=1).to(DEV), normal(2, 20, 12, seed=2).to(DEV)
    w, b = normal(12, seed=3, shift=1.0).to(DEV), normal(12, seed=4).to(DEV)
    dy = normal(2, 20, 12, seed=5).to(DEV)
    f = lambda t: (ops.group_norm_act(t, 3, w, b, act="gelu") * dy).double().sum().item()  # noqa: E731
    xg = x.clone().requires_grad_()
    (g,) = torch.autograd.grad((ops.group_norm_act(xg, 3, w, b, act="gelu") * dy).sum(), xg)
    h = 2.0**-7
    slope = (f(x + h * v) - f(x - h * v)) / (2 * h)
    size = float((g * v).abs().double().sum())
    assert abs(slope - float((g * v).double().sum())) <= size * 2**-10


def test_partial_gradients_and_higher_orders():
    x = normal(2, 9, 8, seed=1).to(DEV).requires_grad_()
    w = normal(8, seed=2).to(DEV).requires_grad_()
    y = ops.group_norm_act(x, 2, w, None)
    dx, dw = torch.autograd.grad(y.sum(), (x, w), retain_graph=True)
    assert torch.equal(torch.autograd.grad(y.sum(), x, retain_graph=True)[0], dx)
    assert torch.equal(torch.autograd.grad(y.sum(), w, retain_graph=True)[0], dw)
    with pytest.raises(RuntimeError, match="not differentiable"):
        torch.autograd.grad(y.sum(), x, create_graph=True)


def test_repeatable_and_on_other_streams():
    x = normal(40, 300, 64, seed=1).to(DEV, torch.bfloat16)
    w, b = normal(64, seed=2).to(DEV), normal(64, seed=3).to(DEV)
    dy = normal(40, 300, 64, seed=4).to(DEV, torch.bfloat16)
    first = check_same_call(x, 8, w, b, None, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = check_same_call(x, 8, w, b, None, dy)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first[0], again[0]) and all(torch.equal(p, q) for p, q in zip(first[1], again[1]))


def test_inside_a_cuda_graph():
    x, w = normal(4, 81, 64, seed=1).to(DEV), normal(64, seed=2).to(DEV)
    want = ops.group_norm_act(x, 8, w)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.group_norm_act(x, 8, w)
    y.zero_()
    graph.replay()
    assert torch.equal(y, want)


@pytest.mark.parametrize("dtype,shift", [(torch.float32, 1e2), (torch.float32, 1e3), (torch.float32, 1e4), (torch.float16, 1e2)])
@pytest.mark.parametrize("n,cells,c,groups", [
    (3, 81, 64, 8), (4, 3481, 32, 4), (2, 20000, 64, 1), (3, 300, 33, 3), (2, 70, 1030, 2)])
def test_means_far_from_zero(dtype, shift, n, cells, c, groups):
    """Data of unit spread far from zero, with bounds that stay well below the outputs' spread.

    far = max |x| rstd.  The mean is at most 64 roundings of |x| off: mean and h by 64 e far (and a rounding
    of x - mean).  The sums of (x - K)^2 of a thread cancel to half on average and take at most 64 additions:
    2 * 2 * 64 e of the variance, doubled for its spread over the threads; a thread's mean, rounded to e |x|,
    enters the merged variance with its distance from the mean (below 1 in units of the spread): 2 e far;
    and the variance about a mean that is off is larger by (64 e far)^2.  rstd takes half of these.
    The gradients carry h's error through their sums, and 64 additions (300 over the samples)."""
    x = normal(n, cells, c, seed=cells, shift=shift).to(DEV, dtype)
    w, b = normal(c, seed=1, scale=0.3, shift=1.0).to(DEV), normal(c, seed=2, scale=0.3).to(DEV)
    dy = normal(n, cells, c, seed=3).to(DEV, dtype)
    leaves = [t.detach().requires_grad_() for t in (x, w, b)]
    y = ops.group_norm_act(leaves[0], groups, leaves[1], leaves[2], act="none")
    got = torch.autograd.grad(y, leaves, dy)
    wy, wdx, wdw, wdb = O.group_norm_act(x.cpu(), groups, w.cpu(), b.cpu(), 1e-5, "none", None, dy.cpu())
    u = UNIT[dtype]
    xs = x.cpu().double().view(n, cells, groups, c // groups)
    mean = xs.mean((1, 3), keepdim=True)
    rstd = 1 / torch.sqrt(xs.var((1, 3), keepdim=True, unbiased=False) + 1e-5)
    h = (xs - mean) * rstd
    wv, bv = (t.cpu().double().view(groups, c // groups) for t in (w, b))
    g = dy.cpu().double().view(xs.shape)
    wg = wv * g
    far = float((xs.abs() * rstd).max())
    assert 0.5 * shift < far < 4 * shift
    off = 65 * E * far                                    # of h
    r = 256 * E + E * far + 0.5 * (64 * E * far) ** 2     # of rstd, relative
    flat = lambda t: t.reshape(n, cells, c)  # noqa: E731
    ty = flat(wv.abs() * (off + h.abs() * r) + 4 * E * ((wv * h).abs() + bv.abs())) + u * wy.abs()
    assert float(ty.max()) < 0.25 * float(wy.std())
    close(y, wy, ty, "y")
    m = lambda t: t.mean((1, 3), keepdim=True)  # noqa: E731
    bn = m(wg * h).abs()
    tb = m(wg.abs()) * off + r * bn + 64 * E * m((wg * h).abs())
    tx = rstd * (64 * E * m(wg.abs()) + h.abs() * tb + (off + h.abs() * r) * (bn + tb) + 4 * E * (wg.abs() + bn * h.abs()))
    tx = flat(tx * (1 + r)) + (r + u) * wdx.abs()
    assert float(tx.max()) < 0.25 * float(wdx.std())
    close(got[0], wdx, tx, "dx")
    s = lambda t: t.sum((0, 1)).reshape(c)  # noqa: E731
    tw = s(g.abs() * (off + h.abs() * r)) + 300 * E * s((g * h).abs()) + UNIT[w.dtype] * wdw.abs()
    if shift < 1e3:
        assert float(tw.max()) < 0.5 * float(wdw.std())
    close(got[1], wdw, tw, "dweight")
    close(got[2], wdb, 300 * E * s(g.abs()) + UNIT[b.dtype] * wdb.abs(), "dbias")


def test_the_most_channels():
    """2^30 channels in one group.  Tiles of 2048 channels hold +-k, k from 1 to 4: every sum is a whole
    number below 2^24 times 2048, so mean and variance are exact and rstd carries its last roundings."""
    c = 1 << 30
    k = torch.randint(1, 5, (c // 2048, 1), generator=torch.Generator().manual_seed(8)).to(DEV, torch.float16)
    x = (k * torch.tensor([1.0, -1.0], device=DEV, dtype=torch.float16).repeat(1024)).view(1, 1, c)
    y = torch.empty_like(x)
    stats = torch.zeros(2, device=DEV)
    d = L.NcaNormDesc(n=1, cells=1, channels=c, groups=1, dtype=2, param_dtype=0, act=0, eps=0.0, x_stride_n=c, x_stride_cell=c)
    lib, size, p = L.lib(), C.c_size_t(0), lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    assert lib.nca_b200_group_norm_workspace(C.byref(d), 0, C.byref(size)) == 0
    ws = torch.empty(size.value, device=DEV, dtype=torch.uint8)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert lib.nca_b200_group_norm(C.byref(d), p(x), None, None, None, p(y), p(stats), p(ws), ws.numel(), stream) == 0
    rstd = 1 / float((k.double() ** 2).mean().sqrt())
    assert stats[0].item() == 0 and abs(stats[1].item() - rstd) <= 4 * E * rstd
    # y: one product and the rounding to fp16
    want = x.double() * rstd
    assert ((y.double() - want).abs() <= 2.0**-11 * want.abs() * 1.01).all()
    with pytest.raises(ValueError, match="channels"):
        ops.group_norm_act(torch.zeros((1, 1, 1), device=DEV).expand(1, 1, (1 << 30) + 8), 1)
    with pytest.raises(ValueError, match="channels"):
        ops.group_norm_act(torch.zeros((1, 1, 1), device=DEV).expand(1, 1, (1 << 32) + 8), 1)


def test_forward_mode_tangents_are_refused():
    x, w = torch.ones((2, 3, 8), device=DEV), torch.ones(8, device=DEV)
    with fwd.dual_level():
        dual = lambda t: fwd.make_dual(t, torch.ones_like(t))  # noqa: E731
        for args in ((dual(x), 2, w, w), (x, 2, dual(w), w), (x, 2, w, dual(w))):
            with pytest.raises(ValueError, match="tangent"):
                ops.group_norm_act(*args)
        leaf = x.clone().requires_grad_()
        y = ops.group_norm_act(leaf, 2, w, w)
        with pytest.raises(ValueError, match="tangent"):
            torch.autograd.grad(y, leaf, dual(torch.ones_like(y)))


def test_refusals():
    x = torch.zeros(2, 3, 8, device=DEV)
    for kw, exc, text in [
        (dict(groups=3), ValueError, "divide"), (dict(groups=0), ValueError, "divide"),
        (dict(weight=torch.ones(7, device=DEV)), ValueError, "weight"),
        (dict(bias=torch.ones(8)), ValueError, "CUDA"),
        (dict(weight=torch.ones(8, device=DEV, dtype=torch.float16)), TypeError, "weight"),
        (dict(weight=torch.ones(8, device=DEV, dtype=torch.float64)), TypeError, "weight"),
        (dict(act="tanh"), ValueError, "act"), (dict(eps=-1.0), ValueError, "eps"),
        (dict(mask=torch.ones(2, 3, 8, device=DEV, dtype=torch.bool)), ValueError, "mask"),
        (dict(mask=torch.ones(2, 3, device=DEV)), TypeError, "mask"),
        (dict(x=torch.zeros(8, device=DEV)), ValueError, "x must be"),
        (dict(x=x.double()), TypeError, "float32"), (dict(x=x.long()), TypeError, "float32"),
    ]:
        args = dict(x=x, groups=2, weight=None, bias=None)
        args.update(kw)
        with pytest.raises(exc, match=text):
            ops.group_norm_act(args.pop("x"), args.pop("groups"), args.pop("weight"), args.pop("bias"), **args)
