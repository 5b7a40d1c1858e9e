"""sample on the GPU against the 64-bit oracle.

The kernels' weights carry 2^-50 of themselves (argument, four terms of the exponential, products), or in the fixed point of
the histograms 2^-44 of the largest at these sizes; sums of n <= 2^17 of them at most n 2^-52 more.  Where no draw and no cut lies within
1e-11 of the mass of a border, which each test checks, the classes have to be equal.  Probabilities are rounded to
fp32 once: 2^-24 of themselves and the 1e-11."""

import ctypes as C
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

import oracle.cell_operators as O
from ncas_b200 import _lib as L
from ncas_b200 import operators as ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
TYPES = [torch.float32, torch.bfloat16, torch.float16]


def inputs(rows, classes, draws, dtype, seed=0, scale=2.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn((rows, classes), generator=g) * scale).to(dtype), torch.rand((rows, draws), generator=g)


def check(z, u, put=lambda t: t.to(DEV), **kw):
    want, probs, nearest = O.sample(z, u, **kw)
    assert nearest > 1e-11  # the inputs decide
    got, p = ops.sample(put(z), u.to(DEV), **kw)
    assert got.dtype == torch.int64 and p.dtype == torch.float32 and got.shape == u.shape == p.shape
    assert torch.equal(got.cpu(), want), (got.cpu() != want).sum()
    assert ((p.cpu().double() - probs).abs() <= probs * 2.0**-24 + 1e-10).all()
    return got


CUTS = [dict(), dict(temperature=0.5, top_k=3), dict(top_p=0.8), dict(min_p=0.1), dict(temperature=1.5, top_k=20, top_p=0.9),
        dict(temperature=0.7, top_k=7, top_p=0.6, min_p=0.05), dict(top_p=0.3, min_p=0.02), dict(temperature=0.0), dict(top_k=1)]


@pytest.mark.parametrize("cut", CUTS)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,draws", [(1, 1, 1), (70, 2, 3), (33, 3, 9), (81, 9, 40), (20, 16, 2), (9, 17, 33), (5, 32, 1),
                                                (7, 33, 2), (6, 100, 5)])
def test_few_classes(rows, classes, draws, dtype, cut):
    check(*inputs(rows, classes, draws, dtype, seed=classes), **cut)


@pytest.mark.parametrize("cut", [dict(), dict(top_k=50), dict(top_p=0.9), dict(top_k=50, top_p=0.9), dict(min_p=0.05),
                                 dict(top_k=1000), dict(top_k=1000, top_p=0.7, min_p=0.001), dict(top_k=1), dict(temperature=0.0),
                                 dict(top_k=256, temperature=2.0), dict(top_k=257), dict(top_p=0.999, temperature=0.3)])
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,classes,draws", [(4, 1000, 3), (3, 1025, 2), (3, 4096, 2), (3, 4097, 2), (2, 20001, 3), (1, 131072, 4)])
def test_many_classes(rows, classes, draws, dtype, cut):
    check(*inputs(rows, classes, draws, dtype, seed=classes, scale=1.5), **cut)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [5, 700, 5000, 40000])
@pytest.mark.parametrize("cut", [dict(), dict(top_k=3), dict(top_k=300, top_p=0.501), dict(top_k=3001), dict(top_p=0.40037)])
def test_ties_go_to_the_lower_index(classes, dtype, cut):
    # all equal; two values; a few values far apart
    u = torch.rand((1, 7), generator=torch.Generator().manual_seed(1))
    g = torch.Generator().manual_seed(2)
    flat = torch.full((1, classes), 1.25)
    two = (torch.rand((1, classes), generator=g) < 0.6).float()
    far = torch.randint(0, 3, (1, classes), generator=g) * 8.0 - 30
    for z in (flat, two, far):
        check(z.to(dtype), u, **cut)


def test_zeros_of_both_signs_are_equal():
    z = torch.tensor([[0.0, -0.0, 0.0, -0.0] * 300])
    u = torch.tensor([[0.0, 0.26, 0.76, 0.999]])
    check(z, u, top_k=4)
    check(z[:, :4], u, top_k=2)


@pytest.mark.parametrize("classes", [9, 50, 3000, 9000])
def test_impossible_classes_and_empty_rows(classes):
    inf, nan = float("inf"), float("nan")
    z, u = inputs(6, classes, 11, torch.float32, seed=3)
    z[0] = -inf
    z[1, : classes - 1] = -inf
    z[2, ::2] = -inf
    z[3, ::2] = nan
    z[4] = nan
    z[5, [1, classes - 2]] = inf
    u[:, 0], u[:, 1], u[:, 2] = 0.0, 1.0, 1.0 - 2.0**-24
    for cut in (dict(), dict(top_k=4), dict(top_p=0.9), dict(top_k=2000, top_p=0.51), dict(min_p=0.3)):
        got = check(z, u, **cut)
        assert (got[0] == -1).all() and (got[4] == -1).all() and (got[1] == classes - 1).all()
        assert set(got[5].tolist()) <= {1, classes - 2}
    uniform = torch.tensor([[-1.0, 2.0, nan]]).expand(6, 3)
    got, _ = ops.sample(z.to(DEV), uniform.to(DEV))
    low, high = ops.sample(z.to(DEV), u[:, :2].to(DEV))[0].T
    assert torch.equal(got[:, 0], low) and torch.equal(got[:, 1], high) and torch.equal(got[:, 2], low)


def test_ranges_of_the_types():
    for z in (torch.tensor([[3e38, -3e38, 1e-38, 0.0, 2.9e38]]), torch.tensor([[1e-40, 2e-40, 0.0, -1e-40]]),
              torch.linspace(-3e38, 3e38, 5000)[None], torch.cat([torch.full((1, 4999), -1e30), torch.zeros(1, 1)], 1)):
        u = torch.tensor([[0.1, 0.4, 0.7, 0.95]])
        for cut in (dict(), dict(temperature=1e30), dict(temperature=1e-30), dict(top_k=2, temperature=1e30), dict(top_p=0.55, temperature=1e30)):
            check(z, u, **cut)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [9, 777, 5003])
def test_strides_alignment_and_shapes(classes, dtype):
    z, u = inputs(6, classes, 4, dtype, seed=4)
    for put in (lambda t: t.T.contiguous().to(DEV).T, lambda t: torch.cat([t, t], 1).to(DEV)[:, :classes],
                lambda t: torch.cat([t[:, :1], t], 1).to(DEV)[:, 1:], lambda t: t.to(DEV)):
        for cut in (dict(), dict(top_k=20), dict(top_p=0.8)):
            want = check(z, u, put, **cut)
    z3, u3 = z.reshape(2, 3, classes).to(DEV), u.reshape(2, 3, 4).to(DEV)
    got, p = ops.sample(z3, u3, top_p=0.8)
    assert got.shape == (2, 3, 4) and torch.equal(got.reshape(6, 4), want)
    one, _ = ops.sample(z3, u3[..., 1], top_p=0.8)
    assert one.shape == (2, 3) and torch.equal(one, got[..., 1])
    single, _ = ops.sample(z3[1, 2], u3[1, 2, 3], top_p=0.8)
    assert single.shape == () and single == got[1, 2, 3]


def test_frequencies_follow_the_probabilities():
    z = torch.tensor([[1.0, 0.0, 2.0, -1.0, 0.5]])
    n = 200000
    u = (torch.arange(n) + 0.5)[None] / n  # evenly spread: counts are the probabilities within 1 of n
    got, p = ops.sample(z.to(DEV), u.float().to(DEV), temperature=0.8)
    share = torch.bincount(got[0].cpu(), minlength=5).double() / n
    want = torch.softmax(z.double() / 0.8, 1)[0]
    assert (share - want).abs().max() <= 2 / n + 2.0**-23


@pytest.mark.parametrize("shape", [(0, 5, 3), (4, 5, 0), (0, 5000, 1), (2, 5000, 0)])
def test_sizes_of_zero(shape):
    rows, classes, draws = shape
    got, p = ops.sample(torch.zeros((rows, classes), device=DEV), torch.zeros((rows, draws), device=DEV))
    assert got.shape == p.shape == (rows, draws)


def test_repeats_on_other_streams_and_in_a_graph():
    z, u = (t.to(DEV) for t in inputs(40, 30011, 3, torch.float16, seed=5))
    cuts = [dict(top_k=50, top_p=0.9), dict(top_p=0.95), dict(top_k=4000), dict()]
    want = [ops.sample(z, u, **c) for c in cuts]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in cuts]
    got = []
    for _ in range(3):
        for s, c in zip(streams, cuts):
            with torch.cuda.stream(s):
                got.append(ops.sample(z, u, **c))
    torch.cuda.synchronize()
    for i, g in enumerate(got):
        assert all(torch.equal(a, b) for a, b in zip(g, want[i % len(cuts)]))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = [ops.sample(z, u, **c) for c in cuts]
    u.copy_(1 - u)
    graph.replay()
    for o, c in zip(outs, cuts):
        assert all(torch.equal(a, b) for a, b in zip(o, ops.sample(z, u, **c)))


def test_refusals():
    z, u = torch.zeros((3, 5), device=DEV), torch.zeros((3, 2), device=DEV)
    cases = [(ValueError, "CUDA", z.cpu(), u, {}), (TypeError, "logits", z.double(), u, {}), (TypeError, "uniforms", z, u.double(), {}),
             (ValueError, "uniforms", z, u[:2], {}), (ValueError, "uniforms", z, u[0, 0], {}), (ValueError, "uniforms", z, u.cpu(), {}),
             (ValueError, "classes", z[:, :0], u, {}), (ValueError, "temperature", z, u, dict(temperature=-1.0)),
             (ValueError, "temperature", z, u, dict(temperature=float("nan"))), (ValueError, "temperature", z, u, dict(temperature=1e-31)),
             (ValueError, "top_k", z, u, dict(top_k=-1)), (ValueError, "top_p", z, u, dict(top_p=0.0)),
             (ValueError, "top_p", z, u, dict(top_p=1.01)), (ValueError, "min_p", z, u, dict(min_p=-0.1)),
             (ValueError, "min_p", z, u, dict(min_p=float("nan"))), (ValueError, "gradient", z.clone().requires_grad_(), u, {})]
    for kind, match, a, b, kw in cases:
        with pytest.raises(kind, match=match):
            ops.sample(a, b, **kw)
    with fwd.dual_level(), pytest.raises(ValueError, match="tangent"):
        ops.sample(fwd.make_dual(z, z), u)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes", [2049, 30000])
@pytest.mark.parametrize("shape", ["peaked", "flat", "two levels", "steps", "far", "tail"])
def test_rows_of_many_shapes(shape, classes, dtype):
    # rows for which the counts over the weights estimate the cut badly: one class with almost all mass, differences below
    # a bin, ties across the border, values far from zero, half of the classes impossible
    g = torch.Generator().manual_seed(11)
    z = torch.randn((2, classes), generator=g)
    if shape == "peaked":
        z[:, classes // 3] = 14.0
    elif shape == "flat":
        z = 3.0 + z * 1e-3
    elif shape == "two levels":
        z = (z > 0.5).float() * 2.0
    elif shape == "steps":
        z = torch.floor(z * 2.0)
    elif shape == "far":
        z = z * 3.0 + 900.0
    else:
        z = torch.where(z > 0, -z * 20, -float("inf"))
        z[:, 7] = 0.0
    z = z.to(dtype)
    u = torch.rand((2, 3), generator=g)
    for cut in (dict(top_p=0.95003), dict(top_p=0.30007, temperature=0.2), dict(top_p=0.99931, temperature=3.0),
                dict(top_p=0.01031), dict(top_p=0.77003, min_p=0.031), dict(top_k=700), dict(top_k=1501, top_p=0.61),
                dict(top_k=1900, min_p=0.2), dict(top_p=0.87004, temperature=1e6)):
        check(z, u, **cut)


@pytest.mark.parametrize("cut", [dict(top_p=0.95), dict(top_k=50, top_p=0.9), dict(top_k=900), dict(min_p=0.02), dict()])
def test_many_rows_at_once(cut):
    z, u = inputs(1500, 2500, 2, torch.bfloat16, seed=12)
    want, _ = ops.sample(z.to(DEV), u.to(DEV), **cut)
    some = torch.arange(0, 1500, 149)
    assert torch.equal(want.cpu()[some], O.sample(z[some], u[some], **cut)[0])
    again, _ = ops.sample(z.to(DEV)[700:], u.to(DEV)[700:], **cut)
    assert torch.equal(again, want[700:])


def test_offsets_beyond_32_bits():
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 16 GB")
    big = torch.empty(2**31 + 2**13, dtype=torch.bfloat16, device=DEV)
    z = big.as_strided((2, 3000), (2**31, 1))
    v, u = inputs(2, 3000, 4, torch.bfloat16, seed=13)
    z.copy_(v)
    for cut in (dict(), dict(top_k=40), dict(top_p=0.8)):
        assert torch.equal(ops.sample(z, u.to(DEV), **cut)[0], ops.sample(v.to(DEV), u.to(DEV), **cut)[0])


def near_cuts(z, top_p, temperature, bins):
    """The min_p whose border lies `bins` hundredths of an exponent above that of top_p."""
    w = torch.exp((z.double() - z.double().max()) / temperature).sort(descending=True).values
    border = w[int((w.cumsum(0) < top_p * w.sum()).sum())]
    min_p = min(1.0, float(border) * math.exp(0.01 * bins))
    assert ((w / min_p - 1).abs() > 1e-11).all()  # no class within rounding of it
    return min_p


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("classes,scale,top_p,temperature", [(131072, 0.8, 0.95, 1.0), (131072, 0.3, 0.9, 0.7), (65536, 1.0, 0.95, 1.5),
                                                             (40000, 0.56, 0.7, 1.0), (2500, 0.5, 0.9, 1.0)])
def test_min_p_beside_the_border_of_top_p(classes, scale, top_p, temperature, dtype):
    for seed in range(3):
        z, u = inputs(1, classes, 12, dtype, seed=100 + seed, scale=scale)
        for bins in (-1.37, 0.23, 0.71, 1.37, 2.41, 3.7, 6.1, 9.3, 14.7):
            check(z, u, temperature=temperature, top_p=top_p, min_p=near_cuts(z[0], top_p, temperature, bins))


@pytest.mark.parametrize("classes,scale,min_p,dtype", [(131072, 0.8, 0.02003, torch.bfloat16), (131072, 0.56, 0.05003, torch.float32),
                                                       (65536, 0.8, 0.02003, torch.float16)])
def test_every_output_is_written(classes, scale, min_p, dtype):
    # through the C ABI into buffers that hold what no draw gives
    z, u = inputs(60, classes, 6, dtype, seed=21, scale=scale)
    zd, ud = z.to(DEV), u.to(DEV)
    tokens, probs = torch.full(u.shape, -7, dtype=torch.int64, device=DEV), torch.full(u.shape, -7.0, device=DEV)
    d = L.NcaSampleDesc(rows=60, classes=classes, draws=6, logits_stride=classes, dtype=TYPES.index(dtype), top_k=0, temperature=1.0,
                        top_p=0.95, min_p=min_p)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    assert L.lib().nca_b200_sample(C.byref(d), p(zd), p(ud), p(tokens), p(probs), stream) == 0
    assert (tokens >= 0).all() and (probs > 0).all()
    want, share, nearest = O.sample(z, u, top_p=0.95, min_p=min_p)
    assert nearest > 1e-11
    assert torch.equal(tokens.cpu(), want)
    assert ((probs.cpu().double() - share).abs() <= share * 2.0**-24 + 1e-10).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("classes,tail", [(131072, 46.03), (131072, 45.51), (2**19, 44.1), (2**19 + 3, 44.1), (2**20 + 1, 43.2), (2**23, 40.6),
                                          (2**23 + 7, 30.2), (2**23, 3.0)])
def test_one_class_above_a_long_tail_of_equal_ones(classes, tail, dtype):
    # a peak of weight 1 and the others at 2^-tail, about half a unit of the fixed point that so many heavy classes would need.
    # Weights are rounded to 2^-bits of the largest: 62 bits less those of the number of classes (51 at most), from 2^19 classes on
    # less those of the weights' sum.  A draw is off by half a unit of every class at most.
    low = torch.tensor(-tail * math.log(2.0)).to(dtype)
    w = math.exp(float(low))
    total = 1 + (classes - 1) * w
    bits = 62 - math.ceil(math.log2(classes if classes <= 2**19 else 2 * total))
    slack = classes * 2.0 ** -(min(bits, 51) + 1) + 1e-13 * total
    peak = classes // 3
    z = torch.full((1, classes), float(low))
    z[0, peak] = 0.0
    inner = (torch.arange(1, 40, dtype=torch.float64) / 40 * (peak * w)) / total
    outer = 1 - (torch.arange(1, 40, dtype=torch.float64) / 40 * ((classes - 1 - peak) * w)) / total
    u = torch.cat([inner, outer, torch.linspace(0, 1, 40, dtype=torch.float64)[:-1]]).float()
    tokens, probs = ops.sample(z.to(dtype).to(DEV), u[None].to(DEV))
    at = tokens[0].cpu().double()
    before = at * w + torch.where(at > peak, 1 - w, 0.0)  # the mass before the class that was drawn
    own = torch.where(at == peak, 1.0, w)
    t = u.double() * total
    assert ((at >= 0) & (at < classes)).all()
    assert (before - slack <= t).all() and (t < before + own + slack).all()
    assert ((probs[0].cpu().double() - own / total).abs() <= own / total * 2.0**-24 + slack / total).all()
