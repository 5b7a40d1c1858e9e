"""orthogonalize on the GPU against the 64-bit oracle.

The kernels round to fp16 in documented places (operands of the products; X to 22 bits) and sum in fp32.  The oracle
can make the same roundings, everything else exact: its distance r from the exact result is what they cost.  The
kernels' roundings fall on values that differ in the last place of fp32, so their errors are of the same size and
otherwise independent: in the Frobenius norm, of n values, within a factor 1 + 6 / sqrt(n) of each other, and 4 for
the smallest matrices here, whose few roundings do not average.  Sums of k <= 4096 products in fp32 add
2^-24 sqrt(k) < 2^-18 of a norm, amplified like r, which is made of roundings of 2^-12: covered by the factor 4 too.
The result adds half a step of its type in every value."""

import ctypes as C

import pytest
import torch

import oracle.cell_operators as O
from ncas_b200 import _lib as L
from ncas_b200 import operators as ops

pytestmark = pytest.mark.gpu

DEV = "cuda"
UNIT = {torch.bfloat16: 2.0**-8, torch.float16: 2.0**-11}
TYPES = [torch.bfloat16, torch.float16]


def matrix(shape, dtype, seed=0, scale=0.02):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * scale).to(dtype)


def check(m, steps=5, put=lambda t: t.to(DEV), **kw):
    got = ops.orthogonalize(put(m), steps=steps, **kw)
    ops.check()
    assert got.shape == m.shape and got.dtype == m.dtype and got.is_contiguous()
    flat = lambda t: t.double().cpu().reshape(-1, *m.shape[-2:])  # noqa: E731
    want, near = flat(O.orthogonalize(m, steps, **kw)), flat(O.orthogonalize(m, steps, rounded=True, **kw))
    for g, w, r in zip(flat(got), want, near):
        tol = 4 * (r - w).norm() + UNIT[m.dtype] * w.norm() + 2.0**-25 * w.numel() ** 0.5
        assert (g - w).norm() <= tol, (float((g - w).norm()), float(tol), float((r - w).norm()))
    return got


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [
    (1, 1), (1, 9), (9, 1), (8, 8), (5, 70), (64, 64), (64, 256), (256, 64), (256, 256), (129, 130), (100, 1000),
    (1000, 100), (257, 600), (513, 300), (385, 385), (640, 1288), (1001, 730)])
def test_against_the_oracle(rows, cols, dtype):
    check(matrix((rows, cols), dtype, seed=rows))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 40, 24), (2, 2, 130, 300), (5, 257, 129), (40, 64, 72), (3, 300, 300)])
def test_stacks(shape, dtype):
    m = matrix(shape, dtype, seed=1)
    got = check(m)
    alone = ops.orthogonalize(m.reshape(-1, *shape[-2:])[-1].to(DEV))
    # a matrix of a stack does not see the others: at most the tiles' shapes differ, and with them nothing in a sum's order
    assert torch.equal(alone, got.reshape(-1, *shape[-2:])[-1])


# about the sizes from which a matrix takes one launch, and from which its last steps take operands of 22 bits
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,steps", [
    (128, 256, 5), (128, 257, 5), (129, 256, 5), (256, 129, 5), (256, 257, 5), (140, 200, 5), (200, 141, 5), (17, 33, 7),
    (128, 128, 1), (250, 250, 2), (250, 250, 3), (300, 310, 8), (255, 255, 6), (1, 256, 12)])
def test_about_the_borders(rows, cols, steps, dtype):
    check(matrix((rows, cols), dtype, seed=rows + cols), steps=steps)


def test_a_bad_matrix_stays_alone():
    m = matrix((4, 100, 260), torch.bfloat16, seed=2).to(DEV)
    want = ops.orthogonalize(m)
    for bad in (float("nan"), float("inf")):
        b = m.clone()
        b[1, 50, 3] = bad
        got = ops.orthogonalize(b)
        assert torch.equal(got[[0, 2, 3]], want[[0, 2, 3]]) and got[1].isnan().any()
    z = m.clone()
    z[2] = 0
    got = ops.orthogonalize(z)
    assert (got[2] == 0).all() and torch.equal(got[[0, 1, 3]], want[[0, 1, 3]])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rank", [1, 3])
def test_low_rank(dtype, rank):
    # what a is left in the small directions is amplified by a at every step: X must not be rounded to 11 bits
    g = torch.Generator().manual_seed(3)
    u, v = torch.randint(-3, 4, (300, rank), generator=g), torch.randint(-3, 4, (rank, 520), generator=g)
    m = (u @ v).to(dtype)  # exact in the type: rank `rank`
    got = check(m)
    s = torch.linalg.svdvals(got.double().cpu())
    # five steps bring the large ones to 0.68 to 1.21; nothing but the result's rounding may appear in the others
    assert (s[:rank] > 0.6).all() and (s[:rank] < 1.25).all()
    assert s[rank] <= UNIT[dtype] * 1.25 * rank**0.5 + 4 * float((O.orthogonalize(m, rounded=True) - O.orthogonalize(m)).norm())


@pytest.mark.parametrize("scale", [1e-30, 1e-9, 1e30, 3e37])
def test_norms_at_the_ends_of_the_range(scale):
    m = matrix((70, 90), torch.bfloat16, seed=4, scale=scale)
    check(m, eps=1e-7 if scale > 1 else 0.0)
    if scale < 1e-8:  # the norm counts for little beside eps
        check(m.clone(), eps=1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_strides_and_alignment(dtype):
    m = matrix((3, 80, 136), dtype, seed=5)
    for put in (lambda t: t.to(DEV).transpose(1, 2).contiguous().transpose(1, 2),  # copied
                lambda t: torch.cat([t, t], 2).to(DEV)[..., :136],
                lambda t: torch.cat([t[..., :1], t], 2).to(DEV)[..., 1:],  # odd starts and rows
                lambda t: t.to(DEV).transpose(0, 1).contiguous().transpose(0, 1)):
        check(m, put=put)
    check(m[:1].expand(3, 80, 136))


def test_steps_and_coefficients():
    m = matrix((90, 200), torch.float16, seed=6)
    check(m, steps=1)
    check(m, steps=12)
    check(m, steps=8, coefficients=(1.5, -0.5, 0.0))
    check(m, steps=3, coefficients=(1.875, -1.25, 0.375))
    check(m, steps=2, coefficients=(1.0, 0.0, 0.0), eps=0.0)


@pytest.mark.parametrize("shape", [(0, 4), (4, 0), (0, 4, 4), (3, 0, 5)])
def test_sizes_of_zero(shape):
    assert ops.orthogonalize(torch.zeros(shape, device=DEV, dtype=torch.bfloat16)).shape == shape


def test_repeats_bit_for_bit_on_other_streams_and_in_a_graph():
    m = matrix((600, 1000), torch.bfloat16, seed=7).to(DEV)
    want = ops.orthogonalize(m)
    torch.cuda.synchronize()
    got, streams = [], [torch.cuda.Stream() for _ in range(3)]
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(ops.orthogonalize(m))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want) for g in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.orthogonalize(m)
    m.neg_()
    graph.replay()
    assert torch.equal(y, -want)
    ops.check()


def test_refusals():
    m = torch.zeros((4, 8), device=DEV, dtype=torch.bfloat16)
    cases = [(ValueError, "CUDA", m.cpu(), {}), (TypeError, "matrix", m.float(), {}), (ValueError, "matrix", m[0], {}),
             (ValueError, "steps", m, dict(steps=0)), (ValueError, "steps", m, dict(steps=1001)),
             (ValueError, "three", m, dict(coefficients=(1.0, 2.0))),
             (ValueError, "finite", m, dict(coefficients=(float("nan"), 0.0, 0.0))),
             (ValueError, "grow", m, dict(coefficients=(3.0, 0.0, 0.0))),
             (ValueError, "grow", m, dict(coefficients=(3.4445, -4.775, 3.0))),
             (ValueError, "eps", m, dict(eps=-1.0)), (ValueError, "eps", m, dict(eps=float("inf"))),
             (ValueError, "gradient", m.clone().requires_grad_(), {})]
    for kind, match, t, kw in cases:
        with pytest.raises(kind, match=match):
            ops.orthogonalize(t, **kw)


def test_a_failure_that_nobody_has_read_does_not_end_it():
    """The C ABI on one row of 2^27 values with control words that an earlier call has set, which end nothing and stay for
    whoever asks."""
    lib = L.lib()
    wide = 1 << 27
    m = torch.ones((1, wide), device=DEV, dtype=torch.bfloat16)
    out = torch.zeros_like(m)
    d = L.NcaOrthoDesc(batch=1, rows=1, cols=wide, dtype=1, steps=2, eps=0.0)
    d.coefficients[:] = [1.5, -0.5, 0.0]
    d.stride[:] = [wide, wide]
    size = C.c_size_t(0)
    assert lib.nca_b200_orthogonalize_workspace(C.byref(d), C.byref(size)) == 0
    ws = torch.empty(size.value, device=DEV, dtype=torch.uint8)
    ctrl = torch.tensor([4, 77, 0, 1], device=DEV, dtype=torch.int32)
    stream = C.c_void_p(torch.cuda.current_stream().cuda_stream)
    p = lambda t: C.c_void_p(t.data_ptr())  # noqa: E731
    detail = C.c_int32(0)
    st = lib.nca_b200_orthogonalize(C.byref(d), p(m), p(out), p(ws), ws.numel(), p(ctrl), 20000, stream)
    assert st == 0
    assert lib.nca_b200_ctrl_status(p(ctrl), C.byref(detail), stream) == 4 and detail.value == 77
    # the one singular value is 1, a fixed point of 1.5 x - 0.5 x^3, and each entry 2^-13.5.  A is off by 2^-8 at most, X by
    # half of that in each step; operands and result round by 2^-8 at most
    assert ((out.float() * 2.0**13.5 - 1).abs() <= 2.0**-7).all()


# sums of more terms than one product adds up, or of pieces for more CTAs, of one sign on A's diagonal and (equal rows) everywhere
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(3, 200001), (200001, 3), (150, 70000), (65600, 300), (2, 40, 131072 + 8), (2, 65537, 130),
                                   (64, 16384), (16385, 100), (300, 8190), (5, 30, 2500), (2, 3001, 9), (270, 5000), (1000, 4100), (2730, 1001)])
def test_long_sums(shape, dtype):
    m = matrix(shape, dtype, seed=12)
    check(m)
    m = m.abs()
    m[..., : m.shape[-2] // 2, :] = 0.02
    check(m)


def test_a_very_long_row():
    for dtype in TYPES:
        got = ops.orthogonalize(torch.full((1, 1 << 22), 3.0, device=DEV, dtype=dtype), steps=3, coefficients=(1.5, -0.5, 0.0), eps=0.0)
        ops.check()
        # as above; the 256 products lose 3e-4 at most, in each step half of it, and the values round
        assert ((got.double() * 2.0**11 - 1).abs() <= 3 * 1.5e-4 + UNIT[dtype]).all()


def test_a_backward_pass_elsewhere_does_not_disturb_it():
    # orthogonalize under a graph of autograd: its input is detached, and nothing is recorded
    w = torch.randn((40, 60), device=DEV).to(torch.bfloat16).requires_grad_()
    loss = (w.float() ** 2).sum()
    with torch.no_grad():
        u = ops.orthogonalize(w)
    assert not u.requires_grad
    loss.backward()
    assert torch.equal(w.grad, (2 * w.detach().float()).to(torch.bfloat16))
    assert torch.equal(ops.orthogonalize(w.detach()), u)


def test_more_matrices_than_a_launch_takes_are_refused():
    with pytest.raises(ValueError, match="65535"):
        ops.orthogonalize(torch.zeros((65536, 2, 2), device=DEV, dtype=torch.bfloat16))


@pytest.mark.parametrize("shape", [(64, 9000), (100, 200), (2, 200, 180)])
def test_two_graphs_in_turn_and_another_stream(shape):
    # each graph has its own workspace: replays of one between those of the other change nothing
    a, b = (matrix(shape, torch.bfloat16, seed=s).to(DEV) for s in (20, 21))
    want = [ops.orthogonalize(t) for t in (a, b)]
    graphs, got = [], []
    for t in (a, b):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            got.append(ops.orthogonalize(t))
        graphs.append(g)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0].replay()
        graphs[1].replay()
        with torch.cuda.stream(side):  # beside them
            beside = ops.orthogonalize(a)
        graphs[0].replay()
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(beside, want[0])
    ops.check()


def strong_and_weak(rows, cols, dtype, seed):
    """A strong direction over noise, as a momentum."""
    g = torch.Generator().manual_seed(seed)
    return ((torch.randn((rows, 1), generator=g) @ torch.randn((1, cols), generator=g) + 0.5 * torch.randn((rows, cols), generator=g)) * 0.01).to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols,steps", [(16, 24, 6), (24, 16, 5), (13, 19, 6), (8, 12, 6), (8, 300, 5), (40, 400, 6), (63, 90, 5)])
def test_small_matrices_are_as_exact_as_their_type(rows, cols, steps, dtype):
    # all operands have 22 bits: what is left is the result's own rounding, whose norm over n values is within a factor
    # 1 + 6 / sqrt(n) of that of the exact result, and the roundings that the oracle can make (factor 4, above).  A whole stack at
    # once: some of its matrices were off by 2 to 4 times the rounding with 11 bits in the first step
    m = torch.stack([strong_and_weak(rows, cols, dtype, seed) for seed in range(20)] +
                    [matrix((rows, cols), dtype, seed=seed) for seed in range(20)])
    got = ops.orthogonalize(m.to(DEV), steps=steps).double().cpu()
    ops.check()
    want, near = O.orthogonalize(m, steps), O.orthogonalize(m, steps, rounded=True)
    norm = lambda t: t.flatten(1).norm(dim=1)  # noqa: E731
    tol = (1 + 6 / (rows * cols) ** 0.5) * norm(want.to(dtype).double() - want) + 4 * norm(near - want) + 2.0**-25 * (rows * cols) ** 0.5
    assert (norm(got - want) <= tol).all(), float((norm(got - want) / tol).max())


@pytest.mark.parametrize("steps", [1, 2])
@pytest.mark.parametrize("rows,cols", [(64, 141), (425, 274), (100, 3000)])
def test_few_steps_of_a_strong_direction(rows, cols, steps):
    # fp16, a direction with nearly all of the norm: as above, all operands have 22 bits
    noise = matrix((5, rows, cols), torch.float32, seed=rows, scale=0.005)
    g = torch.Generator().manual_seed(cols)
    m = (noise + 0.2 * torch.randn((5, rows, 1), generator=g) @ torch.randn((5, 1, cols), generator=g)).half()
    got = ops.orthogonalize(m.to(DEV), steps=steps).double().cpu()
    ops.check()
    want, near = O.orthogonalize(m, steps), O.orthogonalize(m, steps, rounded=True)
    norm = lambda t: t.flatten(1).norm(dim=1)  # noqa: E731
    tol = (1 + 6 / (rows * cols) ** 0.5) * norm(want.half().double() - want) + 4 * norm(near - want) + 2.0**-25 * norm(want)
    assert (norm(got - want) <= tol).all(), float((norm(got - want) / tol).max())
