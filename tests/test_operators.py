"""The cell-training operators without a GPU: the 64-bit oracle against finite differences, the
arguments that the operators refuse, and the C ABI's argument checks."""

import ctypes as C

import pytest
import torch

import oracle.cell_operators as O
from ncas_b200 import _lib as L
from ncas_b200 import operators as ops
from ncas_b200.build import build


@pytest.fixture(scope="module")
def lib():
    build()
    return L.lib()


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def difference(f, x, v, h=1e-5):
    """Directional derivative of the scalar f by central differences (error O(h^2), about 1e-9 here)."""
    return float(f(x + h * v) - f(x - h * v)) / (2 * h)


@pytest.mark.parametrize("name", ["none", "silu", "gelu", "sigmoid"])
def test_oracle_norm_gradient_against_differences(name):
    x, dy, w, b = rand(3, 5, 6), rand(3, 5, 6, seed=1), rand(6, seed=2), rand(6, seed=3)
    mask = torch.tensor([[1, 1, 0, 1, 1], [0, 0, 0, 0, 0], [1, 0, 1, 1, 1]])
    _, dx, dw, db = O.group_norm_act(x, 2, w, b, 1e-3, name, mask, dy)
    f = lambda x, w, b: (O.group_norm_act(x, 2, w, b, 1e-3, name, mask) * dy).sum()  # noqa: E731
    v = rand(3, 5, 6, seed=4)
    assert difference(lambda t: f(t, w, b), x, v) == pytest.approx(float((dx * v).sum()), rel=1e-6, abs=1e-7)
    assert difference(lambda t: f(x, t, b), w, v[0, 0]) == pytest.approx(float((dw * v[0, 0]).sum()), rel=1e-6, abs=1e-7)
    assert difference(lambda t: f(x, w, t), b, v[0, 0]) == pytest.approx(float((db * v[0, 0]).sum()), rel=1e-6, abs=1e-7)
    assert (dx[1] == 0).all() and (dx[0, 2] == 0).all()


@pytest.mark.parametrize("name", ["silu", "gelu", "sigmoid"])
def test_oracle_gated_gradient_against_differences(name):
    a = dict(x=rand(4, 3), w_gate=rand(5, 3, seed=1), w_up=rand(5, 3, seed=2), w_down=rand(2, 5, seed=3),
             b_gate=rand(5, seed=4), b_up=rand(5, seed=5), b_down=rand(2, seed=6))
    dy = rand(4, 2, seed=7)
    g = O.gated_ffn(*a.values(), name=name, dy=dy)
    for k in a:
        v = rand(*a[k].shape, seed=8)
        f = lambda t: (O.gated_ffn(*{**a, k: t}.values(), name=name) * dy).sum()  # noqa: B023, E731
        assert difference(f, a[k], v) == pytest.approx(float((g[k] * v).sum()), rel=1e-6, abs=1e-7), k


def test_oracle_distill_gradient_against_differences():
    s, t = rand(4, 7), rand(4, 3, seed=1)
    i = torch.tensor([[0, 3, 6], [2, 2, -1], [-1, -1, -1], [5, 9, 1]])
    w = torch.tensor([1.0, 0.5, 2.0, 0.0], dtype=torch.float64)
    loss, grad = O.distill(s, t, i, 1.7, w)
    assert loss[2] == 0 and loss[3] == 0 and (grad[2:] == 0).all()
    v = rand(4, 7, seed=2)
    assert difference(lambda x: O.distill(x, t, i, 1.7, w)[0].sum(), s, v) == pytest.approx(
        float((grad * v).sum()), rel=1e-6, abs=1e-7)
    # a teacher equal to the student on all classes has no loss and no gradient
    loss, grad = O.distill(s, s, torch.arange(7).expand(4, 7), 2.0)
    assert loss.abs().max() < 1e-12 and grad.abs().max() < 1e-12


# ------------------------------------------------------------------------------- refusals
def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.group_norm_act(x, 2)
    w = torch.zeros(4, 4, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_ffn(w, w, w, w)
    with pytest.raises(ValueError, match="CUDA"):
        ops.distill_loss(torch.zeros(2, 4), torch.zeros(2, 1), torch.zeros(2, 1, dtype=torch.int32))


def norm_desc(**kw):
    d = L.NcaNormDesc(n=2, cells=4, channels=8, groups=2, dtype=0, param_dtype=0, act=2, eps=1e-5, x_stride_n=32,
                      x_stride_cell=8, dy_stride_n=32, dy_stride_cell=8)
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_norm_descriptor_checks(lib):
    n = C.c_size_t(0)
    ask = lambda **kw: lib.nca_b200_group_norm_workspace(C.byref(norm_desc(**kw)), 1, C.byref(n))  # noqa: E731
    assert ask() == 0 and n.value > 0
    for bad in (dict(groups=3), dict(groups=0), dict(channels=0), dict(n=-1), dict(cells=-1), dict(dtype=3),
                dict(dtype=1, param_dtype=2), dict(act=5), dict(act=-1), dict(eps=-1.0), dict(eps=float("nan"))):
        assert ask(**bad) == 1, bad
    assert lib.nca_b200_group_norm_workspace(None, 0, C.byref(n)) == 1
    # no work, no pointers needed; with work, missing pointers and a short workspace are refused
    d = norm_desc(n=0)
    assert lib.nca_b200_group_norm(C.byref(d), *[None] * 7, 0, None) == 0
    d = norm_desc()
    assert lib.nca_b200_group_norm(C.byref(d), *[None] * 7, 0, None) == 1


def test_norm_channel_numbers_fit_32_bits(lib):
    n = C.c_size_t(0)
    ask = lambda c: lib.nca_b200_group_norm_workspace(  # noqa: E731
        C.byref(norm_desc(n=1, cells=1, channels=c, groups=1)), 1, C.byref(n))
    assert ask(1 << 30) == 0 and ask((1 << 30) + 1) == 2 and ask((1 << 31) - 1) == 2


def gated_desc(**kw):
    d = L.NcaGatedDesc(rows=5, d_in=16, hidden=24, d_out=8, dtype=1, bias_dtype=0, act=2)
    for name, ld in (("x_stride", 16), ("w_gate_stride", 16), ("w_up_stride", 16), ("w_down_stride", 24),
                     ("dy_stride", 8)):
        getattr(d, name)[0], getattr(d, name)[1] = ld, 1
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(d, k)[0], getattr(d, k)[1] = v
        else:
            setattr(d, k, v)
    return d


def test_gated_descriptor_checks(lib):
    n = C.c_size_t(0)
    ask = lambda bwd=0, **kw: lib.nca_b200_gated_workspace(C.byref(gated_desc(**kw)), bwd, C.byref(n))  # noqa: E731
    assert ask() == 0
    plain = n.value
    assert ask(x_stride=(1, 5)) == 0 and n.value > plain  # a transposed x is copied
    assert ask(unaligned=1) == 0 and n.value > plain
    assert ask(bwd=1) == 0 and n.value > plain
    for bad in (dict(rows=-1), dict(d_in=0), dict(hidden=0), dict(d_out=0), dict(bias_dtype=2), dict(act=0),
                dict(act=7)):
        assert ask(**bad) == 1, bad
    assert ask(dtype=0) == 2  # no fp32 products
    assert ask(rows=1 << 31) == 2
    assert lib.nca_b200_gated_saved_bytes(C.byref(gated_desc()), C.byref(n)) == 0 and n.value >= 4 * 5 * 24 * 2
    d = gated_desc(rows=0)
    assert lib.nca_b200_gated_ffn(C.byref(d), *[None] * 10, 0, None, 0, None) == 0
    d = gated_desc()
    assert lib.nca_b200_gated_ffn(C.byref(d), *[None] * 10, 0, None, 0, None) == 1


def test_gated_backward_without_biases_needs_no_room_for_their_sums(lib):
    def ask(bwd, rows):
        n = C.c_size_t(0)
        assert lib.nca_b200_gated_workspace(C.byref(gated_desc(rows=rows)), bwd, C.byref(n)) == 0
        return n.value

    for rows in (1, 5, 1000, 100000):  # a sum of every 32 rows of the tiles of 128, of both matrices, in fp32
        assert ask(1, rows) - ask(2, rows) == 4 * -(-rows // 128) * 2 * 24 * 4


def test_distill_descriptor_checks(lib):
    n = C.c_size_t(0)

    def ask(**kw):
        d = L.NcaDistillDesc(rows=4, classes=9, top=3, dtype=0, teacher_dtype=0, index_bits=32, temperature=1.0,
                             logits_stride=9, teacher_stride=3, index_stride=3)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.nca_b200_distill_workspace(C.byref(d), C.byref(n))

    assert ask() == 0 and ask(top=0) == 0 and ask(rows=0) == 0
    for bad in (dict(rows=-1), dict(classes=0), dict(top=-1), dict(dtype=4), dict(teacher_dtype=-1),
                dict(index_bits=16), dict(temperature=0.0), dict(temperature=-1.0), dict(temperature=float("nan")),
                dict(temperature=float("inf"))):
        assert ask(**bad) == 1, bad
    assert ask(classes=1 << 31) == 2


def test_distill_temperatures_whose_reciprocal_overflows_are_refused(lib):
    n = C.c_size_t(0)
    ask = lambda t: lib.nca_b200_distill_workspace(C.byref(L.NcaDistillDesc(  # noqa: E731
        rows=4, classes=9, top=3, dtype=0, teacher_dtype=0, index_bits=32, temperature=t, logits_stride=9,
        teacher_stride=3, index_stride=3)), C.byref(n))
    assert ask(1e-29) == 0 and ask(1e29) == 0
    for t in (1e-39, 1e-44, 9e-31, 1.1e30):
        assert ask(t) == 1, t


def test_operators_are_registered_with_their_schemas(lib):
    from ncas_b200._ops import ops as torch_ops

    o = torch_ops()
    for name in ("group_norm_act", "gated_ffn", "distill_loss", "distill_loss_and_grad", "operators_status"):
        assert hasattr(o, name)
    assert str(o.group_norm_act.default._schema) == (
        "nca_b200::group_norm_act(Tensor x, int groups, Tensor? weight, Tensor? bias, float eps, str act, "
        "Tensor? mask) -> Tensor")
