"""gated_scan, orthogonalize and sample without a GPU: the 64-bit oracle against differences and definitions, the
arguments that the operators refuse, and the C ABI's argument checks."""

import ctypes as C
import math

import pytest
import torch

import oracle.cell_operators as O
from ncas_b200 import _lib as L
from ncas_b200 import operators as ops
from ncas_b200.build import build
from ncas_b200.student import Muon, near_one


@pytest.fixture(scope="module")
def lib():
    build()
    return L.lib()


def rand(*shape, seed=0):
    return torch.randn(shape, generator=torch.Generator().manual_seed(seed), dtype=torch.float64)


def difference(f, x, v, h=1e-5):
    """Directional derivative of the scalar f by central differences (error O(h^2), about 1e-9 here)."""
    return float(f(x + h * v) - f(x - h * v)) / (2 * h)


@pytest.mark.parametrize("dim,reverse", [(1, False), (1, True), (0, False), (2, True)])
def test_oracle_scan_gradient_against_differences(dim, reverse):
    x, gate, dy = rand(3, 4, 5, 2), rand(3, 4, 5, 2, seed=1), rand(3, 4, 5, 2, seed=2)
    edge = [n for i, n in enumerate((3, 4, 5, 2)) if i != dim]
    state, dlast = rand(*edge, seed=3), rand(*edge, seed=4)
    mask = torch.rand((3, 4, 5), generator=torch.Generator().manual_seed(5)) < 0.7
    got = O.gated_scan(x, gate, state, dim, reverse, mask, dy, dlast)

    def value(x, gate, state):
        y, last = O.gated_scan(x, gate, state, dim, reverse, mask)
        return (y * dy).sum() + (last * dlast).sum()

    for name, at, f in (("x", x, lambda t: value(t, gate, state)), ("gate", gate, lambda t: value(x, t, state)),
                        ("state", state, lambda t: value(x, gate, t))):
        v = rand(*at.shape, seed=6)
        assert difference(f, at, v) == pytest.approx(float((got[name] * v).sum()), rel=1e-6, abs=1e-7), name
    assert (got["y"][~mask] == 0).all() and (got["x"][~mask] == 0).all() and (got["gate"][~mask] == 0).all()


def test_oracle_scan_of_open_and_closed_gates():
    x = rand(1, 6, 3)
    y, last = O.gated_scan(x, torch.full((1, 6, 3), -1e9, dtype=torch.float64), dim=1)
    assert torch.equal(y, x) and torch.equal(last, x[:, -1])
    h = rand(1, 3, seed=1)
    y, last = O.gated_scan(x, torch.full((1, 6, 3), 1e9, dtype=torch.float64), h, dim=1)
    assert torch.equal(last, h) and (y == h[:, None]).all()


def test_oracle_orthogonalize_works_on_the_singular_values():
    m = rand(12, 20)
    u, s, v = torch.linalg.svd(m, full_matrices=False)
    x = s / (s.norm() + 1e-7)
    for _ in range(5):
        x = 3.4445 * x - 4.775 * x**3 + 2.0315 * x**5
    for t in (m, m.T):
        got = O.orthogonalize(t)
        want = (u * x) @ v
        assert ((got if t is m else got.T) - want).abs().max() < 1e-11
    near = O.orthogonalize(m.bfloat16(), rounded=True)
    assert 0 < (near - O.orthogonalize(m.bfloat16())).norm() / near.norm() < 3e-3


def test_oracle_sample_is_the_definition():
    z = torch.tensor([[0.0, 2.0, 1.0, 2.0, -1.0]])
    w = torch.exp(z[0].double() - 2)
    # order: 1, 3 (a tie, by index), 2, 0, 4
    pick = lambda u, **kw: O.sample(z, torch.tensor([[u]]), **kw)[0].item()  # noqa: E731
    c = (w.cumsum(0) / w.sum()).tolist()
    assert [pick(c[i] + 1e-6) for i in range(4)] == [1, 2, 3, 4] and pick(0.0) == 0
    assert pick(0.49, top_k=2) == 1 and pick(0.51, top_k=2) == 3 and pick(0.99, top_k=1) == 1
    assert {pick(u, top_p=0.7) for u in (0.0, 0.3, 0.6, 0.9)} == {1, 3}
    assert {pick(u / 20, min_p=0.3) for u in range(20)} == {1, 2, 3}
    assert pick(0.7, temperature=0.0) == 1 and pick(1.0) == 4 and pick(1.0, top_k=3) == 3
    tokens, probs, _ = O.sample(torch.full((1, 3), -math.inf), torch.tensor([[0.5, 0.1]]))
    assert tokens.tolist() == [[-1, -1]] and probs.tolist() == [[0.0, 0.0]]


# ------------------------------------------------------------------------------- the optimiser
def test_muon_takes_parameter_groups():
    matrix = lambda: torch.nn.Parameter(torch.zeros(4, 6, dtype=torch.bfloat16))  # noqa: E731
    opt = Muon([{"params": [matrix()], "lr": 0.1}, {"params": [matrix(), matrix()], "momentum": 0.5}], lr=0.02)
    assert [(g["lr"], g["momentum"], len(g["params"])) for g in opt.param_groups] == [(0.1, 0.95, 1), (0.02, 0.5, 2)]
    opt.add_param_group({"params": matrix(), "steps": 3})
    for bad in (torch.zeros(4, dtype=torch.bfloat16), torch.zeros(4, 4)):
        with pytest.raises(ValueError, match="Muon"):
            opt.add_param_group({"params": [matrix(), torch.nn.Parameter(bad)]})
        with pytest.raises(ValueError, match="Muon"):
            Muon([{"params": [torch.nn.Parameter(bad)]}])
    assert len(opt.param_groups) == 3 and opt.param_groups[2]["steps"] == 3


@pytest.fixture
def plain_orthogonalize(monkeypatch):
    """Muon on the CPU: the operator's formula in 64 bits in its place."""
    monkeypatch.setattr(ops, "orthogonalize", lambda m, **kw: O.orthogonalize(m, **kw).to(m.dtype))


def gradients(params, seed):
    for i, p in enumerate(params):
        p.grad = rand(*p.shape, seed=seed + i).to(p.dtype)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_a_resumed_muon_goes_on_as_if_never_stopped(plain_orthogonalize, dtype, tmp_path):
    def fresh():
        params = [torch.nn.Parameter(rand(6, 9, seed=i).to(dtype)) for i in range(3)]
        return params, Muon([{"params": params[:2], "lr": 0.1}, {"params": params[2:]}], lr=0.05)

    one, opt = fresh()
    for step in range(4):
        gradients(one, 10 * step)
        opt.step()
        if step == 1:
            torch.save((one, opt.state_dict()), tmp_path / "at_two")
            kept = opt.state_dict()
    two, resumed = fresh()
    weights, state = torch.load(tmp_path / "at_two", weights_only=False)
    resumed.load_state_dict(state)
    for p, w in zip(two, weights):
        p.data.copy_(w.data)
        assert resumed.state[p]["momentum"].dtype == torch.float32
    for step in (2, 3):
        gradients(two, 10 * step)
        resumed.step()
    for a, b in zip(one, two):
        assert torch.equal(a, b) and torch.equal(opt.state[a]["momentum"], resumed.state[b]["momentum"])
    assert resumed.param_groups[0]["lr"] == 0.1 and resumed.param_groups[1]["lr"] == 0.05
    # the dict that was given is not the resumed optimiser's own state; a state without momenta is one of no steps
    live = kept["state"][0]["momentum"].clone()
    resumed.load_state_dict(kept)
    gradients(two, 50)
    resumed.step()
    assert torch.equal(kept["state"][0]["momentum"], live)
    resumed.load_state_dict(fresh()[1].state_dict())
    assert not resumed.state


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("size", [1e-7, 1e-30, 3e4, 1e36])
def test_an_update_does_not_depend_on_the_size_of_its_gradients(plain_orthogonalize, size, dtype):
    # the same gradients times a power of two give the same bits, but for eps = 1e-7 of the smaller one's norm, which the
    # largest entry's scale keeps near 1; the optimiser's grad is of the matrix's type, whose range the sizes stay in
    exponent = math.floor(math.log2(size if dtype == torch.bfloat16 else min(max(size, 2.0**-11), 3e4)))

    def run(scale):
        p = torch.nn.Parameter(torch.zeros(5, 7, dtype=dtype))
        opt = Muon([p], lr=1.0)
        for seed in range(3):
            p.grad = ((rand(5, 7, seed=seed).clamp(-1, 1) * 64).round() / 64 * scale).to(dtype)
            opt.step()
        return p.detach()

    got, want = run(2.0**exponent), run(1.0)
    assert want.abs().max() > 0.1 and torch.equal(got, want)


def test_tiny_and_huge_fp16_momenta(plain_orthogonalize):
    # gradients at the ends of fp16: the momentum of many of 3e4 passes 65504, the update of one of 6e-8 is one step of the type
    for size, steps in ((3e4, 20), (6e-8, 1)):
        p = torch.nn.Parameter(torch.zeros(4, 4, dtype=torch.float16))
        opt = Muon([p], lr=0.5, nesterov=False)
        p.grad = (torch.eye(4) * size).half()
        for _ in range(steps):
            p.data.zero_()
            opt.step()
        # singular values of a multiple of the identity: 0.5 to begin with, then five steps of the polynomial
        want = -0.5 * O.orthogonalize(torch.eye(4))
        assert (p.double() - want).abs().max() <= 2.0**-10
    zero = torch.nn.Parameter(torch.ones(3, 4, dtype=torch.float16))
    zero.grad = torch.zeros_like(zero)
    Muon([zero]).step()
    assert (zero == 1).all()


@pytest.mark.parametrize("shape", [(0, 4), (4, 0)])
def test_muon_of_empty_matrices(monkeypatch, shape):
    monkeypatch.setattr(ops, "orthogonalize", lambda m, **kw: m)
    p = torch.nn.Parameter(torch.zeros(shape, dtype=torch.bfloat16))
    p.grad = torch.zeros_like(p)
    Muon([p]).step()


def test_near_one_multiplies_by_powers_of_two():
    ends = torch.tensor([2.0**-149, -(2.0**-126), 3.0, 3.4e38, -1.0, 0.5, 0.0])
    got = near_one(ends[:, None, None] * torch.tensor([[1.0, 0.5]]))
    top = got.abs().amax((-2, -1))
    assert ((top >= 0.5) & (top < 1))[:-1].all() and (got[-1] == 0).all()
    assert (torch.frexp(got[:-1, 0, 0].abs()).mantissa == torch.frexp(ends[:-1].abs()).mantissa).all()
    assert torch.equal(got[1:, 0, 1], got[1:, 0, 0] / 2)
    assert near_one(torch.zeros(2, 0, 4)).shape == (2, 0, 4)


# ------------------------------------------------------------------------------- refusals
def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 3, 4)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gated_scan(x, x)
    with pytest.raises(ValueError, match="CUDA"):
        ops.orthogonalize(x.bfloat16())
    with pytest.raises(ValueError, match="CUDA"):
        ops.sample(x, torch.zeros(2, 3))


def scan_desc(**kw):
    d = L.NcaScanDesc(n=2, m=3, steps=40, channels=8, dtype=1)
    for name in ("x_stride", "gate_stride", "dy_stride", "y_stride"):
        getattr(d, name)[:] = [40 * 3 * 8, 8, 3 * 8]
    d.mask_stride[:] = [120, 1, 3]
    for k, v in kw.items():
        setattr(d, k, v)
    return d


def test_scan_descriptor_checks(lib):
    n = C.c_size_t(0)
    ask = lambda **kw: lib.nca_b200_gated_scan_workspace(C.byref(scan_desc(**kw)), 1, C.byref(n))  # noqa: E731
    saved = lambda **kw: lib.nca_b200_gated_scan_saved_bytes(C.byref(scan_desc(**kw)), C.byref(n))  # noqa: E731
    assert ask() == 0 and saved() == 0
    for ok in (dict(n=0), dict(m=0), dict(steps=0), dict(channels=0)):
        assert ask(**ok) == 0 and n.value == 0
        assert saved(**ok) == 0 and n.value == 0
    # a state of every 8 steps but the first, for every line and channel
    assert saved(steps=8) == 0 and n.value == 0
    assert saved(steps=9) == 0 and n.value == 4 * 6 * 8
    assert saved(steps=1000) == 0 and n.value == 4 * 6 * 8 * 124
    for bad in (dict(n=-1), dict(m=-1), dict(steps=-1), dict(channels=-1), dict(dtype=3), dict(dtype=-1)):
        assert ask(**bad) == 1 and saved(**bad) == 1, bad
    assert ask(n=1 << 41) == 2 and ask(n=1 << 30, m=1 << 30) == 2 and ask(n=1 << 30, steps=1 << 30) == 2
    # a long line of few channels is cut into pieces, whose maps need room
    assert ask(n=1, m=1, steps=100000) == 0 and n.value > 0 and n.value % (2 * 4 * 8) == 0
    assert lib.nca_b200_gated_scan_workspace(None, 0, C.byref(n)) == 1
    d = scan_desc()
    assert lib.nca_b200_gated_scan(C.byref(d), *[None] * 8, 0, None) == 1
    assert lib.nca_b200_gated_scan_backward(C.byref(d), *[None] * 11, 0, None) == 1
    d = scan_desc(n=0)
    assert lib.nca_b200_gated_scan(C.byref(d), *[None] * 8, 0, None) == 0
    assert lib.nca_b200_gated_scan_backward(C.byref(d), *[None] * 11, 0, None) == 0


def test_scan_pointers_and_workspace_are_checked_before_a_launch(lib):
    d = scan_desc(n=1, m=1, steps=100000)
    p = 1 << 20  # an address that nothing reads: the checks come first
    call = lambda d, x=p, ws=p, size=1 << 30: lib.nca_b200_gated_scan(  # noqa: E731
        C.byref(d), x, p, None, None, p, p, None, ws, size, None)
    assert call(d, x=p + 2) == 1  # pairs of channels start on 4 bytes, or `unaligned` says so
    assert call(d, ws=None) != 0
    assert call(d, size=8) != 0
    d.masked = 1
    assert call(d) == 1


def test_scan_buffers_of_pairs_start_on_8_bytes(lib):
    # an address that nothing reads: the checks come before a launch; without room for the maps even a right call ends there
    d = scan_desc(n=1, m=1, steps=100000)
    p = 1 << 20
    forward = lambda saved, ws, size: lib.nca_b200_gated_scan(C.byref(d), p, p, None, None, p, p, saved, ws, size, None)  # noqa: E731
    backward = lambda saved, ws, size: lib.nca_b200_gated_scan_backward(  # noqa: E731
        C.byref(d), p, p, None, None, saved, p, None, p, p, None, ws, size, None)
    for call in (forward, backward):
        assert call(p + 4, p, 8) == 1
        assert call(p, p + 4, 1 << 30) == 1
        assert call(p, p, 8) == call(p, None, 1 << 30) == 7


def ortho_desc(**kw):
    d = L.NcaOrthoDesc(batch=2, rows=30, cols=50, dtype=1, steps=5, eps=1e-7)
    d.coefficients[:] = [3.4445, -4.775, 2.0315]
    d.stride[:] = [1500, 50]
    for k, v in kw.items():
        if k == "coefficients":
            d.coefficients[:] = v
        else:
            setattr(d, k, v)
    return d


def test_orthogonalize_descriptor_checks(lib):
    n = C.c_size_t(0)
    ask = lambda **kw: lib.nca_b200_orthogonalize_workspace(C.byref(ortho_desc(**kw)), C.byref(n))  # noqa: E731
    assert ask() == 0 and n.value == 0  # one launch, which holds everything itself
    assert ask(cols=300) == 0 and n.value >= 2 * 4 * 30 * 304 * 2  # X twice, each as two planes
    assert ask(batch=0) == 0 and n.value == 0
    for bad in (dict(batch=-1), dict(rows=-1), dict(cols=-1), dict(steps=0), dict(dtype=5), dict(eps=-1.0),
                dict(eps=float("nan")), dict(coefficients=[float("inf"), 0, 0])):
        assert ask(**bad) == 1, bad
    assert ask(dtype=0) == 2 and ask(steps=1001) == 2 and ask(rows=(1 << 30) + 1) == 2 and ask(batch=65536) == 2
    d = ortho_desc()
    assert lib.nca_b200_orthogonalize(C.byref(d), None, None, None, 0, None, 0, None) == 1
    d = ortho_desc(rows=0)
    assert lib.nca_b200_orthogonalize(C.byref(d), None, None, None, 0, None, 0, None) == 0


def test_coefficients_that_let_singular_values_grow_are_refused(lib):
    n = C.c_size_t(0)
    ask = lambda *c, steps=5: lib.nca_b200_orthogonalize_workspace(  # noqa: E731
        C.byref(ortho_desc(coefficients=c, steps=steps)), C.byref(n))

    def grows(a, b, c, steps):  # the largest value of the map on a fine grid of [0, what came before]
        most = 1.0
        for _ in range(steps):
            x = torch.linspace(0, most, 20001, dtype=torch.float64)
            most = float((x * (a + x**2 * (b + x**2 * c))).abs().max())
            if most > 2:
                return True
        return False

    g = torch.Generator().manual_seed(0)
    refused = 0
    for _ in range(300):
        a, b, c = (torch.rand(3, generator=g, dtype=torch.float64) * torch.tensor([4.0, 10.0, 6.0]) - torch.tensor([0.0, 8.0, 2.0])).tolist()
        steps = int(torch.randint(1, 7, (1,), generator=g))
        if abs(a) < 1e-3 or abs(c) < 1e-3:
            continue
        want = grows(a, b, c, steps)
        assert (ask(a, b, c, steps=steps) == 2) == want, (a, b, c, steps)
        refused += want
    assert 50 < refused < 250
    assert ask(1.5, -0.5, 0.0) == 0 and ask(1.0, 0.0, 0.0) == 0 and ask(0.0, 0.0, 0.0) == 0 and ask(2.1, 0.0, 0.0) == 2


def test_sample_descriptor_checks(lib):
    def call(**kw):
        d = L.NcaSampleDesc(rows=4, classes=9, draws=2, logits_stride=9, dtype=0, top_k=0, temperature=1.0, top_p=1.0, min_p=0.0)
        for k, v in kw.items():
            setattr(d, k, v)
        return lib.nca_b200_sample(C.byref(d), None, None, None, None, None)

    assert call(rows=0) == 0 and call(draws=0) == 0
    for bad in (dict(), dict(rows=-1), dict(classes=0), dict(draws=-1), dict(dtype=3), dict(top_k=-1), dict(temperature=-1.0),
                dict(temperature=float("nan")), dict(temperature=1e-31), dict(temperature=1e31), dict(top_p=0.0),
                dict(top_p=1.5), dict(top_p=float("nan")), dict(min_p=-0.1), dict(min_p=1.1)):
        assert call(**bad) == 1, bad
    assert call(classes=(1 << 30) + 1) == 2
    assert lib.nca_b200_sample(None, None, None, None, None, None) == 1


def test_operators_are_registered_with_their_schemas(lib):
    from ncas_b200._ops import ops as torch_ops

    o = torch_ops()
    assert str(o.gated_scan.default._schema) == (
        "nca_b200::gated_scan(Tensor x, Tensor gate, Tensor? state, int dim, bool reverse, Tensor? mask) -> (Tensor, Tensor)")
    assert str(o.orthogonalize.default._schema) == (
        "nca_b200::orthogonalize(Tensor matrix, int steps, float[] coefficients, float eps) -> Tensor")
    assert str(o.sample.default._schema) == (
        "nca_b200::sample(Tensor logits, Tensor uniforms, float temperature, int top_k, float top_p, float min_p) -> "
        "(Tensor, Tensor)")


def test_workloads_of_the_operators():
    import random

    import perf.more_operators as M

    cases = M.listed()
    assert len({c["name"] for c in cases}) == len(cases)
    rng = random.Random(1)
    most = max(M.work(c)["flops"] for c in cases if c["op"] == "ortho")
    for _ in range(200):
        c = M.draw(rng)
        w = M.work(c)
        assert w["bytes"] > 0 and w["flops"] > 0
        assert c["op"] != "ortho" or w["flops"] <= most
