"""GPU: Newton-Schulz steps and the optimiser step around them, against the formulas in 64 bits.

What may be off, as Frobenius norms.  The first operand is rounded where the matrix is small against its norm: a unit u of it grows by at
most the product of the steps' factors a, 3.4445^5 = 485, however small the result.  Every product's operands are rounded too, three products a
step, with factors of a + |b| + |c| = 10 at most between them, 150 u of the result in all; measured on matrices of independent entries it
is a tenth of that, as roundings are independent.  Float32 is held in pairs of half precision, u = 2^-22.  16-bit matrices are held in
pairs where the steps that follow could make more than 16 out of the rounding, and else in half precision, u = 2^-12: 16 of them from the
last rounding with that much to come, and 25 of the products' (b and c after one another); and the result is rounded to its type."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from f2cgt_b200 import ops  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
UNIT = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}


def define(g, steps=5, coefficients=ops.NEWTON_SCHULZ, eps=1e-7):
    x = g.double()
    x = x / (x.square().sum((-2, -1), keepdim=True).sqrt() + eps)
    tall = x.shape[-2] > x.shape[-1]
    x = x.mT if tall else x
    for t in range(steps):
        a, b, c = coefficients[t] if isinstance(coefficients[0], (tuple, list)) else coefficients
        p = x @ x.mT
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.mT if tall else x


def room(want, dtype, gain=485.0):
    """Frobenius norm that the result may be off by, per matrix"""
    norm = want.norm(dim=(-2, -1))
    if dtype == torch.float32:
        return 2.0 ** -22 * (gain + 150 * norm)
    return 2.0 ** -22 * gain + (2.0 ** -12 * (16 + 25) + UNIT[dtype]) * norm


def near(got, want, dtype, gain=485.0):
    off = (got.double() - want).norm(dim=(-2, -1))
    assert (off <= room(want, dtype, gain)).all(), (off / want.norm(dim=(-2, -1))).max()


def matrices(batch, rows, cols, dtype, kind="normal", seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed * 31 + rows * 7 + cols)
    x = torch.randn(batch, rows, cols, generator=g, device="cuda")
    if kind == "decay":
        x = x * (torch.arange(1, rows + 1, device="cuda") ** -1.0)[:, None]
    if kind == "low":
        x = torch.randn(batch, rows, 3, generator=g, device="cuda") @ torch.randn(batch, 3, cols, generator=g, device="cuda")
    return (x * 0.02).to(dtype)


SIZES = [(1, 1), (1, 9), (9, 1), (5, 3), (16, 16), (31, 33), (64, 100), (100, 64), (127, 127), (128, 128), (128, 256), (256, 128), (172, 128), (64, 256),
         (129, 129), (128, 257), (256, 256), (250, 130), (300, 1000), (1000, 300), (64, 2000), (2000, 48), (513, 515), (1031, 602), (1, 5000), (1024, 1024)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", SIZES)
def test_against_the_formula(rows, cols, dtype):
    g = matrices(2 if rows * cols < 500_000 else 1, rows, cols, TYPES[dtype])
    out = ops.orthogonalize(g)
    assert out.dtype == g.dtype and out.shape == g.shape
    near(out, define(g), g.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(128, 128), (100, 256), (400, 600), (700, 200)])
@pytest.mark.parametrize("kind", ["decay", "low"])
def test_matrices_of_few_large_singular_values(rows, cols, kind, dtype):
    g = matrices(3, rows, cols, TYPES[dtype], kind)
    near(ops.orthogonalize(g), define(g), g.dtype)


# few tiles and a long K, of which the CTAs of a cluster take parts
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(200, 2000), (1501, 64), (1000, 1031), (33, 2999)])
def test_long_sums(rows, cols, dtype):
    test_against_the_formula(rows, cols, dtype)


@pytest.mark.parametrize("dtype", TYPES)
def test_zero_and_not_finite_among_long_sums(dtype):
    test_zero_and_matrices_that_are_not_finite_leave_the_others_alone(70, 1200, dtype)


@pytest.mark.parametrize("rows,cols", [(40, 60), (128, 130), (300, 200)])
def test_scale_does_not_matter(rows, cols):
    g = matrices(1, rows, cols, torch.float32)
    want = define(g, eps=0.0)
    for by in (1e-30, 1e-12, 1.0, 1e20, 1e36):
        near(ops.orthogonalize(g * by, eps=0.0), define(g * by, eps=0.0), torch.float32)
        near(ops.orthogonalize(g * by, eps=0.0), want, torch.float32, 485 + 485 * 4)  # g * by is rounded itself


@pytest.mark.parametrize("rows,cols", [(40, 60), (128, 130), (300, 200)])
def test_matrices_smaller_than_eps(rows, cols):
    for norm in (1e-6, 1e-7, 1e-9, 1e-11, 1e-13):
        g = matrices(1, rows, cols, torch.float32)
        g = g / g.norm() * norm
        want = define(g)
        off = float((ops.orthogonalize(g).double() - want).norm())
        assert off <= 2.0 ** -22 * (485 * min(1.0, norm / 1e-7) + 150 * float(want.norm()))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(20, 30), (128, 128), (200, 300), (300, 140)])
def test_zero_and_matrices_that_are_not_finite_leave_the_others_alone(rows, cols, dtype):
    g = matrices(6, rows, cols, TYPES[dtype])
    want = define(g)
    g[1] = 0
    g[2, rows // 2, cols - 1] = float("nan")
    g[4, 0, 0] = float("inf")
    g[5, rows - 1, 0] = -float("inf")
    out = ops.orthogonalize(g)
    assert (out[1] == 0).all() and torch.isnan(out[2]).all() and torch.isnan(out[4]).all() and torch.isnan(out[5]).all()
    near(out[[0, 3]], want[[0, 3]], g.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,cols", [(50, 70), (300, 160)])
def test_steps_and_their_coefficients(rows, cols, dtype):
    g = matrices(2, rows, cols, TYPES[dtype])
    near(ops.orthogonalize(g, steps=0), define(g, 0), g.dtype, 1.0)
    near(ops.orthogonalize(g, steps=1), define(g, 1), g.dtype, 3.4445)
    cubic = (1.5, -0.5, 0.0)
    near(ops.orthogonalize(g, steps=12, coefficients=cubic), define(g, 12, cubic), g.dtype, 1.5 ** 12)
    each = [(3.4445, -4.7750, 2.0315)] * 3 + [(1.875, -1.25, 0.375)] * 2
    near(ops.orthogonalize(g, coefficients=each), define(g, 5, each), g.dtype)
    near(ops.orthogonalize(g, coefficients=[list(c) for c in each]), define(g, 5, each), g.dtype)


def test_result_in_place_batches_and_streams():
    g = matrices(6, 96, 200, torch.float32).reshape(2, 3, 96, 200)
    want = ops.orthogonalize(g)
    near(want, define(g), torch.float32)
    out = torch.empty_like(g)
    assert ops.orthogonalize(g, out=out) is not None and torch.equal(out, want)
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        again = [ops.orthogonalize(g) for _ in range(10)]
    st.synchronize()
    assert all(torch.equal(a, want) for a in again)
    ops.orthogonalize(g, out=g)
    assert torch.equal(g, want)
    assert ops.orthogonalize(torch.zeros(0, 4, 5, device="cuda")).shape == (0, 4, 5)
    assert ops.orthogonalize(torch.zeros(3, 0, 5, device="cuda")).shape == (3, 0, 5)


def test_a_call_can_be_captured():
    g = matrices(1, 150, 300, torch.float32)
    ops.orthogonalize(g)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.orthogonalize(g)
    g.mul_(torch.rand_like(g))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, ops.orthogonalize(g))


LISTS = [[(128, 128)] * 4 + [(172, 128)] * 2, [(1, 1), (7, 1), (1, 30), (5, 200)], [(256, 256)] * 4 + [(64, 256)] * 2, [(300, 700), (700, 300), (40, 50)],
         [(16, 16)] * 70, [(1024, 512), (128, 128), (130, 900), (20, 20)]]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("which", range(len(LISTS)))
@pytest.mark.parametrize("nesterov", [True, False])
def test_optimiser_steps(which, dtype, nesterov):
    dt = TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(which)
    ws = [(torch.randn(r, c, generator=g, device="cuda") / math.sqrt(c)).to(dt) for r, c in LISTS[which]]
    ms = [torch.zeros(r, c, device="cuda") for r, c in LISTS[which]]
    lr, mu, decay = 0.03, 0.9, 0.1
    for step in range(3):
        gs = [(torch.randn(r, c, generator=g, device="cuda") * 0.01).to(dt) for r, c in LISTS[which]]
        wants = []
        for w, gr, m in zip(ws, gs, ms):
            v = mu * m.double() + gr.double()
            u = gr.double() + mu * v if nesterov else v
            o = define(u)
            gain = lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
            wants.append((w.double() * (1 - lr * decay) - gain * o, v, gain * float(room(o, dt))))
        ops.muon_step(ws, gs, ms, lr, momentum=mu, nesterov=nesterov, weight_decay=decay)
        for w, m, (want, v, off) in zip(ws, ms, wants):
            assert (m.double() - v).abs().max() <= 2.0 ** -23 * (v.abs().max() + 1e-30)
            # the update's error, the result's rounding and three of single precision
            assert float((w.double() - want).norm()) <= off + (UNIT[dt] + 3 * 2.0 ** -24) * float(want.norm())


def test_a_step_writes_weights_and_momenta_only():
    ws, gs, ms = ([torch.randn(150, 90, device="cuda") for _ in range(3)] for _ in range(3))
    kept = [g.clone() for g in gs]
    version = ws[0]._version, ms[0]._version
    ops.muon_step(ws, gs, ms, 0.01)
    assert all(torch.equal(a, b) for a, b in zip(gs, kept))
    assert ws[0]._version > version[0] and ms[0]._version > version[1]
    ops.muon_step([], [], [], 0.01)


def test_refusals():
    g = torch.randn(4, 6, device="cuda")
    w, m = torch.randn(4, 6, device="cuda"), torch.zeros(4, 6, device="cuda")
    bad = [lambda: ops.orthogonalize(g.cpu()), lambda: ops.orthogonalize(g.double()), lambda: ops.orthogonalize(g.t()), lambda: ops.orthogonalize(g[0]),
           lambda: ops.orthogonalize(g, steps=-1), lambda: ops.orthogonalize(g, steps=17), lambda: ops.orthogonalize(g, coefficients=(1.0, 2.0)),
           lambda: ops.orthogonalize(g, coefficients=[(1.0, 2.0, 3.0)] * 4), lambda: ops.orthogonalize(g, coefficients=(50.0, 0.0, 0.0)),
           lambda: ops.orthogonalize(g, coefficients=(float("nan"), 0.0, 0.0)), lambda: ops.orthogonalize(g, eps=-1.0),
           lambda: ops.orthogonalize(g, out=torch.empty(6, 4, device="cuda")), lambda: ops.orthogonalize(g, out=torch.empty(4, 6, device="cuda").half()),
           lambda: ops.orthogonalize(g.clone().requires_grad_()),
           lambda: ops.muon_step([w], [g], [], 0.1), lambda: ops.muon_step([w], [g.half()], [m], 0.1), lambda: ops.muon_step([w], [g], [m.half()], 0.1),
           lambda: ops.muon_step([w], [g[:3]], [m], 0.1), lambda: ops.muon_step([w.clone().requires_grad_()], [g], [m], 0.1),
           lambda: ops.muon_step([w, w.half()], [g, g.half()], [m, m.clone()], 0.1), lambda: ops.muon_step([w[None]], [g[None]], [m[None]], 0.1),
           lambda: ops.muon_step([w.t()], [g.t().contiguous()], [m.t().contiguous()], 0.1)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        ops.orthogonalize(g, coefficients=3.0)
    with pytest.raises(TypeError):
        ops.orthogonalize(None)
