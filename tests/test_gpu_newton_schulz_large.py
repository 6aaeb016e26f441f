"""GPU: Newton-Schulz steps by the kernels of larger matrices - pairs of CTAs, half of the symmetric products, several rounds of tiles, stages of 128
elements - and of matrices at odd addresses, against the formula in 64 bits; and float16, held in pairs of half precision throughout.

What may be off, as Frobenius norms: float32 and bfloat16 as test_gpu_newton_schulz.py derives it.  Float16 is float32's (its operands are the
same pairs, u = 2^-22) and the result's rounding: 2^-11 of it, or half of the smallest float16, 2^-25, of each element."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from f2cgt_b200 import ops  # noqa: E402
from test_gpu_newton_schulz import SIZES, TYPES, UNIT, define, matrices, room  # noqa: E402


def bound(want, dtype, gain=485.0):
    if dtype != torch.float16:
        return room(want, dtype, gain)
    return room(want, torch.float32, gain) + 2.0 ** -11 * want.norm(dim=(-2, -1)) + 2.0 ** -25 * math.sqrt(want.shape[-1] * want.shape[-2])


def near(got, want, dtype, gain=485.0):
    off = (got.double() - want).norm(dim=(-2, -1))
    assert (off <= bound(want, dtype, gain)).all(), (off / bound(want, dtype, gain)).max()


@pytest.mark.parametrize("rows,cols", SIZES)
def test_float16_keeps_its_bits(rows, cols):
    g = matrices(2 if rows * cols < 500_000 else 1, rows, cols, torch.float16)
    near(ops.orthogonalize(g), define(g), torch.float16)


@pytest.mark.parametrize("rows,cols", [(128, 128), (100, 256), (400, 600), (700, 200), (200, 2000)])
@pytest.mark.parametrize("kind", ["decay", "low"])
def test_float16_of_few_large_singular_values(rows, cols, kind):
    g = matrices(3, rows, cols, torch.float16, kind)
    near(ops.orthogonalize(g), define(g), torch.float16)


# one round of pairs; symmetric products by halves; stages of 128 elements (float32, float16 over 1024); several rounds; and tall ones
LARGE = [(1, 1300, 1100), (1, 1100, 1500), (6, 520, 700), (6, 700, 520), (12, 516, 700), (12, 700, 516), (2, 1500, 1100), (12, 1024, 1024), (1, 2050, 2300)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", LARGE)
def test_large_matrices(batch, rows, cols, dtype):
    g = matrices(batch, rows, cols, TYPES[dtype])
    out = ops.orthogonalize(g)
    near(out, define(g), g.dtype)
    assert all(torch.equal(ops.orthogonalize(g), out) for _ in range(5))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(6, 520, 700), (12, 700, 516)])
@pytest.mark.parametrize("kind", ["decay", "low"])
def test_large_matrices_of_few_large_singular_values(batch, rows, cols, kind, dtype):
    g = matrices(batch, rows, cols, TYPES[dtype], kind)
    near(ops.orthogonalize(g), define(g), g.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(6, 520, 700), (12, 700, 516), (2, 1500, 1100)])
def test_zero_and_matrices_that_are_not_finite_among_large_ones(batch, rows, cols, dtype):
    g = matrices(batch, rows, cols, TYPES[dtype])
    want = define(g)
    g[1, 7, 3] = float("nan")
    if batch > 4:
        g[2] = 0
        g[4, rows - 1, cols - 1] = float("inf")
    out = ops.orthogonalize(g)
    rest = [i for i in range(batch) if i not in ((1,) if batch <= 4 else (1, 2, 4))]
    assert torch.isnan(out[1]).all() and (batch <= 4 or (torch.isnan(out[4]).all() and (out[2] == 0).all()))
    near(out[rest], want[rest], g.dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,rows,cols", [(3, 64, 96), (3, 33, 41), (2, 300, 400), (2, 301, 203), (6, 520, 700)])
@pytest.mark.parametrize("lead", [1, 2, 3])
def test_matrices_at_odd_addresses(batch, rows, cols, lead, dtype):
    g = matrices(batch, rows, cols, TYPES[dtype])
    size = g.numel()
    room_in, room_out = (torch.full((size + 8,), 7.0, dtype=g.dtype, device="cuda") for _ in range(2))
    at, out = room_in[lead:lead + size].view(g.shape), room_out[4 - lead:4 - lead + size].view(g.shape)
    at.copy_(g)
    ops.orthogonalize(at, out=out)
    near(out, define(g), g.dtype)
    assert torch.equal(at, g)
    for t, first in ((room_in, lead), (room_out, 4 - lead)):
        assert (t[:first] == 7).all() and (t[first + size:] == 7).all()


def step(shapes, dtype, where, nesterov=True):
    """One step of ops.muon_step on tensors that ``where`` places, against the formula."""
    g = torch.Generator(device="cuda").manual_seed(len(shapes))
    ws = where([(torch.randn(s, generator=g, device="cuda") / math.sqrt(s[1])).to(dtype) for s in shapes])
    gs = where([(torch.randn(s, generator=g, device="cuda") * 0.01).to(dtype) for s in shapes])
    ms = where([torch.randn(s, generator=g, device="cuda") * 0.02 for s in shapes])
    lr, mu, decay = 0.03, 0.9, 0.1
    wants = []
    for w, gr, m in zip(ws, gs, ms):
        v = mu * m.double() + gr.double()
        o = define(gr.double() + mu * v if nesterov else v)
        gain = lr * math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        wants.append((w.double() * (1 - lr * decay) - gain * o, v, gain * float(bound(o, dtype))))
    ops.muon_step(ws, gs, ms, lr, momentum=mu, nesterov=nesterov, weight_decay=decay)
    for w, m, (want, v, off) in zip(ws, ms, wants):
        assert (m.double() - v).abs().max() <= 2.0 ** -23 * (v.abs().max() + 1e-30)
        tiny = 2.0 ** -25 * math.sqrt(w.numel()) if dtype == torch.float16 else 0.0
        assert float((w.double() - want).norm()) <= off + (UNIT[dtype] + 3 * 2.0 ** -24) * float(want.norm()) + tiny


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", [[(1100, 1300)], [(700, 516)] * 12 + [(128, 128)], [(520, 700)] * 6 + [(1500, 1100)] * 2])
def test_optimiser_steps_of_large_matrices(shapes, dtype):
    step(shapes, TYPES[dtype], lambda tensors: tensors)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shapes", [[(33, 41), (64, 64), (5, 3)], [(301, 203), (300, 400), (301, 203)]])
def test_optimiser_steps_in_flat_buffers(shapes, dtype):
    """Views of one buffer behind one another, as the gradients of the data-parallel trainer are: at addresses of every kind."""
    def flat(tensors):
        buffer = torch.cat([tensors[0].new_zeros(1)] + [t.flatten() for t in tensors])
        ends = [1]
        for t in tensors:
            ends.append(ends[-1] + t.numel())
        return [buffer[a:b].view(t.shape) for t, a, b in zip(tensors, ends, ends[1:])]

    step(shapes, TYPES[dtype], flat)
