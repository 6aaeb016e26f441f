"""GPU: what the dense operators leave behind a bounded wait that has run out.  With ``F2C_NO_WAITS`` nothing is issued that a wait could be for,
and all run out (at once, or those of a product of matrices that one SM does not hold after their full limit): results are NaN, the device
status has the kernel's code, and the next ordinary call has the bits of the one before."""
import ctypes

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from f2cgt_b200 import _lib, ops  # noqa: E402
from f2cgt_b200._lib import check, lib  # noqa: E402

TAGS = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
COEFFICIENTS = (ctypes.c_float * 48)(*ops.NEWTON_SCHULZ * 16)
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def stream():
    return torch.cuda.current_stream().cuda_stream


def lost(out, code):
    assert ops.device_status() == code
    assert torch.isnan(out).all()
    assert ops.device_status() == 0


# a CTA a tile, parts of K over a cluster, pairs of CTAs
@pytest.mark.parametrize("out_type", TYPES)
@pytest.mark.parametrize("m,n,k", [(1000, 172, 256), (16, 4096, 4096), (4000, 700, 1600)])
@pytest.mark.parametrize("relu", [0, 1])
def test_8_bit_products(m, n, k, relu, out_type):
    g = torch.Generator(device="cuda").manual_seed(m)
    q, w = (torch.randint(-127, 128, (r, k), generator=g, dtype=torch.int8, device="cuda") for r in (m, n))
    s, ws = torch.rand(m, generator=g, device="cuda"), torch.rand(n, generator=g, device="cuda")
    ops.device_status()
    want = ops.int8_mm(q, s, w, ws, relu=bool(relu), out_dtype=out_type)
    out = torch.zeros(m, n, dtype=out_type, device="cuda")
    check(lib.f2c_int8_mm(q.data_ptr(), k, s.data_ptr(), w.data_ptr(), k, ws.data_ptr(), None, relu | _lib.NO_WAITS, out.data_ptr(), TAGS[out_type],
                          m, n, k, None, 0, stream()))
    lost(out, 4)
    assert torch.equal(ops.int8_mm(q, s, w, ws, relu=bool(relu), out_dtype=out_type), want)
    assert ops.device_status() == 0


# one launch; codes first (weights are asked for ahead), with a CTA a tile, parts of K and pairs
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,n,k,code", [(1024, 172, 256, 7), (20_000, 128, 256, 4), (16, 4096, 4096, 4), (4000, 700, 1600, 4)])
def test_8_bit_layers(m, n, k, code, dtype):
    g = torch.Generator(device="cuda").manual_seed(m)
    x = torch.randn(m, k, generator=g, device="cuda").to(dtype)
    w, ws = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8, device="cuda"), torch.rand(n, generator=g, device="cuda")
    ops.device_status()
    want = ops.int8_linear(x, w, ws)
    out = torch.zeros(m, n, dtype=dtype, device="cuda")
    need = lib.f2c_int8_linear_workspace(x.data_ptr(), k, k, None, 0, 0, TAGS[dtype], w.data_ptr(), k, m, n)
    space = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")
    check(lib.f2c_int8_linear(x.data_ptr(), k, k, None, 0, 0, TAGS[dtype], w.data_ptr(), k, ws.data_ptr(), None, _lib.NO_WAITS, out.data_ptr(), TAGS[dtype],
                              m, n, space.data_ptr() if need else None, need, stream()))
    lost(out, code)
    assert torch.equal(ops.int8_linear(x, w, ws), want)
    assert ops.device_status() == 0


# one CTA a matrix; a CTA a tile, parts of K, pairs of CTAs with half of the symmetric products
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("batch,rows,cols,code", [(3, 100, 128, 6), (2, 128, 200, 6), (1, 300, 400, 5), (1, 1031, 602, 5), (6, 520, 700, 5), (2, 1500, 1100, 5)])
def test_orthogonalised_matrices(batch, rows, cols, code, dtype):
    g = torch.randn(batch, rows, cols, generator=torch.Generator(device="cuda").manual_seed(rows), device="cuda").to(dtype)
    ops.device_status()
    want = ops.orthogonalize(g)
    out = torch.zeros_like(g)
    need = lib.f2c_orthogonalize_workspace(TAGS[dtype], batch, rows, cols)
    space = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")
    for steps in (1, 3) if code == 6 else (1,):
        out.zero_()
        check(lib.f2c_orthogonalize(g.data_ptr(), out.data_ptr(), TAGS[dtype], batch, rows, cols, COEFFICIENTS, steps | _lib.NO_WAITS, 1e-7,
                                    space.data_ptr() if need else None, need, stream()))
        lost(out, code)
    assert torch.equal(ops.orthogonalize(g), want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("rows,cols,code", [(100, 128, 6), (300, 400, 5)])
def test_weights_of_an_optimiser_step(rows, cols, code):
    """The momentum has moved; the weights are not to be used."""
    g, w = torch.randn(rows, cols, device="cuda"), torch.randn(rows, cols, device="cuda")
    momentum = torch.zeros_like(w)
    ops.device_status()
    one = (_lib.MuonMatrix * 1)(_lib.MuonMatrix(w.data_ptr(), g.data_ptr(), momentum.data_ptr(), rows, cols))
    need = lib.f2c_muon_workspace(one, 1, _lib.F32)
    space = torch.zeros(max(need, 1), dtype=torch.uint8, device="cuda")
    check(lib.f2c_muon_step(one, 1, _lib.F32, 0.02, 0.95, 1, 0.0, COEFFICIENTS, 1 | _lib.NO_WAITS, 1e-7, space.data_ptr() if need else None, need, stream()))
    lost(w, code)
    assert torch.equal(momentum, g)
