"""CPU: the 8-bit products and the orthogonalised updates refuse bad arguments before any CUDA call, and do nothing on nothing."""
import ctypes as C

import pytest

from f2cgt_b200 import _lib

lib = _lib.lib
INVALID, UNSUPPORTED, LIMIT = 1, 2, 4
AT = 0x10000  # an address that is never looked at


def quantize(x1=AT, ld1=8, k1=8, x2=0, ld2=0, k2=0, dtype=_lib.F32, m=4, codes=AT, ldq=16, scales=AT):
    return lib.f2c_int8_quantize(x1, ld1, k1, x2, ld2, k2, dtype, m, codes, ldq, scales, None)


def mm(codes=AT, ldq=16, scales=AT, w=AT, ldw=16, ws=AT, bias=0, relu=0, out=AT, dtype=_lib.F32, m=4, n=4, k=16, work=0, size=0):
    return lib.f2c_int8_mm(codes, ldq, scales, w, ldw, ws, bias, relu, out, dtype, m, n, k, work, size, None)


def linear(x1=AT, ld1=16, k1=16, dtype=_lib.F32, w=AT, ldw=16, ws=AT, out=AT, out_dtype=_lib.F32, m=4, n=4, work=0, size=0):
    return lib.f2c_int8_linear(x1, ld1, k1, 0, 0, 0, dtype, w, ldw, ws, 0, 0, out, out_dtype, m, n, work, size, None)


@pytest.mark.parametrize("call,status", [
    (lambda: quantize(dtype=_lib.F64), UNSUPPORTED), (lambda: quantize(m=-1), INVALID), (lambda: quantize(k1=131072, ld1=131072), LIMIT),
    (lambda: quantize(ld1=7), INVALID), (lambda: quantize(x1=0), INVALID), (lambda: quantize(k2=4, ld2=4), INVALID), (lambda: quantize(ldq=7), INVALID),
    (lambda: quantize(scales=0), INVALID), (lambda: quantize(m=0, x1=0, codes=0, scales=0), 0),
    (lambda: mm(dtype=_lib.I8), UNSUPPORTED), (lambda: mm(k=131072, ldq=131072, ldw=131072), LIMIT), (lambda: mm(ldq=15), INVALID), (lambda: mm(ldw=15), INVALID),
    (lambda: mm(n=-1), INVALID), (lambda: mm(out=0), INVALID), (lambda: mm(w=0), INVALID), (lambda: mm(codes=AT + 1), INVALID),
    (lambda: mm(codes=AT + 1, work=AT + 8, size=1 << 20), INVALID), (lambda: mm(n=(1 << 21) + 1), LIMIT), (lambda: mm(m=0, codes=0, out=0), 0), (lambda: mm(n=0), 0),
    (lambda: linear(dtype=_lib.I8), UNSUPPORTED), (lambda: linear(out_dtype=_lib.I32), UNSUPPORTED), (lambda: linear(x1=0), INVALID), (lambda: linear(ldw=8), INVALID),
    (lambda: linear(m=100000), INVALID), (lambda: linear(m=0), 0), (lambda: linear(n=0), 0)])
def test_8_bit_products(call, status):
    assert call() == status
    assert status == 0 or b"int8" in lib.f2c_last_error()


def test_workspaces_of_the_8_bit_products():
    assert lib.f2c_int8_mm_workspace(AT, 16, AT, 16, 100, 50, 16) == 0
    assert lib.f2c_int8_mm_workspace(AT, 17, AT, 16, 100, 50, 16) == 1792  # 1600 bytes of codes, to the next 256
    assert lib.f2c_int8_mm_workspace(AT + 4, 16, AT, 19, 100, 50, 19) == 3328 + 1792  # and 32 a row of both
    assert lib.f2c_int8_linear_workspace(AT, 256, 256, None, 0, 0, _lib.F32, AT, 256, 1, 172) == 0
    assert lib.f2c_int8_linear_workspace(AT, 256, 256, None, 0, 0, _lib.F32, AT, 256, 100000, 172) == 400128 + 25600000
    assert lib.f2c_int8_linear_workspace(AT, 256, 256, None, 0, 0, _lib.F32, AT, 256, 0, 172) == 0
    # rows that cannot be encoded on the way, by their start, their stride or their length, need a place for their codes
    codes = 4096 + 1024 * 256
    assert lib.f2c_int8_linear_workspace(AT, 256, 256, None, 0, 0, _lib.F32, AT, 256, 1024, 172) == 0
    assert lib.f2c_int8_linear_workspace(AT + 4, 256, 256, None, 0, 0, _lib.F32, AT, 256, 1024, 172) == codes
    assert lib.f2c_int8_linear_workspace(AT, 257, 256, None, 0, 0, _lib.F32, AT, 256, 1024, 172) == codes
    assert lib.f2c_int8_linear_workspace(AT, 128, 128, AT + 8, 128, 128, _lib.F32, AT, 256, 1024, 172) == codes
    assert lib.f2c_int8_linear_workspace(AT, 254, 254, None, 0, 0, _lib.F32, AT, 256, 1024, 172) == codes


COEFFICIENTS = (C.c_float * 15)(*[3.4445, -4.7750, 2.0315] * 5)


def orthogonalize(dtype=_lib.F32, batch=1, rows=300, cols=300, co=COEFFICIENTS, steps=5, eps=1e-7, work=AT, size=1 << 40, g=AT, out=AT):
    return lib.f2c_orthogonalize(g, out, dtype, batch, rows, cols, co, steps, eps, work, size, None)


def step(list_, dtype=_lib.F32, work=AT, size=1 << 40, steps=5, co=COEFFICIENTS):
    return lib.f2c_muon_step((_lib.MuonMatrix * max(1, len(list_)))(*list_), len(list_), dtype, 0.02, 0.95, 1, 0.0, co, steps, 1e-7, work, size, None)


def grow(*co):
    return (C.c_float * 15)(*co * 5)


@pytest.mark.parametrize("call,status", [
    (lambda: orthogonalize(dtype=_lib.F64), UNSUPPORTED), (lambda: orthogonalize(batch=-1), INVALID), (lambda: orthogonalize(batch=65536), LIMIT),
    (lambda: orthogonalize(rows=65537), LIMIT), (lambda: orthogonalize(steps=17), LIMIT), (lambda: orthogonalize(steps=-1), LIMIT),
    (lambda: orthogonalize(co=None), INVALID), (lambda: orthogonalize(eps=-1.0), INVALID), (lambda: orthogonalize(eps=float("nan")), INVALID),
    (lambda: orthogonalize(co=grow(9.0, 0.0, 0.0)), LIMIT), (lambda: orthogonalize(co=grow(1.0, 70.0, 0.0)), LIMIT),
    (lambda: orthogonalize(co=grow(float("nan"), 0.0, 0.0)), LIMIT), (lambda: orthogonalize(co=grow(2.0, 0.0, 0.0)), LIMIT),
    (lambda: orthogonalize(g=0), INVALID), (lambda: orthogonalize(work=0), INVALID), (lambda: orthogonalize(work=AT + 16), INVALID), (lambda: orthogonalize(size=100), INVALID),
    (lambda: orthogonalize(batch=0, g=0), 0), (lambda: orthogonalize(rows=0, work=0), 0),
    (lambda: step([(AT, AT, AT, 300, 300)], dtype=_lib.I8), UNSUPPORTED), (lambda: step([(AT, AT, 0, 300, 300)]), INVALID),
    (lambda: step([(AT, AT, AT, 300, -1)]), INVALID), (lambda: step([(AT, AT, AT, 300, 300)], work=0), INVALID), (lambda: step([(AT, AT, AT, 300, 300)], size=10), INVALID),
    (lambda: step([]), 0), (lambda: step([(0, 0, 0, 0, 300)]), 0)])
def test_orthogonalised_updates(call, status):
    assert call() == status
    assert status == 0 or b"orthogonalize" in lib.f2c_last_error() or b"muon_step" in lib.f2c_last_error()


def test_workspaces_of_the_updates():
    assert lib.f2c_orthogonalize_workspace(_lib.F32, 7, 128, 256) == 0 and lib.f2c_orthogonalize_workspace(_lib.F32, 7, 256, 128) == 0
    one, two = (lib.f2c_orthogonalize_workspace(_lib.F32, b, 300, 400) for b in (1, 2))
    assert one >= 4 * 2 * 300 * 400 and two > one
    small = _lib.MuonMatrix(AT, AT, AT, 64, 64)
    large = _lib.MuonMatrix(AT, AT, AT, 300, 400)
    assert lib.f2c_muon_workspace((_lib.MuonMatrix * 2)(small, small), 2, _lib.F32) == 0
    assert lib.f2c_muon_workspace((_lib.MuonMatrix * 3)(large, small, large), 3, _lib.F32) == two


A, B, G, M = (0x1000000 * i for i in range(1, 5))  # 300 x 300 float32 are 360,000 bytes


@pytest.mark.parametrize("list_", [
    [(A, G, M, 300, 300), (A, G + 400_000, M + 400_000, 300, 300)], [(A, G, M, 300, 300), (B, G, M, 300, 300)], [(A, A, M, 300, 300)], [(A, G, A, 300, 300)],
    [(A, G, G, 300, 300)], [(A, G, M, 300, 300), (A + 359_996, G, M + 400_000, 300, 300)], [(A, G, M, 300, 300), (B, A + 4, M + 400_000, 20, 20)],
    [(A, G, M, 1, 1), (B, G, M, 1, 1)], [(A, G, M, 300, 300), (B, M + 100, M + 400_000, 20, 20)], [(B, G, M, 20, 20), (A, G, B - 16, 20, 20)]])
def test_matrices_of_a_step_that_share_memory_are_refused(list_):
    assert step(list_) == INVALID and b"shares memory" in lib.f2c_last_error()


@pytest.mark.parametrize("list_", [
    [(A, G, M, 300, 300), (A + 360_000, G + 360_000, M + 360_000, 300, 300)], [(A, G, M, 300, 300), (B, G, M + 360_000, 300, 300)],
    [(A, G, M, 300, 300), (B, G + 100, M + 360_000, 20, 20)], [(A, A, A, 0, 300), (B, B, B, 300, 0)]])
def test_neighbours_and_shared_gradients_are_not(list_):
    assert step(list_, work=0) == (0 if 0 in list_[0] else INVALID)
    assert 0 in list_[0] or b"workspace" in lib.f2c_last_error()


@pytest.mark.parametrize("rows,cols", [(30, 50), (300, 300)])
@pytest.mark.parametrize("dtype,item", [(_lib.F32, 4), (_lib.BF16, 2)])
def test_results_that_share_a_part_of_the_matrices_are_refused(rows, cols, dtype, item):
    size = 2 * rows * cols * item
    for at in (item, size // 2, size - item):
        for g, out in ((A, A + at), (A + at, A)):
            assert orthogonalize(dtype=dtype, batch=2, rows=rows, cols=cols, g=g, out=out) == INVALID
            assert b"memory" in lib.f2c_last_error()
    if rows == 300:  # (goes on to what is refused next)
        for g, out in ((A, A), (A, A + size), (A + size, A)):
            assert orthogonalize(dtype=dtype, batch=2, rows=rows, cols=cols, g=g, out=out, work=0) == INVALID
            assert b"workspace" in lib.f2c_last_error()
