"""CPU: layer norm, 8-bit activations and learned rows refuse bad arguments before any CUDA call, and do nothing on nothing."""
import pytest

from f2cgt_b200 import _lib

lib = _lib.lib
OK, INVALID, UNSUPPORTED, LIMIT = 0, 1, 2, 4
AT = 0x10000  # an address that is never looked at


def encode(x=AT, ldx=40, dtype=_lib.F32, m=4, d=40, codes=AT, ldq=48, scales=AT):
    return lib.f2c_checkpoint_int8(x, ldx, dtype, m, d, codes, ldq, scales, None)


def values(codes=AT, ldq=48, scales=AT, m=4, d=40, out=AT, ldo=40, dtype=_lib.F32):
    return lib.f2c_checkpoint_values(codes, ldq, scales, m, d, out, ldo, dtype, None)


def norm(x=AT, ldx=40, dtype=_lib.F32, m=4, d=40, eps=1e-5, y=AT, mean=0, rstd=0, active=0, codes=0, ldq=0, scales=0):
    return lib.f2c_layer_norm(x, ldx, dtype, m, d, 0, 0, eps, 0, y, mean, rstd, active, codes, ldq, scales, None)


def backward(dy=AT, ldy=40, dtype=_lib.F32, x=AT, ldx=40, codes=0, ldq=0, scales=0, mean=AT, rstd=AT, m=4, d=40, dx=AT, work=AT, size=1 << 30):
    return lib.f2c_layer_norm_backward(dy, ldy, dtype, x, ldx, codes, ldq, scales, mean, rstd, 0, 0, m, d, dx, AT, AT, work, size, None)


@pytest.mark.parametrize("call,status", [
    (lambda: encode(dtype=_lib.F64), UNSUPPORTED), (lambda: encode(m=-1), INVALID), (lambda: encode(d=(1 << 20) + 1, ldx=1 << 21, ldq=1 << 21), LIMIT), (lambda: encode(ldx=39), INVALID),
    (lambda: encode(x=0), INVALID), (lambda: encode(codes=0), INVALID), (lambda: encode(codes=AT + 8), INVALID), (lambda: encode(ldq=40), INVALID), (lambda: encode(ldq=32), INVALID),
    (lambda: encode(scales=0), INVALID), (lambda: encode(scales=AT + 4), INVALID), (lambda: encode(m=1 << 30, d=1 << 10, ldx=1 << 10, ldq=1 << 10), LIMIT),
    (lambda: encode(m=0, x=0, codes=0, scales=0), OK), (lambda: encode(d=0, x=0, codes=0, scales=0), OK),
    (lambda: values(dtype=_lib.I8), UNSUPPORTED), (lambda: values(out=0), INVALID), (lambda: values(ldo=39), INVALID), (lambda: values(codes=AT + 4), INVALID), (lambda: values(m=0, out=0), OK),
    (lambda: norm(dtype=_lib.I32), UNSUPPORTED), (lambda: norm(eps=-1e-9), INVALID), (lambda: norm(eps=float("nan")), INVALID), (lambda: norm(mean=AT), INVALID), (lambda: norm(x=0), INVALID),
    (lambda: norm(y=0), INVALID), (lambda: norm(ldx=39), INVALID), (lambda: norm(codes=AT), INVALID), (lambda: norm(codes=AT, ldq=40, scales=AT), INVALID),
    (lambda: norm(m=1 << 31), LIMIT), (lambda: norm(m=0, x=0, y=0), OK), (lambda: norm(d=0, x=0, y=0), OK),
    (lambda: backward(dtype=_lib.U8), UNSUPPORTED), (lambda: backward(x=0), INVALID), (lambda: backward(codes=AT, ldq=48, scales=AT), INVALID), (lambda: backward(dy=0), INVALID),
    (lambda: backward(mean=0), INVALID), (lambda: backward(rstd=0), INVALID), (lambda: backward(dx=0), INVALID), (lambda: backward(ldy=39), INVALID), (lambda: backward(ldx=39), INVALID),
    (lambda: backward(work=0), INVALID), (lambda: backward(work=AT + 16), INVALID), (lambda: backward(size=100), INVALID), (lambda: backward(d=0), OK)])
def test_norms_and_8_bit_activations(call, status):
    assert call() == status
    assert status == OK or b"checkpoint" in lib.f2c_last_error() or b"layer_norm" in lib.f2c_last_error()


def test_workspaces_of_the_norms_gradient():
    assert lib.f2c_layer_norm_backward_workspace(0, 128) == 0 and lib.f2c_layer_norm_backward_workspace(10, 0) == 0
    assert lib.f2c_layer_norm_backward_workspace(8, 128) == 1024  # one CTA's two sums of 128 columns
    assert lib.f2c_layer_norm_backward_workspace(1 << 20, 128) >= 148 * 1024


def lookup(table=AT, ld=8, dtype=_lib.F32, rows=10, d=8, ids=AT, index=_lib.I64, m=4, out=AT):
    return lib.f2c_embedding(table, ld, dtype, rows, d, ids, index, m, 1.0, out, None)


def rows_gradient(dy=AT, ldy=8, dtype=_lib.F32, ids=AT, index=_lib.I64, m=4, rows=10, d=8, grad=AT, looked_up=AT, count=AT, work=AT, size=1 << 40):
    return lib.f2c_embedding_backward(dy, ldy, dtype, ids, index, m, rows, d, 1.0, grad, looked_up, count, work, size, None)


@pytest.mark.parametrize("call,status", [
    (lambda: lookup(dtype=_lib.F64), UNSUPPORTED), (lambda: lookup(index=_lib.I16), UNSUPPORTED), (lambda: lookup(m=-1), INVALID), (lambda: lookup(rows=1 << 31), LIMIT),
    (lambda: lookup(m=(1 << 30) + 1), LIMIT), (lambda: lookup(m=1 << 30, d=1 << 12, ld=1 << 12), LIMIT), (lambda: lookup(d=(1 << 20) + 1, ld=1 << 21), LIMIT), (lambda: lookup(ld=7), INVALID), (lambda: lookup(table=0), INVALID),
    (lambda: lookup(ids=0), INVALID), (lambda: lookup(out=0), INVALID), (lambda: lookup(m=0, ids=0, out=0), OK), (lambda: lookup(d=0, out=0), OK),
    (lambda: rows_gradient(dtype=_lib.I8), UNSUPPORTED), (lambda: rows_gradient(index=_lib.U8), UNSUPPORTED), (lambda: rows_gradient(d=-1), INVALID), (lambda: rows_gradient(dy=0), INVALID),
    (lambda: rows_gradient(ids=0), INVALID), (lambda: rows_gradient(grad=0), INVALID), (lambda: rows_gradient(looked_up=0), INVALID), (lambda: rows_gradient(ldy=7), INVALID),
    (lambda: rows_gradient(m=5000, work=0), INVALID), (lambda: rows_gradient(m=5000, work=AT + 8), INVALID), (lambda: rows_gradient(m=5000, size=1000), INVALID),
    (lambda: rows_gradient(count=0, looked_up=0, rows=1 << 25, d=1 << 20, ldy=1 << 20, m=1), LIMIT), (lambda: rows_gradient(count=0, grad=0), INVALID),
    (lambda: rows_gradient(count=0, rows=0, m=0, dy=0, ids=0, work=0, grad=0), OK)])
def test_learned_rows(call, status):
    assert call() == status
    assert status == OK or b"embedding" in lib.f2c_last_error()


def test_workspaces_of_learned_rows():
    few, many, large = (lib.f2c_embedding_backward_workspace(m, rows, 128) for m, rows in ((1025, 1000), (100_000, 1000), (100_000, 1 << 30)))
    assert 0 < few < many < large and lib.f2c_embedding_backward_workspace(0, 10, 10) == lib.f2c_embedding_backward_workspace(1024, 1000, 128) == 0
    assert many < 100_000 * 128 * 4  # less than the rows themselves


def weights(dy=AT, ldy=8, dtype=_lib.F32, codes=AT, ldq=48, scales=AT, m=4, n=8, k=40, dw=AT, db=AT, flags=0, work=AT, size=1 << 40):
    return lib.f2c_checkpoint_weight_grad(dy, ldy, dtype, codes, ldq, scales, m, n, k, dw, db, flags, work, size, None)


@pytest.mark.parametrize("call,status", [
    (lambda: weights(dtype=_lib.F64), UNSUPPORTED), (lambda: weights(n=-1), INVALID), (lambda: weights(m=1 << 31), LIMIT), (lambda: weights(n=(1 << 17) + 1, ldy=1 << 18), LIMIT),
    (lambda: weights(k=(1 << 17) + 1, ldq=1 << 18), LIMIT), (lambda: weights(flags=1), INVALID), (lambda: weights(codes=AT + 8), INVALID), (lambda: weights(ldq=40), INVALID), (lambda: weights(scales=0), INVALID),
    (lambda: weights(dy=0), INVALID), (lambda: weights(dw=0), INVALID), (lambda: weights(db=0), INVALID), (lambda: weights(ldy=7), INVALID), (lambda: weights(k=0), INVALID),
    (lambda: weights(m=10000, work=0), INVALID), (lambda: weights(m=10000, work=AT + 64), INVALID), (lambda: weights(m=10000, size=1 << 16), INVALID), (lambda: weights(n=0, dw=0, db=0), OK)])
def test_weight_gradients(call, status):
    assert call() == status
    assert status == OK or b"checkpoint_weight_grad" in lib.f2c_last_error()


def test_workspaces_of_weight_gradients():
    size = lib.f2c_checkpoint_weight_grad_workspace
    assert size(AT, 8, _lib.F32, 0, 8, 8) == size(AT, 8, _lib.F32, 8, 0, 8) == size(AT, 128, _lib.F32, 32, 128, 128) == 0  # one part
    assert size(AT, 128, _lib.F32, 59_000, 128, 128) % (65536 + 512) == 0 and size(AT, 2048, _lib.BF16, 16_384, 2048, 4096) == 0
    assert size(AT, 4096, _lib.BF16, 16_384, 4096, 4096) == 68 * 2 * 131_072  # 512 tiles: three rounds of 148 SMs, and halves of the other 68
    # rows that do not start on 16 bytes are copied
    assert size(AT + 4, 128, _lib.F32, 32, 128, 128) == 32 * 512 and size(AT, 41, _lib.BF16, 100, 41, 128) >= 100 * 96 and size(AT, 41, _lib.F16, 1, 41, 16) == 0


def test_relu_of_bits_keeps_infinities_where_it_is_open():
    import torch
    from f2cgt_b200 import sage
    x = torch.tensor([-1.0, 2.0, 0.0, 3.0], requires_grad=True)
    y = sage._ReluBits.apply(x)
    y.backward(torch.tensor([float("inf"), float("inf"), float("nan"), -2.0]))
    assert y.tolist() == [0.0, 2.0, 0.0, 3.0] and x.grad.tolist() == [0.0, float("inf"), 0.0, -2.0]
