"""The gradient of a linear layer whose input was kept in 8 bits, against sums in 64 bits of the values that the codes stand for."""
import ctypes as C

import pytest
import torch

import learn_reference as R

pytestmark = pytest.mark.gpu


def ops():
    from f2cgt_b200 import ops
    return ops


def matrix(m, d, dtype, seed=0, pad=0, start=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(m, d + pad + start, generator=g, device="cuda").to(dtype)[:, start:start + d]


def check(dy, c):
    m, n = dy.shape
    x, d = R.decode(c.codes, c.scales), dy.double()
    step = c.scales[:, :, 0].double().repeat_interleave(128, 1)[:, :x.shape[1]]
    low = x - step * c.codes.double()
    dw, db = ops().checkpoint_weight_grad(dy, c)
    assert dw.dtype is db.dtype is dy.dtype and dw.shape == (n, x.shape[1]) and db.shape == (n,)
    coded, lows = d.abs().t() @ (x - low).abs(), d.abs().t() @ low.abs()
    # a product of 16 rows leaves at most 2^-23 of the sums' and the products' sizes, an accumulator takes three for every 16 of 256 rows (float32), or two for every
    # 16 of all rows; dy times the step is rounded to single precision (and to 16 bits; with bfloat16 it is x that is); every 256 rows and every part of the
    # rows add a rounding
    f32 = dy.dtype is torch.float32
    tensor = 48 * 2.0 ** -23 if f32 else (m / 8 + 2) * 2.0 ** -23 + 2.0 ** -17
    links = m / 128 + 160
    R.near(dw, d.t() @ x, (tensor + (links + 2) * R.U) * (coded + lows) + (m / 32 + 24 + links) * R.U * lows, dy.dtype)
    R.near(db, d.sum(0), (m / 32 + 24 + 160) * R.U * d.abs().sum(0), dy.dtype)
    return dw, db


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 128, 128), (5, 3, 200), (31, 130, 16), (32, 128, 128), (33, 127, 129), (257, 64, 300), (1000, 172, 128), (1024, 172, 256), (4000, 41, 602),
                                   (9000, 128, 128), (8200, 1, 128), (20000, 256, 256), (300, 1500, 1100), (2500, 2100, 1700), (2001, 1700, 1665), (2100, 3350, 1700)])
def test_gradients(m, n, k, dtype):
    x = matrix(m, k, dtype, seed=1).relu()
    x[:, ::3] -= 0.5  # groups whose lowest value is not zero
    check(matrix(m, n, dtype, seed=2), ops().checkpoint_int8(x))


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("n,pad,start", [(128, 1, 0), (128, 0, 1), (100, 4, 4), (126, 2, 2), (9, 8, 8), (172, 3, 1)])
def test_rows_at_odd_places(n, pad, start, dtype):
    check(matrix(700, n, dtype, pad=pad, start=start), ops().checkpoint_int8(matrix(700, 140, dtype, seed=3)))


def test_every_other_row_and_wider_rows_of_codes():
    c = ops().checkpoint_int8(matrix(900, 200, torch.float32))
    part = type(c)(c.codes[::2], c.scales[::2].contiguous())
    check(matrix(450, 60, torch.float32, seed=4), part)
    room = torch.zeros(450, 512, dtype=torch.uint8, device="cuda")
    room[:, :200] = c.codes[::2]
    room[:, 200:] = 255  # not the operator's
    a, b = ops().checkpoint_weight_grad(matrix(450, 60, torch.float32, seed=4), part), ops().checkpoint_weight_grad(matrix(450, 60, torch.float32, seed=4), type(c)(room[:, :200], part.scales))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,n,k", [(100, 128, 128), (1500, 200, 256), (777, 77, 130), (520, 1300, 1300)])
def test_small_whole_numbers_are_exact(m, n, k, dtype):
    """Steps of one, a lowest value of zero or minus two and dy of -1, 0 and 1: every product and sum is a whole number below 2^24."""
    g = torch.Generator(device="cuda")
    g.manual_seed(8)
    codes = torch.randint(0, 256, (m, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.uint8)[:, :k]
    scales = torch.ones(m, (k + 127) // 128, 2, device="cuda")
    scales[:, :, 1] = -2.0 * torch.randint(0, 2, scales.shape[:2], generator=g, device="cuda")
    dy = torch.randint(-1, 2, (m, n), generator=g, device="cuda").to(dtype)
    want = dy.double().t() @ R.decode(codes, scales)
    dw, db = ops().checkpoint_weight_grad(dy, ops().Int8Checkpoint(codes, scales))
    assert torch.equal(dw, want.to(dtype)) and torch.equal(db, dy.double().sum(0).to(dtype))


def test_single_precision_is_kept():
    """Products that need all 24 bits, of one row.  Rounded or cut are the product of dy and the step (2^-24 of it), what its three parts leave (2^-27), the sum of
    the two small parts' products (2^-23 of it, 2^-31 of all), and that sum plus the large part's product, which is cut off: less than a unit of the last of
    24 bits, 2^-23."""
    x, dy = matrix(1, 256, torch.float32), matrix(1, 300, torch.float32, seed=2)
    c = ops().checkpoint_int8(x)
    c.scales[:, :, 1] = 0
    want = dy.double().t() @ R.decode(c.codes, c.scales)
    dw, _ = ops().checkpoint_weight_grad(dy, c)
    assert ((dw.double() - want).abs() <= want.abs() * (2.0 ** -24 + 2.0 ** -23 + 2.0 ** -26)).all()


def test_rows_in_large_numbers():
    """More rows than a thousand accumulations would keep to single precision: sums are taken out on the way.  Errors add up like roundings that go
    all one way, three of 2^-23 for every 16 of 256 rows where sums are cut, of the sizes; those of one sign make the most of it."""
    m = 300_000
    x = matrix(m, 128, torch.float32).abs()
    dy = torch.ones(m, 3, device="cuda")
    c = ops().checkpoint_int8(x)
    want = R.decode(c.codes, c.scales).sum(0)
    dw, db = ops().checkpoint_weight_grad(dy, c)
    assert ((dw.double() - want).abs() <= 48 * 2.0 ** -23 * want).all() and torch.equal(db, torch.full((3,), float(m), device="cuda"))


def test_numbers_that_are_none_stay_where_they_are():
    x, dy = matrix(400, 300, torch.float32), matrix(400, 20, torch.float32, seed=2)
    x[17, 200], dy[5, 3] = float("inf"), float("nan")
    dw, db = ops().checkpoint_weight_grad(dy, ops().checkpoint_int8(x))
    want = torch.zeros(20, 300, dtype=torch.bool, device="cuda")
    want[:, 128:256] = want[3] = True
    assert torch.equal(torch.isnan(dw), want) and torch.isnan(db).tolist() == [i == 3 for i in range(20)]


def test_nothing():
    o = ops()
    dw, db = o.checkpoint_weight_grad(torch.empty(0, 7, device="cuda"), o.checkpoint_int8(torch.empty(0, 33, device="cuda")))
    assert dw.shape == (7, 33) and not dw.any() and not db.any()
    dw, db = o.checkpoint_weight_grad(torch.empty(9, 0, device="cuda"), o.checkpoint_int8(matrix(9, 33, torch.float32)))
    assert dw.shape == (0, 33) and db.shape == (0,)


def test_against_differences():
    """A layer is linear in its weight: the difference of sum(dy * (x W^T)) along a direction t is <dW, t>."""
    m, n, k = 300, 20, 50
    c, dy, t = ops().checkpoint_int8(matrix(m, k, torch.float32)), matrix(m, n, torch.float32, seed=2), matrix(n, k, torch.float32, seed=3).double()
    x = ops().checkpoint_values(c).double()
    w = matrix(n, k, torch.float32, seed=4).double()
    loss = [float((dy.double() * (x @ (w + e * t).t())).sum()) for e in (1.0, -1.0)]
    dw, _ = ops().checkpoint_weight_grad(dy, c)
    assert abs((loss[0] - loss[1]) / 2 - float((dw.double() * t).sum())) <= 2.0 ** -18 * float(((dy.double().abs().t() @ x.abs()) * t.abs()).sum())


def test_the_same_bits_every_time_in_a_graph_and_beside_another():
    x, dy = matrix(5000, 256, torch.float32), matrix(5000, 172, torch.float32, seed=2)
    c = ops().checkpoint_int8(x)
    first = ops().checkpoint_weight_grad(dy, c)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = [ops().checkpoint_weight_grad(dy, c) for _ in range(3)]
    here = [ops().checkpoint_weight_grad(dy, c) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    for got in beside + here:
        assert torch.equal(got[0], first[0]) and torch.equal(got[1], first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops().checkpoint_weight_grad(dy, ops().checkpoint_int8(x))
    x.copy_(matrix(5000, 256, torch.float32, seed=40))
    dy.copy_(matrix(5000, 172, torch.float32, seed=41))
    graph.replay()
    again = ops().checkpoint_weight_grad(dy, ops().checkpoint_int8(x))
    assert torch.equal(captured[0], again[0]) and torch.equal(captured[1], again[1])


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,n,k", [(5000, 128, 128), (300, 1500, 1500), (2000, 3400, 1700)])
def test_waits_that_run_out_leave_nan_and_a_status(m, n, k, dtype):
    from f2cgt_b200 import _lib
    o = ops()
    dy, c = matrix(m, n, dtype), o.checkpoint_int8(matrix(m, k, dtype, seed=1))
    want = o.checkpoint_weight_grad(dy, c)
    dw, db = torch.zeros(n, k, dtype=dtype, device="cuda"), torch.zeros(n, dtype=dtype, device="cuda")
    tag = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}[dtype]
    size = _lib.lib.f2c_checkpoint_weight_grad_workspace(dy.data_ptr(), n, tag, m, n, k)
    work = torch.empty(size + 256, dtype=torch.uint8, device="cuda")
    assert o.device_status() == 0
    rc = _lib.lib.f2c_checkpoint_weight_grad(dy.data_ptr(), n, tag, c.codes.data_ptr(), c.codes.stride(0), c.scales.data_ptr(), m, n, k, dw.data_ptr(), db.data_ptr(), _lib.NO_WAITS,
                                             work.data_ptr(), size, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0 and o.device_status() == 8 and torch.isnan(dw).all()
    got = o.checkpoint_weight_grad(dy, c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and o.device_status() == 0


def test_refusals():
    o = ops()
    dy, c = matrix(20, 8, torch.float32), o.checkpoint_int8(matrix(20, 40, torch.float32))
    bad = [lambda: o.checkpoint_weight_grad(dy[:19], c), lambda: o.checkpoint_weight_grad(dy.double(), c), lambda: o.checkpoint_weight_grad(dy.cpu(), c),
           lambda: o.checkpoint_weight_grad(dy.t(), c), lambda: o.checkpoint_weight_grad(dy[0], c), lambda: o.checkpoint_weight_grad(dy.clone().requires_grad_(), c),
           lambda: o.checkpoint_weight_grad(dy, (c.codes, c.scales[:19])), lambda: o.checkpoint_weight_grad(dy, (c.codes.contiguous(), c.scales)),
           lambda: o.checkpoint_weight_grad(dy, (c.codes.int(), c.scales)), lambda: o.checkpoint_weight_grad(dy, (c.codes, c.scales.double()))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
