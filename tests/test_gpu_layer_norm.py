"""Layer norm on the GPU against its definition in 64 bits: forward, what is kept, backward, at sizes where rows change hands."""
import pytest
import torch

import learn_reference as R

pytestmark = pytest.mark.gpu

SIZES = [(1, 1), (1, 128), (3, 7), (33, 100), (257, 128), (1300, 128), (130, 130), (65, 256), (40, 512), (21, 602), (700, 641), (9, 1024), (17, 1100), (601, 2048), (5, 4096), (4, 4100),
         (3, 8192), (2, 8196), (2, 16384), (70, 20001)]


def ops():
    from f2cgt_b200 import ops
    return ops


def rows(m, d, dtype, seed=0, spread=1.0, offset=0.0, pad=0, start=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(m, d + pad + start, generator=g, device="cuda") * spread + offset
    return x.to(dtype)[:, start:start + d]


def vectors(d, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return 1 + 0.3 * torch.randn(d, generator=g, device="cuda"), 0.3 * torch.randn(d, generator=g, device="cuda")


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,d", SIZES)
def test_forward(m, d, dtype):
    x, (w, b) = rows(m, d, dtype, offset=0.5), vectors(d)
    (y, _, _, _), (y_off, _, _) = R.norm(x, w, b, 1e-5)
    R.near(ops().layer_norm(x, w, b), y, y_off, dtype)
    R.near(ops().layer_norm(x, w, b, relu=True), y.clamp_min(0), y_off, dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,d,pad,start", [(37, 128, 3, 0), (37, 128, 8, 4), (29, 126, 6, 2), (29, 602, 1, 1), (5, 1500, 0, 5), (3, 9001, 2, 3), (6, 256, 250, 0)])
def test_rows_at_odd_places(m, d, pad, start, dtype):
    x, (w, b) = rows(m, d, dtype, pad=pad, start=start), vectors(d)
    (y, _, _, _), (y_off, _, _) = R.norm(x, w, b, 1e-5)
    R.near(ops().layer_norm(x, w, b), y, y_off, dtype)
    dy = rows(m, d, dtype, seed=5, pad=start, start=pad)
    got, saved = ops().layer_norm_train(x, w, b)
    want, off = R.norm_backward(dy, x.double(), saved.mean, saved.rstd, w)
    for a, q, o, t in zip(ops().layer_norm_backward(dy, saved, w), want, off, (dtype, torch.float32, torch.float32)):
        R.near(a, q, o, t)


@pytest.mark.parametrize("offset,spread", [(1000.0, 1.0), (-3e4, 0.01), (0.0, 1e-4), (0.0, 1e10)])
@pytest.mark.parametrize("d", [128, 300, 3000])
def test_means_that_are_large_and_rows_that_are_flat(offset, spread, d):
    x, (w, b) = rows(9, d, torch.float32, offset=offset, spread=spread), vectors(d)
    (y, mean, rstd, _), (y_off, mean_off, rstd_off) = R.norm(x, w, b, 1e-5)
    got, saved = ops().layer_norm_train(x, w, b)
    R.near(got, y, y_off)
    R.near(saved.mean, mean, mean_off)
    R.near(saved.rstd, rstd, rstd_off)


def test_weights_that_are_not_there_and_weights_at_odd_places():
    x = rows(11, 200, torch.float32)
    w, b = (t[1:] for t in vectors(201))  # 4 bytes off
    for weight, bias in ((None, None), (w, None), (None, b), (w, b)):
        (y, _, _, _), (off, _, _) = R.norm(x, weight, bias, 0.1)
        R.near(ops().layer_norm(x, weight, bias, eps=0.1), y, off)
        got, saved = ops().layer_norm_train(x, weight, bias, eps=0.1)
        dy = rows(11, 200, torch.float32, seed=2)
        want, offs = R.norm_backward(dy, x.double(), saved.mean, saved.rstd, weight)
        for a, q, o in zip(ops().layer_norm_backward(dy, saved, weight), want, offs):
            R.near(a, q, o)


def test_equal_values_have_the_bias():
    w, b = vectors(130)
    x = torch.full((3, 130), 7.0, device="cuda")
    y, saved = ops().layer_norm_train(x, w, b)
    assert torch.equal(y, b.expand(3, 130)) and torch.equal(saved.mean, torch.full((3,), 7.0, device="cuda"))
    # without eps there is no such result
    assert torch.isnan(ops().layer_norm(x, w, b, eps=0.0)).all()


@pytest.mark.parametrize("d", [128, 700, 5000])
def test_numbers_that_are_none_stay_in_their_rows(d):
    x, (w, b) = rows(8, d, torch.float32), vectors(d)
    want = ops().layer_norm(x, w, b, relu=True)
    x[2, d // 2] = float("nan")
    x[5, 0] = float("inf")
    got = ops().layer_norm(x, w, b, relu=True)
    sound = [0, 1, 3, 4, 6, 7]
    assert torch.equal(got[sound], want[sound]) and torch.isnan(got[2]).all() and torch.isnan(got[5]).any()


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,d", SIZES)
@pytest.mark.parametrize("int8", [False, True])
def test_backward(m, d, dtype, int8):
    x, (w, b), dy = rows(m, d, dtype, offset=0.5), vectors(d), rows(m, d, dtype, seed=3)
    for relu in (False, True):
        (y, mean, rstd, _), (y_off, mean_off, rstd_off) = R.norm(x, w, b, 1e-5)
        got, saved = ops().layer_norm_train(x, w, b, relu=relu, int8=int8)
        R.near(got, y.clamp_min(0) if relu else y, y_off, dtype)
        R.near(saved.mean, mean, mean_off)
        R.near(saved.rstd, rstd, rstd_off)
        kept, g = x.double(), dy
        if int8:
            codes, scales = R.encode(x)
            assert torch.equal(saved.x.codes, codes) and torch.equal(saved.x.scales, scales)
            kept = R.decode(codes, scales)
        if relu:
            open_ = R.bits_of(saved.active, d)
            assert torch.equal(open_, got > 0) or dtype is not torch.float32  # (a half may round to zero)
            assert not (open_ != (y > 0))[(y.abs() > y_off)].any()
            assert saved.active.shape == (m, (d + 7) // 8) and not (saved.active[:, -1].int() >> ((d - 1) % 8 + 1)).any()
            g = dy * open_
        else:
            assert saved.active is None
        want, off = R.norm_backward(g, kept, saved.mean, saved.rstd, w)
        for a, q, o, t in zip(ops().layer_norm_backward(dy, saved, w), want, off, (dtype, torch.float32, torch.float32)):
            R.near(a, q, o, t)


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("m,d", [(7, 33), (5, 1300)])
def test_gradient_against_differences(m, d, relu):
    """Along a direction t, L(x + e t) - L(x - e t) over 2 e is <dx, t> up to e^2 times third derivatives and what the values' roundings are over e:
    y's are 2^-22 of |y| <= 4 times |dy|, so below 2^-20 sqrt(m d) / e in all for directions and gradients of size one each value."""
    x, (w, b), dy, t = rows(m, d, torch.float32, spread=2.0), vectors(d), rows(m, d, torch.float32, seed=3), rows(m, d, torch.float32, seed=4)
    e = 2.0 ** -9
    y, saved = ops().layer_norm_train(x, w, b, relu=relu)
    if relu:  # no difference crosses the ReLU's corner: values near it have no say
        dy = dy * (y > 0.1) + 0
    dx, dw, db = ops().layer_norm_backward(dy, saved, w)

    def loss(x, w, b):
        return float((ops().layer_norm(x, w, b, relu=relu).double() * dy.double()).sum())

    room = 2.0 ** -20 * (m * d) ** 0.5 / e + e * e * 50 * (m * d) ** 0.5
    assert abs((loss(x + e * t, w, b) - loss(x - e * t, w, b)) / (2 * e) - float((dx.double() * t.double()).sum())) < room
    for grad, vary in ((dw, lambda s: loss(x, w + s * t[0], b)), (db, lambda s: loss(x, w, b + s * t[0]))):
        assert abs((vary(e) - vary(-e)) / (2 * e) - float((grad.double() * t[0].double()).sum())) < room


def test_rows_of_which_there_are_none():
    w, b = vectors(64)
    x = torch.empty(0, 64, device="cuda")
    y, saved = ops().layer_norm_train(x, w, b, relu=True, int8=True)
    dx, dw, db = ops().layer_norm_backward(x, saved, w)
    assert y.shape == dx.shape == (0, 64) and not dw.any() and not db.any()
    x = torch.empty(5, 0, device="cuda")
    assert ops().layer_norm(x).shape == (5, 0)


def test_the_same_bits_every_time_and_in_a_graph():
    w, b = vectors(300)
    x, dy = rows(3000, 300, torch.bfloat16), rows(3000, 300, torch.bfloat16, seed=9)

    def both():
        y, saved = ops().layer_norm_train(x, w, b, relu=True, int8=True)
        return (y,) + tuple(ops().layer_norm_backward(dy, saved, w))

    first = both()
    assert all(torch.equal(a, q) for a, q in zip(first, both()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        both()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = both()
    x.copy_(rows(3000, 300, torch.bfloat16, seed=21))
    dy.copy_(rows(3000, 300, torch.bfloat16, seed=22))
    graph.replay()
    assert all(torch.equal(a, q) for a, q in zip(captured, both()))


def test_refusals():
    o = ops()
    x, (w, b) = rows(4, 16, torch.float32), vectors(16)
    y, saved = o.layer_norm_train(x, w, b, relu=True)
    bad = [lambda: o.layer_norm(x.cpu()), lambda: o.layer_norm(x.double()), lambda: o.layer_norm(x[0]), lambda: o.layer_norm(x.t()), lambda: o.layer_norm(x, w[:8]),
           lambda: o.layer_norm(x, w.half()), lambda: o.layer_norm(x, w, b[None]), lambda: o.layer_norm(x, w.cpu()), lambda: o.layer_norm(x, eps=-1.0),
           lambda: o.layer_norm(x, eps=float("nan")), lambda: o.layer_norm(x.clone().requires_grad_()), lambda: o.layer_norm(x, w.clone().requires_grad_()),
           lambda: o.layer_norm(x[:1].expand(4, 16)),
           lambda: o.layer_norm_backward(x.half(), saved, w), lambda: o.layer_norm_backward(x[:3], saved, w), lambda: o.layer_norm_backward(x, saved._replace(mean=saved.mean[:3]), w),
           lambda: o.layer_norm_backward(x, saved._replace(rstd=saved.rstd.double()), w), lambda: o.layer_norm_backward(x, saved._replace(active=saved.active[:, :1]), w),
           lambda: o.layer_norm_backward(x, saved, w[:3]), lambda: o.layer_norm_backward(x.clone().requires_grad_(), saved, w)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        o.layer_norm([1.0])
    with torch.no_grad():
        assert torch.equal(o.layer_norm(x.clone().requires_grad_(), w, b, relu=True), y)
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(RuntimeError, match="tangent"):
            o.layer_norm(fwd.make_dual(x, x))


@pytest.mark.parametrize("m,d", [((1 << 21) + 3, 1100), ((1 << 25) + 3, 66)])
def test_offsets_beyond_32_bits(m, d):
    """More than 2^31 values, 2^32 bytes: the last rows are those of a call of their own."""
    o = ops()
    x = torch.zeros(m, d, dtype=torch.bfloat16, device="cuda")
    dy = torch.zeros(m, d, dtype=torch.bfloat16, device="cuda")
    x[-300:], dy[-300:] = rows(300, d, torch.bfloat16, offset=0.5), rows(300, d, torch.bfloat16, seed=3)
    w, b = vectors(d)
    y, saved = o.layer_norm_train(x, w, b, relu=True, int8=True)
    y_last, last = o.layer_norm_train(x[-300:], w, b, relu=True, int8=True)
    assert torch.equal(y[-300:], y_last) and torch.equal(saved.x.codes[-300:], last.x.codes) and torch.equal(saved.x.scales[-300:], last.x.scales)
    assert torch.equal(saved.mean[-300:], last.mean) and torch.equal(saved.rstd[-300:], last.rstd) and torch.equal(saved.active[-300:], last.active)
    del y
    dx, dw, db = o.layer_norm_backward(dy, saved, w)
    dx_last, dw_last, db_last = o.layer_norm_backward(dy[-300:], last, w)
    assert torch.equal(dx[-300:], dx_last) and not dx[:-300].any()
    # the same 300 summands and zeros, added up in another order
    h = (o.checkpoint_values(last.x).double() - last.mean.double()[:, None]) * last.rstd.double()[:, None]
    assert ((dw - dw_last).abs() <= 2 * 303 * R.U * (dy[-300:].double() * h).abs().sum(0)).all() and ((db - db_last).abs() <= 2 * 303 * R.U * dy[-300:].double().abs().sum(0)).all()
    del dx
    kept = o.checkpoint_int8(x)
    assert torch.equal(kept.codes[-300:], last.x.codes) and torch.equal(kept.scales[-300:], last.x.scales)
    del x, saved
    narrow = dy[:, :8].contiguous()
    del dy
    dweight, dbias = o.checkpoint_weight_grad(narrow, kept)
    values, grads = o.checkpoint_values(last.x).double(), narrow[-300:].double()
    # the values to 16 bits; the result and the sums of the last part's 300 rows
    assert ((dweight.double() - grads.T @ values).abs() <= 2.0 ** -8 * (grads.T @ values).abs() + 2.0 ** -16 * grads.abs().T @ values.abs()).all()
    assert ((dbias.double() - grads.sum(0)).abs() <= 2.0 ** -8 * grads.sum(0).abs() + 2.0 ** -16 * grads.abs().sum(0)).all()
    values = o.checkpoint_values(kept, torch.bfloat16)
    assert torch.equal(values[-300:], o.checkpoint_values(last.x, torch.bfloat16)) and not values[:-300].any()
