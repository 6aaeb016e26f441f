"""Layer norm of rows whose mean is far larger than their deviation: what the sum loses of the mean has no part in the result."""
import pytest
import torch

import learn_reference as R

pytestmark = pytest.mark.gpu

WIDTHS = [100, 128, 200, 256, 300, 602, 768, 1000, 1024, 1500, 2048, 4096, 5000, 8192, 9001, 16384]  # of every kernel, even and not


def ops():
    from f2cgt_b200 import ops
    return ops


def vectors(d, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return 1 + 0.3 * torch.randn(d, generator=g, device="cuda"), 0.3 * torch.randn(d, generator=g, device="cuda")


def links(d):
    """Of a row's sum: a lane has two packed pairs of every 128 columns of its warp - of one warp up to 1024 columns, 4 to 4096, 8 to 8192, 16 beyond -, a pair's two
    numbers, 5 exchanges in the warp, up to 4 between warps; and the division by the columns, of two roundings."""
    warps = 1 if d <= 1024 else 4 if d <= 4096 else 8 if d <= 8192 else 16
    chunks = (d + 127) // 128
    return 2 * ((chunks + warps - 1) // warps) + 1 + 5 + 4 + 2


def norm(x, weight, bias, eps):
    """y, mean, rstd in 64 bits, and the most that they are off.  The first mean is off by `first`; the mean of the differences from it corrects it, off by what a sum of that
    many links loses of the differences.  A difference of two near numbers, and the correction's product, are a rounding each."""
    x = x.double()
    k = links(x.shape[1])
    mean = x.mean(1)
    z = x - mean[:, None]
    var = (z * z).mean(1)
    rstd = (var + eps) ** -0.5
    h = z * rstd[:, None]
    y = h * weight.double() + bias.double()
    first = k * R.U * x.abs().mean(1)
    size = z.abs().mean(1) + first  # of a difference, on average
    left = (k + 2) * R.U * size  # of the mean's error
    z_off = left[:, None] + R.U * (2 * z.abs() + first[:, None])
    # the variance: mean of the squares less the square of the correction
    var_off = (k + 6) * R.U * (var + first ** 2) + 2 * first * left
    rstd_off = rstd * (0.5 * var_off * rstd ** 2 + 4 * R.U)
    h_off = rstd[:, None] * (z_off + R.U * first[:, None]) + z.abs() * rstd_off[:, None] + 2 * R.U * h.abs()
    y_off = weight.double().abs() * h_off + 2 * R.U * (h * weight.double()).abs() + 2 * R.U * y.abs()
    return (y, mean, rstd), (y_off, left, rstd_off)


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("value", [33.3, 1000.3, 12345.6, -100000.7])
def test_rows_of_one_value_have_the_bias(value, d):
    w, b = vectors(d)
    x = torch.full((9, d), value, device="cuda")
    (y, _, _), (off, _, _) = norm(x, w, b, 1e-5)
    assert off.max() < 2e-3  # of a deviation
    got, saved = ops().layer_norm_train(x, w, b)
    R.near(got, y, off)
    R.near(ops().layer_norm(x, w, b), y, off)
    assert torch.equal(saved.mean, x[:, 0])
    assert ((saved.rstd.double() * 1e-5 ** 0.5 - 1).abs() < 1e-4).all()


@pytest.mark.parametrize("d", WIDTHS)
@pytest.mark.parametrize("offset,spread", [(1000.0, 0.01), (-3e4, 0.01), (1e5, 1.0), (4.0, 1.0), (0.0, 1.0)])
def test_rows_around_a_large_mean(offset, spread, d):
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    x, (w, b) = torch.randn(9, d, generator=g, device="cuda") * spread + offset, vectors(d)
    (y, mean, rstd), (y_off, mean_off, rstd_off) = norm(x, w, b, 1e-5)
    assert y_off.max() < 2e-2 and (rstd_off < 1e-2 * rstd).all()  # of a deviation
    got, saved = ops().layer_norm_train(x, w, b)
    R.near(got, y, y_off)
    R.near(saved.mean, mean, mean_off)
    R.near(saved.rstd, rstd, rstd_off)
    R.near(ops().layer_norm(x, w, b, relu=True), y.clamp_min(0), y_off)


@pytest.mark.parametrize("d", [128, 602, 2048, 9001])
@pytest.mark.parametrize("dtype,offset", [(torch.float16, 2000.0), (torch.bfloat16, -500.0)])
def test_16_bit_rows_around_a_large_mean(dtype, offset, d):
    g = torch.Generator(device="cuda")
    g.manual_seed(4)
    x, (w, b) = (torch.randn(9, d, generator=g, device="cuda") * 4 + offset).to(dtype), vectors(d)
    (y, mean, rstd), (y_off, mean_off, rstd_off) = norm(x, w, b, 1e-5)
    got, saved = ops().layer_norm_train(x, w, b)
    R.near(got, y, y_off, dtype)
    R.near(saved.mean, mean, mean_off)
    R.near(saved.rstd, rstd, rstd_off)


@pytest.mark.parametrize("d", [128, 700, 3000, 5000, 9000])
def test_squares_beyond_the_type_and_no_eps(d):
    """An infinite variance leaves the bias, equal values without eps have no result, and neither has a row with a NaN."""
    w, b = vectors(d)
    x = torch.full((4, d), 1000.3, device="cuda")
    x[0, ::2], x[0, 1::2] = 1e25, -1e25
    x[1, 3] = float("nan")
    got, saved = ops().layer_norm_train(x, w, b)
    assert torch.equal(got[0], b) and float(saved.rstd[0]) == 0
    assert torch.isnan(got[1]).all() and torch.isnan(saved.mean[1]) and torch.isnan(saved.rstd[1])
