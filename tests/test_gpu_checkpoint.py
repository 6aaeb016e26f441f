"""Activations in 8 bits on the GPU against the definition: the same codes and scales bit for bit, values one rounding off."""
import pytest
import torch

import learn_reference as R

pytestmark = pytest.mark.gpu


def ops():
    from f2cgt_b200 import ops
    return ops


def rows(m, d, dtype, seed=0, pad=0, start=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    x = torch.randn(m, d + pad + start, generator=g, device="cuda") * (0.1 + 3 * torch.rand(m, 1, generator=g, device="cuda"))
    return x.to(dtype)[:, start:start + d]


def check(x):
    c = ops().checkpoint_int8(x)
    codes, scales = R.encode(x)
    assert c.codes.dtype is torch.uint8 and c.codes.shape == x.shape and torch.equal(c.codes, codes)
    assert torch.equal(c.scales.nan_to_num(-1.0, -2.0, -3.0), scales.nan_to_num(-1.0, -2.0, -3.0))
    return c


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,d", [(1, 1), (1, 128), (5, 3), (70, 128), (33, 129), (2500, 128), (9, 256), (50, 602), (3, 4096), (2, 10001), (300, 17)])
def test_codes_and_values(m, d, dtype):
    x = rows(m, d, dtype)
    c = check(x)
    want = R.decode(c.codes, c.scales)
    for out in R.TYPES:
        got = ops().checkpoint_values(c, out)
        assert got.dtype is out
        R.near(got, want, R.U * want.abs(), out)
    # half a step, and what the roundings of the difference, the quotient and the step are off
    step = c.scales[:, :, 0].double().repeat_interleave(128, 1)[:, :d]
    assert ((want - x.double()).abs() <= step * (0.5 + 255 * 4 * R.U) + 2 * R.U * x.double().abs().amax()).all()


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("pad,start", [(1, 0), (0, 1), (2, 2), (4, 0), (6, 4), (0, 3)])
def test_rows_at_odd_places(pad, start, dtype):
    for d in (5, 128, 300):
        check(rows(21, d, dtype, pad=pad, start=start))


def test_ties_go_to_even():
    """Values that lie between two codes: low 0, step 2^-3, values (j + 0.5) step."""
    j = torch.arange(126, device="cuda", dtype=torch.float32)
    x = torch.cat([torch.tensor([0.0, 255 / 8], device="cuda"), (j + 0.5) / 8])[None].repeat(3, 1)
    c = check(x)
    assert (c.codes[:, 2:].int() % 2 == 0).all() and float(c.scales[0, 0, 0]) == 0.125


def test_values_all_over_the_type():
    """Steps from nothing to the largest, in single precision's whole range."""
    g = torch.Generator(device="cuda")
    g.manual_seed(3)
    e = torch.arange(-149, 128, device="cuda", dtype=torch.float64)
    x = (torch.rand(e.numel(), 131, generator=g, device="cuda").double() * 2.0 ** e[:, None]).float()
    x[:, 128:] *= -1
    c = check(x)
    assert not torch.isnan(c.scales).any()


def test_groups_of_equal_values():
    x = torch.full((4, 200), -3.25, device="cuda", dtype=torch.bfloat16)
    c = check(x)
    assert not c.codes.any() and torch.equal(ops().checkpoint_values(c, torch.bfloat16), x)
    check(torch.zeros(3, 40, device="cuda"))


def test_numbers_that_are_none_stay_in_their_group():
    x = rows(6, 384, torch.float32)
    x[1, 130], x[2, 0], x[3, 383] = float("nan"), float("inf"), -float("inf")
    x[4, 200], x[4, 201] = 3e38, -3e38  # more than the type's range apart
    x[5, 5], x[5, 6] = float("inf"), -float("inf")
    c = check(x)
    lost = torch.isnan(ops().checkpoint_values(c))
    want = torch.zeros_like(lost)
    want[1, 128:256] = want[2, :128] = want[3, 256:] = want[4, 128:256] = want[5, :128] = True
    assert torch.equal(lost, want)


def test_rows_of_which_there_are_none():
    for shape in ((0, 77), (9, 0)):
        c = ops().checkpoint_int8(torch.empty(shape, device="cuda"))
        assert c.codes.shape == shape and ops().checkpoint_values(c).shape == shape


def test_refusals():
    o = ops()
    x = rows(4, 40, torch.float32)
    c = o.checkpoint_int8(x)
    bad = [lambda: o.checkpoint_int8(x.cpu()), lambda: o.checkpoint_int8(x.double()), lambda: o.checkpoint_int8(x[0]), lambda: o.checkpoint_int8(x.t()),
           lambda: o.checkpoint_int8(x.clone().requires_grad_()), lambda: o.checkpoint_values((c.codes, c.scales[:3])), lambda: o.checkpoint_values((c.codes, c.scales.half())),
           lambda: o.checkpoint_values((c.codes.view(torch.int8), c.scales)), lambda: o.checkpoint_values((c.codes[:, 1:], c.scales)),
           lambda: o.checkpoint_values((c.codes.contiguous(), c.scales)), lambda: o.checkpoint_values((c.codes[:1].clone(), c.scales[:1])),
           lambda: o.checkpoint_values(c, torch.float64), lambda: o.checkpoint_values((c.codes, c.scales[:, :, :1]))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        o.checkpoint_values(c, "float32")
    assert torch.equal(o.checkpoint_values((c.codes[2:], c.scales[2:])), o.checkpoint_values(c)[2:])
    assert torch.equal(o.checkpoint_values((c.codes[::3], c.scales[::3].contiguous())), o.checkpoint_values(c)[::3])
