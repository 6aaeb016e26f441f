"""Sums of checkpoint_weight_grad over many rows: what the tensor cores' accumulators cut off is bounded by the rows between two takings out, not by all rows.

S is the sum of |dy||x|.  An accumulator takes two products of 16 rows each (three beside float32), each of which leaves at most 2^-23 of the sizes that it adds;
what is taken out is added up in single precision."""
import pytest
import torch

import learn_reference as R

pytestmark = pytest.mark.gpu

TAKEN = {torch.float32: 256, torch.float16: 1024, torch.bfloat16: 2048}  # rows between two takings out
CUTS = {torch.float32: 3 / 16, torch.float16: 2 / 16, torch.bfloat16: 2 / 16}  # a row
# what the operands are rounded to, of one product: dy times the step to single precision, and to two numbers of eight bits; x to two such, and to single precision
OPERANDS = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -18 + 2.0 ** -24, torch.bfloat16: 2.0 ** -18 + 2.0 ** -24}


def ops():
    from f2cgt_b200 import ops
    return ops


def positive(m, d, dtype, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.rand(m, d, generator=g, device="cuda").add_(0.5).to(dtype)


def half_step(value, dtype):
    """Half the distance between the type's numbers around a value (normal ones)."""
    digits = {torch.float32: 24, torch.float16: 11, torch.bfloat16: 8}[dtype]
    return torch.ldexp(torch.ones_like(value), torch.frexp(value).exponent - digits - 1)


def rounded_once(got, want, off):
    """Half a step of the type, exactly, and what the sum is off (1 % for what is of second order)."""
    bad = ~((got.double() - want).abs() <= half_step(want, got.dtype) + 1.01 * off)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, by up to {float(((got.double() - want).abs() - half_step(want, got.dtype))[bad].max() / want.abs().max()):.3g} more than a rounding"


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m", [65536, 70_000, 9000])
def test_summands_of_one_sign(m, dtype):
    """148 tiles, one of each an SM, whose rows are not split but beyond 65,536: every sum is rounded once to the type, and is off by the cuts between two
    takings out, the operands' roundings and an addition a taking out.  (Cut over all rows, sums of 9000 were 4e-5 off.)"""
    n, k = 148 // 37 * (256 if dtype is torch.bfloat16 else 128), 37 * 128
    x, dy = positive(m, k, dtype, 1), positive(m, n, dtype, 2) / 64
    x[:, ::128] = 0  # (nothing is left beside whole steps)
    c = ops().checkpoint_int8(x)
    del x
    dw, db = ops().checkpoint_weight_grad(dy, c)
    want = dy.double().t() @ R.decode(c.codes, c.scales)
    off = (CUTS[dtype] * min(m, TAKEN[dtype]) * 2.0 ** -23 + OPERANDS[dtype] + (m / TAKEN[dtype] + 4) * R.U) * want
    rounded_once(dw, want, off)
    R.near(db, dy.double().sum(0), (m / 4 + 8) * R.U * dy.double().sum(0), dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m", [255, 257, 1023, 1024, 1025, 1057, 2047, 2048, 2049, 2081, 4096, 4129, 10_000])
def test_rows_around_a_taking_out(m, dtype):
    """Whole numbers below 2^24 are exact however the rows fall into takings out: codes with a step of one and dy of -1, 0 and 1, the columns of dy and of x odd in number."""
    n, k = 4 * (256 if dtype is torch.bfloat16 else 128) - 3, 37 * 128 - 5
    g = torch.Generator(device="cuda")
    g.manual_seed(m)
    codes = torch.randint(0, 256, (m, (k + 15) // 16 * 16), generator=g, device="cuda", dtype=torch.uint8)[:, :k]
    scales = torch.ones(m, (k + 127) // 128, 2, device="cuda")
    scales[:, :, 1] = -100.0 * torch.randint(0, 2, scales.shape[:2], generator=g, device="cuda")
    dy = torch.randint(-1, 2, (m, n), generator=g, device="cuda").to(dtype)
    want = dy.double().t() @ R.decode(codes, scales)
    dw, db = ops().checkpoint_weight_grad(dy, ops().Int8Checkpoint(codes, scales))
    assert torch.equal(dw, want.to(dtype)) and torch.equal(db, dy.double().sum(0).to(dtype))
    again = ops().checkpoint_weight_grad(dy, ops().Int8Checkpoint(codes, scales))
    assert torch.equal(again[0], dw) and torch.equal(again[1], db)


def parts(c, dy):
    """x, the sum's sizes S, and those of its two parts when the code nearest to zero is the origin: no more than S and twice S."""
    x, d = R.decode(c.codes, c.scales), dy.double().abs()
    step, low = (c.scales[:, :, i].double().repeat_interleave(128, 1)[:, :x.shape[1]] for i in (0, 1))
    zero = torch.round(-low / step).clamp(0, 255)
    whole, base, coded = d.t() @ x.abs(), d.t() @ (low + step * zero).abs(), d.t() @ (step * (c.codes.double() - zero)).abs()
    assert (base <= 1.01 * whole).all() and (coded <= 2.01 * whole).all()
    return x, whole, base, coded


def check_about_zero(dy, c):
    """Against sums in 64 bits, by the sizes of what is added up: takings out and their sum, and up to 160 parts; base times dy a thread's chain of an eighth of the rows."""
    dtype, m = dy.dtype, dy.shape[0]
    x, whole, base, coded = parts(c, dy)
    dw, _ = ops().checkpoint_weight_grad(dy, c)
    if dtype is torch.bfloat16:
        coded, base = whole, 0 * whole
    off = (CUTS[dtype] * min(m, TAKEN[dtype]) * 2.0 ** -23 + OPERANDS[dtype]) * coded + (m / TAKEN[dtype] + 160) * R.U * (coded + base) + (m / 8 + 8) * R.U * base
    R.near(dw, dy.double().t() @ x, off, dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
def test_small_values_beside_large_ones_of_both_signs(dtype):
    """Two columns of every group 128 and -127 steps from zero, the others none or one: the sums of the others have the size of a step, whatever the range of their groups."""
    m, n, k = 16_384, 100, 256
    g = torch.Generator(device="cuda")
    g.manual_seed(5)
    x = torch.randint(-1, 2, (m, k), generator=g, device="cuda").float()
    x[:, ::128], x[:, 1::128] = 128, -127
    x *= 0.1 + torch.rand(m, 1, generator=g, device="cuda")
    check_about_zero(positive(m, n, dtype, 6) / 64, ops().checkpoint_int8(x.to(dtype)))


@pytest.mark.parametrize("shift", [0.0, 0.7, 30.0, -30.0])
@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,n,k", [(16_384, 100, 200), (3000, 1300, 1400), (70, 128, 128), (1, 5, 300)])
def test_both_signs_and_one_sign_far_away(m, n, k, dtype, shift):
    g = torch.Generator(device="cuda")
    g.manual_seed(7)
    x = torch.randn(m, k, generator=g, device="cuda") + shift
    check_about_zero(positive(m, n, dtype, 8) / 64, ops().checkpoint_int8(x.to(dtype)))


def test_groups_of_equal_values_and_of_none():
    """No step: the value is the base.  A step beside which zero has no code: the nearest one."""
    x = torch.full((500, 300), -3.25, device="cuda")
    x[::2] = 0
    x[1::4, 128:] = 1e-40
    x[3::4, 256:] = 1e30
    dy = positive(500, 40, torch.float32, 9)
    dw, _ = ops().checkpoint_weight_grad(dy, ops().checkpoint_int8(x))
    R.near(dw, dy.double().t() @ x.double(), (500 / 8 + 200) * R.U * (dy.double().abs().t() @ x.double().abs()))


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("m,split", [(9000, False), (9000, True), (40, False)])
def test_waits_that_run_out_around_a_taking_out(m, split, dtype):
    """With all waits run out: NaN in all of both results, a status, and nothing of it in the next call."""
    import ctypes as C

    from f2cgt_b200 import _lib
    o = ops()
    n, k = (100, 200) if split else (4 * (256 if dtype is torch.bfloat16 else 128), 37 * 128)
    dy, c = positive(m, n, dtype, 3), o.checkpoint_int8(positive(m, k, dtype, 4) - 1)
    want = o.checkpoint_weight_grad(dy, c)
    dw, db = torch.zeros(n, k, dtype=dtype, device="cuda"), torch.zeros(n, dtype=dtype, device="cuda")
    tag = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}[dtype]
    size = _lib.lib.f2c_checkpoint_weight_grad_workspace(dy.data_ptr(), n, tag, m, n, k)
    assert (size > 0) is split
    work = torch.empty(size + 256, dtype=torch.uint8, device="cuda")
    rc = _lib.lib.f2c_checkpoint_weight_grad(dy.data_ptr(), n, tag, c.codes.data_ptr(), c.codes.stride(0), c.scales.data_ptr(), m, n, k, dw.data_ptr(), db.data_ptr(), _lib.NO_WAITS,
                                             work.data_ptr(), size, C.c_void_p(torch.cuda.current_stream().cuda_stream))
    assert rc == 0 and o.device_status() == 8 and torch.isnan(dw).all() and torch.isnan(db).all()
    got = o.checkpoint_weight_grad(dy, c)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and o.device_status() == 0


@pytest.mark.parametrize("dtype", R.TYPES)
def test_numbers_that_are_none_before_a_taking_out(dtype):
    """They stay in their column of dy and in their group of x."""
    m, n, k = 5000, 4 * (256 if dtype is torch.bfloat16 else 128), 37 * 128
    x, dy = positive(m, k, dtype, 1) - 1, positive(m, n, dtype, 2)
    x[17, 200], x[4000, 1000], dy[5, 3] = float("inf"), float("nan"), float("nan")
    dw, db = ops().checkpoint_weight_grad(dy, ops().checkpoint_int8(x))
    want = torch.zeros(n, k, dtype=torch.bool, device="cuda")
    want[:, 128:256] = want[:, 896:1024] = want[3] = True
    assert torch.equal(torch.isnan(dw), want) and torch.isnan(db).nonzero().flatten().tolist() == [3]


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("tiles", [37, 40])
def test_the_same_bits_beside_another_and_in_a_graph(tiles, dtype):
    """148 tiles, whole, and 160, of which 12 have their rows split."""
    m, n, k = 5000, 4 * (256 if dtype is torch.bfloat16 else 128), tiles * 128
    x, dy = positive(m, k, dtype, 1) - 1, positive(m, n, dtype, 2)
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
        captured = ops().checkpoint_weight_grad(dy, c)
    dy.copy_(positive(m, n, dtype, 41))
    graph.replay()
    again = ops().checkpoint_weight_grad(dy, c)
    assert torch.equal(captured[0], again[0]) and torch.equal(captured[1], again[1])
