"""GPU: 8-bit quantisation of rows and products with a scale for every row and channel, against the definition in 64 bits.

Codes have to be equal.  The integer sum is exact; the result is rounded when the sum becomes a float, when the scales are multiplied,
when they are applied and when the bias is added (2^-24 of the magnitudes each), and once more to the output's type."""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from f2cgt_b200 import _lib, ops  # noqa: E402

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
HALF_ULP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 0.0, torch.float16: 2.0 ** -25, torch.bfloat16: 0.0}


def define(x):
    """codes and scales of float32 rows in numpy's single precision"""
    x = x.float().cpu().numpy()
    with np.errstate(all="ignore"):
        top = np.abs(x).max(1) if x.shape[1] else np.zeros(len(x), np.float32)
        bad = ~np.isfinite(x).all(1)
        scale = (top / np.float32(127)).astype(np.float32)
        q = np.clip(np.rint(x / scale[:, None]), -127, 127)
    q[bad | (scale == 0)] = 0
    scale[bad] = np.nan
    return q.astype(np.int8), scale


def rows(m, k, dtype, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + m * 31 + k)
    return (torch.randn(m, k, generator=g) * torch.rand(m, 1, generator=g) * 3).to(dtype)


def weights(n, k, seed=1):
    g = torch.Generator().manual_seed(seed + n * 131 + k)
    q = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    return q, torch.rand(n, generator=g) * 0.01 + 1e-4, torch.randn(n, generator=g)


def check(got, q, s, wq, ws, bias, relu):
    y = q.astype(np.float64) @ wq.numpy().astype(np.float64).T * s.astype(np.float64)[:, None] * ws.numpy().astype(np.float64)
    b = bias.numpy().astype(np.float64) if bias is not None else 0.0
    room = 4 * 2.0 ** -24 * (np.abs(y) + np.abs(b))
    want = y + b
    if relu:
        want = np.where(want <= 0, 0.0, want)
    room = room + HALF_ULP[got.dtype] * (np.abs(want) + room) + TINY[got.dtype]
    have = got.double().cpu().numpy()
    assert have.shape == want.shape
    assert np.array_equal(np.isnan(have), np.isnan(want))
    fine = ~np.isnan(want)
    assert (np.abs(have - want)[fine] <= room[fine]).all()


SIZES = [(0, 4), (1, 1), (1, 256), (2, 3), (7, 16), (33, 100), (64, 128), (129, 255), (300, 602), (5, 4099), (2, 131071), (1000, 17)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("m,k", SIZES)
def test_codes_and_scales_are_the_definition(m, k, dtype):
    x = rows(m, k, TYPES[dtype])
    codes, scales = ops.int8_quantize(x.cuda())
    q, s = define(x)
    assert codes.shape == (m, k) and codes.dtype == torch.int8 and scales.dtype == torch.float32
    assert m <= 1 or codes.stride(0) % 16 == 0
    assert np.array_equal(codes.cpu().numpy(), q) and np.array_equal(scales.cpu().numpy(), s)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("k1,k2", [(128, 128), (100, 3), (1, 64), (37, 0), (0, 20), (2048, 2048), (5, 4000)])
def test_two_tensors_side_by_side(k1, k2, dtype):
    x = rows(77, k1 + k2, TYPES[dtype], 3)
    codes, scales = ops.int8_quantize(x[:, :k1].contiguous().cuda(), x[:, k1:].contiguous().cuda())
    q, s = define(x)
    assert np.array_equal(codes.cpu().numpy(), q) and np.array_equal(scales.cpu().numpy(), s)
    wq, ws, b = weights(50, k1 + k2)
    y = ops.int8_linear(x[:, :k1].contiguous().cuda(), wq.cuda(), ws.cuda(), b.cuda(), x2=x[:, k1:].contiguous().cuda())
    check(y, q, s, wq, ws, b, False)


@pytest.mark.parametrize("k", [5, 64, 200, 2000])
def test_ties_zero_rows_and_rows_that_are_not_finite(k):
    x = torch.zeros(12, k)
    x[1] = torch.arange(k) % 255 - 127 + 0.5      # halfway between codes where the scale is one
    x[1, 0] = 127
    x[2, k // 2] = float("nan")
    x[3, k - 1] = float("inf")
    x[4, 0] = -float("inf")
    x[5] = 1e-45 * (torch.arange(k) % 3)          # no scale can be represented
    x[6] = 3e-44 * (torch.arange(k) % 7 - 3)      # a subnormal scale
    x[7] = 1e-38 * (torch.arange(k) % 11 - 5)
    x[8] = 3.4e38 * (torch.arange(k) % 2 * 2 - 1)
    x[9, 0] = -5.0
    x[10] = -0.0
    x[11] = torch.linspace(-1, 1, k)
    q, s = define(x)
    codes, scales = ops.int8_quantize(x.cuda())
    assert np.array_equal(codes.cpu().numpy(), q)
    assert np.array_equal(scales.cpu().numpy(), s, equal_nan=True)
    wq, ws, b = weights(130, k)
    y = ops.int8_linear(x.cuda(), wq.cuda(), ws.cuda(), b.cuda(), relu=True)
    have = y.cpu()
    assert torch.isnan(have[2:5]).all()
    assert torch.equal(have[0], b.clamp_min(0)) and torch.equal(have[10], b.clamp_min(0))
    keep = [0, 1, 5, 6, 7, 9, 10, 11]
    check(y[keep], q[keep], s[keep], wq, ws, b, True)


def test_codes_next_to_a_tie():
    # quotients within a few units in the last place of a half, for scales that are no powers of two
    g = np.random.default_rng(5)
    x = np.zeros((400, 96), np.float32)
    for i in range(400):
        top = np.float32(g.uniform(0.1, 300))
        scale = np.float32(top / np.float32(127))
        half = (g.integers(-126, 126, 95) + 0.5).astype(np.float32) * scale
        off = g.integers(-3, 4, 95).astype(np.int32)
        x[i, 0] = top
        x[i, 1:] = (half.view(np.int32) + off).view(np.float32)
    q, s = define(torch.from_numpy(x))
    codes, scales = ops.int8_quantize(torch.from_numpy(x).cuda())
    assert np.array_equal(codes.cpu().numpy(), q) and np.array_equal(scales.cpu().numpy(), s)


MM = [(1, 1, 1), (1, 172, 256), (1, 4096, 512), (3, 5, 7), (8, 128, 128), (16, 1000, 4096), (17, 129, 33), (64, 64, 64), (100, 41, 602), (129, 257, 130),
      (255, 128, 256), (256, 256, 2048), (257, 130, 4097), (1000, 172, 256), (3000, 7, 16), (4096, 512, 48), (20000, 128, 256), (2, 1000, 20000),
      (700, 300, 1000), (33, 40, 131071)]


@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,n,k", MM)
def test_products(m, n, k, out):
    x, (wq, ws, b) = rows(m, k, torch.float32, 9), weights(n, k)
    q, s = define(x)
    with_bias, relu = (m + n) % 2 == 0, (n + k) % 2 == 0
    qd, sd = torch.from_numpy(q).cuda(), torch.from_numpy(s).cuda()
    y = ops.int8_mm(qd, sd, wq.cuda(), ws.cuda(), b.cuda() if with_bias else None, relu, TYPES[out])
    assert y.dtype == TYPES[out]
    check(y, q, s, wq, ws, b if with_bias else None, relu)
    xd = x.to(TYPES[out])
    q, s = define(xd)
    y = ops.int8_linear(xd.cuda(), wq.cuda(), ws.cuda(), b.cuda() if with_bias else None, relu)
    assert y.dtype == TYPES[out]
    check(y, q, s, wq, ws, b if with_bias else None, relu)


# many tiles and a long K, where pairs of CTAs share one: odd numbers of channel tiles (the last half of a pair has none), tails everywhere
@pytest.mark.parametrize("out", TYPES)
@pytest.mark.parametrize("m,n,k", [(4000, 700, 1600), (7001, 1100, 1333), (20001, 390, 1500)])
def test_many_tiles_and_a_long_k(m, n, k, out):
    test_products(m, n, k, out)


def test_extreme_codes_do_not_overflow():
    for m, n in ((3, 5), (200, 130)):
        q, w = torch.full((m, 131071), -128, dtype=torch.int8), torch.full((n, 131071), -128, dtype=torch.int8)
        s, ws = torch.full((m,), 0.5), torch.full((n,), 0.25)
        y = ops.int8_mm(q.cuda(), s.cuda(), w.cuda(), ws.cuda())
        assert (y.cpu().double() - 131071 * 16384 / 8.0).abs().max() <= 4 * 2.0 ** -24 * 131071 * 2048


@pytest.mark.parametrize("m,n,k", [(40, 70, 96), (300, 200, 130), (1, 33, 50)])
def test_strided_and_unaligned_operands(m, n, k):
    x, (wq, ws, b) = rows(m, k, torch.float32, 4), weights(n, k)
    q, s = define(x)
    for lead, gap in ((0, 0), (0, 13), (1, 16), (16, 32), (3, 5)):
        big = torch.full((m, k + lead + gap), 77, dtype=torch.int8)
        big[:, lead:lead + k] = torch.from_numpy(q)
        wide = torch.full((n, k + gap + lead), -99, dtype=torch.int8)
        wide[:, gap:gap + k] = wq
        y = ops.int8_mm(big.cuda()[:, lead:lead + k], torch.from_numpy(s).cuda(), wide.cuda()[:, gap:gap + k], ws.cuda(), b.cuda())
        check(y, q, s, wq, ws, b, False)
        xs = torch.full((m, k + lead + gap), float("nan"))
        xs[:, lead:lead + k] = x
        y = ops.int8_linear(xs.cuda()[:, lead:lead + k], wide.cuda()[:, gap:gap + k], ws.cuda(), b.cuda())
        check(y, q, s, wq, ws, b, False)
    # vectors that do not start on 16 bytes
    off = lambda t: torch.cat([torch.zeros(1), t]).cuda()[1:]  # noqa: E731
    y = ops.int8_mm(torch.from_numpy(q).cuda(), off(torch.from_numpy(s)), wq.cuda(), off(ws), off(b))
    check(y, q, s, wq, ws, b, False)


@pytest.mark.parametrize("m,n,k", [(1, 172, 256), (40, 70, 96), (1024, 172, 256), (300, 41, 602), (2000, 300, 1000)])
def test_workspaces_are_kept_to(m, n, k):
    lib, stream = _lib.lib, torch.cuda.current_stream().cuda_stream
    x, (wq, ws, _) = rows(m, k, torch.float32, 4), weights(n, k)
    q, s = define(x)
    for lead, gap in ((0, 0), (1, 0), (0, 1), (4, 4)):
        xs = torch.zeros(m, lead + k + gap).cuda()
        xs[:, lead:lead + k] = x.cuda()
        wide = torch.zeros(n, lead + k + gap, dtype=torch.int8).cuda()
        wide[:, lead:lead + k] = wq.cuda()
        scales, out = ws.cuda(), torch.empty(m, n).cuda()
        xp, wp, ld = xs.data_ptr() + 4 * lead, wide.data_ptr() + lead, lead + k + gap
        need = lib.f2c_int8_linear_workspace(xp, ld, k, None, 0, 0, _lib.F32, wp, ld, m, n)
        space = torch.full((need + 65536,), 85, dtype=torch.uint8).cuda()
        assert lib.f2c_int8_linear(xp, ld, k, None, 0, 0, _lib.F32, wp, ld, scales.data_ptr(), None, 0, out.data_ptr(), _lib.F32, m, n,
                                   space.data_ptr() if need else None, need, stream) == 0
        assert (space[need:] == 85).all()
        check(out, q, s, wq, ws, None, False)


def test_no_columns_no_rows():
    b = torch.randn(6)
    y = ops.int8_mm(torch.zeros(4, 0, dtype=torch.int8).cuda(), torch.ones(4).cuda(), torch.zeros(6, 0, dtype=torch.int8).cuda(), torch.ones(6).cuda(), b.cuda())
    assert torch.equal(y.cpu(), b.expand(4, 6))
    assert ops.int8_mm(torch.zeros(0, 8, dtype=torch.int8).cuda(), torch.ones(0).cuda(), torch.zeros(6, 8, dtype=torch.int8).cuda(), torch.ones(6).cuda()).shape == (0, 6)
    assert ops.int8_linear(torch.zeros(3, 8).cuda(), torch.zeros(0, 8, dtype=torch.int8).cuda(), torch.ones(0).cuda()).shape == (3, 0)


def test_a_call_writes_nothing_but_its_output():
    m, n, k = 203, 45, 70
    x, (wq, ws, b) = rows(m, k, torch.float32, 8), weights(n, k)
    before = [t.clone() for t in (x, wq, ws, b)]
    d = [t.cuda() for t in (x, wq, ws, b)]
    ops.int8_linear(*d)
    assert all(torch.equal(t.cpu(), u) for t, u in zip(d, before))


def test_many_rows_whose_outputs_pass_32_bit_offsets():
    m, n, k = 1_100_000, 2048, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    q = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8, device="cuda")
    s = torch.rand(m, generator=g, device="cuda")
    wq, ws, _ = weights(n, k)
    y = ops.int8_mm(q, s, wq.cuda(), ws.cuda(), out_dtype=torch.bfloat16)
    for lo in (0, m // 2, m - 1000):
        part = slice(lo, lo + 1000)
        check(y[part], q[part].cpu().numpy(), s[part].cpu().numpy(), wq, ws, None, False)


def test_another_stream_and_the_same_bits_again():
    x, (wq, ws, b) = rows(500, 300, torch.float32, 6), weights(200, 300)
    d = [t.cuda() for t in (x, wq, ws, b)]
    torch.cuda.synchronize()
    st = torch.cuda.Stream()
    with torch.cuda.stream(st):
        ys = [ops.int8_linear(*d) for _ in range(20)]
    st.synchronize()
    first = ops.int8_linear(*d)
    assert all(torch.equal(y, first) for y in ys)


def test_a_call_can_be_captured():
    x, (wq, ws, b) = rows(40, 512, torch.float32, 6), weights(300, 512)
    d = [t.cuda() for t in (x, wq, ws, b)]
    want = ops.int8_linear(*d)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.int8_linear(*d)
    d[0].mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(y, ops.int8_linear(*d)) and not torch.equal(y, want)


def test_refusals():
    x, (wq, ws, b) = rows(4, 8, torch.float32), weights(6, 8)
    x, wq, ws, b = (t.cuda() for t in (x, wq, ws, b))
    q, s = ops.int8_quantize(x)
    bad = [lambda: ops.int8_quantize(x.cpu()), lambda: ops.int8_quantize(x.double()), lambda: ops.int8_quantize(x[0]), lambda: ops.int8_quantize(x.t()),
           lambda: ops.int8_quantize(x, x.half()), lambda: ops.int8_quantize(x, x[:2]), lambda: ops.int8_quantize(x[:, ::2]),
           lambda: ops.int8_mm(q, s[:3], wq, ws), lambda: ops.int8_mm(q, s, wq[:, :4], ws), lambda: ops.int8_mm(q, s, wq, ws[:5]),
           lambda: ops.int8_mm(q, s, wq, ws, b[:5]), lambda: ops.int8_mm(q, s, wq, ws, out_dtype=torch.int32), lambda: ops.int8_mm(q.float(), s, wq, ws),
           lambda: ops.int8_mm(q, s, wq.t(), ws), lambda: ops.int8_mm(q, s, wq.cpu(), ws), lambda: ops.int8_mm(q, s.double(), wq, ws),
           lambda: ops.int8_linear(x, wq, ws, b.half()), lambda: ops.int8_linear(x.expand(2, 4, 8), wq, ws),
           lambda: ops.int8_linear(x[:1].expand(4, 8), wq, ws), lambda: ops.int8_linear(x.clone().requires_grad_(), wq, ws),
           lambda: ops.int8_quantize(torch.zeros(1, 131072, device="cuda"))]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        ops.int8_quantize(None)
    with pytest.raises(TypeError):
        ops.int8_mm(q, s, wq, ws, out_dtype="float32")
    with torch.no_grad():
        ops.int8_linear(x.clone().requires_grad_(), wq, ws)
