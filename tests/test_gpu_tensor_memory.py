"""GPU: kernels that hold tensor memory, back to back and on two streams: each has to get its columns, whoever else is on the SM."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def test_kernels_with_tensor_memory_in_a_row_and_side_by_side(capi):
    from f2cgt_b200 import ops
    from f2cgt_b200._lib import check, lib
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    # short rows in one launch: CTAs of 25 KB of shared memory and 64 columns, which fit on an SM beside all the others
    rows = rnd(8000, 64)
    codes, scales = ops.int8_quantize(rnd(128, 64))
    stack, points, centres = rnd(200, 100, 128), rnd(60_000, 16), rnd(256, 16)
    x1, x2, w1, w2, b = rnd(7000, 64), rnd(7000, 64), rnd(96, 64), rnd(96, 64), rnd(96)

    def layer():
        y = torch.empty(7000, 96, device="cuda")
        check(lib.f2c_sage_forward(x1.data_ptr(), x2.data_ptr(), w1.data_ptr(), w2.data_ptr(), b.data_ptr(), y.data_ptr(), 7000, 96, 64, 0, ops._stream(y)))
        return y

    calls = [lambda: ops.int8_linear(rows, codes, scales), lambda: ops.orthogonalize(stack), lambda: ops.kmeans_assign(points, centres, "l2"), layer,
             lambda: ops.orthogonalize(stack[:1, :, :64].contiguous())]
    want = [call() for call in calls]
    torch.cuda.synchronize()
    ops.device_status()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for i in range(60):
        for s, stream in enumerate(streams):
            with torch.cuda.stream(stream):
                for j in range(len(calls)):
                    at = (j * (1 + s) + i) % len(calls)
                    got.append((at, calls[at]()))
    torch.cuda.synchronize()
    assert ops.device_status() == 0
    assert all(torch.equal(out, want[at]) for at, out in got)
