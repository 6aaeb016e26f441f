"""Learned rows on the GPU: the lookup against one rounding of the product, the gradient against sums in 64 bits."""
import pytest
import torch

import learn_reference as R

pytestmark = pytest.mark.gpu


def ops():
    from f2cgt_b200 import ops
    return ops


def table_of(rows, d, dtype, seed=0, pad=0, start=0):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return torch.randn(rows, d + pad + start, generator=g, device="cuda").to(dtype)[:, start:start + d]


def ids_of(m, rows, how, dtype=torch.int64, seed=1):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    if how == "one":
        ids = torch.full((m,), rows - 1, device="cuda")
    elif how == "skew":
        ids = (torch.rand(m, generator=g, device="cuda").double() ** 6 * rows).long().clamp(max=rows - 1)
    elif how == "outside":
        ids = torch.randint(-2 * rows - 2, 3 * rows + 2, (m,), generator=g, device="cuda")
    elif how == "nowhere":
        ids = torch.full((m,), -1, device="cuda")
    elif how == "descending":
        ids = (torch.arange(m, device="cuda").flip(0) // 3) % rows
    else:
        ids = torch.randint(0, rows, (m,), generator=g, device="cuda")
    return ids.to(dtype)


@pytest.mark.parametrize("dtype", R.TYPES)
@pytest.mark.parametrize("rows,d,pad,start", [(1, 1, 0, 0), (50, 128, 0, 0), (50, 100, 0, 0), (50, 602, 0, 0), (31, 33, 2, 1), (31, 128, 8, 4), (9, 4100, 0, 0), (31, 126, 0, 2)])
def test_lookup(rows, d, pad, start, dtype):
    table = table_of(rows, d, dtype, pad=pad, start=start)
    for m, how, scale, index in ((1, "any", 1.0, torch.int64), (777, "any", d ** 0.5, torch.int32), (300, "outside", -0.3, torch.int64), (300, "outside", 2.0, torch.int32)):
        ids = ids_of(m, rows, how, index)
        inside = (ids >= 0) & (ids < rows)
        by = float(torch.tensor(scale, dtype=torch.float32))  # the scale is single precision
        want = torch.where(inside[:, None], table.double()[ids.clamp(0, rows - 1).long()] * by, 0.0)
        got = ops().embedding(table, ids, scale)
        assert got.dtype is dtype
        R.near(got, want, R.U * want.abs(), dtype)
        if scale == 1.0:
            assert torch.equal(got, table[ids])


def test_ids_of_any_shape():
    table = table_of(20, 16, torch.float32)
    ids = ids_of(24, 20, "any")
    for shape in ((), (1,), (2, 3, 4), (0, 5)):
        part = ids[:max(1, 0)].reshape(()) if shape == () else ids[:torch.Size(shape).numel()].reshape(shape)
        assert torch.equal(ops().embedding(table, part, 3.0), table[part] * 3.0)
        dy = torch.ones(tuple(shape) + (16,), device="cuda")
        assert torch.equal(ops().embedding_backward(dy, part, 20)[:, 0], torch.bincount(part.reshape(-1), minlength=20).float())


def check_gradient(dy, ids, rows, scale):
    m, d = ids.numel(), dy.shape[-1]
    by = float(torch.tensor(scale, dtype=torch.float32))
    flat, grads = ids.reshape(-1).long(), dy.reshape(m, d).double()
    inside = (flat >= 0) & (flat < rows)
    want = torch.zeros(rows, d, dtype=torch.float64, device="cuda").index_put_((flat[inside],), grads[inside], accumulate=True)
    sizes = torch.zeros_like(want).index_put_((flat[inside],), grads[inside].abs(), accumulate=True)
    # a stretch has up to 32 places; those of one row are joined in up to 16 steps, or a CTA's eight warps take an eighth of them each.  Few rows: a CTA's 16 warps
    # take 25 of its places each, or one takes 32, and then every 16th CTA's
    links = max(32 + 16 + 8 + m / 32 / 8, 25 + 16 + 148 / 16 + 1 + 16)
    dense = ops().embedding_backward(dy, ids, rows, scale)
    assert dense.dtype is dy.dtype and dense.shape == (rows, d)
    R.near(dense, want * by, (links * R.U * sizes + 2 * R.U * want.abs()) * abs(by), dy.dtype)
    looked_up, part, count = ops().embedding_backward_rows(dy, ids, rows, scale)
    there = torch.unique(flat[inside])
    n = there.numel()
    assert looked_up.shape == (m,) and part.shape == (m, d) and int(count) == n
    assert torch.equal(looked_up[:n], there) and (looked_up[n:] == -1).all() and not part[n:].any()
    assert torch.equal(part[:n], dense[there])
    R.near(part[:n], want[there] * by, (links * R.U * sizes[there] + 2 * R.U * want[there].abs()) * abs(by), dy.dtype)
    untouched = torch.ones(rows, dtype=torch.bool, device="cuda")
    untouched[there] = False
    assert not dense[untouched].any()
    return dense


@pytest.mark.parametrize("how", ["any", "one", "skew", "outside", "nowhere", "descending"])
@pytest.mark.parametrize("m,rows,d", [(1, 1, 1), (1, 1000, 128), (7, 3, 5), (8, 8, 128), (33, 5, 130), (255, 3000, 64), (1024, 172, 128), (1024, 3, 4096), (1000, 100_000, 12), (1025, 172, 128), (4096, 100, 36), (4097, 100, 36),
                                      (5000, 2047, 8), (5000, 2048, 8), (5000, 512, 130), (5000, 513, 130), (59001, 172, 128), (59200, 1024, 20), (59201, 1024, 20), (59200, 1025, 20), (6400, 1, 1030), (1026, 9, 4100), (20000, 5_000_000, 4), (16385, 172, 260), (40001, 7, 128), (70000, 60000, 16)])
def test_gradient(m, rows, d, how):
    dy = table_of(m, d, torch.float32, seed=2)
    check_gradient(dy, ids_of(m, rows, how), rows, 1.7)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("m,rows,d,pad,start", [(100, 9, 128, 0, 0), (5000, 700, 301, 0, 0), (5000, 700, 64, 3, 1), (17000, 100, 4, 4, 0), (30_000, 90, 300, 4, 2), (2000, 5000, 129, 1, 1)])
def test_gradient_of_other_types_and_places(m, rows, d, pad, start, dtype, index):
    check_gradient(table_of(m, d, dtype, seed=2, pad=pad, start=start), ids_of(m, rows, "skew", index), rows, 0.5)


def test_keys_that_need_three_digits():
    """2^22 rows and more: three digits of the sort."""
    rows, m = (1 << 23) + 5, 9000
    ids = ids_of(m, rows, "any")
    ids[::7] = rows - 1
    ids[1::7] = 1 << 22
    check_gradient(table_of(m, 4, torch.float32), ids, rows, 1.0)


def test_offsets_beyond_32_bits():
    """A table of 2^32 + bytes: the last rows' places are beyond what 32 bits address."""
    rows, d = 40_000_000, 128
    table = torch.empty(rows, d, dtype=torch.float16, device="cuda")
    last = table_of(5, d, torch.float16)
    table[-5:] = last
    table[:5] = 2 * last
    ids = torch.tensor([rows - 1, 0, rows - 5, 4, rows], device="cuda")
    got = ops().embedding(table, ids)
    assert torch.equal(got[:4], torch.stack([last[4], 2 * last[0], last[0], 2 * last[4]])) and not got[4].any()
    del table
    grad = ops().embedding_backward(last, ids, rows)
    assert torch.equal(grad[ids[:4]], last[:4]) and int(grad.view(torch.int16).count_nonzero()) == int(last[:4].view(torch.int16).count_nonzero())
    looked_up, part, count = ops().embedding_backward_rows(last, ids, rows)
    assert looked_up.tolist() == [0, 4, rows - 5, rows - 1, -1] and torch.equal(part[:4], last[[1, 3, 2, 0]])


def test_gradient_against_differences():
    """The lookup is linear: its difference along a direction is the gradient's product with it, up to roundings."""
    table, t, ids, dy = table_of(40, 24, torch.float32), table_of(40, 24, torch.float32, seed=5), ids_of(300, 40, "skew"), table_of(300, 24, torch.float32, seed=6)
    grad = ops().embedding_backward(dy, ids, 40, 1.5)
    change = (ops().embedding(table + t, ids, 1.5).double() - ops().embedding(table, ids, 1.5).double()) * dy.double()
    room = 2.0 ** -21 * float((dy.abs().double() * (ops().embedding(table.abs() + t.abs(), ids, 1.5).double())).sum()) + 60 * R.U * float((grad.abs() * t.abs()).sum())
    assert abs(float(change.sum()) - float((grad.double() * t.double()).sum())) < room


def test_numbers_that_are_none_stay_in_their_row():
    ids, dy = ids_of(5000, 50, "any"), table_of(5000, 8, torch.float32)
    dy[ids == 7] = float("nan")
    grad = ops().embedding_backward(dy, ids, 50)
    assert torch.isnan(grad[7]).all() and int(torch.isnan(grad).sum()) == 8
    dy[:] = float("nan")
    assert not ops().embedding_backward(dy, ids_of(5000, 50, "nowhere"), 50).any()


def test_nothing():
    o = ops()
    none = torch.empty(0, dtype=torch.int64, device="cuda")
    assert o.embedding(table_of(3, 4, torch.float32), none).shape == (0, 4)
    assert not o.embedding_backward(torch.empty(0, 4, device="cuda"), none, 3).any()
    looked_up, rows, count = o.embedding_backward_rows(torch.empty(0, 4, device="cuda"), none, 3)
    assert looked_up.shape == (0,) and rows.shape == (0, 4) and int(count) == 0
    ids = torch.tensor([0, -1], device="cuda")
    assert not o.embedding(torch.empty(0, 4, device="cuda"), ids).any()
    assert o.embedding_backward(torch.ones(2, 4, device="cuda"), ids, 0).shape == (0, 4)
    looked_up, rows, count = o.embedding_backward_rows(torch.ones(2, 4, device="cuda"), ids, 0)
    assert looked_up.tolist() == [-1, -1] and not rows.any() and int(count) == 0
    looked_up, rows, count = o.embedding_backward_rows(torch.ones(5000, 4, device="cuda"), ids_of(5000, 3, "any"), 0)
    assert (looked_up == -1).all() and not rows.any() and int(count) == 0
    looked_up, rows, count = o.embedding_backward_rows(torch.ones(2, 0, device="cuda"), ids, 5)
    assert int(count) == 0 and rows.shape == (2, 0)


def test_the_same_bits_every_time_and_in_a_graph():
    ids, dy, table = ids_of(30000, 400, "skew"), table_of(30000, 128, torch.float32), table_of(400, 128, torch.float32)

    def all_of():
        return (ops().embedding(table, ids, 2.0), ops().embedding_backward(dy, ids, 400, 2.0)) + tuple(ops().embedding_backward_rows(dy, ids, 400, 2.0))

    first = all_of()
    assert all(torch.equal(a, b) for a, b in zip(first, all_of()))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        all_of()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = all_of()
    ids.copy_(ids_of(30000, 400, "outside", seed=77))
    dy.copy_(table_of(30000, 128, torch.float32, seed=78))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, all_of()))


def test_refusals():
    o = ops()
    table, ids, dy = table_of(10, 8, torch.float32), ids_of(6, 10, "any"), table_of(6, 8, torch.float32)
    bad = [lambda: o.embedding(table.cpu(), ids), lambda: o.embedding(table, ids.cpu()), lambda: o.embedding(table.double(), ids), lambda: o.embedding(table, ids.float()),
           lambda: o.embedding(table, ids.to(torch.int16)), lambda: o.embedding(table[0], ids), lambda: o.embedding(table.t(), ids), lambda: o.embedding(table, ids[::2]),
           lambda: o.embedding(table.clone().requires_grad_(), ids), lambda: o.embedding_backward(dy[:5], ids, 10), lambda: o.embedding_backward(dy.t(), ids, 10),
           lambda: o.embedding_backward(dy, ids, -1), lambda: o.embedding_backward(dy, ids, 2 ** 31), lambda: o.embedding_backward(dy[0], ids, 10),
           lambda: o.embedding_backward(dy.clone().requires_grad_(), ids, 10), lambda: o.embedding_backward_rows(dy.double(), ids, 10)]
    for call in bad:
        with pytest.raises(RuntimeError):
            call()
    with pytest.raises(TypeError):
        o.embedding(table, [1, 2])
