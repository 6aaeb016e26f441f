"""The rows alone of a gradient of many places: numbered right, and in a time that grows with the places."""
import pytest
import torch

from test_gpu_embedding import check_gradient, ids_of, ops, table_of

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("how", ["any", "one", "skew", "outside", "nowhere", "descending"])
@pytest.mark.parametrize("m,rows,d", [(256 * 1024, 300_000, 4), (256 * 1024 + 1, 300_000, 4), (1_100_003, 5_000_000, 4), (1_100_003, 3000, 4), (300_000, 70_000, 130)])
def test_gradient(m, rows, d, how):
    check_gradient(table_of(m, d, torch.float32, seed=2), ids_of(m, rows, how), rows, 1.7)


def test_time_grows_with_the_places():
    """2^24 places are 16 times 2^20.  Reading every tile's number for every stretch would make it 256 times for that part, 69 GB."""
    times = []
    for m in (1 << 20, 1 << 24):
        ids, dy = ids_of(m, 1 << 24, "any"), torch.ones(m, 4, dtype=torch.bfloat16, device="cuda")
        best = float("inf")
        for _ in range(4):
            a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
            a.record()
            looked_up, rows, count = ops().embedding_backward_rows(dy, ids, 1 << 24)
            b.record()
            torch.cuda.synchronize()
            best = min(best, a.elapsed_time(b))
        times.append(best)
        assert int(rows.float().sum() / 4) == m
        del looked_up, rows, dy, ids
    assert times[1] < 24 * times[0], times


def test_the_same_in_a_graph_and_beside_another():
    """Places whose tiles are numbered by a launch of its own, in captured calls and two at once."""
    m, rows = 300_000, 1 << 20
    ids, dy = ids_of(m, rows, "outside"), table_of(m, 4, torch.float32)
    first = ops().embedding_backward_rows(dy, ids, rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        beside = [ops().embedding_backward_rows(dy, ids, rows) for _ in range(3)]
    here = [ops().embedding_backward_rows(dy, ids, rows) for _ in range(3)]
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for got in beside + here for a, b in zip(got, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = ops().embedding_backward_rows(dy, ids, rows)
    ids.copy_(ids_of(m, rows, "skew", seed=5))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, ops().embedding_backward_rows(dy, ids, rows)))
