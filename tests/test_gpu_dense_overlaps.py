"""GPU: tensors of one call that share memory are refused where the call writes one of them, and neighbours of one buffer are not."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from f2cgt_b200 import ops  # noqa: E402


@pytest.mark.parametrize("shape", [(64, 96), (300, 200)])
def test_matrices_of_a_step(shape):
    rnd = lambda: torch.randn(shape, device="cuda")  # noqa: E731
    w, v, g, m, n = rnd(), rnd(), rnd(), rnd(), rnd()
    kept = [t.clone() for t in (w, v, g, m, n)]
    for weights, grads, momenta in (([w, w], [g, g], [m, n]), ([w, v], [g, g], [m, m]), ([w], [w], [m]), ([w], [g], [w]), ([w], [g], [g])):
        with pytest.raises(RuntimeError, match="shares memory"):
            ops.muon_step(weights, grads, momenta, 0.1)
    assert all(torch.equal(a, b) for a, b in zip((w, v, g, m, n), kept))
    ops.muon_step([w, v], [g, g], [m, n], 0.1)  # one gradient for two weights is read only
    # gradients, weights and momenta that are views of flat buffers, as a data-parallel trainer's are
    size = w.numel()
    flat = [torch.cat([a.flatten(), b.flatten()]) for a, b in ((kept[0], kept[1]), (g, g), (kept[3], kept[4]))]
    views = [[f[:size].view(shape), f[size:].view(shape)] for f in flat]
    ops.muon_step(*views, 0.1)
    assert torch.equal(views[0][0], w) and torch.equal(views[0][1], v) and torch.equal(views[2][0], m) and torch.equal(views[2][1], n)


@pytest.mark.parametrize("rows,cols", [(64, 96), (300, 200)])
def test_results_of_matrices(rows, cols):
    stack = torch.randn(4, rows, cols, device="cuda")
    kept = stack.clone()
    want = ops.orthogonalize(stack)
    for g, out in ((stack[:3], stack[1:]), (stack[1:], stack[:3]), (stack[0], stack.view(-1)[4:4 + rows * cols].view(rows, cols))):
        with pytest.raises(RuntimeError, match="memory"):
            ops.orthogonalize(g, out=out)
    assert torch.equal(stack, kept)
    ops.orthogonalize(stack[:2], out=stack[2:])
    assert torch.equal(stack[2:], want[:2]) and torch.equal(stack[:2], kept[:2])
    ops.orthogonalize(stack[:2], out=stack[:2])
    assert torch.equal(stack[:2], want[:2])
