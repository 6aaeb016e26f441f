"""Layer norm, 8-bit activations and learned rows at the ends of what they take."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def ops():
    from f2cgt_b200 import ops
    return ops


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("int8", [False, True])
def test_rows_without_columns(int8, relu):
    """The mean of no values is NaN, not what the memory held before."""
    held = [torch.full((5,), 7.0, device="cuda") for _ in range(8)]
    torch.cuda.synchronize()
    del held
    y, saved = ops().layer_norm_train(torch.empty(5, 0, device="cuda"), relu=relu, int8=int8)
    assert y.shape == (5, 0) and torch.isnan(saved.mean).all() and torch.isnan(saved.rstd).all()
    dx, dweight, dbias = ops().layer_norm_backward(torch.empty(5, 0, device="cuda"), saved)
    assert dx.shape == (5, 0) and dweight.shape == dbias.shape == (0,)


def test_what_is_refused_at_the_ends():
    from f2cgt_b200 import sage
    o = ops()
    with pytest.raises(RuntimeError, match="no columns"):
        o.checkpoint_weight_grad(torch.ones(9, 3, device="cuda"), o.checkpoint_int8(torch.empty(9, 0, device="cuda")))
    ids = torch.arange(12, device="cuda")[::2]
    rows = sage.NodeEmbedding(20, 8, device="cuda")
    for call in (lambda: rows(ids), lambda: o.embedding_backward(torch.ones(6, 8, device="cuda"), ids, 20), lambda: o.embedding_backward_rows(torch.ones(6, 8, device="cuda"), ids, 20)):
        with pytest.raises(RuntimeError, match="contiguous"):
            call()
    rows(ids.contiguous()).sum().backward()
    assert torch.equal(rows.weight.grad[:, 0], torch.bincount(ids, minlength=20).float())
