"""CPU: the learning rates of Muon, on parameters that are no matrices (which Adam updates)."""
import pytest

torch = pytest.importorskip("torch")


def muon(**kw):
    from f2cgt_b200.muon import Muon
    return Muon([torch.zeros(3, requires_grad=True)], **kw)


def moved(optimizer):
    """what one step changes a parameter by, of gradients of one: Adam's rate"""
    p = optimizer.adam.params[0]
    before = p.detach().clone()
    p.grad = torch.ones_like(p)
    optimizer.step()
    return float((before - p.detach()).max())


def test_adam_s_rate_moves_with_the_rate():
    o = muon(lr=0.02, adam_lr=0.004)
    assert moved(o) == pytest.approx(0.004, rel=1e-5)
    o.lr = 0.01
    assert moved(o) == pytest.approx(0.002, rel=1e-4)
    o.lr = 0.0
    assert moved(o) == 0.0
    o.lr = 0.02
    assert moved(o) == pytest.approx(0.004, rel=1e-4)


def test_a_rate_of_zero_at_first_leaves_adam_s_alone():
    o = muon(lr=0.0, adam_lr=0.004)
    assert moved(o) == pytest.approx(0.004, rel=1e-5)
    for lr in (0.001, 0.01, 0.02):
        o.lr = lr
        assert o.lr == lr and moved(o) == pytest.approx(0.004, rel=1e-4)


@pytest.mark.parametrize("first,then", [((0.02, 0.004), (0.5, 0.3)), ((0.02, 0.004), (0.0, 0.3)), ((0.0, 0.004), (0.5, 0.3))])
def test_a_state_goes_on_with_its_own_rates(first, then):
    """in an optimiser that was built with others"""
    a, b = (muon(lr=lr, adam_lr=adam_lr) for lr, adam_lr in (first, then))
    a.lr = 0.01
    moved(a)
    b.load_state_dict(a.state_dict())
    assert b.lr == 0.01 and b.adam.lr == a.adam.lr
    for lr in (0.01, 0.03, 0.0, 0.02):
        a.lr = b.lr = lr
        assert b.adam.lr == a.adam.lr and moved(b) == pytest.approx(moved(a), rel=1e-5)


def test_a_state_without_adam_s_rate_is_taken():
    a, b = muon(lr=0.02, adam_lr=0.004), muon(lr=0.01, adam_lr=0.004)
    state = {k: v for k, v in a.state_dict().items() if k not in ("adam_lr", "adam_ratio")}
    b.load_state_dict(state)
    assert b.lr == 0.02 and b.adam.lr == pytest.approx(0.008)


def test_a_torch_without_the_fused_kernel(monkeypatch):
    """The same updates, to the rounding of a step of 0.004 on values of one: 10 steps, 2^-23 of one each and of the steps themselves."""
    def run():
        g = torch.Generator().manual_seed(0)
        o = muon(lr=0.02, adam_lr=0.004)
        p = o.adam.params[0]
        with torch.no_grad():
            p.copy_(torch.rand(3, generator=g))
        for _ in range(10):
            p.grad = torch.randn(3, generator=g)
            o.step()
        return p.detach().clone()

    want = run()
    monkeypatch.delattr(torch, "_fused_adam_")
    assert float((run() - want).abs().max()) <= 20 * 2.0 ** -23
