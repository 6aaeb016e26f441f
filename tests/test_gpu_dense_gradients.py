"""GPU: the dense operators have no derivative, and refuse every floating-point input that asks for one instead of dropping it."""
import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")

from f2cgt_b200 import ops  # noqa: E402


def calls():
    """(operator, its floating-point inputs by name, call)"""
    g = torch.Generator(device="cuda").manual_seed(0)
    rnd = lambda *s: torch.rand(*s, generator=g, device="cuda")  # noqa: E731
    codes, w = torch.zeros(4, 16, dtype=torch.int8, device="cuda"), torch.ones(6, 16, dtype=torch.int8, device="cuda")
    return [("int8_quantize", dict(x=rnd(4, 16), x2=rnd(4, 8)), lambda x, x2: ops.int8_quantize(x, x2)),
            ("int8_mm", dict(scales=rnd(4), w_scales=rnd(6), bias=rnd(6)), lambda scales, w_scales, bias: ops.int8_mm(codes, scales, w, w_scales, bias)),
            ("int8_linear", dict(x=rnd(4, 10), x2=rnd(4, 6), w_scales=rnd(6), bias=rnd(6)),
             lambda x, x2, w_scales, bias: ops.int8_linear(x, w, w_scales, bias, x2=x2)),
            ("orthogonalize", dict(g=rnd(4, 6), out=rnd(4, 6)), lambda g, out: ops.orthogonalize(g, out=out)),
            ("muon_step", dict(w=rnd(4, 6), g=rnd(4, 6), m=rnd(4, 6)), lambda w, g, m: ops.muon_step([w], [g], [m], 0.1))]


INPUTS = [(i, name) for i, names in enumerate(("x x2", "scales w_scales bias", "x x2 w_scales bias", "g out", "w g m")) for name in names.split()]


@pytest.mark.parametrize("which,name", INPUTS)
def test_inputs_that_require_a_gradient(which, name):
    op, inputs, call = calls()[which]
    call(**inputs)
    asking = dict(inputs, **{name: inputs[name].clone().requires_grad_()})
    with pytest.raises(RuntimeError, match=f"{op} has no gradient"):
        call(**asking)
    with torch.no_grad():
        call(**asking)


@pytest.mark.parametrize("which,name", INPUTS)
def test_inputs_with_a_tangent(which, name):
    from torch.autograd import forward_ad
    op, inputs, call = calls()[which]
    with forward_ad.dual_level():
        call(**inputs)
        dual = dict(inputs, **{name: forward_ad.make_dual(inputs[name], torch.ones_like(inputs[name]))})
        with pytest.raises(RuntimeError, match=f"{op} has no forward-mode derivative"):
            call(**dual)
        with torch.no_grad(), pytest.raises(RuntimeError):  # which leaves that mode alone
            call(**dual)
        with forward_ad._set_fwd_grad_enabled(False):
            call(**dual)
