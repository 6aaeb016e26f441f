"""GPU: a GraphSAGE network trained with orthogonalised updates and answering in 8-bit integers."""
import math

import pytest

pytestmark = pytest.mark.gpu
torch = pytest.importorskip("torch")


def network(layers=3, hidden=64, classes=10, bias=True, seed=0):
    from f2cgt_b200 import sage, synth
    n, D = 20000, 128
    indptr, indices = synth.power_law_graph(n, 12, 2.1, seed=1, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, 4), generator=g, dtype=torch.uint8, device="cuda")
    books = torch.randn(4, 256, 32, generator=g, device="cuda")
    cm = sage.CompressionManager(D, ["vq"], [(32, 8)], [books], [codes])
    torch.manual_seed(seed)
    model = sage.SAGE(D, hidden, classes, layers, 0.5, cm).cuda()
    with torch.no_grad():
        for layer in model.layers:
            layer.fc_self.bias.normal_(0, 0.3)
    if not bias:
        for layer in model.layers:
            layer.fc_self.bias = None
    seeds = torch.randperm(n, generator=g, device="cuda")[:300]
    loader = sage.GPUSamplingDataloader(indptr, indices, seeds, 300, (5, 4, 3)[:layers], shuffle=False)
    return model, next(iter(loader))[2]


@pytest.mark.parametrize("bias", [True, False])
@pytest.mark.parametrize("layers", [1, 2, 3])
def test_answers_in_8_bits_are_near_the_network_s(capi, layers, bias):
    # rows of some 256 values are rounded to steps of max / 127: 1 % of their norm at most, and as much for the weights, in three layers: 4 %
    from f2cgt_b200 import sage
    model, blocks = network(layers, bias=bias)
    model.eval()
    with torch.no_grad():
        want = model(blocks)
    got = sage.Int8SAGE(model)(blocks)
    assert got.shape == want.shape and got.dtype == torch.float32
    assert float((got - want).norm() / want.norm()) < 0.04


def test_an_8_bit_layer_is_quantisation_and_product(capi):
    from f2cgt_b200 import ops, sage
    model, blocks = network()
    answer = sage.Int8SAGE(model)
    first = blocks[0]
    cm = model.layers[0].sm
    own, mean = cm.decode_rows(first["dst_nodes"]), cm.aggregate(first["indptr"], first["indices_global"])
    codes, scales, bias = answer.layers[0]
    h = ops.int8_mm(*ops.int8_quantize(own, mean), codes, scales, bias, relu=True)
    assert torch.equal(h, ops.int8_linear(own, codes, scales, bias, relu=True, x2=mean))
    for (codes, scales, bias), block, relu in zip(answer.layers[1:], blocks[1:], (True, False)):
        mean = ops.spmm_csr(h, block["indptr"], block["indices_local"])
        h = ops.int8_mm(*ops.int8_quantize(h[:block["dst_nodes"].numel()], mean), codes, scales, bias, relu=relu)
    assert torch.equal(h, answer(blocks))
    with pytest.raises(RuntimeError):
        answer(blocks[:2])


def test_the_optimiser_is_its_step_and_adam(capi):
    from f2cgt_b200 import ops
    from f2cgt_b200.muon import Muon
    from f2cgt_b200.train_graphsage import DirectFusedAdam
    torch.manual_seed(1)
    shapes = [(64, 128), (172, 64), (300, 40)]
    a = [torch.randn(s, device="cuda", requires_grad=True) for s in shapes] + [torch.randn(64, device="cuda", requires_grad=True)]
    b = [t.detach().clone() for t in a]
    mine = Muon(a, lr=0.05, weight_decay=0.1, adam_lr=0.01)
    vector = b[3].requires_grad_(True)
    adam, momenta = DirectFusedAdam([vector], lr=0.01), [torch.zeros(s, device="cuda") for s in shapes]
    for step in range(3):
        grads = [torch.randn_like(t) for t in a]
        for t, g in zip(a, grads):
            t.grad = g.clone()
        vector.grad = grads[3].clone()
        mine.step()
        with torch.no_grad():
            ops.muon_step(b[:3], grads[:3], momenta, mine.lr, weight_decay=0.1)
        adam.step()
        mine.lr *= 0.9
        adam.lr *= 0.9
    assert all(torch.equal(t, u) for t, u in zip(a, b))
    # what is saved goes on where it was
    c = [t.detach().clone().requires_grad_(True) for t in a]
    other = Muon(c, lr=1.0, weight_decay=0.1, adam_lr=0.2)
    other.load_state_dict({k: [x.clone() for x in v] if isinstance(v, list) else v for k, v in mine.state_dict().items()})
    for t, u in zip(a, c):
        t.grad = torch.randn_like(t)
        u.grad = t.grad.clone()
    mine.step()
    other.step()
    assert all(torch.equal(t, u) for t, u in zip(a, c))
    a[0].grad = None
    kept = a[0].detach().clone()
    mine.step()
    assert torch.equal(a[0], kept)
    mine.zero_grad()
    assert all(t.grad is None for t in a)
    mine.step()
    with pytest.raises(RuntimeError):
        Muon([torch.randn(4, 4, device="cuda").t().requires_grad_(), torch.randn(3, 5, requires_grad=True)])
    with pytest.raises(RuntimeError):
        other.load_state_dict(Muon(a[:2]).state_dict())


def test_weights_learn_as_under_the_formula(capi):
    """The losses of 150 steps are those of the same network whose updates are computed in 64 bits.  An update is 2^-20 off or so, of size 0.02 in
    weights of size 1; a hundred of them, each of which the later ones could double at most tenfold, leave the loss well within one per cent."""
    from f2cgt_b200.muon import Muon
    from f2cgt_b200.train_graphsage import DirectFusedAdam
    from test_gpu_newton_schulz import define

    def plain_step(matrices, momenta, lr):
        with torch.no_grad():
            for p, m in zip(matrices, momenta):
                m.mul_(0.95).add_(p.grad.double())
                p.sub_((lr * math.sqrt(max(1.0, p.shape[0] / p.shape[1])) * define(p.grad.double() + 0.95 * m)).float())

    def run(own):
        torch.manual_seed(2)
        x = torch.randn(2048, 96, device="cuda")
        y = torch.relu(x @ torch.randn(96, 48, device="cuda") / math.sqrt(96)) @ torch.randn(48, 8, device="cuda")
        net = torch.nn.Sequential(torch.nn.Linear(96, 64), torch.nn.ReLU(), torch.nn.Linear(64, 8)).cuda()
        matrices, vectors = [p for p in net.parameters() if p.dim() == 2], [p for p in net.parameters() if p.dim() == 1]
        optimizer = Muon(net.parameters(), lr=0.02) if own else DirectFusedAdam(vectors, lr=0.003)
        momenta = [torch.zeros_like(p, dtype=torch.float64) for p in matrices]
        losses = []
        for _ in range(150):
            loss = torch.nn.functional.mse_loss(net(x), y)
            net.zero_grad()
            loss.backward()
            if not own:
                plain_step(matrices, momenta, 0.02)
            optimizer.step()
            losses.append(float(loss.detach()))
        return losses

    mine, plain = run(True), run(False)
    assert all(abs(a - b) <= 0.01 * b for a, b in zip(mine, plain))
    assert mine[-1] < mine[0]


def test_training_with_orthogonalised_updates(capi, monkeypatch):
    from f2cgt_b200 import train_graphsage as tg
    monkeypatch.setitem(tg.PRESETS, "small", dict(tg.PRESETS["small"], nodes=5000, degree=10, train=512, fan_out=(3, 3)))
    record = tg.train(epochs=2, batch_size=256, optimizer="muon", answer_int8=True)
    assert record["optimizer"] == "muon" and all(math.isfinite(v) for v in record["loss_last_step_per_epoch"])
    assert record["int8"]["relative_error"] < 0.04
    assert "int8" not in tg.train(epochs=1, batch_size=256, max_steps=1)
    with pytest.raises(ValueError):
        tg.train(epochs=1, batch_size=256, max_steps=1, optimizer="sgd")
