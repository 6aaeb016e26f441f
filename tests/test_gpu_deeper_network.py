"""GraphSAGE with learned rows, norm between the layers and activations in 8 bits: the modules, a network of all of them, its gradients and memory."""
import math

import pytest
import torch

import learn_reference as R

pytestmark = pytest.mark.gpu


def minibatch(layers=3, n=20000, seed=1, batch=300):
    from f2cgt_b200 import sage, synth
    indptr, indices = synth.power_law_graph(n, 12, 2.1, seed=1, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (n, 4), generator=g, dtype=torch.uint8, device="cuda")
    books = torch.randn(4, 256, 32, generator=g, device="cuda")
    cm = sage.CompressionManager(128, ["vq"], [(32, 8)], [books], [codes])
    seeds = torch.randperm(n, generator=g, device="cuda")[:batch]
    return cm, next(iter(sage.GPUSamplingDataloader(indptr, indices, seeds, batch, (5, 4, 3)[:layers], shuffle=False)))[2]


@pytest.mark.parametrize("relu", [False, True])
@pytest.mark.parametrize("int8", [False, True])
@pytest.mark.parametrize("dtype", R.TYPES)
def test_layer_norm_module(dtype, int8, relu):
    from f2cgt_b200 import ops, sage
    torch.manual_seed(0)
    norm = sage.LayerNorm(200, relu=relu, int8=int8).cuda()
    with torch.no_grad():
        norm.weight.normal_(1, 0.2)
        norm.bias.normal_(0, 0.2)
    x = torch.randn(300, 200, device="cuda").to(dtype).requires_grad_()
    y = norm(x)
    assert torch.equal(y, ops.layer_norm(x.detach(), norm.weight.detach(), norm.bias.detach(), relu=relu)) and y.requires_grad
    y.sum().backward()  # (a gradient whose rows are all one number)
    _, saved = ops.layer_norm_train(x.detach(), norm.weight.detach(), norm.bias.detach(), relu=relu, int8=int8)
    dx, dw, db = ops.layer_norm_backward(torch.ones_like(x), saved, norm.weight.detach())
    assert torch.equal(x.grad, dx) and torch.equal(norm.weight.grad, dw) and torch.equal(norm.bias.grad, db)
    with torch.no_grad():
        assert torch.equal(norm(x), y)
    norm.requires_grad_(False)
    assert not norm(x.detach()).requires_grad
    (again,) = torch.autograd.grad(norm(x).float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):
        again.sum().backward()


@pytest.mark.parametrize("sparse", [False, True])
def test_node_embedding_module(sparse):
    from f2cgt_b200 import ops, sage
    torch.manual_seed(0)
    rows = sage.NodeEmbedding(500, 32, scale=2.0, sparse=sparse, device="cuda")
    ids = torch.randint(-1, 500, (40, 30), device="cuda")
    y = rows(ids)
    dy = torch.randn_like(y)
    y.backward(dy)
    want = ops.embedding_backward(dy, ids, 500, 2.0)
    assert torch.equal(y, ops.embedding(rows.weight.detach(), ids, 2.0))
    if sparse:
        grad = rows.weight.grad
        looked_up, part, count = ops.embedding_backward_rows(dy, ids, 500, 2.0)
        assert grad.is_sparse and torch.equal(grad._indices()[0], torch.unique(ids[ids >= 0])) and torch.equal(grad._values(), part[:int(count)])
        assert torch.equal(grad._indices()[0], looked_up[:int(count)]) and torch.equal(grad.to_dense(), want)
        before = rows.weight.detach().clone()
        torch.optim.SparseAdam(list(rows.parameters()), lr=0.1).step()
        touched = torch.zeros(500, dtype=torch.bool, device="cuda")
        touched[ids[ids >= 0]] = True
        assert torch.equal((rows.weight != before).any(1), touched)
    else:
        assert torch.equal(rows.weight.grad, want)
        # gradients of two lookups of the same rows add up
        rows(ids).backward(dy)
        assert torch.equal(rows.weight.grad, want + want)
    with torch.no_grad():
        assert torch.equal(rows(ids), ops.embedding(rows.weight.detach(), ids, 2.0))


def plain(model, blocks, weights):
    """The network's definition in 64 bits over ``weights`` (by name), in torch operations, without dropout."""
    h = weights["embedding.weight"] * model.embedding.scale
    h = h[blocks[0]["src_nodes"]]
    for i, block in enumerate(blocks):
        n = block["dst_nodes"].numel()
        deg = (block["indptr"][1:] - block["indptr"][:-1]).long()
        dst = torch.repeat_interleave(torch.arange(n, device="cuda"), deg)
        mean = torch.zeros(n, h.shape[1], dtype=h.dtype, device="cuda").index_add(0, dst, h[block["indices_local"][:dst.numel()].long()]) / deg.clamp(min=1)[:, None]
        at = f"layers.{i}."
        h = h[:n] @ weights[at + "fc_self.weight"].t() + weights[at + "fc_self.bias"] + mean @ weights[at + "fc_neigh.weight"].t()
        if i + 1 < len(blocks):
            z = h - h.mean(1, keepdim=True)
            h = z / ((z * z).mean(1, keepdim=True) + 1e-5).sqrt() * weights[f"norms.{i}.weight"] + weights[f"norms.{i}.bias"]
            h = h.relu()
    return h


def network(cm, norm=True, activations="float", embedding=True, dropout=0.0, hidden=64, seed=0):
    from f2cgt_b200 import sage
    torch.manual_seed(seed)
    rows = sage.NodeEmbedding(20000, 128, scale=0.5) if embedding else None
    model = sage.SAGE(128, hidden, 10, 3, dropout, None if embedding else cm, norm=norm, activations=activations, embedding=rows).cuda()
    with torch.no_grad():
        for name, p in model.named_parameters():
            if "norms" in name or name.endswith("bias"):
                p.add_(0.2 * torch.randn_like(p))
    return model


@pytest.mark.parametrize("activations", ["float", "int8"])
def test_a_network_of_all_of_them(activations):
    """Answers and gradients against the definition in 64 bits.  Products of at most 128 terms in single precision, three layers: 1e-5 of the norms
    with room; in the gradients a value within such a rounding of a ReLU's corner may fall on the other side - of some 600,000 of deviation one, 0.5 are
    expected within 1e-6 -, and one of n open ones is 1 / sqrt(n) of the norm, 2e-3: 5e-3.  With 8 bits a kept value is half a step off, at most 7 deviations / 255 / 2 of them and 1 / 12 squared on average: 0.8 % of the deviation; a gradient
    is a product of one such with another that went through two more: below 3 % of its norm."""
    cm, blocks = minibatch()
    model = network(cm, activations=activations)
    weights = {k: v.detach().double().requires_grad_() for k, v in model.named_parameters()}
    want = plain(model, blocks, weights)
    dy = torch.randn(want.shape, device="cuda", dtype=torch.float64)
    (want * dy).sum().backward()
    got = model(blocks)
    assert float((got.double() - want).norm() / want.norm()) < 1e-5
    got.backward(dy.float())
    for name, p in model.named_parameters():
        off = float((p.grad.double() - weights[name].grad).norm() / weights[name].grad.norm())
        assert off < (5e-3 if activations == "float" else 0.03), (name, off)
    again = network(cm, activations=activations)
    again(blocks).backward(dy.float())
    assert torch.equal(model.layers[2].fc_self.weight.grad, again.layers[2].fc_self.weight.grad)


@pytest.mark.parametrize("norm,embedding", [(False, False), (True, False), (False, True), (True, True)])
def test_8_bit_gradients_are_near_the_others(norm, embedding):
    """(the bound of the test above)"""
    cm, blocks = minibatch()
    grads = []
    for activations in ("float", "int8"):
        model = network(cm, norm=norm, activations=activations, embedding=embedding)
        loss = torch.nn.functional.cross_entropy(model(blocks), torch.arange(300, device="cuda") % 10)
        loss.backward()
        grads.append([p.grad.clone() for p in model.parameters()])
    for a, b in zip(*grads):
        assert float((a - b).norm() / a.norm()) < 0.03


def test_what_was_there_is_as_it_was():
    """Without the options the network is the same object and takes the same path: no names of its state change."""
    from f2cgt_b200 import sage
    cm, blocks = minibatch()
    torch.manual_seed(0)
    model = sage.SAGE(128, 64, 10, 3, 0.0, cm).cuda()
    assert sorted(model.state_dict()) == sorted(f"layers.{i}.{n}" for i in range(3) for n in ("fc_self.weight", "fc_self.bias", "fc_neigh.weight"))
    assert model._plain_weights() is not None and network(cm)._plain_weights() is None
    assert network(cm, norm=False, activations="int8", embedding=False)._plain_weights() is None


def test_memory_of_kept_activations():
    """What a forward pass holds for the backward pass: a value of 4 bytes each from the product, the norm and the own rows becomes little more than one."""
    cm, blocks = minibatch(n=200000, batch=8000)
    held = {}
    for activations in ("float", "int8"):
        model = network(cm, activations=activations, embedding=False, hidden=256)
        model(blocks).sum().backward()
        torch.cuda.synchronize()
        before = torch.cuda.memory_allocated()
        out = model(blocks)
        torch.cuda.synchronize()
        held[activations] = torch.cuda.memory_allocated() - before
        del out, model
    assert held["int8"] < 0.4 * held["float"], held


@pytest.mark.parametrize("norm,embedding", [(True, False), (False, True), (True, True)])
def test_answers_in_8_bits(norm, embedding):
    """Products in 8 bits: the bound of the plain network's test, 4 % of the norm."""
    from f2cgt_b200 import sage
    cm, blocks = minibatch()
    model = network(cm, norm=norm, embedding=embedding).eval()
    with torch.no_grad():
        want = model(blocks)
    got = sage.Int8SAGE(model)(blocks)
    assert float((got - want).norm() / want.norm()) < 0.04


def test_dropout_training_and_refusals():
    from f2cgt_b200 import sage
    cm, blocks = minibatch()
    model, other = network(cm, activations="int8", dropout=0.5), network(cm, dropout=0.5)
    torch.manual_seed(3)
    a = model(blocks)
    torch.manual_seed(3)
    assert torch.equal(other(blocks), a)  # what is kept has no say in the answer
    a.sum().backward()
    assert all(torch.isfinite(p.grad).all() for p in model.parameters())
    rows = sage.NodeEmbedding(10, 64)
    for call in (lambda: sage.SAGE(128, 8, 3, 2, 0.0, cm, activations="int4"), lambda: sage.SAGE(128, 8, 3, 2, 0.0, None, embedding=rows), lambda: sage.SAGE(64, 8, 3, 2, 0.0, cm, embedding=rows)):
        with pytest.raises(ValueError):
            call()


def test_training_command(monkeypatch):
    from f2cgt_b200 import train_graphsage as tg
    monkeypatch.setitem(tg.PRESETS, "small", dict(tg.PRESETS["small"], nodes=5000, degree=10, train=512, fan_out=(3, 3)))
    for options in (dict(norm=True), dict(norm=True, activations="int8"), dict(activations="int8", optimizer="muon", norm=True), dict(norm=True, activations="int8", embedding=64, answer_int8=True)):
        record = tg.train(epochs=2, batch_size=256, **options)
        assert all(math.isfinite(v) for v in record["loss_last_step_per_epoch"])
        assert record["norm"] is options.get("norm", False) and record["activations"] == options.get("activations", "float") and record["embedding"] == options.get("embedding", 0)
    with pytest.raises(ValueError):
        tg.train(epochs=1, max_steps=1, embedding=64, optimizer="muon")
    with pytest.raises(ValueError):
        tg.train(epochs=1, max_steps=1, activations="int4")


def test_a_step_in_a_graph():
    """Forward and backward of the modules, captured and replayed on other inputs: what eager calls give on them."""
    from f2cgt_b200 import sage
    torch.manual_seed(0)
    rows, norm = sage.NodeEmbedding(300, 96, scale=2.0, device="cuda"), sage.LayerNorm(96, relu=True, int8=True).cuda()
    ids, dy = torch.randint(-1, 300, (5000,), device="cuda"), torch.randn(5000, 96, device="cuda")
    parameters = [rows.weight, norm.weight, norm.bias]

    def step():
        return torch.autograd.grad(norm(rows(ids)), parameters, dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    ids.copy_(torch.randint(-1, 300, (5000,), device="cuda"))
    dy.copy_(torch.randn(5000, 96, device="cuda"))
    graph.replay()
    assert all(torch.equal(a, b) for a, b in zip(captured, step()))


def test_other_streams_and_threads():
    """The modules' backward pass runs on the stream of the forward one, and from several threads at once."""
    import threading
    from f2cgt_b200 import sage
    cm, blocks = minibatch()
    model = network(cm, activations="int8")
    dy = torch.randn(300, 10, device="cuda")
    want = torch.autograd.grad(model(blocks), list(model.parameters()), dy)
    torch.cuda.synchronize()
    found, errors = [None] * 3, []

    def one(i):
        try:
            stream = torch.cuda.Stream()
            with torch.cuda.stream(stream):
                for _ in range(3):
                    found[i] = torch.autograd.grad(model(blocks), list(model.parameters()), dy)
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=one, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    for got in found:
        for a, b, (name, _) in zip(got, want, model.named_parameters()):
            # the aggregation's gradient adds with atomics: everything behind it may differ in its roundings
            assert float((a - b).norm()) <= 1e-5 * float(b.norm()), name
