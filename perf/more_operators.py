"""What a deeper GraphSAGE network trains with, as operators: learned rows for nodes, layer norm between layers, and activations kept
in 8 bits until the backward pass.  ``listed`` and ``draw`` say on which sizes, ``run`` makes one call or one call and its gradient.

Kinds:
  norm     ops.layer_norm: y = (x - mean) / sqrt(var + eps) * weight + bias over rows, with or without ReLU
  train    ops.layer_norm_train and ops.layer_norm_backward: the same with its gradients; ``keep`` says what stays for the backward
           pass: the rows as they are, or in 8 bits
  back     ops.layer_norm_backward alone, from rows in 8 bits and the ReLU's bits
  pack     ops.checkpoint_int8 and ops.checkpoint_values: rows to 8 bits and back
  wgrad    ops.checkpoint_weight_grad: the gradient of a linear layer's weight and bias, its input in 8 bits
  embed    ops.embedding and ops.embedding_backward or ops.embedding_backward_rows: rows of a table, scaled, and the table's gradient:
           dense, or the ids that were looked up, ascending, -1 behind them, and their rows, zeros behind them; an id outside the table
           (padding: -1) is a row of zeros and has no gradient

Definitions.  8 bits: of every row, 128 columns at a time are a group; low = its smallest value, step = (largest - low) / 255, code =
round-to-even((x - low) / step), the differences and quotients in single precision; a code stands for low + step * code.
Bits of ReLU: column c of a row is bit c % 8 of its byte c // 8.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS, GROUP = 1e-5, 128


def listed():
    return [
        # one node's hidden row: the smallest call, latency only
        dict(name="norm_row", kind="norm", m=1, d=128, dtype="f32", relu=True),
        # a wide layer over many rows: bound by memory
        dict(name="norm_wide", kind="norm", m=16_384, d=4096, dtype="bf16", relu=False),
        # the hidden layer over the outermost block of a minibatch, forward and backward
        dict(name="train_block", kind="train", m=59_000, d=128, dtype="f32", keep="rows"),
        # a width that is no multiple of anything, the rows kept in 8 bits
        dict(name="train_ragged", kind="train", m=5003, d=602, dtype="f16", keep="int8"),
        # the backward pass of norm and ReLU in the 256-column preset, everything it needs in 9 bits a value
        dict(name="back_block", kind="back", m=37_237, d=256, dtype="f32"),
        # the outermost block's activations to 8 bits and back
        dict(name="pack_block", kind="pack", m=59_000, d=128, dtype="f32"),
        # activations of a wide layer
        dict(name="pack_wide", kind="pack", m=8192, d=4096, dtype="bf16"),
        # the last layer's weights from the seeds of a minibatch: latency
        dict(name="wgrad_seeds", kind="wgrad", m=1024, n=172, k=128, dtype="f32"),
        # a hidden layer's weights from the outermost block
        dict(name="wgrad_block", kind="wgrad", m=59_000, n=128, k=128, dtype="f32"),
        # a wide layer: bound by the tensor cores
        dict(name="wgrad_wide", kind="wgrad", m=16_384, n=2048, k=4096, dtype="bf16"),
        # labels as inputs: few rows, each looked up hundreds of times
        dict(name="embed_labels", kind="embed", rows=172, m=59_000, d=128, dtype="f32", sparse=False, skew=1.5, pad=0.0),
        # learned rows of every node, looked up for a hop's neighbours: the table's gradient only where it is not zero
        dict(name="embed_nodes", kind="embed", rows=2_449_029, m=121_000, d=128, dtype="f32", sparse=True, skew=2.0, pad=0.02),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["norm", "train", "back", "pack", "wgrad", "wgrad", "embed", "embed"])
    dtype = rng.choice(["f32", "f16", "bf16"])
    if kind == "wgrad":
        m, n, k = log(1, 65_536), log(1, 4096), log(1, 4096)
        if rng.random() < 0.5:
            n, k = max(4, n // 4 * 4), max(16, k // 16 * 16)
        return dict(kind=kind, m=max(1, min(m, 60_000_000_000 // (n * k))), n=n, k=k, dtype=dtype)
    if kind == "embed":
        rows, d = log(1, 2_449_029), log(1, 4096)
        if rng.random() < 0.5:
            d = max(8, d // 8 * 8)
        rows = max(1, min(rows, 300_000_000 // d))
        m = max(1, min(log(1, 262_144), 16_000_000 // d))
        return dict(kind=kind, rows=rows, m=m, d=d, dtype=dtype, sparse=rows * d > 60_000_000 or rng.random() < 0.4, skew=rng.choice([1.0, 1.5, 2.0, 6.0]),
                    pad=rng.choice([0.0, 0.02]))
    m, d = log(1, 65_536), log(8, 8192)
    if rng.random() < 0.5:
        d = max(8, d // 8 * 8)
    m = max(1, min(m, (60_000_000 if kind == "norm" else 16_000_000) // d))
    c = dict(kind=kind, m=m, d=d, dtype=dtype)
    if kind == "norm":
        c["relu"] = rng.random() < 0.5
    if kind == "train":
        c["keep"] = rng.choice(["rows", "int8"])
    return c


def _activations(m, d, g, dev):
    """Rows as a linear layer gives them: columns of different means and widths."""
    return torch.randn(m, d, generator=g, device=dev) * (0.5 + torch.rand(d, generator=g, device=dev)) + 0.3 * torch.randn(d, generator=g, device=dev)


def _rows16(codes):
    """The codes with rows that start on 16-byte boundaries, as ops.checkpoint_int8 lays them out."""
    rows, d = codes.shape
    room = torch.zeros((rows, (d + 15) // 16 * 16), dtype=torch.uint8, device=codes.device)
    room[:, :d] = codes
    return room[:, :d]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "embed":
        s["table"] = torch.randn(c["rows"], c["d"], generator=g, device=dev).to(dt)
        # popular rows are looked up more often; which ones they are has nothing to do with their place in the table
        u = torch.rand(c["m"], generator=g, device=dev, dtype=torch.float64)
        popular = (u ** c["skew"] * c["rows"]).long().clamp_(max=c["rows"] - 1)
        ids = (popular * 1_000_003 + 7) % c["rows"]
        s["ids"] = torch.where(torch.rand(c["m"], generator=g, device=dev) < c["pad"], torch.full_like(ids, -1), ids)
        s["scale"] = math.sqrt(c["d"])
        s["dy"] = (torch.randn(c["m"], c["d"], generator=g, device=dev) / c["m"]).to(dt)
        return s
    if c["kind"] == "wgrad":
        x = _activations(c["m"], c["k"], g, dev).relu_()
        codes, s["scales"] = _encode(x.to(dt))
        s["codes"] = _rows16(codes)
        s["dy"] = torch.randn(c["m"], c["n"], generator=g, device=dev).to(dt)
        return s
    m, d = c["m"], c["d"]
    s["x"] = _activations(m, d, g, dev).to(dt)
    if c["kind"] == "pack":
        return s
    s["weight"] = 1 + 0.2 * torch.randn(d, generator=g, device=dev)
    s["bias"] = 0.2 * torch.randn(d, generator=g, device=dev)
    if c["kind"] != "norm":
        s["dy"] = torch.randn(m, d, generator=g, device=dev).to(dt)
    if c["kind"] == "back":
        y, s["mean"], s["rstd"] = _norm(s["x"].float(), s["weight"], s["bias"])
        bits = torch.zeros(m, (d + 7) // 8 * 8, dtype=torch.int32, device=dev)
        bits[:, :d] = y > 0
        s["active"] = (bits.view(m, -1, 8) << torch.arange(8, dtype=torch.int32, device=dev)).sum(2).to(torch.uint8)
        codes, s["scales"] = _encode(s.pop("x"))
        s["codes"] = _rows16(codes)
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from f2cgt_b200 import ops
    c = s["case"]
    if c["kind"] == "norm":
        return ops.layer_norm(s["x"], s["weight"], s["bias"], eps=EPS, relu=c["relu"])
    if c["kind"] == "train":
        y, saved = ops.layer_norm_train(s["x"], s["weight"], s["bias"], eps=EPS, int8=c["keep"] == "int8")
        return (y,) + tuple(ops.layer_norm_backward(s["dy"], saved, s["weight"]))
    if c["kind"] == "back":
        saved = ops.NormSaved(ops.Int8Checkpoint(s["codes"], s["scales"]), s["mean"], s["rstd"], s["active"])
        return tuple(ops.layer_norm_backward(s["dy"], saved, s["weight"]))
    if c["kind"] == "pack":
        return ops.checkpoint_values(ops.checkpoint_int8(s["x"]), dtype=s["x"].dtype)
    if c["kind"] == "wgrad":
        return tuple(ops.checkpoint_weight_grad(s["dy"], ops.Int8Checkpoint(s["codes"], s["scales"])))
    y = ops.embedding(s["table"], s["ids"], scale=s["scale"])
    if c["sparse"]:
        looked_up, grad, _ = ops.embedding_backward_rows(s["dy"], s["ids"], c["rows"], scale=s["scale"])
        return y, looked_up, grad
    return y, ops.embedding_backward(s["dy"], s["ids"], c["rows"], scale=s["scale"])


# ---------------------------------------------------------------- the operators in elementary operations, 32 bits
def _groups(x, fill):
    """[m, groups, 128] of the rows, missing columns of the last group filled with what ``fill`` gives."""
    m, d = x.shape
    n = (d + GROUP - 1) // GROUP
    room = x.new_full((m, n * GROUP), fill)
    room[:, :d] = x
    return room.view(m, n, GROUP)


def _encode(x):
    x = x.float()
    low = _groups(x, math.inf).amin(2)
    step = (_groups(x, -math.inf).amax(2) - low) / torch.full_like(low, 255.0)
    q = (_groups(x, 0.0) - low[:, :, None]) / step[:, :, None]
    q = torch.where(step[:, :, None] > 0, torch.round(q), torch.zeros_like(q)).clamp(0, 255)
    codes = q.reshape(x.shape[0], -1)[:, :x.shape[1]].to(torch.uint8)
    return codes, torch.stack([step, low], dim=2)


def _decode(codes, scales):
    m, d = codes.shape
    q = _groups(codes.float(), 0.0)
    return (scales[:, :, 1:] + scales[:, :, :1] * q).reshape(m, -1)[:, :d]


def _norm(x, weight, bias):
    mean = x.mean(1)
    centred = x - mean[:, None]
    rstd = (centred.square().mean(1) + EPS).rsqrt()
    return centred * rstd[:, None] * weight + bias, mean, rstd


def _norm_backward(dy, x, mean, rstd, weight):
    hat = (x - mean[:, None]) * rstd[:, None]
    g = dy * weight
    dx = (g - g.mean(1, keepdim=True) - hat * (g * hat).mean(1, keepdim=True)) * rstd[:, None]
    return dx, (dy * hat).sum(0), dy.sum(0)


def _run_plain(s):
    c = s["case"]
    dt = DTYPES[c["dtype"]]
    if c["kind"] == "norm":
        y = _norm(s["x"].float(), s["weight"], s["bias"])[0]
        return (y.clamp_min(0) if c["relu"] else y).to(dt)
    if c["kind"] == "train":
        x = s["x"].float()
        y, mean, rstd = _norm(x, s["weight"], s["bias"])
        kept = _decode(*_encode(x)) if c["keep"] == "int8" else x
        dx, dw, db = _norm_backward(s["dy"].float(), kept, mean, rstd, s["weight"])
        return y.to(dt), dx.to(dt), dw, db
    if c["kind"] == "back":
        bits = (s["active"][:, :, None].int() >> torch.arange(8, dtype=torch.int32, device=s["active"].device)) & 1
        dy = s["dy"].float() * bits.reshape(bits.shape[0], -1)[:, :c["d"]]
        dx, dw, db = _norm_backward(dy, _decode(s["codes"], s["scales"]), s["mean"], s["rstd"], s["weight"])
        return dx.to(dt), dw, db
    if c["kind"] == "pack":
        return _decode(*_encode(s["x"])).to(dt)
    if c["kind"] == "wgrad":
        dy = s["dy"].float()
        return (dy.t() @ _decode(s["codes"], s["scales"])).to(dt), dy.sum(0).to(dt)
    ids = s["ids"]
    inside = (ids >= 0) & (ids < c["rows"])
    y = torch.where(inside[:, None], s["table"][ids.clamp(0, c["rows"] - 1)].float() * s["scale"], 0.0).to(dt)
    key, order = torch.sort(torch.where(inside, ids, c["rows"]), stable=True)
    dy = torch.where((key < c["rows"])[:, None], s["dy"][order].float() * s["scale"], 0.0)
    if not c["sparse"]:
        return y, torch.zeros(c["rows"] + 1, c["d"], device=dy.device).index_add_(0, key, dy)[:c["rows"]].to(dt)
    place = torch.cat([torch.zeros_like(key[:1]), (key[1:] != key[:-1]).cumsum(0)])
    looked_up = torch.full_like(key, -1)
    looked_up[place] = torch.where(key < c["rows"], key, -1)
    return y, looked_up, torch.zeros_like(dy).index_add_(0, place, dy).to(dt)


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_values(x):
    """What the 8-bit codes of the rows stand for; the codes by their definition in single precision."""
    parts = []
    for part in x.to(torch.float32).split(GROUP, dim=1):
        low, high = part.min(dim=1, keepdim=True).values, part.max(dim=1, keepdim=True).values
        step = torch.sub(high, low).div(torch.tensor(255.0, device=x.device).expand_as(low))
        code = torch.nan_to_num(torch.sub(part, low).div(step)).round().clamp(max=255)
        parts.append(torch.addcmul(low.double().expand(part.shape), step.double().expand(part.shape), code.double()))
    return torch.cat(parts, dim=1)


def _exact_kept(codes, scales):
    width = codes.shape[1]
    each = scales.double().repeat_interleave(GROUP, dim=1)[:, :width]
    return torch.addcmul(each[:, :, 1], each[:, :, 0], codes.double())


def _exact_gradients(dy, hat, inverse, weight):
    """Gradients by the chain rule through z = x - mean(x) and y = z / sqrt(mean(z^2) + eps)."""
    g = dy * weight
    along = torch.einsum("md,md->m", g, hat).div(dy.shape[1]).unsqueeze(1)
    through = torch.addcmul(g, hat, along, value=-1)
    return torch.sub(through, through.mean(dim=1, keepdim=True) + along * hat.mean(dim=1, keepdim=True)) * inverse.unsqueeze(1), \
        torch.einsum("md,md->d", dy, hat), torch.einsum("md->d", dy)


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] == "pack":
        return _exact_values(s["x"])
    if c["kind"] == "wgrad":
        return torch.matmul(s["dy"].double().mT, _exact_kept(s["codes"], s["scales"])), s["dy"].double().sum(dim=0)
    if c["kind"] == "embed":
        padded = torch.nn.functional.pad(s["table"].double(), (0, 0, 0, 1)) if s["table"].numel() < 2 ** 26 else None
        ids = torch.where((s["ids"] < 0) | (s["ids"] >= c["rows"]), torch.full_like(s["ids"], c["rows"]), s["ids"])
        if padded is not None:
            y = padded.index_select(0, ids) * s["scale"]
        else:
            y = s["table"].index_select(0, ids.clamp(max=c["rows"] - 1)).double() * s["scale"]
            y[ids == c["rows"]] = 0
        order = torch.argsort(ids, stable=True)
        sorted_ids, counts = torch.unique_consecutive(ids[order], return_counts=True)
        ends = counts.cumsum(0)
        sums = torch.cat([torch.zeros(1, c["d"], dtype=torch.float64, device=ids.device), s["dy"][order].double().cumsum(0)])
        rows = (sums[ends] - sums[ends - counts]) * s["scale"]
        here = sorted_ids < c["rows"]
        sorted_ids, rows = sorted_ids[here], rows[here]
        if c["sparse"]:
            behind = c["m"] - sorted_ids.numel()
            return y, torch.nn.functional.pad(sorted_ids, (0, behind), value=-1), torch.nn.functional.pad(rows, (0, 0, 0, behind))
        dense = torch.zeros(c["rows"], c["d"], dtype=torch.float64, device=ids.device)
        dense[sorted_ids] = rows
        return y, dense
    weight, bias = s["weight"].double(), s["bias"].double()
    if c["kind"] == "back":
        mean, inverse = s["mean"].double(), s["rstd"].double()
        hat = torch.sub(_exact_kept(s["codes"], s["scales"]), mean.unsqueeze(1)) * inverse.unsqueeze(1)
        places = torch.arange(c["d"], device=hat.device)
        open_ = s["active"][:, places // 8].bitwise_right_shift((places % 8).to(torch.uint8)).bitwise_and(1)
        return _exact_gradients(s["dy"].double() * open_.double(), hat, inverse, weight)
    x = s["x"].double()
    variance, mean = torch.var_mean(x, dim=1, correction=0)
    inverse = (variance + EPS).pow(-0.5)
    hat = torch.sub(x, mean.unsqueeze(1)) * inverse.unsqueeze(1)
    y = torch.addcmul(bias, hat, weight)
    if c["kind"] == "norm":
        return y.relu() if c["relu"] else y
    if c["keep"] == "int8":
        hat = torch.sub(_exact_values(s["x"]), mean.unsqueeze(1)) * inverse.unsqueeze(1)
    return (y,) + tuple(_exact_gradients(s["dy"].double(), hat, inverse, weight))


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    c, item = case, DTYPES[case["dtype"]].itemsize
    if c["kind"] == "embed":
        size = c["m"] * c["d"] * item
        touched = min(c["rows"], c["m"])
        grad = c["m"] * (c["d"] * item + 8) if c["sparse"] else c["rows"] * c["d"] * item
        return {"bytes": touched * c["d"] * item + 2 * size + grad + 8 * c["m"], "flops": 2 * c["m"] * c["d"]}
    if c["kind"] == "wgrad":
        m, n, k = c["m"], c["n"], c["k"]
        return {"bytes": m * n * item + m * k + 8 * m * ((k + GROUP - 1) // GROUP) + n * k * item + n * item, "flops": 2 * m * n * k}
    m, d = c["m"], c["d"]
    if c["kind"] == "pack":
        return {"bytes": 2 * m * d * item, "flops": 6 * m * d}
    if c["kind"] == "norm":
        return {"bytes": 2 * m * d * item + 8 * d, "flops": 7 * m * d}
    if c["kind"] == "train":
        return {"bytes": 4 * m * d * item + 16 * d, "flops": 18 * m * d}
    return {"bytes": 2 * m * d * item + m * d + m * ((d + 7) // 8) + 8 * m * ((d + GROUP - 1) // GROUP) + 8 * m + 12 * d, "flops": 13 * m * d}
