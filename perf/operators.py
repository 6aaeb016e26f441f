"""The dense half of a GraphSAGE layer as operators: its product in 8-bit integers (how a trained network answers) and the
orthogonalised update of its weights (how it learns).  ``listed`` and ``draw`` say on which sizes, ``run`` makes one call.

Kinds:
  mm       ops.int8_mm: int8 codes [m, k] times int8 codes [n, k], a scale for every row of each, bias and ReLU
  linear   ops.int8_linear: the same from rows in floating point, whose codes and scales it computes; ``pair``: the rows are
           the columns of two tensors side by side (a SAGE layer's own row and its neighbours' mean)
  ortho    ops.orthogonalize: Newton-Schulz steps X <- aX + (bA + cA^2)X, A = XX^T, from X = G / (|G| + eps)
  muon     ops.muon_step: momentum, orthogonalised update and decay of a list of weight matrices, in place

Definitions.  Codes of a row x: scale = max|x| / 127 and code = round-to-even(x / scale), both quotients in single precision.
Coefficients, steps and eps are those of the calls' defaults.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
STEPS, COEFFICIENTS, EPS = 5, (3.4445, -4.7750, 2.0315), 1e-7
LR, MOMENTUM, DECAY = 0.02, 0.95, 0.01


def listed():
    return [
        # hidden layer over the outermost block of a minibatch: 59,000 rows, 128 own + 128 neighbour columns, codes in hand
        dict(name="mm_block", kind="mm", m=59_000, n=128, k=256, out="f32", bias=True, relu=True),
        # a wide layer over many rows: the largest product, bound by the tensor cores
        dict(name="mm_wide", kind="mm", m=16_384, n=4096, k=4096, out="bf16", bias=False, relu=False),
        # one node's answer from the last layer: the smallest call, latency only
        dict(name="linear_row", kind="linear", m=1, n=172, k=256, dtype="f32", pair=False, bias=True, relu=False),
        # the seeds of a minibatch through the last layer, own row and neighbours' mean side by side
        dict(name="linear_seeds", kind="linear", m=1024, n=172, k=256, dtype="f32", pair=True, bias=True, relu=False),
        # a few rows through a wide layer: bound by reading the weights
        dict(name="linear_few", kind="linear", m=16, n=4096, k=4096, dtype="bf16", pair=False, bias=True, relu=False),
        # feature widths and class counts that are no multiple of anything
        dict(name="linear_ragged", kind="linear", m=5003, n=41, k=602, dtype="f16", pair=False, bias=True, relu=True),
        # a hidden weight matrix of the 128-column presets alone
        dict(name="ortho_hidden", kind="ortho", batch=1, m=128, n=128, dtype="f32"),
        # a tall odd matrix: the first layer of wide features
        dict(name="ortho_ragged", kind="ortho", batch=1, m=1031, n=602, dtype="f32"),
        # a stack of square matrices, one of each layer
        dict(name="ortho_stack", kind="ortho", batch=12, m=1024, n=1024, dtype="bf16"),
        # the largest: bound by the tensor cores
        dict(name="ortho_wide", kind="ortho", batch=1, m=4096, n=4096, dtype="bf16"),
        # a step over all weight matrices of the 3-layer network with 128 hidden columns and 172 classes
        dict(name="muon_sage", kind="muon", shapes="128x128*4,172x128*2", dtype="f32"),
        # a step over two layers of a wide network in 32 bits
        dict(name="muon_wide", kind="muon", shapes="2048x2048*1,2048x8192*1", dtype="f32"),
    ]


def draw(rng):
    def log(lo, hi):
        return max(lo, min(hi, round(math.exp(rng.uniform(math.log(lo), math.log(hi))))))

    kind = rng.choice(["mm", "linear", "ortho", "muon"])
    if kind in ("mm", "linear"):
        m, n, k = log(1, 65_536), log(1, 4096), log(8, 4096)
        if rng.random() < 0.5:
            n, k = max(8, n // 8 * 8), max(16, k // 16 * 16)
        m = min(m, 40_000_000 // max(n, k))
        c = dict(kind=kind, m=m, n=n, k=k, bias=rng.random() < 0.7, relu=rng.random() < 0.5)
        if kind == "mm":
            return dict(c, out=rng.choice(["f32", "bf16", "f16"]))
        pair = rng.random() < 0.4
        return dict(c, k=k // 2 * 2 if pair else k, dtype=rng.choice(["f32", "bf16", "f16"]), pair=pair)
    dtype = rng.choice(["f32", "bf16", "f16"] if kind == "ortho" else ["f32", "bf16"])
    m, n = log(16, 2500), log(16, 2500)
    if rng.random() < 0.5:
        m, n = max(16, m // 16 * 16), max(16, n // 16 * 16)
    if kind == "ortho":
        return dict(kind=kind, batch=log(1, max(1, min(32, 20_000_000 // (m * n)))), m=m, n=n, dtype=dtype)
    m2, n2 = log(16, 2500), log(16, 2500)
    return dict(kind=kind, shapes=f"{m}x{n}*{rng.randint(1, 3)},{m2}x{n2}*{rng.randint(1, 2)}", dtype=dtype)


def _shapes(text):
    out = []
    for part in text.split(","):
        size, count = part.split("*")
        out += [tuple(int(v) for v in size.split("x"))] * int(count)
    return out


def _rows16(codes):
    """The codes with rows that start on 16-byte boundaries, as ops.int8_quantize lays them out."""
    rows, k = codes.shape
    room = torch.zeros((rows, (k + 15) // 16 * 16), dtype=torch.int8, device=codes.device)
    room[:, :k] = codes
    return room[:, :k]


def _gradient(rows, cols, g, dev):
    """A weight gradient as a training step makes it: the product of output gradients with ReLU activations over many rows."""
    t = 2 * max(rows, cols, 512)
    dy = torch.randn(t, rows, generator=g, device=dev)
    x = torch.randn(t, cols, generator=g, device=dev).relu_() * (0.25 + torch.rand(cols, generator=g, device=dev))
    return dy.t() @ x / t


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(device=dev)
    g.manual_seed(seed)
    c = dict(case)
    s = {"case": c}
    if c["kind"] in ("mm", "linear"):
        m, n, k = c["m"], c["n"], c["k"]
        w = torch.randn(n, k, generator=g, device=dev) / math.sqrt(k)
        q, s["ws"] = _codes(w)
        s["w"] = _rows16(q)
        s["bias"] = torch.randn(n, generator=g, device=dev) if c["bias"] else None
        x = torch.randn(m, k, generator=g, device=dev) * (0.5 + torch.rand(k, generator=g, device=dev))
        if c["kind"] == "mm":
            q, s["xs"] = _codes(x)
            s["x"] = _rows16(q)
        else:
            x = x.to(DTYPES[c["dtype"]])
            s["x"], s["x2"] = (x[:, :k // 2].contiguous(), x[:, k // 2:].contiguous()) if c["pair"] else (x, None)
    elif c["kind"] == "ortho":
        s["g"] = torch.stack([_gradient(c["m"], c["n"], g, dev) for _ in range(c["batch"])]).to(DTYPES[c["dtype"]])
    else:
        dt = DTYPES[c["dtype"]]
        sizes = _shapes(c["shapes"])
        s["weights"] = [(torch.randn(r, q, generator=g, device=dev) / math.sqrt(q)).to(dt) for r, q in sizes]
        s["grads"] = [_gradient(r, q, g, dev).to(dt) for r, q in sizes]
        s["momenta"] = [8 * _gradient(r, q, g, dev) for r, q in sizes]
    return s


def run(state):
    return _run_own(state) if own else _run_plain(state)


def _run_own(s):
    from f2cgt_b200 import ops
    c = s["case"]
    if c["kind"] == "mm":
        return ops.int8_mm(s["x"], s["xs"], s["w"], s["ws"], bias=s["bias"], relu=c["relu"], out_dtype=DTYPES[c["out"]])
    if c["kind"] == "linear":
        return ops.int8_linear(s["x"], s["w"], s["ws"], bias=s["bias"], relu=c["relu"], x2=s["x2"])
    if c["kind"] == "ortho":
        return ops.orthogonalize(s["g"])
    ops.muon_step(s["weights"], s["grads"], s["momenta"], lr=LR, momentum=MOMENTUM, weight_decay=DECAY)
    return s["weights"], s["momenta"]


# ---------------------------------------------------------------- the operators in elementary operations, 32 bits
def _codes(x):
    top = x.abs().amax(1, keepdim=True)
    scale = top / torch.full_like(top, 127.0)
    q = torch.where(scale > 0, torch.round(x / scale), torch.zeros_like(x))
    return q.clamp(-127, 127).to(torch.int8), scale.reshape(-1)


def _product(q, qs, w, ws, bias, relu, dtype):
    y = (q.float() @ w.float().t()) * (qs[:, None] * ws)
    if bias is not None:
        y = y + bias
    return (y.clamp_min(0) if relu else y).to(dtype)


def _newton_schulz(g):
    a, b, c = COEFFICIENTS
    x = g.float()
    x = x / (x.square().sum(dim=(-2, -1), keepdim=True).sqrt() + EPS)
    tall = x.shape[-2] > x.shape[-1]
    if tall:
        x = x.transpose(-2, -1)
    for _ in range(STEPS):
        p = x @ x.transpose(-2, -1)
        x = a * x + (b * p + c * (p @ p)) @ x
    return x.transpose(-2, -1) if tall else x


def _run_plain(s):
    c = s["case"]
    if c["kind"] == "mm":
        return _product(s["x"], s["xs"], s["w"], s["ws"], s["bias"], c["relu"], DTYPES[c["out"]])
    if c["kind"] == "linear":
        x = s["x"] if s["x2"] is None else torch.cat([s["x"], s["x2"]], dim=1)
        q, qs = _codes(x.float())
        return _product(q, qs, s["w"], s["ws"], s["bias"], c["relu"], x.dtype)
    if c["kind"] == "ortho":
        return _newton_schulz(s["g"]).contiguous().to(s["g"].dtype)
    for w, g, v in zip(s["weights"], s["grads"], s["momenta"]):
        v.mul_(MOMENTUM).add_(g.float())
        o = _newton_schulz(g.float() + MOMENTUM * v)
        gain = math.sqrt(max(1.0, w.shape[0] / w.shape[1]))
        w.copy_(w.float() * (1 - LR * DECAY) - LR * gain * o)
    return s["weights"], s["momenta"]


# ---------------------------------------------------------------- the definitions in 64 bits
def _exact_polar(g):
    """The singular values go through the polynomial, the singular vectors stay: sigma <- a sigma + b sigma^3 + c sigma^5, written as
    products with the smaller Gram matrix."""
    rows, cols = g.shape[-2:]
    z = g / (torch.linalg.vector_norm(g, dim=(-2, -1), keepdim=True) + EPS)
    a, b, c = COEFFICIENTS
    eye = torch.eye(min(rows, cols), dtype=z.dtype, device=z.device)
    for _ in range(STEPS):
        if rows <= cols:
            gram = torch.matmul(z, z.mT)
            z = torch.matmul(a * eye + torch.matmul(gram, b * eye + c * gram), z)
        else:
            gram = torch.matmul(z.mT, z)
            z = torch.matmul(z, a * eye + torch.matmul(gram, b * eye + c * gram))
    return z


def exact(case, seed):
    s, c = prepare(case, seed), case
    if c["kind"] in ("mm", "linear"):
        if c["kind"] == "mm":
            codes, scales = s["x"].double(), s["xs"].double()
        else:
            rows = torch.cat([t.to(torch.float32) for t in (s["x"], s["x2"]) if t is not None], dim=1)
            scale = torch.linalg.vector_norm(rows, ord=math.inf, dim=1).div(torch.tensor(127.0, device=rows.device).expand(rows.shape[0]))
            ratio = torch.div(rows, scale.unsqueeze(1))  # single precision: the definition of the codes
            codes, scales = torch.nan_to_num(ratio).round().double(), scale.double()
        y = torch.matmul(codes * scales.unsqueeze(1), (s["w"].double() * s["ws"].double().unsqueeze(1)).t())
        if s["bias"] is not None:
            y += s["bias"].double()
        return y.relu() if c["relu"] else y
    if c["kind"] == "ortho":
        return _exact_polar(s["g"].double())
    weights, momenta = [], []
    for w, g, v in zip(s["weights"], s["grads"], s["momenta"]):
        v = MOMENTUM * v.double() + g.double()
        o = _exact_polar(g.double() + MOMENTUM * v)
        weights.append((1 - LR * DECAY) * w.double() - LR * max(1.0, w.shape[0] / w.shape[1]) ** 0.5 * o)
        momenta.append(v)
    return weights, momenta


# ---------------------------------------------------------------- what a pass cannot do without
def _newton_schulz_flops(rows, cols):
    """Per step with p <= q: the symmetric products XX^T (half of 2ppq) and A^2 (half of 2ppp), and the full one onto X (2ppq)."""
    p, q = min(rows, cols), max(rows, cols)
    return STEPS * (3 * p * p * q + p * p * p)


def work(case):
    c = case
    if c["kind"] in ("mm", "linear"):
        m, n, k = c["m"], c["n"], c["k"]
        rows = m * k + 4 * m if c["kind"] == "mm" else m * k * DTYPES[c["dtype"]].itemsize
        out = m * n * DTYPES[c["out" if c["kind"] == "mm" else "dtype"]].itemsize
        return {"bytes": rows + n * k + 4 * n + (4 * n if c["bias"] else 0) + out, "flops": 2 * m * n * k}
    if c["kind"] == "ortho":
        return {"bytes": 2 * c["batch"] * c["m"] * c["n"] * DTYPES[c["dtype"]].itemsize, "flops": c["batch"] * _newton_schulz_flops(c["m"], c["n"])}
    sizes, item = _shapes(c["shapes"]), DTYPES[c["dtype"]].itemsize
    return {"bytes": sum(r * q * (3 * item + 8) for r, q in sizes), "flops": sum(_newton_schulz_flops(r, q) for r, q in sizes)}
