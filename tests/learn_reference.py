"""Definitions in 64 bits, and how far single precision may be from them, for layer norm, 8-bit activations and learned rows.

U is half a step of single precision relative to a value: the most that one rounding is off.  A sum of n values whose longest chain of additions has k
links is at most k U times the sum of their absolute values off (to first order)."""
import torch

U = 2.0 ** -24
GROUP = 128
# half a step of the types: relative, and of their smallest values
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def rounded(value, dtype):
    """The most that one rounding to ``dtype`` moves values of this size."""
    return value.abs() * HALF[dtype] + TINY[dtype]


def chain(d):
    """Links of a row's sum: a lane's own columns (4 of every 128, over at least one warp), 5 exchanges in a warp, up to 16 warps, and a division."""
    return 4 * ((d + 127) // 128) + 5 + 16 + 2


def encode(x):
    """(codes uint8, scales [m, groups, 2]) by the definition, in single precision, group by group."""
    codes, scales = [], []
    for part in x.float().split(GROUP, dim=1):
        low, high = part.amin(1, keepdim=True), part.amax(1, keepdim=True)
        step = (high - low) / torch.full_like(low, 255.0)
        q = torch.round((part - low) / step)
        q = torch.where(step > 0, q, torch.zeros_like(q)).clamp(0, 255)
        lost = ~torch.isfinite(high - low)
        codes.append(torch.where(lost, torch.zeros_like(q), q).to(torch.uint8))
        scales.append(torch.where(lost, torch.full_like(low, float("nan")), torch.cat([step, low], 1)))
    return torch.cat(codes, 1), torch.stack(scales, 1)


def decode(codes, scales):
    """Values in 64 bits."""
    each = scales.double().repeat_interleave(GROUP, dim=1)[:, :codes.shape[1]]
    return each[:, :, 1] + each[:, :, 0] * codes.double()


def bits_of(active, d):
    places = torch.arange(d, device=active.device)
    return ((active[:, places // 8].int() >> (places % 8).int()) & 1).bool()


def norm(x, weight, bias, eps):
    """y, mean, rstd in 64 bits, and the most that single precision is off for each."""
    x = x.double()
    d = x.shape[1]
    k = chain(d)
    w = torch.ones(d, dtype=torch.float64, device=x.device) if weight is None else weight.double()
    b = torch.zeros(d, dtype=torch.float64, device=x.device) if bias is None else bias.double()
    mean = x.mean(1)
    z = x - mean[:, None]
    var = (z * z).mean(1)
    rstd = (var + eps) ** -0.5
    h = z * rstd[:, None]
    y = h * w + b
    mean_off = k * U * x.abs().mean(1)
    # the variance: its sum's chain, the squares and differences, and the mean's error, which enters squared (its linear part sums to nothing but roundings)
    var_off = (k + 6) * U * var + mean_off ** 2 + 2 * mean_off * U * z.abs().mean(1)
    rstd_off = rstd * (0.5 * var_off * rstd ** 2 + 4 * U)
    h_off = rstd[:, None] * (mean_off[:, None] + U * z.abs()) + z.abs() * rstd_off[:, None] + 2 * U * h.abs()
    y_off = w.abs() * h_off + 2 * U * (h * w).abs() + 2 * U * y.abs()
    return (y, mean, rstd, h), (y_off, mean_off, rstd_off)


def norm_backward(dy, x, mean, rstd, weight):
    """dx, dweight, dbias in 64 bits from what was kept, and the most that single precision is off.  ``x``: values in 64 bits; those that were decoded
    in single precision are U of their size off."""
    dy, mean, rstd = dy.double(), mean.double()[:, None], rstd.double()[:, None]
    m, d = dy.shape
    k, rows = chain(d) + 4, 80 + m / 100
    w = torch.ones(d, dtype=torch.float64, device=dy.device) if weight is None else weight.double()
    h = (x - mean) * rstd
    h_off = 2 * U * h.abs() + rstd * U * (x.abs() + (x - mean).abs())
    g = dy * w
    u, v = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    u_off = k * U * g.abs().mean(1, keepdim=True)
    v_off = (k + 2) * U * (g * h).abs().mean(1, keepdim=True) + (g.abs() * h_off).mean(1, keepdim=True)
    dx = rstd * (g - u - h * v)
    dx_off = rstd * (3 * U * (g.abs() + u.abs() + (h * v).abs()) + u_off + h.abs() * v_off + h_off * v.abs()) + 2 * U * dx.abs()
    dw, db = (dy * h).sum(0), dy.sum(0)
    dw_off = (rows + 2) * U * (dy * h).abs().sum(0) + (dy.abs() * h_off).sum(0)
    db_off = rows * U * dy.abs().sum(0)
    return (dx, dw, db), (dx_off, dw_off, db_off)


def near(got, want, off, dtype=torch.float32):
    """Every value within ``off``, and a rounding to ``dtype``, of what it should be."""
    got = got.double()
    room = off * 1.01 + rounded(want.abs() + off, dtype)
    bad = ~((got - want).abs() <= room)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()} values off, the worst {float(((got - want).abs() / room)[bad].max()):.3g} times what is allowed"
