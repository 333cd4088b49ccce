"""The operators on channels-last maps in float64, from their definitions, with bounds on what the float32 sums and the
roundings to the map's type may change (elementwise, from the operands' magnitudes)."""
import math

import torch

ACTIVATIONS = ("none", "relu", "silu", "gelu")
# largest slope and curvature of the activations (gelu: 1.129, 0.798; silu: 1.0998, 0.5)
SLOPE, CURVE = 1.13, 0.8
F32 = 2.0 ** -24
# the activation functions' own error, of the argument: the error function to 1.5e-7, exponentials to a few last bits
ACT = 1e-6


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def tiny(dtype):
    """half of the smallest step of the type's subnormals"""
    return torch.finfo(dtype).tiny * torch.finfo(dtype).eps / 2


def value(z, activation):
    return {"none": lambda: z, "relu": lambda: z.clamp(min=0), "silu": lambda: z * torch.sigmoid(z),
            "gelu": lambda: z * torch.special.ndtr(z)}[activation]()


def slope(z, activation):
    s = torch.sigmoid(z)
    return {"none": lambda: torch.ones_like(z), "relu": lambda: (z > 0).double(), "silu": lambda: s + z * s * (1 - s),
            "gelu": lambda: torch.special.ndtr(z) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)}[activation]()


def kept(rows, dtype):
    """What the 8-bit form of (..., channels) rows stands for."""
    out = torch.empty_like(rows)
    most = torch.finfo(dtype).max
    for c in range(0, rows.shape[-1], 32):
        block = rows[..., c:c + 32]
        big = block.abs().amax(-1, keepdim=True)
        k = torch.ceil(torch.log2(big / 127)).clamp(min=-126)
        v = (torch.round(block / torch.exp2(k)) * torch.exp2(k)).clamp(-most, most)
        out[..., c:c + 32] = torch.where(torch.isfinite(big), v, math.nan)
    return out


def as_rows(x):
    return x.movedim(1, -1).reshape(-1, x.shape[1])


def as_map(rows, like, channels):
    return rows.reshape(like.shape[0], *like.shape[2:], channels).movedim(-1, 1)


def _slope_error(z, ez, activation):
    e = CURVE * ez + ACT if activation != "none" else torch.zeros_like(z)
    if activation == "relu":
        e = torch.where(z.abs() <= ez, torch.ones_like(z), torch.zeros_like(z))   # on which side of zero it falls
    return e


def norm(x, groups, weight, bias, eps, activation, grad=None, keep_int8=False):
    """[(result, bound)]: y, then the gradients of the input, the weight and the bias where `grad` is given."""
    dtype, shape = x.dtype, x.shape
    u, t = half_step(dtype), tiny(dtype)
    b, c = shape[:2]
    cg = c // groups

    def view(v):
        return v.double().movedim(1, -1).reshape(b, -1, groups, cg)

    def back(v):
        return as_map(v.reshape(-1, c), x, c)

    X = view(x)
    w = (torch.ones(c, device=x.device) if weight is None else weight).double().view(groups, cg)
    s = (torch.zeros(c, device=x.device) if bias is None else bias).double().view(groups, cg)
    mean = X.mean((1, 3), keepdim=True)
    rstd = ((X - mean).square().mean((1, 3), keepdim=True) + eps).rsqrt()
    # the sums of a lane's few hundred float32 deviations: under 256 roundings of the spread
    def z_of(X):
        h = (X - mean) * rstd
        z = h * w + s
        ez = F32 * (16 * (w.abs() * rstd * (X.abs() + mean.abs()) + z.abs() + s.abs()) + 256 * w.abs() * (1 + h.abs()))
        return h, z, ez

    h, z, ez = z_of(X)
    y = value(z, activation)
    got = [(back(y), back(SLOPE * ez + ACT * z.abs() + u * y.abs() + t))]
    if grad is None:
        return got
    if keep_int8:
        X = kept(x.double().movedim(1, -1), dtype).reshape(X.shape)
        h, z, ez = z_of(X)
    dy = view(grad)
    dz = dy * slope(z, activation)
    edz = dy.abs() * _slope_error(z, ez, activation) + 8 * F32 * dz.abs()
    eh = F32 * (16 * rstd * (X.abs() + mean.abs()) + 256 * (1 + h.abs()))
    dn, edn = dz * w, edz * w.abs()

    def avg(v):
        return v.mean((1, 3), keepdim=True)

    dx = rstd * (dn - avg(dn) - h * avg(dn * h))
    sums = 64 * F32   # relative to the sums of magnitudes
    edx = rstd * (edn + avg(edn) + h.abs() * avg(edn * h.abs() + dn.abs() * eh) + eh * avg(dn * h).abs()
                  + sums * (dn.abs() + avg(dn.abs()) + h.abs() * avg((dn * h).abs())))
    edx = edx + 256 * F32 * dx.abs()
    dw, db = (dz * h).sum((0, 1)), dz.sum((0, 1))
    edw = (edz * h.abs() + dz.abs() * eh + sums * (dz * h).abs()).sum((0, 1))
    edb = (edz + sums * dz.abs()).sum((0, 1))
    return got + [(back(dx), back(edx + u * dx.abs() + t)), (dw.view(c), (edw + u * dw.abs() + t).view(c)),
                  (db.view(c), (edb + u * db.abs() + t).view(c))]


def _sum_error(n, dtype):
    """n products summed in float32 (six products of pieces each for float32, with what the pieces leave out): eight
    standard deviations of as many independent roundings, of a step each."""
    return 8 * math.sqrt(n * (6 if dtype == torch.float32 else 1)) * 2 * F32 + (F32 if dtype == torch.float32 else 0)


def pointwise(x, weight, bias, residual, activation, grad=None, keep_int8=False):
    """[(result, bound)]: y, then the gradients of the input, the weight and the bias where `grad` is given."""
    dtype = x.dtype
    u, t = half_step(dtype), tiny(dtype)
    X, W = as_rows(x.double()), weight.double().flatten(1)
    n, k = W.shape
    z = X @ W.t()
    ez = _sum_error(k, dtype) * (X.abs() @ W.abs().t())
    if bias is not None:
        z = z + bias.double()
        ez = ez + 2 * F32 * z.abs()
    y = value(z, activation)
    ey = SLOPE * ez + (ACT * z.abs() if activation != "none" else 0)
    if residual is not None:
        y = y + as_rows(residual.double())
        ey = ey + F32 * y.abs()
    got = [(as_map(y, x, n), as_map(ey + u * y.abs() + t, x, n))]
    if grad is None:
        return got
    if keep_int8:
        X = kept(X, dtype)
    dy = as_rows(grad.double())
    dz = dy * slope(z, activation)
    # the argument is kept in the map's type, and dz is rounded to it for the products (float32: kept whole)
    ez = ez + (u * z.abs() + t if activation != "none" else 0)
    edz = dy.abs() * _slope_error(z, ez, activation) + 8 * F32 * dz.abs()
    erz = edz + (u * (dz.abs() + edz) + t if dtype != torch.float32 and activation != "none" else 0)
    rows = X.shape[0]
    dx, dw, db = dz @ W, dz.t() @ X, dz.sum(0)
    edx = erz @ W.abs() + _sum_error(n, dtype) * (dz.abs() @ W.abs())
    edw = erz.t() @ X.abs() + _sum_error(rows, dtype) * (dz.abs().t() @ X.abs())
    edb = edz.sum(0) + 64 * F32 * dz.abs().sum(0)
    return got + [(as_map(dx, x, k), as_map(edx + u * dx.abs() + t, x, k)), (dw, edw + u * dw.abs() + t),
                  (db, edb + u * db.abs() + t)]


def check(got, expected, what=""):
    """Every value within its bound; the whole within what independent roundings leave of it."""
    for i, (g, (r, bound)) in enumerate(zip(got, expected)):
        assert g is not None and g.shape == r.shape, (what, i, None if g is None else g.shape, r.shape)
        d = (g.double() - r).abs()
        worst = (d - bound).max().item() if d.numel() else 0.0
        assert worst <= 0, (what, i, "over its bound by", worst, "at", d.argmax().item(), "of", r.abs().max().item())


def make(shape, dtype, seed, device="cuda", spread=1.0, shift=0.0):
    """A channels-last map (or a vector or matrix) of normal values."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(*shape, generator=g, dtype=torch.float64) * spread + shift
    if len(shape) > 2:
        x = x.movedim(1, -1).contiguous().movedim(-1, 1)
    return x.to(dtype).to(device)


def layouts(device, dtype, shape, groups, out):
    """Shape, strides and type of every result of every operator, the internal ones among them, for maps of this shape."""
    ops = torch.ops.tvdcn
    x, w = torch.zeros(shape, device=device, dtype=dtype), torch.zeros(out, shape[1], device=device, dtype=dtype)
    p, b = torch.zeros(shape[1], device=device, dtype=dtype), torch.zeros(out, device=device, dtype=dtype)
    every = [True] * 3
    got = []
    for act in range(len(ACTIVATIONS)):
        y, stats = ops._group_norm_act_forward(x, groups, p, p, 1e-5, act)
        got += [y, stats, *ops._group_norm_act_backward(y, x, None, None, p, p, stats, act, every)]
        y, pre = ops._pointwise_conv_forward(x, w, b, None, act, True)
        got += [y, pre, *ops._pointwise_conv_backward(y, x, None, None, w, pre, act, every)]
        if dtype != torch.float64:
            codes, exponents = ops.compress_activation(x)
            got += [codes, exponents, ops.expand_activation(codes, exponents, dtype)]
            got += ops._group_norm_act_backward(x, None, codes, exponents, p, p, stats, act, every)
            got += ops._pointwise_conv_backward(y, None, codes, exponents, w, pre, act, every)
    return [(tuple(t.shape), t.stride(), t.dtype) for t in got]


LAYOUT_SHAPES = [((3, 42, 4, 5), 7, 10), ((1, 8, 9), 1, 8), ((5, 6), 2, 3), ((2, 3, 1, 2, 4), 3, 1), ((0, 6, 4), 2, 4), ((2, 6, 0), 3, 4)]
