"""The operators that take a pixel's channels as one vector, in float64 from their definitions, with bounds on what float32 sums
and the roundings to the map's type may change (elementwise, from the operands' magnitudes)."""
import numpy as np
import torch

from map_reference import ACT, F32, SLOPE, as_map, as_rows, half_step, tiny, value

LEAST_SCALE, MOST_SCALE = 2.0 ** -126, 2.6793883890187504e+36


def _sum_steps(channels):
    """Roundings on the way of a term of a row's sum: a lane's terms one after another (32 at most, or its share of 1024
    lanes'), then a tree over the lanes and the waves one by one."""
    return max(32, -(-channels // 1024)) + 6 + 16


def rms(x, residual, weight, eps, total=None, grad=None, grad_sum=None):
    """[(result, bound)]: y and the sum (with a residual; `total`: the sum as it was rounded, which is what is normalised), then the
    gradients of the input and the weight where `grad` is given."""
    dtype, c = x.dtype, x.shape[1]
    u, t = half_step(dtype), tiny(dtype)
    s = as_rows(x.double())
    got = []
    if residual is not None:
        exact = s + as_rows(residual.double())
        got = [(as_map(exact, x, c), as_map((u + F32) * exact.abs() + t, x, c))]
        s = as_rows(total.double())
    w = (torch.ones(c, device=x.device) if weight is None else weight).double()
    rstd = (s.square().mean(1, keepdim=True) + eps).rsqrt()
    # the mean: its sum's roundings, the product with 1 / channels (rounded) and the addition of eps; the root halves them; then
    # the root, the quotient, and float32's subnormals where the reciprocal root is one
    er = (_sum_steps(c) + 3) / 2 * F32 + 2 * F32 + 2.0 ** -149 / rstd
    h = s * rstd
    y = h * w
    ey = y.abs() * (er + 2 * F32)
    got = [(as_map(y, x, c), as_map(ey + u * y.abs() + t, x, c))] + got
    if grad is None:
        return got
    dy = as_rows(grad.double())
    eh = er + F32
    dh = dy * w
    m = (dh * h).mean(1, keepdim=True)
    em = (dh * h).abs().mean(1, keepdim=True) * (eh + (_sum_steps(c) + 3) * F32)
    inner = dh - h * m
    e_inner = 2 * F32 * dh.abs() + h.abs() * em + h.abs() * m.abs() * (eh + 2 * F32)
    dx = rstd * inner
    edx = rstd * (e_inner + inner.abs() * er) + F32 * dx.abs()
    if grad_sum is not None:
        dx = dx + as_rows(grad_sum.double())
        edx = edx + 2 * F32 * dx.abs()
    dw = (dy * h).sum(0)
    # a lane's rows one after another (a 256th of the rows at most), then 16 chunks and a tree
    edw = ((dy * h).abs() * (eh + (64 + s.shape[0] / 256) * F32)).sum(0)
    return got + [(as_map(dx, x, c), as_map(edx + u * dx.abs() + t, x, c)), (dw, edw + u * dw.abs() + t)]


def quantize(rows):
    """Codes and scales of (..., channels) float64 rows that hold values of a map's type: exact."""
    big = rows.abs().amax(-1)
    scales = (big.float() * torch.tensor(1 / 127, device=rows.device)).clamp(LEAST_SCALE, MOST_SCALE)   # (float32's product)
    scales = torch.where(torch.isfinite(big), scales, torch.ones_like(scales))
    codes = torch.round(rows / scales.double().unsqueeze(-1))
    codes = torch.where(torch.isfinite(big).unsqueeze(-1), codes, torch.zeros_like(codes))
    return codes, torch.where(torch.isfinite(big), scales, torch.full_like(scales, float("nan")))


def dequantize(codes, scales, dtype):
    """(result, bound): the product rounded to the type, in float32 before that or not."""
    y = codes.double() * scales.double().unsqueeze(1)
    return y, (half_step(dtype) * (1 + 2 * F32) + F32) * y.abs() + tiny(dtype)


def check_rms_int8(codes, scales, s, weight, eps):
    """The 8-bit form of the normalised rows of s, whose codes may fall to either side of a border by float32's last bits."""
    c = s.shape[1]
    rows = as_rows(s.double())
    rstd = (rows.square().mean(1, keepdim=True) + eps).rsqrt()
    v = rows * rstd * (1.0 if weight is None else weight.double())
    ev = (_sum_steps(c) + 3) / 2 * F32 + 4 * F32 + 2.0 ** -149 / rstd
    want = (v.abs().amax(1) / 127).clamp(LEAST_SCALE, MOST_SCALE)
    got = scales.reshape(-1).double()
    assert ((got - want).abs() <= want * (ev[:, 0] + 3 * F32)).all()
    q = as_rows(codes).double()
    assert ((q - v / got[:, None]).abs() <= 0.5 + 128 * (ev + 2 * F32)).all()
    assert q.abs().max() <= 127


def pointwise_int8(codes, scales, weight_codes, weight_scales, bias, residual, activation, dtype):
    """(result, bound)"""
    sums = as_rows(codes).double() @ weight_codes.double().t()
    z = sums * scales.reshape(-1, 1).double() * weight_scales.double()
    ez = 3 * F32 * z.abs()
    if bias is not None:
        z = z + bias.double()
        ez = ez + F32 * z.abs()
    y = value(z, activation)
    ey = SLOPE * ez + (ACT * z.abs() if activation != "none" else 0)
    if residual is not None:
        y = y + as_rows(residual.double())
        ey = ey + F32 * y.abs()
    n = weight_codes.shape[0]
    return as_map(y, codes, n), as_map(ey + half_step(dtype) * y.abs() + tiny(dtype), codes, n)


def philox(counter, key):
    """Philox4x32-10 of (n, 4) counters and one key of two words, from the generator's published definition."""
    c = [np.asarray(counter)[..., i].astype(np.uint64) for i in range(4)]
    k = [int(key[0]), int(key[1])]
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    for _ in range(10):
        a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
        c = [(b >> half) ^ c[1] ^ np.uint64(k[0]), b & low, (a >> half) ^ c[3] ^ np.uint64(k[1]), a & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, -1)


def kept(n, p, seed, first=0):
    """Which of the values first .. first + n - 1 (first: a multiple of eight) are kept."""
    groups = np.arange(first // 8, (first + n + 7) // 8, dtype=np.uint64)
    counter = np.zeros((len(groups), 4), np.uint64)
    counter[:, 0], counter[:, 1] = groups & np.uint64(0xFFFFFFFF), groups >> np.uint64(32)
    key = seed % 2 ** 64
    words = philox(counter, (key % 2 ** 32, key >> 32))
    bits = np.stack([words & np.uint64(0xFFFF), words >> np.uint64(16)], -1).reshape(-1)[:n]
    return torch.from_numpy(bits >= round(65536 * p))


def dropout(x, p, seed, residual=None):
    """(result, bound, mask as a map)"""
    c = x.shape[1]
    mask = as_map(kept(x.numel(), p, seed).view(-1, c), x, c).to(x.device)
    drop = round(65536 * p)
    y = torch.where(mask, x.double() * (65536 / (65536 - drop) if drop < 65536 else 0.0), 0.0)
    e = 2 * F32 * y.abs()   # the scale and the product
    if residual is not None:
        y = y + residual.double()
        e = e + F32 * y.abs()
    return y, e + half_step(x.dtype) * y.abs() + tiny(x.dtype), mask
