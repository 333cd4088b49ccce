"""The operators that take a pixel's channels as one vector on the GPU, against their definitions in float64 (row_reference.py):
every type and direction, from single pixels to maps beyond 32-bit offsets, channels of any count up to the longest rows, other
memory orders, values that are not finite, streams, graphs."""
import math

import pytest
import torch

import tvdcn
from map_reference import ACTIVATIONS, as_map, as_rows, check, make, pointwise
from row_reference import check_rms_int8, dequantize, dropout, kept, pointwise_int8, quantize, rms
from test_rows_cpu import SHAPES, Block, layouts

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]
SEED = 0x123456789ABCDEF
OPS = torch.ops.tvdcn


def leaf(t):
    return None if t is None else t.detach().requires_grad_(True)


def seed_of(v=SEED):
    return torch.tensor([v], device="cuda")


# one lane to a row, several rows to a wave, whole waves, whole workgroups, rows beyond their registers; channels that make no
# whole accesses among all of them
NORM_SHAPES = [
    (2, 3, 5, 3), (1, 1, 7), (4097, 1), (3, 7, 9), (37, 8), (1, 40, 1), (3, 71, 11, 13), (1000, 16, 2), (5, 130, 3, 1, 2), (1, 256),
    (2, 257, 9), (3, 512, 33), (7, 513), (1, 600, 30), (3, 1000, 5), (2, 1024, 17), (2, 1500, 9), (5, 2047), (3, 2048, 4), (2, 2056, 3),
    (1, 2100, 5), (3, 4097), (2, 8192, 2), (2, 9001), (3, 16384), (2, 16392), (1, 20001), (2, 32776), (1, 70001, 2), (300, 96, 1, 1),
    (2, 64, 60, 70), (1, 1 << 17),
]


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_norms(shape, dtype):
    x, r, w = make(shape, dtype, 1), make(shape, dtype, 2), make((shape[1],), dtype, 3, spread=0.3, shift=1.0)
    dy, ds = make(shape, dtype, 4), make(shape, dtype, 5)
    t = [leaf(v) for v in (x, r, w)]
    y, s = tvdcn.add_rms_norm(*t)
    dx, dr, dw = torch.autograd.grad([y, s], t, [dy, ds])
    check([y, s, dx, dw], rms(x, r, w, 1e-6, s.detach(), dy, ds), shape)
    assert torch.equal(dx, dr)
    t = [leaf(v) for v in (x, w)]
    y = tvdcn.rms_norm(*t, 0.1)
    check([y, *torch.autograd.grad(y, t, dy)], rms(x, None, w, 0.1, None, dy), shape)
    check([tvdcn.rms_norm(x)], rms(x, None, None, 1e-6), shape)
    codes, scales, s = tvdcn.add_rms_norm_int8(x, r, w)
    check([s], rms(x, r, w, 1e-6, s)[1:])
    check_rms_int8(codes, scales, s, w, 1e-6)
    check_rms_int8(*tvdcn.rms_norm_int8(x, None, 0.5), x, None, 0.5)


@pytest.mark.parametrize("shape", NORM_SHAPES, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_8_bits(shape, dtype):
    x = make(shape, dtype, 1, spread=3.0)
    codes, scales = tvdcn.quantize_int8(x)
    q, s = quantize(x.movedim(1, -1).double())
    assert torch.equal(codes.movedim(1, -1).double(), q) and torch.equal(scales, s)
    for out in DTYPES:
        check([tvdcn.dequantize_int8(codes, scales, out)], [dequantize(codes, scales, out)], out)


@pytest.mark.parametrize("dtype", DTYPES)
def test_8_bits_at_rounding_borders_and_range_ends(dtype):
    """Codes of values on, next to and between the borders, of rows from the smallest to the largest, are those of exact quotients."""
    g = torch.Generator().manual_seed(1)
    low, high = (-24, 15) if dtype == torch.float16 else (-149, 127)
    rows = []
    for e in (low, low + 1, low + 9, -20, -7, -1, 0, 3, high - 8, high - 7):
        for scale in (1.0, 1 + 2 ** -7, 1.37, 127 / 128, 1.9921875):
            half = torch.arange(-254, 255, dtype=torch.float64) / 2 * scale * 2.0 ** e
            rows.append(torch.cat([half, torch.tensor([127.0 * scale * 2.0 ** e])]))
            rows.append(rows[-1] * (1 + torch.randint(-2, 3, (510,), generator=g) * 2.0 ** -24))
    x = torch.stack(rows).to(dtype)
    x = x[torch.isfinite(x).all(1)].cuda()
    assert len(x) > 60
    codes, scales = tvdcn.quantize_int8(x)
    q, s = quantize(x.double())
    assert torch.equal(scales, s) and torch.equal(codes.double(), q)
    cpu = tvdcn.quantize_int8(x.cpu())
    assert torch.equal(cpu[0], codes.cpu()) and torch.equal(cpu[1], scales.cpu())
    # the largest finite value comes back finite
    x = torch.full((2, 40), torch.finfo(dtype).max, device="cuda", dtype=dtype)
    x[1, ::2] *= -1
    codes, scales = tvdcn.quantize_int8(x)
    back = tvdcn.dequantize_int8(codes, scales, dtype)
    assert (codes.abs() == 127).all() and torch.isfinite(back).all() and ((back / x - 1).abs() < 2 * torch.finfo(dtype).eps).all()


@pytest.mark.parametrize("shape", [(4, 24, 6), (4, 71, 6), (3, 2500, 2), (3, 9001, 2), (3, 40000, 2)], ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_values_that_are_not_finite_stay_in_their_pixel(shape, dtype):
    x, w = make(shape, dtype, 1), make((shape[1],), dtype, 2, shift=1.0)
    bad = x.clone()
    bad[0, shape[1] // 2, 0], bad[1, shape[1] - 1, 1], bad[-1, 0, 1] = math.nan, math.inf, -math.inf
    touched = ~torch.isfinite(bad).all(1)
    y, want = tvdcn.rms_norm(bad, w), tvdcn.rms_norm(x, w)
    clean = ~touched.unsqueeze(1).expand_as(x)
    assert touched.sum() == 3 and torch.equal(y[clean], want[clean])
    # the formula's: all NaN for a NaN; for an infinity it is NaN and the others are zero
    assert y[0, :, 0].isnan().all() and y[-1, 0, 1].isnan() and not y[-1, 1:, 1].any()
    codes, scales = tvdcn.rms_norm_int8(bad, w)
    codes2, scales2 = tvdcn.quantize_int8(bad)
    for q, s in ((codes, scales), (codes2, scales2)):
        assert torch.equal(s.isnan(), touched) and not q.movedim(1, -1)[touched].any()
        assert torch.equal(tvdcn.dequantize_int8(q, s, dtype).isnan().all(1), touched)
    b = leaf(bad)
    dx, = torch.autograd.grad(tvdcn.rms_norm(b, w), b, torch.ones_like(b))
    a = leaf(x)
    dx0, = torch.autograd.grad(tvdcn.rms_norm(a, w), a, torch.ones_like(a))
    assert torch.equal(dx[clean], dx0[clean]) and dx[0, :, 0].isnan().all()


@pytest.mark.parametrize("channels", [24, 71, 2500, 9001, 40000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norms_of_values_whose_squares_are_no_float32(channels, dtype):
    x, w = make((6, channels), dtype, 1), make((channels,), dtype, 2, shift=1.0)
    x = x * torch.tensor([1e30, 1e36, 6e37, 1e19, 1e-30, 0.0], device="cuda")[:, None].to(dtype)
    assert torch.isfinite(x).all()
    for eps in (1e-6, 1e-37, 1e36):
        check([tvdcn.rms_norm(x, w, eps)], rms(x, None, w, eps), eps)
        check_rms_int8(*tvdcn.rms_norm_int8(x, w, eps), x, w, eps)
    assert not tvdcn.rms_norm(x, w)[5].any()
    a, dy = leaf(x[:4]), make((4, channels), dtype, 3)
    dx, = torch.autograd.grad(tvdcn.rms_norm(a, w), a, dy)
    check([dx], rms(x[:4], None, w, 1e-6, None, dy)[1:2])


PRODUCTS = [((1, 1), 1), ((1, 256), 1024), ((3, 7, 5), 9), ((1, 16, 1), 8), ((2, 71, 11, 13), 101), ((1, 64, 63), 65), ((300, 33), 130),
            ((1, 128, 257), 64), ((17, 2048), 96), ((1, 4100), 40), ((2, 512, 40, 41), 256), ((5, 100, 9, 2, 3), 3), ((1, 48, 5000), 4),
            ((1, 20000), 24), ((64, 1000), 1000), ((33, 15), 520), ((15, 272), 1001)]


def codes_of(shape, seed):
    """An 8-bit map whose every byte value occurs, -128 too."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-128, 128, (shape[0], *shape[2:], shape[1]), generator=g, dtype=torch.int8).movedim(-1, 1)
    s = torch.rand(shape[0], *shape[2:], generator=g) * 0.02 + 0.001
    return q.cuda(), s.cuda()


@pytest.mark.parametrize("shape,out", PRODUCTS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_int8_products(shape, out, dtype):
    a = [*codes_of(shape, 1), *codes_of((out, shape[1]), 2)]
    b, r = make((out,), dtype, 3), make((shape[0], out, *shape[2:]), dtype, 4)
    for act, bias, res in (("none", None, None), ("relu", b, r), ("silu", None, r), ("gelu", b, None)):
        y = tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype)
        check([y], [pointwise_int8(*a, bias, res, act, dtype)], (shape, out, act))


@pytest.mark.parametrize("rows,channels,out", [(65536, 64, 256), (65536, 144, 520), (40000, 512, 264), (70001, 71, 72), (66000, 256, 136),
                                               (16391, 320, 300), (20000, 1024, 1024), (8200, 128, 33), (4096, 80, 2048)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_int8_products_of_many_pixels(rows, channels, out, dtype):
    a = [*codes_of((rows, channels), 1), *codes_of((out, channels), 2)]
    b, r = make((out,), dtype, 3), make((rows, out), dtype, 4)
    for act, bias, res in (("none", None, None), ("gelu", b, r)):
        y = tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype)
        check([y], [pointwise_int8(*a, bias, res, act, dtype)], act)


def test_int8_products_are_summed_exactly():
    """The longest sums of the largest products, which only whole numbers hold."""
    c = 131071
    q = torch.full((3, c), -128, dtype=torch.int8, device="cuda")
    q[1] = 127
    q[2, ::2] = 127
    w = torch.full((9, c), -128, dtype=torch.int8, device="cuda")
    w[4] = 127
    one = torch.ones(9, device="cuda")
    y = tvdcn.pointwise_conv_int8(q, one[:3], w, one, dtype=torch.float32)
    assert torch.equal(y, (q.double() @ w.double().t()).float())
    # a result that cancels: exact where float32's sums would not be
    w[:, 1::2] = 127
    y = tvdcn.pointwise_conv_int8(q, one[:3], w, one, dtype=torch.float32)
    assert torch.equal(y, (q.double() @ w.double().t()).float())


DROPS = [(1, 1), (3, 37, 4, 3), (5, 3), (2, 8, 3), (1, 1001), (4, 64, 50), (1, 3, 3, 3, 3), (2, 512, 640)]


@pytest.mark.parametrize("shape", DROPS, ids=str)
@pytest.mark.parametrize("dtype", DTYPES)
def test_dropout(shape, dtype):
    for p, seed in ((0.1, SEED), (0.5, -1), (0.9, -2 ** 63), (0.0, 7), (1.0, 2 ** 63 - 1)):
        x, r, dy = (make(shape, dtype, i) for i in (1, 2, 3))
        for res in (None, r):
            t = [leaf(v) for v in (x, res) if v is not None]
            y = tvdcn.seeded_dropout(t[0], p, seed_of(seed), *t[1:])
            want, bound, mask = dropout(x, p, seed, res)
            check([y], [(want, bound)], (shape, p))
            dx, *dr = torch.autograd.grad(y, t, dy)
            check([dx], [dropout(dy, p, seed)[:2]])
            assert all(torch.equal(g, dy) for g in dr) and not dx[~mask].any()


def test_dropout_drops_what_is_not_finite():
    x = torch.full((64, 65), math.nan, device="cuda")
    x[:, ::3] = math.inf
    y = tvdcn.seeded_dropout(x, 0.5, seed_of(), torch.ones_like(x))
    mask = dropout(torch.ones_like(x), 0.5, SEED)[2]
    assert torch.equal(~y.isfinite(), mask) and (y[~mask] == 1).all()


def test_dropout_draws_its_seed_from_the_generator():
    x = torch.ones(64, 64, device="cuda")
    torch.manual_seed(5)
    a, b = tvdcn.seeded_dropout(x, 0.5), tvdcn.seeded_dropout(x, 0.5)
    torch.manual_seed(5)
    assert torch.equal(tvdcn.seeded_dropout(x, 0.5), a) and not torch.equal(a, b)


def test_memory_orders_and_alignment():
    """Strided, offset and NC<spatial> maps, parameters, scales and gradients: the results of their channels-last copies."""
    x, r, dy, ds = (make((3, 40, 6, 7), torch.bfloat16, i) for i in range(4))
    w = make((40,), torch.bfloat16, 9, shift=1.0)

    def others(t):
        off = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")[1:].view(3, 6, 7, 40)
        off.copy_(t.movedim(1, -1))
        wide = torch.empty(3, 50, 6, 7, dtype=t.dtype, device="cuda")
        wide[:, 5:45] = t
        return [t.contiguous(), off.movedim(-1, 1), wide[:, 5:45], t.transpose(2, 3).contiguous().transpose(2, 3)]

    def all_of(x, r, w, dy, ds):
        t = [leaf(v) for v in (x, r, w)]
        y, s = tvdcn.add_rms_norm(*t)
        got = [y, s, *torch.autograd.grad([y, s], t, [dy, ds]), *tvdcn.add_rms_norm_int8(x, r, w), *tvdcn.quantize_int8(x)]
        codes, scales = got[-2:]
        got += [tvdcn.seeded_dropout(x, 0.3, seed_of(), r), tvdcn.dequantize_int8(codes, scales, torch.half)]
        a = leaf(x)
        got += torch.autograd.grad(tvdcn.seeded_dropout(a, 0.3, seed_of()), a, dy)
        return [t.detach() for t in got]

    want = all_of(x, r, w, dy, ds)
    for v in zip(*[others(t) for t in (x, r, dy, ds)]):
        odd = torch.empty(81, dtype=w.dtype, device="cuda")[1:]
        odd[::2] = w
        for g, e in zip(all_of(v[0], v[1], odd[::2], v[2], v[3]), want):
            assert torch.equal(g, e)
    # codes and scales of the product
    q, s = codes_of((3, 40, 6, 7), 5)
    wq, ws = codes_of((24, 40), 6)
    b, res = make((24,), torch.bfloat16, 7), make((3, 24, 6, 7), torch.bfloat16, 8)
    want = tvdcn.pointwise_conv_int8(q, s, wq, ws, b, res, "silu")
    offset = torch.empty(24 * 40 + 3, dtype=torch.int8, device="cuda")[3:].view(24, 40)
    offset.copy_(wq)
    strided = torch.stack([s, s], -1)[..., 0]
    got = tvdcn.pointwise_conv_int8(q.contiguous(), strided, offset, torch.stack([ws, ws], 1)[:, 0], b, res.contiguous(), "silu")
    assert torch.equal(got, want)
    assert torch.equal(tvdcn.dequantize_int8(q.contiguous(), strided, torch.float32), tvdcn.dequantize_int8(q, s, torch.float32))


def test_gradients_that_are_expanded():
    """A sum's gradient: one value for the whole map."""
    x, w = make((3, 40, 6, 7), torch.float32, 1), make((40,), torch.float32, 2, shift=1.0)
    a, b = leaf(x), leaf(w)
    tvdcn.rms_norm(a, b).sum().backward()
    check([a.grad, b.grad], rms(x, None, w, 1e-6, None, torch.ones_like(x))[1:])
    # of one of the two results
    t = [leaf(v) for v in (x, x * 0.5, w)]
    y, s = tvdcn.add_rms_norm(*t)
    got = torch.autograd.grad(s.sum(), t, retain_graph=True, allow_unused=True)
    assert (got[0] == 1).all() and (got[1] == 1).all() and (got[2] is None or not got[2].any())
    got = torch.autograd.grad(y.sum(), t)
    check([got[0], got[2]], rms(x, t[1].detach(), w, 1e-6, s.detach(), torch.ones_like(x))[2:])


def test_gradients_against_differences():
    """The gradients against central differences of the forward, in float32 along random directions."""
    x, r, w = (make(s, torch.float32, i, shift=h) for i, (s, h) in enumerate((((2, 24, 5), 0), ((2, 24, 5), 0), ((24,), 1.0))))
    dy, ds = make((2, 24, 5), torch.float32, 5), make((2, 24, 5), torch.float32, 6)

    def f(x, r, w):
        y, s = tvdcn.add_rms_norm(tvdcn.seeded_dropout(x, 0.25, seed_of(), r), r, w)
        return (y.double() * dy).sum() + (s.double() * ds).sum()

    t = [leaf(v) for v in (x, r, w)]
    grads = torch.autograd.grad(f(*t), t)
    h = 2.0 ** -7
    for i, v in enumerate((x, r, w)):
        d = make(tuple(v.shape), torch.float32, 20 + i)
        args = [x, r, w]
        plus, minus = (f(*args[:i], v + k * h * d, *args[i + 1:]) for k in (1, -1))
        slope = (plus - minus) / (2 * h)
        want = (grads[i].double() * d).sum()
        # the differences' third order, h^2 times terms of the slope's size, and float32's roundings over 2 h of sums of about 500 terms
        assert abs(slope - want) <= 20 * h * h * (grads[i].abs() * d.abs()).sum() + 500 * 2.0 ** -23 / h


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_without_data_have_the_layouts_of_the_results(dtype):
    for shape in SHAPES:
        assert layouts("cuda", dtype, shape) == layouts("meta", dtype, shape), shape


def test_empty_maps():
    for shape in ((0, 6, 4), (2, 6, 0)):
        x, w = torch.zeros(shape, requires_grad=True, device="cuda"), torch.ones(6, requires_grad=True, device="cuda")
        y, s = tvdcn.add_rms_norm(tvdcn.seeded_dropout(x, 0.5, seed_of()), x, w)
        (y.sum() + s.sum()).backward()
        assert x.grad.shape == shape and not w.grad.any()


def test_block_in_training():
    """Norm, two products, dropout and the shortcut together, forward and all gradients, against the chain in float64."""
    torch.manual_seed(11)
    m = Block(40).cuda()
    x, r = make((2, 40, 9, 11), torch.float32, 1), make((2, 40, 9, 11), torch.float32, 2)
    dy = make((2, 40, 9, 11), torch.float32, 3)
    a, b = leaf(x), leaf(r)
    torch.manual_seed(12)
    y = m(a, b)
    params = list(m.parameters())
    got = [y.detach(), *torch.autograd.grad(y, [a, b, *params], dy)]
    torch.manual_seed(12)
    seed = int(torch.randint(0x7FFFFFFFFFFFFFFF, [1], dtype=torch.int64, device="cuda"))
    drop = round(65536 * 0.1)
    mask = dropout(x, 0.1, seed)[2].movedim(1, -1).double() * (65536 / (65536 - drop))
    p = [leaf(t.double()) for t in params]   # norm.weight, wide.weight, wide.bias, narrow.weight, narrow.bias, last.weight
    a, b = leaf(x.double().movedim(1, -1)), leaf(r.double().movedim(1, -1))

    def norm(v, w):
        return v * (v.square().mean(-1, keepdim=True) + 1e-6).rsqrt() * w

    s = a + b
    z = norm(s, p[0]).reshape(-1, 40) @ p[1].t() + p[2]
    z = ((z * torch.special.ndtr(z)) @ p[3].t() + p[4]).view(s.shape)
    y = norm(z * mask + s, p[5])
    want = [y, *torch.autograd.grad(y, [a, b, *p], dy.double().movedim(1, -1))]
    for g, e in zip(got, want):
        e = e.movedim(-1, 1) if e.dim() == 4 else e
        # six operators of float32, sums of up to 198 rows x 160 channels: some hundred roundings of the result's size
        assert (g.double() - e).norm() <= 256 * 2.0 ** -24 * e.norm()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_block_in_8_bits(dtype):
    """A served block: normalised into 8 bits, widened, quantized, narrowed onto the shortcut, each step on what the last gave."""
    c, x, r = 64, make((2, 64, 9, 11), dtype, 1), make((2, 64, 9, 11), dtype, 2)
    w = make((c,), dtype, 3, shift=1.0, spread=0.2)
    wide, narrow = tvdcn.PointwiseConv(c, 4 * c, activation="gelu").to("cuda", dtype), tvdcn.PointwiseConv(4 * c, c).to("cuda", dtype)
    wide8, narrow8 = tvdcn.PointwiseConvInt8.from_float(wide), tvdcn.PointwiseConvInt8.from_float(narrow)
    with torch.no_grad():
        codes, scales, s = tvdcn.add_rms_norm_int8(x, r, w)
        h = wide8(codes, scales)
        y = narrow8(h, residual=s)
    check_rms_int8(codes, scales, s, w, 1e-6)
    check([h], [pointwise_int8(codes, scales, wide8.weight_codes, wide8.weight_scales, wide8.bias, None, "gelu", dtype)])
    q, sc = quantize(h.movedim(1, -1).double())
    q = q.to(torch.int8).movedim(-1, 1)
    check([y], [pointwise_int8(q, sc, narrow8.weight_codes, narrow8.weight_scales, narrow8.bias, s, "none", dtype)])
    # beside the block in 16 bits: each quantization is off by at most half of 1/127 of a row's largest value
    with torch.no_grad():
        plain = narrow(wide(tvdcn.add_rms_norm(x, r, w)[0]), s)
    assert (y - plain).float().norm() < 0.02 * plain.float().norm()


def test_results_do_not_change_from_call_to_call():
    x, r, w = make((4, 200, 50, 41), torch.bfloat16, 1), make((4, 200, 50, 41), torch.bfloat16, 2), make((200,), torch.bfloat16, 3)
    a = [*codes_of((4, 200, 50, 41), 1), *codes_of((160, 200), 2)]

    def run():
        t = [leaf(v) for v in (x, r, w)]
        y, s = tvdcn.add_rms_norm(*t)
        return [y, s, *torch.autograd.grad([y, s], t, [x, r]), *tvdcn.add_rms_norm_int8(x, r, w), tvdcn.pointwise_conv_int8(*a)]

    first = run()
    for _ in range(3):
        for g, e in zip(run(), first):
            assert torch.equal(g, e)


def test_streams():
    """Calls on several streams at once, each with its own results and workspaces, as on one."""
    streams = [torch.cuda.Stream() for _ in range(3)]
    cases = [(make((2, 71, 40, 30), torch.float32, i), make((71,), torch.float32, 10 + i, shift=1.0), codes_of((2, 71, 40, 30), i),
              codes_of((50, 71), 20 + i), seed_of(i)) for i in range(3)]

    def run(x, w, q, wq, seed):
        t = [leaf(x), leaf(w)]
        y = tvdcn.rms_norm(*t)
        return [y.detach(), *torch.autograd.grad(y, t, x), tvdcn.pointwise_conv_int8(*q, *wq), tvdcn.seeded_dropout(x, 0.3, seed, x)]

    want = [run(*c) for c in cases]
    torch.cuda.synchronize()
    for _ in range(3):
        got = []
        for s, c in zip(streams, cases):
            with torch.cuda.stream(s):
                got.append(run(*c))
        torch.cuda.synchronize()
        for g, e in zip(got, want):
            assert all(torch.equal(a, b) for a, b in zip(g, e))


def captured(step):
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    return graph, out


def test_graph_in_training():
    """Forward and backward captured and replayed on new inputs and seeds, with eager calls between, against the eager results."""
    dtype, shape = torch.bfloat16, (2, 72, 24, 20)
    x, r, dy = (make(shape, dtype, i) for i in (1, 2, 3))
    w, seed = make((72,), dtype, 4, shift=1.0), seed_of()

    def step():
        t = [leaf(v) for v in (x, r, w)]
        y, s = tvdcn.add_rms_norm(tvdcn.seeded_dropout(t[0], 0.2, seed, t[1]), t[1], t[2])
        return [y.detach(), s.detach(), *torch.autograd.grad([y, s], t, [dy, dy])]

    graph, out = captured(step)
    for n in (100, 200, 300):
        for k, t in enumerate((x, r, dy)):
            t.copy_(make(shape, dtype, n + k))
        seed.fill_(n)
        want = step()
        graph.replay()
        torch.cuda.synchronize()
        for g, e in zip(out, want):
            assert torch.equal(g, e)


def test_graphs_that_share_a_memory_pool_and_draw_their_own_seeds():
    """Served and drawing steps in two graphs, replayed in turn, on new inputs; every replay of a drawing one drops others."""
    x, w = make((2, 71, 24, 20), torch.float16, 1), make((71,), torch.float16, 2, shift=1.0)
    wq = codes_of((50, 71), 3)

    def served():
        with torch.no_grad():
            codes, scales = tvdcn.rms_norm_int8(x, w)
            return tvdcn.pointwise_conv_int8(codes, scales, *wq, activation="gelu", dtype=torch.float16)

    def drawn():
        return tvdcn.seeded_dropout(torch.ones_like(x), 0.5)

    graphs = [captured(served), captured(drawn)]
    masks = []
    for n in (100, 200, 300):
        x.copy_(make(tuple(x.shape), torch.float16, n))
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(graphs[0][1], served())
        masks.append(graphs[1][1].bool().clone())
        assert abs(masks[-1].float().mean().item() - 0.5) < 0.02
    assert not torch.equal(masks[0], masks[1]) and not torch.equal(masks[1], masks[2])


def test_autocast():
    x, r, w = make((2, 32, 9, 9), torch.float32, 1), make((2, 32, 9, 9), torch.float32, 2), make((32,), torch.float32, 3)
    q, wq, b = codes_of((2, 32, 9, 9), 1), codes_of((16, 32), 2), make((16,), torch.float32, 4)
    h = x.half()
    with torch.autocast("cuda", torch.float16):
        got = [tvdcn.rms_norm(h, w), *tvdcn.add_rms_norm(h, r, w), *tvdcn.rms_norm_int8(h, w), *tvdcn.add_rms_norm_int8(h, r, w),
               tvdcn.pointwise_conv_int8(*q, *wq, b, None, "relu", torch.float16), tvdcn.seeded_dropout(h, 0.5, seed_of(), r)]
    f = h.float()
    want = [tvdcn.rms_norm(h, w.half()), *tvdcn.add_rms_norm(f, r, w), *tvdcn.rms_norm_int8(h, w.half()), *tvdcn.add_rms_norm_int8(f, r, w),
            tvdcn.pointwise_conv_int8(*q, *wq, b.half(), None, "relu", torch.float16), tvdcn.seeded_dropout(f, 0.5, seed_of(), r)]
    for g, e in zip(got, want):
        assert g.dtype == e.dtype and torch.equal(g, e)


def test_compiled_training_step():
    m = Block(24).cuda()
    x, r = leaf(make((2, 24, 9, 5), torch.float32, 1)), leaf(make((2, 24, 9, 5), torch.float32, 2))
    m.drop.p = 0.0
    y = m(x, r)
    want = [y, *torch.autograd.grad(y.square().sum(), [x, r, *m.parameters()])]
    fast = torch.compile(m, backend="aot_eager", fullgraph=True)
    y = fast(x, r)
    got = [y, *torch.autograd.grad(y.square().sum(), [x, r, *m.parameters()])]
    for g, e in zip(got, want):
        assert torch.allclose(g, e, rtol=1e-5, atol=1e-6 * e.abs().max().item())


def test_maps_beyond_32_bit_offsets():
    """More than 2^31 values: the last rows of each result against float64, and the first."""
    rows, c = 4200000, 520
    gen = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(rows, c, generator=gen, device="cuda", dtype=torch.bfloat16)
    w = (1 + 0.2 * torch.randn(c, generator=gen, device="cuda")).bfloat16()
    parts = (slice(0, 300), slice(rows - 300, rows))
    dy = torch.zeros_like(x)
    dy[-200:] = torch.randn(200, c, generator=gen, device="cuda").bfloat16()
    a, b = leaf(x), leaf(w)
    y, s = tvdcn.add_rms_norm(a, x, b)
    for part in parts:
        check([y[part], s[part]], rms(x[part], x[part], w, 1e-6, s[part].detach()))
    dx, dw = torch.autograd.grad(y, [a, b], dy)
    check([dx[-200:], dw], rms(x[-200:], x[-200:], w, 1e-6, s[-200:].detach(), dy[-200:])[2:])
    assert not dx[:-200].any()
    del y, dx, a, dy
    codes, scales = tvdcn.quantize_int8(x)
    for part in parts:
        q, sc = quantize(x[part].double())
        assert torch.equal(codes[part].double(), q) and torch.equal(scales[part], sc)
    back = tvdcn.dequantize_int8(codes, scales, torch.float16)
    for part in parts:
        check([back[part]], [dequantize(codes[part], scales[part], torch.float16)])
    del back
    for out, cc in ((40, c), (24, 519)):   # multiplied as they lie, and from a copy
        q = codes if cc == c else codes[:, :cc].contiguous()
        wq = codes_of((out, cc), 2)
        y = tvdcn.pointwise_conv_int8(q, scales, *wq, dtype=torch.float32)
        for part in parts:
            check([y[part]], [pointwise_int8(q[part], scales[part], *wq, None, None, "none", torch.float32)])
    del codes, y, q
    y = tvdcn.seeded_dropout(x, 0.5, seed_of(), s.detach())
    for part in parts:
        n, first = 300 * c, part.start * c
        mask = kept(n, 0.5, SEED, first).view(300, c).cuda()
        want = torch.where(mask, 2 * x[part].float(), 0.0) + s[part].detach().float()
        assert torch.equal(y[part], want.bfloat16())


def test_a_result_beyond_32_bit_offsets():
    rows, c, out = 1100000, 32, 2000
    q, s = codes_of((rows, c), 1)
    wq = codes_of((out, c), 2)
    y = tvdcn.pointwise_conv_int8(q, s, *wq)
    for part in (slice(0, 300), slice(rows - 300, rows)):
        check([y[part]], [pointwise_int8(q[part], s[part], *wq, None, None, "none", torch.bfloat16)])


def test_kernel_timer_families():
    import ctypes
    lib = ctypes.CDLL(tvdcn.extension.HIP_LIB_PATH)
    x = make((4, 24, 6), torch.float32, 1)
    q, wq = codes_of((4, 24, 6), 1), codes_of((8, 24), 2)
    lib.tvdcn_kernel_timer_enable(1)
    try:
        tvdcn.rms_norm(x), tvdcn.pointwise_conv_int8(*q, *wq), tvdcn.seeded_dropout(x, 0.5, seed_of()), tvdcn.quantize_int8(x)
        ms, n = ctypes.c_double(), ctypes.c_int64()
        for family in (8, 9, 10, 11):
            assert lib.tvdcn_kernel_timer_read(family, ctypes.byref(ms), ctypes.byref(n)) == 0 and n.value == 1
    finally:
        lib.tvdcn_kernel_timer_enable(0)


@pytest.mark.parametrize("seed", range(16))
def test_int8_products_of_random_sizes(seed):
    """Sizes that fill the chip with the largest tiles and end anywhere in them: one stage along the reduction to many, one tile a
    workgroup to several, whole tiles and ragged ones, with and without what is added."""
    import random
    rng = random.Random(seed)
    channels = rng.choice((16, 64, 128, 144, 256, 257, 384, 1040, 2048))
    out = 8 * rng.randint(1, 96) if seed % 4 else rng.randint(1, 700)
    rows = rng.randint(1, 1 << 25) // max(channels, 256) * 256 // out
    rows = max(1, min(rows if seed % 3 else rows // 256 * 256, 120000))
    dtype = DTYPES[seed % 3]
    a = [*codes_of((rows, channels), seed), *codes_of((out, channels), seed + 1)]
    b, r = make((out,), dtype, 3), torch.randn(rows, out, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)
    for act, bias, res in (("none", None, r), ("silu", b, r), ("relu", b, None)):
        y = tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype)
        check([y], [pointwise_int8(*a, bias, res, act, dtype)], (rows, channels, out, act))


def test_int8_products_of_rows_in_several_launches():
    """So many tiles that the rows go out in runs: the rows at the border between them, and the last."""
    rows, channels, out = (1 << 21) // (1 << 14) * 64 + 70, 24, 1 << 20
    q, s = codes_of((rows, channels), 1)
    wq, ws = codes_of((out, channels), 2)
    r = torch.randn(rows, out, generator=torch.Generator("cuda").manual_seed(3), device="cuda", dtype=torch.bfloat16)
    y = tvdcn.pointwise_conv_int8(q, s, wq, ws, None, r)
    for part in (slice(0, 70), slice(rows - 200, rows)):
        for cols in (slice(0, 500), slice(out - 500, out)):
            want = pointwise_int8(q[part], s[part], wq[cols], ws[cols], None, r[part, cols], "none", torch.bfloat16)
            check([y[part, cols]], [want], (part, cols))


@pytest.mark.parametrize("channels", [24, 71, 2500, 4097, 8192, 40000, 1 << 20])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_norms_of_the_largest_finite_values(channels, dtype):
    """Rows at the type's largest finite value, of one sign, of both, beside small values, and alone among zeros, with the least and
    the largest eps."""
    most = torch.finfo(dtype).max
    x = make((6, channels), dtype, 1)
    x[0], x[1], x[2] = most, x[2].sign() * most, 2e38
    x[3, ::2] = -most
    x[4] = 0
    x[4, channels // 2] = most
    x[5] = 0
    x[5, 0] = 1.8e19                # (its square is a float32, the mean of that with the largest eps is none)
    w, dy = make((channels,), dtype, 2, shift=1.0), make((6, channels), dtype, 3)
    assert torch.isfinite(x).all()
    for eps in (1e-6, 2e-38, 3.4e38):
        t = [leaf(x), leaf(w)]
        y = tvdcn.rms_norm(*t, eps)
        want = rms(x, None, w, eps, None, dy)
        # beside the largest values the small ones' product with the reciprocal root is subnormal: it is rounded to a multiple of
        # 2^-149, by up to 2^-150, and then multiplied by the weight
        want[0] = want[0][0], want[0][1] + 2.0 ** -150 * w.double().abs()
        check([y, *torch.autograd.grad(y, t, dy)], want, eps)
        assert y[:5].any(1).all()
        check_rms_int8(*tvdcn.rms_norm_int8(x, w, eps), x, w, eps)
    y, s = tvdcn.add_rms_norm(x, torch.zeros_like(x), w)
    assert torch.equal(s, x) and torch.equal(y, tvdcn.rms_norm(x, w))
    codes, scales, s = tvdcn.add_rms_norm_int8(x, torch.zeros_like(x))
    assert torch.equal(s, x) and (codes[:2].abs() == 127).all()


# of every kernel that takes the products: straight from memory, tiles of 64, of 128, the persistent ones
@pytest.mark.parametrize("rows,channels,out", [(5, 64, 40), (70, 71, 30), (4096, 512, 512), (4100, 333, 264), (65536, 1024, 300), (20000, 64, 128),
                                               (100000, 64, 128), (65536, 64, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_int8_products_of_scales_at_the_range_ends(rows, channels, out, dtype):
    """Scales of 2^112 to 2^120 with some of 2^-126: their product with the sums alone is no float32, the result is an ordinary value.
    On rows among others, and on columns."""
    (q, _), (wq, _) = codes_of((rows, channels), 1), codes_of((out, channels), 2)
    g = torch.Generator().manual_seed(3)

    def scales(n):
        far, near = (torch.exp2(torch.randint(lo, lo + 9, (n,), generator=g)) * (1 + torch.rand(n, generator=g)) for lo in (112, 0))
        return torch.where(torch.rand(n, generator=g) < 0.1, far, near).cuda()

    least = [torch.full((n,), 2.0 ** -126, device="cuda") for n in (rows, out)]
    r = make((rows, out), dtype, 4)
    for s, ws in ((scales(rows), least[1]), (least[0], scales(out))):
        for act, res in (("none", None), ("relu", r)):
            y = tvdcn.pointwise_conv_int8(q, s, wq, ws, None, res, act, dtype)
            assert y.isfinite().all()
            check([y], [pointwise_int8(q, s, wq, ws, None, res, act, dtype)], act)


# Tiles of 128 x 128 (the first three), persistent ones of 256 x 128 and of 256 x 256, these with one stage along the reduction and
# several tiles to a workgroup: whole tiles and ragged ones, rows of codes multiplied as they lie and copied first
@pytest.mark.parametrize("rows,channels,out", [(65536, 1024, 300), (65537, 512, 1001), (50001, 900, 350), (131072, 128, 128), (100000, 64, 128),
                                               (65536, 100, 384), (65536, 64, 512), (66000, 128, 1000), (70001, 64, 520), (70001, 120, 512)])
@pytest.mark.parametrize("dtype", DTYPES)
def test_int8_products_of_many_tiles(rows, channels, out, dtype):
    a = [*codes_of((rows, channels), 1), *codes_of((out, channels), 2)]
    b = make((out,), dtype, 3)
    r = torch.randn(rows, out, device="cuda", generator=torch.Generator("cuda").manual_seed(4)).to(dtype)
    for act, bias, res in (("none", None, None), ("none", None, r), ("relu", b, r), ("gelu", b, None)):
        y = tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype)
        check([y], [pointwise_int8(*a, bias, res, act, dtype)], act)
        # (loads and stores that overlap from tile to tile: again, and beside another product)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype)
        assert torch.equal(tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype), y)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(other, y)


@pytest.mark.parametrize("seed", range(18))
def test_int8_products_of_random_sizes_and_types(seed):
    """As above, each of type, whole tiles of rows, columns by eights, and what is added drawn by itself."""
    import random
    rng = random.Random(1000 + seed)
    channels, dtype = rng.choice((16, 48, 64, 100, 128, 192, 256, 520, 1024)), DTYPES[rng.randrange(3)]
    out = 8 * rng.randint(1, 128) if rng.random() < 0.7 else rng.randint(1, 1000)
    rows = max(1, min(int(2 ** rng.uniform(10, 25)) // out, 140000))
    rows = -(-rows // 256) * 256 if rng.random() < 0.5 else rows
    a = [*codes_of((rows, channels), seed), *codes_of((out, channels), seed + 1)]
    b, r = make((out,), dtype, 3), torch.randn(rows, out, device="cuda", generator=torch.Generator("cuda").manual_seed(seed)).to(dtype)
    for act in ACTIVATIONS:
        bias, res = (b if rng.random() < 0.5 else None), (r if rng.random() < 0.5 else None)
        y = tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype)
        check([y], [pointwise_int8(*a, bias, res, act, dtype)], (rows, channels, out, act, dtype, bias is None, res is None))
