"""The operators that take a pixel's channels as one vector without a GPU: the host kernels against the float64 definitions,
gradients against differences, refusals (Python, operators and C ABI), shapes without data, TorchScript, compilation, modules."""
import ctypes
import math

import numpy as np
import pytest
import torch

import tvdcn
from map_reference import ACTIVATIONS, as_map, as_rows, check, make
from row_reference import check_rms_int8, dropout, kept, philox, pointwise_int8, quantize, rms

DTYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]
OPS = torch.ops.tvdcn
SEED = 0x123456789ABCDEF


def leaf(t):
    return None if t is None else t.detach().requires_grad_(True)


def cpu(shape, dtype, seed, **kw):
    return make(shape, dtype, seed, device="cpu", **kw)


def seed_of(v=SEED):
    return torch.tensor([v])


@pytest.mark.parametrize("dtype", DTYPES)
def test_host_norms(dtype):
    for shape in ((3, 36, 5, 7), (2, 1, 4), (5, 71)):
        x, r, w = cpu(shape, dtype, 1), cpu(shape, dtype, 2), cpu((shape[1],), dtype, 3, shift=1.0)
        dy, ds = cpu(shape, dtype, 4), cpu(shape, dtype, 5)
        t = [leaf(v) for v in (x, r, w)]
        y, s = tvdcn.add_rms_norm(*t)
        dx, dr, dw = torch.autograd.grad([y, s], t, [dy, ds])
        check([y, s, dx, dw], rms(x, r, w, 1e-6, s.detach(), dy, ds))
        assert torch.equal(dx, dr)
        t = [leaf(v) for v in (x, w)]
        y = tvdcn.rms_norm(*t, 0.1)
        check([y, *torch.autograd.grad(y, t, dy)], rms(x, None, w, 0.1, None, dy))
        check([tvdcn.rms_norm(x)], rms(x, None, None, 1e-6))
        if dtype != torch.float64:
            codes, scales, s = tvdcn.add_rms_norm_int8(x, r, w)
            check_rms_int8(codes, scales, s, w, 1e-6)
            check_rms_int8(*tvdcn.rms_norm_int8(x), x, None, 1e-6)


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_host_8_bits(dtype):
    x = cpu((2, 71, 5), dtype, 1, spread=3.0)
    x[0, :, 1] = 0
    x[0, 3, 2], x[1, 0, 0], x[1, 70, 4] = math.inf, math.nan, -math.inf
    codes, scales = tvdcn.quantize_int8(x)
    q, s = quantize(x.movedim(1, -1).double())
    assert codes.dtype == torch.int8 and scales.dtype == torch.float32 and scales.shape == (2, 5)
    assert torch.equal(codes.movedim(1, -1).double(), q) and torch.equal(scales.nan_to_num(-1), s.nan_to_num(-1))
    for out in DTYPES[1:]:
        y = tvdcn.dequantize_int8(codes, scales, out)
        want = (codes.float() * scales.unsqueeze(1)).to(out)
        assert y.dtype == out and torch.equal(y.isnan(), want.isnan()) and torch.equal(y.nan_to_num(0), want.nan_to_num(0))
    assert scales[0, 1] == 2.0 ** -126 and y[0, :, 2].isnan().all() and not codes[0, :, 1].any()


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_host_int8_product(dtype):
    x, w = cpu((3, 37, 4, 3), torch.float32, 1), cpu((10, 37), torch.float32, 2)
    a = [*tvdcn.quantize_int8(x), *tvdcn.quantize_int8(w)]
    b, r = cpu((10,), dtype, 3), cpu((3, 10, 4, 3), dtype, 4)
    for act in ACTIVATIONS:
        for bias, res in ((b, r), (None, None), (b, None)):
            y = tvdcn.pointwise_conv_int8(*a, bias, res, act, dtype)
            check([y], [pointwise_int8(*a, bias, res, act, dtype)], act)
    # near the product of the values: half a step of each, of at most 1/127 of the largest
    near = tvdcn.pointwise_conv_int8(*a, dtype=torch.float32) - tvdcn.pointwise_conv(x, w)
    assert near.abs().max() < 37 * (x.abs().max() * w.abs().max()) / 127


def test_philox_is_the_published_generator():
    """Known answers of Philox4x32-10 that its authors publish with their library (zeros, ones, digits of pi)."""
    ones = 0xFFFFFFFF
    for counter, key, want in (
            ((0, 0, 0, 0), (0, 0), (0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8)),
            ((ones,) * 4, (ones,) * 2, (0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD)),
            ((0x243F6A88, 0x85A308D3, 0x13198A2E, 0x03707344), (0xA4093822, 0x299F31D0),
             (0xD16CFE09, 0x94FDCCEB, 0x5001E420, 0x24126EA1))):
        assert tuple(int(v) for v in philox(np.array([counter], np.uint64), key)[0]) == want


@pytest.mark.parametrize("dtype", DTYPES)
def test_host_dropout(dtype):
    for shape, p, seed in (((3, 37, 4, 3), 0.3, SEED), ((5, 3), 0.5, -1), ((1, 1, 1), 0.9, -2 ** 63), ((2, 8, 3), 0.0, 0),
                           ((2, 8, 3), 1.0, 2 ** 63 - 1), ((2, 8, 3), 2.0 ** -18, 5)):
        x, r = cpu(shape, dtype, 1), cpu(shape, dtype, 2)
        for res in (None, r):
            t = [leaf(v) for v in (x, res) if v is not None]
            y = tvdcn.seeded_dropout(t[0], p, seed_of(seed), *t[1:])
            want, bound, mask = dropout(x, p, seed, res)
            check([y], [(want, bound)], (shape, p))
            dy = cpu(shape, dtype, 3)
            dx, *dr = torch.autograd.grad(y, t, dy)
            check([dx], [dropout(dy, p, seed)[:2]])
            assert all(torch.equal(g, dy) for g in dr) and not dx[~mask].any()
    # a dropped value is zero whatever it holds, and the shortcut goes through
    x = torch.full((64, 64), math.nan)
    y = tvdcn.seeded_dropout(x, 0.5, seed_of(), torch.ones(64, 64))
    mask = dropout(torch.ones(64, 64), 0.5, SEED)[2]
    assert torch.equal(y.isnan(), mask) and (y[~mask] == 1).all()


def test_dropout_masks_do_not_depend_on_memory_order_and_have_the_rate():
    x = torch.ones(4, 30, 20, 7)
    y = tvdcn.seeded_dropout(x, 0.25, seed_of())
    for other in (x.to(memory_format=torch.channels_last), x.transpose(2, 3).contiguous().transpose(2, 3), x.half(), x.double()):
        assert torch.equal(tvdcn.seeded_dropout(other, 0.25, seed_of()).bool(), y.bool())
    n = x.numel()
    assert abs(y.bool().sum().item() - 0.75 * n) < 5 * math.sqrt(n * 0.25 * 0.75)   # five standard deviations
    torch.manual_seed(3)
    a = tvdcn.seeded_dropout(x, 0.25)
    b = tvdcn.seeded_dropout(x, 0.25)
    torch.manual_seed(3)
    assert torch.equal(tvdcn.seeded_dropout(x, 0.25), a) and not torch.equal(a, b)


def test_gradients_against_differences():
    def double(*shape):
        return torch.randn(*shape, dtype=torch.float64, requires_grad=True)
    x, r, w = double(2, 6, 3), double(2, 6, 3), double(6)
    assert torch.autograd.gradcheck(lambda *a: tvdcn.rms_norm(*a), (x, w))
    assert torch.autograd.gradcheck(lambda a: tvdcn.rms_norm(a, None, 0.5), (x,))
    assert torch.autograd.gradcheck(lambda *a: tvdcn.add_rms_norm(*a), (x, r, w))
    assert torch.autograd.gradcheck(lambda *a: tvdcn.add_rms_norm(*a)[0], (x, r, w))
    assert torch.autograd.gradcheck(lambda a: tvdcn.add_rms_norm(a, r.detach(), w.detach())[1], (x,))
    assert torch.autograd.gradcheck(lambda a: tvdcn.add_rms_norm(a, a), (x,))   # the same map twice
    assert torch.autograd.gradcheck(lambda *a: tvdcn.seeded_dropout(a[0], 0.4, seed_of(), a[1]), (x, r))
    assert torch.autograd.gradgradcheck(lambda a: tvdcn.seeded_dropout(a, 0.4, seed_of()), (x,))


def test_only_the_gradients_asked_for():
    x, r, w = (torch.randn(s) for s in ((2, 6, 3), (2, 6, 3), (6,)))
    want = torch.autograd.grad(tvdcn.add_rms_norm(*(t := [leaf(v) for v in (x, r, w)]))[0].sum(), t)
    for i in range(3):
        t = [leaf(v) if j == i else v for j, v in enumerate((x, r, w))]
        y, s = tvdcn.add_rms_norm(*t)
        assert s.requires_grad or i == 2
        g, = torch.autograd.grad(y.sum(), t[i])
        assert torch.equal(g, want[i])
    # of the sum alone: what comes in goes out, and the weight has none
    t = [leaf(v) for v in (x, r, w)]
    g = torch.autograd.grad(tvdcn.add_rms_norm(*t)[1], t, torch.ones_like(x), allow_unused=True)
    assert torch.equal(g[0], torch.ones_like(x)) and torch.equal(g[1], torch.ones_like(x)) and (g[2] is None or not g[2].any())


X, W = torch.zeros(2, 6, 3), torch.zeros(6)
Q, S = torch.zeros(2, 6, 3, dtype=torch.int8), torch.zeros(2, 3)
WQ, WS = torch.zeros(4, 6, dtype=torch.int8), torch.zeros(4)


@pytest.mark.parametrize("args,message", [
    ((torch.zeros(6),), "expected a \\(batch, channels"), ((torch.zeros(2, 0, 3),), "needs channels"),
    ((torch.zeros(2, 6, 3, dtype=torch.int32),), "unsupported dtype"), ((X, torch.zeros(5)), "weight of shape"),
    ((X, W.double()), "weight of dtype"), ((X, W.to("meta")), "weight is on meta"), ((X, W, 0.0), "eps"), ((X, W, -1.0), "eps"),
    ((X, W, math.nan), "eps"), ((X, W, 1e-40), "eps"), ((X, W, 1e39), "eps"),
])
def test_norm_refusals(args, message):
    for f in (tvdcn.rms_norm, tvdcn.rms_norm_int8):
        with pytest.raises(RuntimeError, match=message):
            f(*args)
    for f in (tvdcn.add_rms_norm, tvdcn.add_rms_norm_int8):
        with pytest.raises(RuntimeError, match=message):
            f(args[0], args[0], *args[1:])


def test_residual_refusals():
    for f in (tvdcn.add_rms_norm, tvdcn.add_rms_norm_int8, lambda x, r: tvdcn.seeded_dropout(x, 0.5, seed_of(), r)):
        for r, message in ((torch.zeros(2, 6, 1), "residual of shape"), (X.half(), "residual of dtype"), (X.to("meta"), "residual is on")):
            with pytest.raises(RuntimeError, match=message):
                f(X, r)


@pytest.mark.parametrize("args,message", [
    ((Q.float(), S, WQ, WS), "int8 codes"), ((Q[0, 0], S, WQ, WS), "int8 codes"), ((Q, S.double(), WQ, WS), "float32 scales"),
    ((Q, S[:1], WQ, WS), "float32 scales"), ((Q, S.to("meta"), WQ, WS), "scales is on"), ((Q, S, WQ.int(), WS), "weight codes"),
    ((Q, S, WQ[:, :5], WS), "for 6 input channels"), ((Q, S, WQ[None], WS), "weight codes of shape"), ((Q, S, WQ, WS[:3]), "weight scales"),
    ((Q, S, WQ[:0], WS[:0]), "weight codes"), ((Q, S, WQ.to("meta"), WS.to("meta")), "weight codes is on"),
    ((Q, S, WQ, WS, torch.zeros(6)), "bias of shape"), ((Q, S, WQ, WS, torch.zeros(4)), "bias of dtype"),
    ((Q, S, WQ, WS, None, torch.zeros(2, 4, 1)), "residual of shape"), ((Q, S, WQ, WS, None, torch.zeros(2, 4, 3)), "residual of dtype"),
    ((Q, S, WQ, WS, None, None, "none", torch.float64), "float32, float16 and bfloat16"),
    ((Q, S, WQ, WS, None, None, "none", torch.int8), "float32, float16 and bfloat16"),
    ((torch.zeros(1, 131072, dtype=torch.int8), torch.zeros(1), torch.zeros(1, 131072, dtype=torch.int8), torch.zeros(1)), "131071"),
])
def test_int8_product_refusals(args, message):
    with pytest.raises(RuntimeError, match=message):
        tvdcn.pointwise_conv_int8(*args)


def test_other_refusals():
    for x, message in ((torch.zeros(6), "expected a"), (torch.zeros(2, 0), "needs channels"), (X.double(), "bfloat16 maps only"), (Q, "dtype")):
        with pytest.raises(RuntimeError, match=message):
            tvdcn.quantize_int8(x)
    for f in (tvdcn.rms_norm_int8, lambda x: tvdcn.add_rms_norm_int8(x, x)):
        with pytest.raises(RuntimeError, match="bfloat16 maps only"):
            f(X.double())
    for q, s, t in ((Q.float(), S, torch.float32), (Q, S[:1], torch.float32), (Q, S, torch.float64), (Q, S.half(), torch.float32),
                    (Q.to("meta"), S, torch.float32)):
        with pytest.raises(RuntimeError, match="dequantize_int8"):
            tvdcn.dequantize_int8(q, s, t)
    for p, seed, message in ((-0.1, seed_of(), "p must be"), (1.1, seed_of(), "p must be"), (math.nan, seed_of(), "p must be"),
                             (0.5, torch.zeros(2, dtype=torch.int64), "seed of one"), (0.5, torch.zeros(1), "int64 seed"),
                             (0.5, seed_of().to("meta"), "seed is on")):
        with pytest.raises(RuntimeError, match=message):
            tvdcn.seeded_dropout(X, p, seed)
    for make_bad in (lambda: tvdcn.RMSNorm(0), lambda: tvdcn.PointwiseConvInt8(0, 3), lambda: tvdcn.SeededDropout(1.5),
                     lambda: tvdcn.PointwiseConvInt8(3, 3, activation="tanh"),
                     lambda: tvdcn.pointwise_conv_int8(Q, S, WQ, WS, activation="tanh")):
        with pytest.raises(ValueError):
            make_bad()
    with pytest.raises(RuntimeError, match="unknown activation"):
        OPS.pointwise_conv_int8(Q, S, WQ, WS, None, None, 4, torch.float32)
    # the backward operator checks what it is given
    g, st = torch.zeros(2, 6, 3), torch.zeros(2, 3)
    for a in ((g, None, X[:1], st, None), (g, X[:1], X, st, None), (g, None, X, st[:1], None), (g, None, X, st.double(), None),
              (g, None, X, st, W[:5]), (g.half(), None, X, st, None), (g, None, X.to("meta"), st, None)):
        with pytest.raises(RuntimeError, match="rms_norm"):
            OPS._rms_norm_backward(*a, [True] * 2)


def test_lost_gradients_are_refused():
    """Rounding to 8 bits has no gradient: where one would be lost the call says so, and under no_grad it does not."""
    x, w, b = X + 1, leaf(W + 1), leaf(torch.zeros(4))
    calls = [lambda: tvdcn.rms_norm_int8(x, w), lambda: tvdcn.add_rms_norm_int8(x, leaf(x)), lambda: tvdcn.quantize_int8(leaf(x)),
             lambda: tvdcn.dequantize_int8(Q, leaf(S), torch.float32),
             lambda: tvdcn.pointwise_conv_int8(Q, S, WQ, WS, b, dtype=torch.float32),
             lambda: tvdcn.pointwise_conv_int8(Q, leaf(S), WQ, WS)]
    for f in calls:
        with pytest.raises(RuntimeError, match="has no gradient"):
            f()
        with torch.no_grad():
            f()


def test_second_and_forward_mode_derivatives_are_refused():
    x, w, r = (torch.randn(s, requires_grad=True) for s in ((2, 6, 3), (6,), (2, 6, 3)))
    for y in (tvdcn.rms_norm(x, w), tvdcn.add_rms_norm(x, r, w)[0], sum(tvdcn.add_rms_norm(x, r))):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="double backwards on rms_norm not supported"):
            g.sum().backward()
    ad, match = torch.autograd.forward_ad, "forward-mode derivatives .* not supported"
    x, w, r = x.detach(), w.detach(), r.detach()
    for f, args in ((tvdcn.rms_norm, (x, w)), (tvdcn.add_rms_norm, (x, r, w)), (tvdcn.rms_norm_int8, (x, w)), (tvdcn.quantize_int8, (x,)),
                    (lambda a, b: tvdcn.seeded_dropout(a, 0.5, seed_of(), b), (x, r))):
        for i, t in enumerate(args):
            for grad_mode in (True, False):
                with ad.dual_level(), torch.set_grad_enabled(grad_mode), pytest.raises(RuntimeError, match=match):
                    f(*args[:i], ad.make_dual(t, torch.ones_like(t)), *args[i + 1:])
    for f in (lambda a: tvdcn.rms_norm(a), lambda a: tvdcn.seeded_dropout(a, 0.5, seed_of())):
        a = leaf(x)
        y = f(a)
        with ad.dual_level(), pytest.raises(RuntimeError, match=match):
            torch.autograd.grad(y, a, ad.make_dual(torch.ones_like(y), torch.ones_like(y)))


def test_changes_before_the_backward_are_noticed():
    w, match = torch.randn(6, requires_grad=True), "modified by an inplace operation"
    x = torch.randn(2, 6, 3)
    y = tvdcn.rms_norm(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match=match):
        y.sum().backward()
    y, s = tvdcn.add_rms_norm(x, x.clone(), w)
    x.add_(1)                       # (what is kept is the sum)
    y.sum().backward(retain_graph=True)
    with torch.no_grad():
        s.add_(1)
    with pytest.raises(RuntimeError, match=match):
        y.sum().backward()
    a, seed = torch.randn(2, 6, 3, requires_grad=True), seed_of()
    y = tvdcn.seeded_dropout(a, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match=match):
        y.sum().backward()


SHAPES = [(3, 42, 4, 5), (1, 8, 9), (5, 6), (2, 3, 1, 2, 4), (0, 6, 4), (2, 6, 0), (1, 1)]


def layouts(device, dtype, shape):
    """Shape, strides and type of every result of every operator, the internal ones among them, for maps of this shape."""
    x, w = torch.zeros(shape, device=device, dtype=dtype), torch.zeros(shape[1], device=device, dtype=dtype)
    seed = torch.zeros(1, device=device, dtype=torch.int64)
    got = [tvdcn.rms_norm(x, w), *tvdcn.add_rms_norm(x, x, w), tvdcn.seeded_dropout(x, 0.5, seed, x), OPS._seeded_dropout(x, 0.5, seed, None)]
    y, s, rstd = OPS._rms_norm_forward(x, x, w, 1e-6, True)
    got += [y, s, rstd, *OPS._rms_norm_backward(y, s, s, rstd, w, [True] * 2)]
    if dtype != torch.float64:
        codes, scales = tvdcn.quantize_int8(x)
        got += [codes, scales, *tvdcn.rms_norm_int8(x, w), *tvdcn.add_rms_norm_int8(x, x, w), tvdcn.dequantize_int8(codes, scales, dtype)]
        weight = torch.zeros(10, shape[1], device=device, dtype=torch.int8)
        got.append(tvdcn.pointwise_conv_int8(codes, scales, weight, torch.zeros(10, device=device), dtype=dtype))
    return [(tuple(t.shape), t.stride(), t.dtype) for t in got]


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_without_data_have_the_layouts_of_the_results(dtype):
    for shape in SHAPES:
        got = layouts("cpu", dtype, shape)
        assert layouts("meta", dtype, shape) == got, shape
        for sizes, strides, t in got:
            if len(sizes) > 2 and 0 not in sizes and sizes[1] > 1 and (sizes[1] in (shape[1], 10)) and len(sizes) == len(shape):
                assert strides[1] == 1


def test_empty_maps():
    for shape in ((0, 6, 4), (2, 6, 0)):
        x, w = torch.zeros(shape, requires_grad=True), torch.ones(6, requires_grad=True)
        y, s = tvdcn.add_rms_norm(tvdcn.seeded_dropout(x, 0.5, seed_of()), x, w)
        (y.sum() + s.sum()).backward()
        assert x.grad.shape == shape and not w.grad.any()
        with torch.no_grad():
            codes, scales = tvdcn.rms_norm_int8(x, w)
            assert tvdcn.pointwise_conv_int8(codes, scales, WQ, WS).shape == (shape[0], 4, shape[2])
            assert tvdcn.dequantize_int8(*tvdcn.quantize_int8(x), torch.half).shape == shape


class Block(torch.nn.Module):
    """A residual block over pixels, as these operators are used together in training."""

    def __init__(self, c=6):
        super().__init__()
        self.norm = tvdcn.AddRMSNorm(c)
        self.wide = tvdcn.PointwiseConv(c, 4 * c, activation="gelu")
        self.narrow = tvdcn.PointwiseConv(4 * c, c)
        self.drop = tvdcn.SeededDropout(0.1)
        self.last = tvdcn.RMSNorm(c)

    def forward(self, x, shortcut):
        y, s = self.norm(x, shortcut)
        return self.last(self.drop(self.narrow(self.wide(y)), s))


def test_modules_script_and_compile():
    m, x = Block(), torch.randn(2, 6, 4, 3)
    scripted = torch.jit.script(m)
    torch.manual_seed(1)
    y = m(x, x)
    torch.manual_seed(1)
    assert torch.equal(scripted(x, x), y)
    y.square().sum().backward()
    assert all(p.grad is not None and p.grad.isfinite().all() for p in m.parameters())
    m.eval()
    assert torch.equal(m(x, x), m(x, x))
    meta = Block().to("meta")
    z = torch.zeros(2, 6, 4, 3, device="meta")
    assert torch.compile(meta, backend="aot_eager", fullgraph=True)(z, z).shape == x.shape
    assert "eps=1e-06" in repr(m) and "p=0.1" in repr(m)
    assert tvdcn.RMSNorm(6, affine=False).weight is None
    # served: the products in 8 bits
    with torch.no_grad():
        wide, narrow = tvdcn.PointwiseConvInt8.from_float(m.wide), tvdcn.PointwiseConvInt8.from_float(m.narrow)
        codes, scales, s = tvdcn.add_rms_norm_int8(x, x, m.norm.weight)
        served = m.last(narrow(wide(codes, scales), residual=s))
        exact = m(x, x)
        assert (served - exact).norm() < 0.05 * exact.norm()
        assert torch.equal(torch.jit.script(wide)(codes, scales), wide(codes, scales))
        assert torch.equal(wide(x), wide(*tvdcn.quantize_int8(x)))


def test_int8_module_types():
    m = tvdcn.PointwiseConvInt8.from_float(tvdcn.PointwiseConv(6, 4), torch.float16)
    assert m.weight_codes.dtype == torch.int8 and m.weight_scales.dtype == torch.float32 and m.bias.dtype == torch.float16
    scales = m.weight_scales.clone()
    for to in (torch.bfloat16, torch.float32):
        m = m.to(to)
        assert m.dtype == to and m.bias.dtype == to and m.weight_codes.dtype == torch.int8 and torch.equal(m.weight_scales, scales)
        assert m(torch.zeros(2, 6)).dtype == to
    bare = tvdcn.PointwiseConvInt8.from_float(tvdcn.PointwiseConv(6, 4, bias=False)).half()
    assert bare.bias is None and bare(torch.zeros(2, 6)).dtype == torch.float16
    other = tvdcn.PointwiseConvInt8(6, 4, dtype=torch.float32)
    other.load_state_dict(m.state_dict())
    x = torch.randn(3, 6)
    assert torch.equal(other(x), m(x)) and "bias=False" in repr(bare)


# ---- C ABI ----

class RmsDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("rows", ctypes.c_int64), ("channels", ctypes.c_int64), ("eps", ctypes.c_double)]


class PointDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("activation", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("in_channels", ctypes.c_int64), ("out_channels", ctypes.c_int64)]


SUCCESS, INVALID, SMALL, UNSUPPORTED = 0, 1, 2, 3
P, SIZE, I32, I64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32, ctypes.c_int64


@pytest.fixture(scope="module")
def lib():
    l = ctypes.CDLL(tvdcn.extension.HIP_LIB_PATH)
    l.tvdcn_last_error.restype = ctypes.c_char_p
    for n in ("rms_norm_backward", "pointwise_conv_int8"):
        getattr(l, "tvdcn_%s_workspace_size" % n).restype = SIZE
    l.tvdcn_rms_norm_forward.argtypes = [P] * 8
    l.tvdcn_rms_norm_int8.argtypes = [P] * 8
    l.tvdcn_rms_norm_backward.argtypes = [P] * 9 + [SIZE, P]
    l.tvdcn_quantize_int8.argtypes = l.tvdcn_dequantize_int8.argtypes = [I32, I64, I64, P, P, P, P]
    l.tvdcn_pointwise_conv_int8.argtypes = [P] * 9 + [SIZE, P]
    l.tvdcn_seeded_dropout.argtypes = [I32, I64, ctypes.c_double, P, P, P, P, P]
    return l


def rms_desc(**kw):
    return RmsDesc(**dict(dict(dtype=0, rows=9, channels=8, eps=1e-6), **kw))


def point_desc(**kw):
    return PointDesc(**dict(dict(dtype=0, activation=0, rows=9, in_channels=8, out_channels=16), **kw))


def test_c_abi_refuses_descriptors(lib):
    p, big = P(4096), 1 << 40
    for kw, status in ((dict(dtype=4), INVALID), (dict(dtype=1), UNSUPPORTED), (dict(rows=-1), INVALID), (dict(channels=0), INVALID),
                       (dict(channels=1 << 21), UNSUPPORTED), (dict(rows=1 << 60), UNSUPPORTED), (dict(eps=0.0), INVALID),
                       (dict(eps=-1.0), INVALID), (dict(eps=math.nan), INVALID), (dict(eps=1e-42), INVALID), (dict(eps=1e300), INVALID)):
        d = ctypes.byref(rms_desc(**kw))
        assert lib.tvdcn_rms_norm_backward_workspace_size(d) == 0
        assert lib.tvdcn_rms_norm_forward(d, p, p, p, p, p, p, None) == status, kw
        assert lib.tvdcn_rms_norm_int8(d, p, p, p, p, p, p, None) == status, kw
        assert lib.tvdcn_rms_norm_backward(d, p, p, p, p, p, p, p, p, big, None) == status, kw
        assert lib.tvdcn_last_error()
    for kw, status in ((dict(dtype=-1), INVALID), (dict(dtype=1), UNSUPPORTED), (dict(activation=4), INVALID), (dict(rows=-1), INVALID),
                       (dict(in_channels=0), INVALID), (dict(out_channels=0), INVALID), (dict(in_channels=131072), UNSUPPORTED),
                       (dict(in_channels=1 << 16, out_channels=1 << 16), UNSUPPORTED), (dict(rows=1 << 62), UNSUPPORTED)):
        d = ctypes.byref(point_desc(**kw))
        assert lib.tvdcn_pointwise_conv_int8_workspace_size(d) == 0
        assert lib.tvdcn_pointwise_conv_int8(d, p, p, p, p, p, p, p, p, big, None) == status, kw
    for f in (lib.tvdcn_quantize_int8, lib.tvdcn_dequantize_int8):
        for dtype, rows, c, status in ((1, 2, 8, UNSUPPORTED), (7, 2, 8, INVALID), (0, -1, 8, INVALID), (0, 2, 0, INVALID),
                                       (0, 2, 1 << 21, UNSUPPORTED), (0, 1 << 60, 8, UNSUPPORTED)):
            assert f(dtype, rows, c, p, p, p, None) == status
        assert f(0, 0, 8, None, None, None, None) == SUCCESS
    for dtype, n, prob, status in ((1, 8, 0.5, UNSUPPORTED), (5, 8, 0.5, INVALID), (0, -1, 0.5, INVALID), (0, 8, -0.1, INVALID),
                                   (0, 8, 1.5, INVALID), (0, 8, math.nan, INVALID), (0, 1 << 50, 0.5, UNSUPPORTED)):
        assert lib.tvdcn_seeded_dropout(dtype, n, prob, p, p, p, p, None) == status
    assert lib.tvdcn_seeded_dropout(0, 0, 0.5, None, None, None, None, None) == SUCCESS


def test_c_abi_refuses_pointers_and_workspaces(lib):
    p, odd, two, big = P(4096), P(4104), P(4098), 1 << 40
    d = ctypes.byref(rms_desc())
    f, q, b = lib.tvdcn_rms_norm_forward, lib.tvdcn_rms_norm_int8, lib.tvdcn_rms_norm_backward
    for g in (f, q):
        assert g(None, p, p, p, p, p, p, None) == INVALID and g(d, None, p, p, p, p, p, None) == INVALID
        assert g(d, p, None, p, p, p, p, None) == INVALID and g(d, p, p, p, None, p, p, None) == INVALID   # a residual and its sum
        assert g(d, p, p, p, p, None, p, None) == INVALID and g(d, odd, p, p, p, p, p, None) == INVALID
        assert g(d, p, p, odd, p, p, p, None) == INVALID and g(d, p, p, p, p, p, two, None) == INVALID
    assert q(d, p, p, p, p, p, None, None) == INVALID
    need = lib.tvdcn_rms_norm_backward_workspace_size(d)
    assert need > 0 and b(d, p, p, p, p, p, p, p, p, need - 1, None) == SMALL and b(d, p, p, p, p, p, p, p, None, big, None) == SMALL
    assert b(d, None, p, p, p, p, p, p, p, big, None) == INVALID and b(d, p, p, None, p, p, p, p, p, big, None) == INVALID
    assert b(d, p, p, p, None, p, p, p, p, big, None) == INVALID and b(d, p, odd, p, p, p, p, p, p, big, None) == INVALID
    assert b(d, p, p, p, two, p, p, p, p, big, None) == INVALID and b(d, p, p, p, p, p, p, p, odd, big, None) == INVALID
    assert b(d, p, p, p, p, p, None, None, None, 0, None) == SUCCESS                                   # nothing asked for
    none = ctypes.byref(rms_desc(rows=0))
    assert f(none, None, None, None, None, None, None, None) == SUCCESS and lib.tvdcn_rms_norm_backward_workspace_size(none) == 0
    d, f = ctypes.byref(point_desc(in_channels=9)), lib.tvdcn_pointwise_conv_int8
    for i in range(4):
        assert f(d, *[None if j == i else p for j in range(7)], p, big, None) == INVALID
    assert f(d, p, p, p, p, p, p, None, p, big, None) == INVALID and f(d, odd, p, p, p, p, p, p, p, big, None) == INVALID
    assert f(d, p, two, p, p, p, p, p, p, big, None) == INVALID and f(d, p, p, p, p, odd, p, p, p, big, None) == INVALID
    need = lib.tvdcn_pointwise_conv_int8_workspace_size(d)
    if need:
        assert f(d, p, p, p, p, p, p, p, p, need - 1, None) == SMALL
    assert f(ctypes.byref(point_desc(rows=0)), None, None, None, None, None, None, None, None, 0, None) == SUCCESS
    assert lib.tvdcn_pointwise_conv_int8_workspace_size(ctypes.byref(point_desc(in_channels=32))) == 0
    for g in (lib.tvdcn_quantize_int8, lib.tvdcn_dequantize_int8):
        assert g(0, 2, 8, None, p, p, None) == INVALID and g(0, 2, 8, odd, p, p, None) == INVALID
    assert lib.tvdcn_quantize_int8(0, 2, 8, p, p, two, None) == INVALID and lib.tvdcn_quantize_int8(0, 2, 8, p, p, None, None) == INVALID
    assert lib.tvdcn_dequantize_int8(0, 2, 8, p, two, p, None) == INVALID
    g = lib.tvdcn_seeded_dropout
    assert g(0, 8, 0.5, None, p, p, p, None) == INVALID and g(0, 8, 0.5, P(4100), p, p, p, None) == INVALID
    assert g(0, 8, 0.5, p, None, p, p, None) == INVALID and g(0, 8, 0.5, p, p, odd, p, None) == INVALID


def test_a_sum_that_needs_no_gradient_asks_for_none():
    x, r, w = torch.randn(2, 6, 3), torch.randn(2, 6, 3), torch.randn(6, requires_grad=True)
    y, s = tvdcn.add_rms_norm(x, r, w)
    assert y.requires_grad and not s.requires_grad
    s.add_(1)                       # (what the backward reads has changed)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y, s = tvdcn.add_rms_norm(x, leaf(r), w)
    assert s.requires_grad


def test_a_convolution_weight_in_8_bits():
    conv, x = torch.nn.Conv2d(6, 4, 1), torch.randn(2, 6, 3, 5)
    with torch.no_grad():
        codes, scales = tvdcn.quantize_int8(conv.weight)
        assert codes.shape == (4, 6, 1, 1) and scales.shape == (4, 1, 1)
        a = tvdcn.quantize_int8(x)
        y = tvdcn.pointwise_conv_int8(*a, codes, scales, conv.bias, dtype=torch.float32)
        assert torch.equal(y, tvdcn.pointwise_conv_int8(*a, codes[:, :, 0, 0], scales[:, 0, 0], conv.bias, dtype=torch.float32))
        for q, s in ((codes.expand(4, 6, 2, 1), scales), (codes, scales[:3])):
            with pytest.raises(RuntimeError, match="pointwise_conv_int8: expected"):
                tvdcn.pointwise_conv_int8(*a, q, s)


@pytest.mark.parametrize("requires", [True, False])
def test_operators_are_registered_as_torch_expects(requires):
    """Schemas, autograd registration, shapes without data and traced calls, by torch's own check."""
    x, w, seed = torch.randn(2, 6, 4, 3, requires_grad=requires), torch.randn(6, requires_grad=requires), seed_of()
    calls = [(OPS.rms_norm, (x, w, 1e-6)), (OPS.add_rms_norm, (x, x.detach(), w, 1e-6)), (OPS.seeded_dropout, (x, 0.3, seed, None))]
    if not requires:
        codes, scales = tvdcn.quantize_int8(x)
        q, s = tvdcn.quantize_int8(torch.randn(4, 6))
        calls += [(OPS.rms_norm_int8, (x, w, 1e-6)), (OPS.add_rms_norm_int8, (x, x, w, 1e-6)), (OPS.quantize_int8, (x,)),
                  (OPS.dequantize_int8, (codes, scales, torch.float16)),
                  (OPS.pointwise_conv_int8, (codes, scales, q, s, None, None, 3, torch.bfloat16))]
    for op, args in calls:
        assert set(torch.library.opcheck(op.default, args).values()) == {"SUCCESS"}


def test_host_int8_product_of_scales_at_the_range_ends():
    """A large scale of a pixel with small ones of the weight, and the other way round, where the result is an ordinary value."""
    x, w = cpu((5, 64), torch.float32, 1), cpu((10, 64), torch.float32, 2)
    up = torch.tensor([1e36, 1e37, 1.0, 1e30, 1e37])[:, None]
    for a, b in ((x * up, w * 1e-37), (x * 1e-37, w * up.repeat(2, 1))):
        q = [*tvdcn.quantize_int8(a), *tvdcn.quantize_int8(b)]
        for dtype in DTYPES[1:]:
            y = tvdcn.pointwise_conv_int8(*q, dtype=dtype)
            assert y.isfinite().all()
            check([y], [pointwise_int8(*q, None, None, "none", dtype)], dtype)
    # where the result is no float32, it is infinite
    q = tvdcn.quantize_int8(x * 1e37)
    assert (tvdcn.pointwise_conv_int8(*q, *q, dtype=torch.float32).diagonal() == math.inf).all()


def test_int8_module_takes_its_type_from_a_loaded_bias():
    m = tvdcn.PointwiseConvInt8.from_float(tvdcn.PointwiseConv(6, 4)).half()
    x = torch.randn(3, 6)
    other = tvdcn.PointwiseConvInt8(6, 4, device="meta")
    other.load_state_dict(m.state_dict(), assign=True)
    assert other(x).dtype == torch.float16 and torch.equal(other(x), m(x)) and "float16" in repr(other)
    assert torch.equal(torch.jit.script(other)(x), m(x))
    other = other.to(torch.float32)
    assert other(x).dtype == torch.float32 and other.weight_scales.dtype == torch.float32
    other = tvdcn.PointwiseConvInt8(6, 4, bias=False, device="meta", dtype=torch.float16)
    other.load_state_dict(tvdcn.PointwiseConvInt8.from_float(tvdcn.PointwiseConv(6, 4, bias=False)).state_dict(), assign=True)
    assert other(x).dtype == torch.float16
