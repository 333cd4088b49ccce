"""The operators on channels-last maps without a GPU: the host kernels against the float64 definitions, gradients against
differences, refusals (Python, operators and C ABI), shapes without data, TorchScript, compilation and modules."""
import ctypes
import os
import re

import pytest
import torch

import tvdcn
from map_reference import ACTIVATIONS, LAYOUT_SHAPES, as_map, as_rows, check, kept, layouts, make, norm, pointwise

DTYPES = [torch.float64, torch.float32, torch.float16, torch.bfloat16]
OPS = torch.ops.tvdcn


def leaf(t):
    return None if t is None else t.detach().requires_grad_(True)


def cpu(shape, dtype, seed, **kw):
    return make(shape, dtype, seed, device="cpu", **kw)


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_host_kernels(dtype, keep):
    if dtype == torch.float64 and keep:
        return
    for act in ACTIVATIONS:
        x, w, b = cpu((3, 36, 5, 7), dtype, 1), cpu((36,), dtype, 2, shift=1.0), cpu((36,), dtype, 3)
        dy = cpu((3, 36, 5, 7), dtype, 4)
        t = [leaf(v) for v in (x, w, b)]
        y = tvdcn.group_norm_act(t[0], 4, t[1], t[2], 1e-5, act, keep)
        check([y, *torch.autograd.grad(y, t, dy)], norm(x, 4, w, b, 1e-5, act, dy, keep), act)
        w, b, r = cpu((10, 36), dtype, 5), cpu((10,), dtype, 6), cpu((3, 10, 5, 7), dtype, 7)
        dy = cpu((3, 10, 5, 7), dtype, 8)
        t = [leaf(v) for v in (x, w, b, r)]
        y = tvdcn.pointwise_conv(*t, act, keep)
        *g, dr = torch.autograd.grad(y, t, dy)
        check([y, *g], pointwise(x, w, b, r, act, dy, keep), act)
        assert torch.equal(dr, dy)


@pytest.mark.parametrize("act", ACTIVATIONS)
def test_gradients_against_differences(act):
    x = torch.randn(2, 6, 3, 2, dtype=torch.float64, requires_grad=True)
    w, b = (torch.randn(6, dtype=torch.float64, requires_grad=True) for _ in range(2))
    assert torch.autograd.gradcheck(lambda *a: tvdcn.group_norm_act(a[0], 2, *a[1:], 1e-5, act), (x, w, b))
    assert torch.autograd.gradcheck(lambda a: tvdcn.group_norm_act(a, 2, None, None, 1e-5, act), (x,))
    assert torch.autograd.gradcheck(lambda *a: tvdcn.group_norm_act(a[0], 2, None, a[1], 1e-5, act), (x, b))
    w = torch.randn(4, 6, dtype=torch.float64, requires_grad=True)
    b = torch.randn(4, dtype=torch.float64, requires_grad=True)
    r = torch.randn(2, 4, 3, 2, dtype=torch.float64, requires_grad=True)
    assert torch.autograd.gradcheck(lambda *a: tvdcn.pointwise_conv(*a, act), (x, w, b, r))
    assert torch.autograd.gradcheck(lambda *a: tvdcn.pointwise_conv(a[0], a[1], None, a[2], act), (x, w, r))
    assert torch.autograd.gradcheck(lambda *a: tvdcn.pointwise_conv(*a, None, None, act), (x, w))


@pytest.mark.parametrize("dtype", DTYPES[1:])
def test_round_trip(dtype):
    for shape in ((2, 71, 5), (3, 32), (1, 3, 2, 2)):
        x = cpu(shape, dtype, 1, spread=3.0)
        x[(0,) * x.dim()] = float("nan")
        codes, exps = tvdcn.compress_activation(x)
        assert codes.shape == x.shape and codes.dtype == torch.int8
        assert exps.shape == (shape[0], (shape[1] + 31) // 32, *shape[2:]) and exps.dtype == torch.uint8
        back, want = tvdcn.expand_activation(codes, exps, dtype), as_map(kept(as_rows(x.double()), dtype), x, shape[1])
        assert torch.equal(back.isnan(), want.isnan()) and torch.equal(back.nan_to_num(0).double(), want.nan_to_num(0))
        # no further off than half a step, which is at most 1/127 of the block's largest value
        off = (back - x).abs().nan_to_num(0).max()
        assert off <= x.nan_to_num(0).abs().max() / 127 * (1 + torch.finfo(dtype).eps)


NORM_X, NORM_W = torch.zeros(2, 6, 3), torch.zeros(6)


@pytest.mark.parametrize("args,message", [
    ((torch.zeros(6), 2), "expected a \\(batch, channels"),
    ((torch.zeros(2, 0, 3), 1), "needs channels"),
    ((torch.zeros(2, 6, 3, dtype=torch.int32), 2), "unsupported dtype"),
    ((torch.zeros(2, 6, 3, dtype=torch.complex64), 2), "unsupported dtype"),
    ((NORM_X, 4), "divisible"), ((NORM_X, 0), "divisible"), ((NORM_X, -2), "divisible"), ((NORM_X, 12), "divisible"),
    ((NORM_X, 2, torch.zeros(5)), "weight of shape"), ((NORM_X, 2, None, torch.zeros(6, 1)), "bias of shape"),
    ((NORM_X, 2, NORM_W.double()), "weight of dtype"), ((NORM_X.half(), 2, NORM_W), "weight of dtype"),
    ((NORM_X, 2, NORM_W.to("meta")), "weight is on meta"),
    ((NORM_X, 2, NORM_W, NORM_W, -1.0), "eps"), ((NORM_X, 2, NORM_W, NORM_W, float("nan")), "eps"),
])
def test_norm_refusals(args, message):
    with pytest.raises(RuntimeError, match=message):
        tvdcn.group_norm_act(*args)


@pytest.mark.parametrize("args,message", [
    ((torch.zeros(6), torch.zeros(4, 6)), "expected a \\(batch, channels"),
    ((NORM_X, torch.zeros(4, 5)), "for 6 input channels"), ((NORM_X, torch.zeros(6)), "expected a weight"),
    ((NORM_X, torch.zeros(0, 6)), "expected a weight"), ((NORM_X, torch.zeros(4, 6, 3)), "axes of size one"),
    ((NORM_X, torch.zeros(4, 6), torch.zeros(6)), "bias of shape"),
    ((NORM_X, torch.zeros(4, 6), None, torch.zeros(2, 4, 1)), "residual of shape"),
    ((NORM_X, torch.zeros(4, 6), None, torch.zeros(4, 3)), "residual of shape"),
    ((NORM_X, torch.zeros(4, 6).half()), "weight of dtype"),
    ((NORM_X, torch.zeros(4, 6), None, torch.zeros(2, 4, 3).bfloat16()), "residual of dtype"),
])
def test_pointwise_refusals(args, message):
    with pytest.raises(RuntimeError, match=message):
        tvdcn.pointwise_conv(*args)


def test_other_refusals():
    x, w = torch.zeros(2, 6, 3), torch.zeros(4, 6)
    for f in (lambda a: tvdcn.group_norm_act(x, 2, activation=a), lambda a: tvdcn.pointwise_conv(x, w, activation=a),
              lambda a: tvdcn.GroupNormAct(2, 6, activation=a), lambda a: tvdcn.PointwiseConv(6, 4, activation=a)):
        with pytest.raises(ValueError, match="activation must be"):
            f("tanh")
    for code in (-1, 4):
        with pytest.raises(RuntimeError, match="unknown activation"):
            OPS.pointwise_conv(x, w, None, None, code)
        with pytest.raises(RuntimeError, match="unknown activation"):
            OPS.group_norm_act(x, 2, None, None, 1e-5, code)
    with pytest.raises(ValueError):
        tvdcn.GroupNormAct(4, 6)
    with pytest.raises(ValueError):
        tvdcn.PointwiseConv(0, 6)
    # 8-bit maps have no float64
    d = x.double().requires_grad_(True)
    for f in (lambda: tvdcn.compress_activation(d.detach()), lambda: tvdcn.group_norm_act(d, 2, keep_int8=True),
              lambda: tvdcn.pointwise_conv(d, w.double(), keep_int8=True)):
        with pytest.raises(RuntimeError, match="float64 are not supported|bfloat16 maps only"):
            f()
    codes, exps = tvdcn.compress_activation(x)
    for q, e, t in ((codes.float(), exps, torch.float32), (codes, exps.int(), torch.float32), (codes, exps[:1], torch.float32),
                    (codes[0, 0], exps, torch.float32), (codes, exps, torch.float64), (codes, exps, torch.int8),
                    (codes.to("meta"), exps, torch.float32)):
        with pytest.raises(RuntimeError, match="expand_activation"):
            tvdcn.expand_activation(q, e, t)
    # the backward operators check what they are given
    g, st = torch.zeros(2, 6, 3), torch.zeros(2, 2, 3)
    bad = [(g, None, None, None, st), (g, x, codes, exps, st), (g, None, codes, None, st), (g, x[:1], None, None, st),
           (g, x, None, None, st[:, :1]), (g, x, None, None, st.half()), (g, x, None, None, torch.zeros(2, 2, 4)),
           (g, x, None, None, st[0]), (g, None, codes[:, :4], exps, st)]
    for a in bad:
        with pytest.raises(RuntimeError, match="group_norm_act"):
            OPS._group_norm_act_backward(*a[:4], None, None, a[4], 0, [True] * 3)
    g = torch.zeros(2, 4, 3)
    for a in ((g, None, None, None, w, g, 1), (g, x, None, None, w, None, 2), (g, x, None, None, w, g[:1], 2),
              (g, x, None, None, w[:3], g, 2), (g, x[:, :5], None, None, w, g, 2), (g, None, codes[:1], exps[:1], w, g, 2)):
        with pytest.raises(RuntimeError, match="pointwise_conv"):
            OPS._pointwise_conv_backward(*a, [True] * 3)


def test_double_backward_is_refused():
    x, w = torch.randn(2, 6, 3, requires_grad=True), torch.randn(4, 6, requires_grad=True)
    for y in (tvdcn.group_norm_act(x, 2, activation="silu"), tvdcn.pointwise_conv(x, w, activation="gelu")):
        g, = torch.autograd.grad(y.square().sum(), x, create_graph=True)
        with pytest.raises(RuntimeError, match="double backwards on .* not supported"):
            g.sum().backward()


@pytest.mark.parametrize("grad_mode", [True, False])
def test_forward_mode_derivatives_are_refused(grad_mode):
    """A tangent of any input, with gradients recorded or not, through torch.func, and of the gradient in a backward."""
    ad = torch.autograd.forward_ad
    x, p, r = torch.randn(2, 6, 3), torch.randn(6), torch.randn(2, 4, 3)
    w, b = torch.randn(4, 6), torch.randn(4)
    match = "forward-mode derivatives .* not supported"
    for f, args in ((lambda *a: tvdcn.group_norm_act(a[0], 2, *a[1:], activation="silu"), (x, p, p)),
                    (lambda *a: tvdcn.pointwise_conv(*a, activation="gelu"), (x, w, b, r))):
        for i, t in enumerate(args):
            with ad.dual_level(), torch.set_grad_enabled(grad_mode):
                dual = ad.make_dual(t, torch.ones_like(t))
                with pytest.raises(RuntimeError, match=match):
                    f(*args[:i], dual, *args[i + 1:])
            with pytest.raises(RuntimeError, match=match), torch.set_grad_enabled(grad_mode):
                torch.func.jvp(lambda v: f(*args[:i], v, *args[i + 1:]), (t,), (torch.ones_like(t),))
        first = leaf(args[0])
        y = f(first, *args[1:])
        with ad.dual_level(), pytest.raises(RuntimeError, match=match):
            torch.autograd.grad(y, first, ad.make_dual(torch.ones_like(y), torch.ones_like(y)))
        assert f(*args).shape == y.shape


def test_input_changed_before_the_backward_is_noticed():
    x, w = torch.randn(2, 6, 3), torch.randn(4, 6, requires_grad=True)
    y = tvdcn.pointwise_conv(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()
    y = tvdcn.pointwise_conv(x, w, keep_int8=True)   # what is kept is a copy
    x.add_(1)
    y.sum().backward()


@pytest.mark.parametrize("keep", [False, True])
@pytest.mark.parametrize("act", ACTIVATIONS)
def test_a_frozen_weight_keeps_no_input(act, keep):
    """Only the weight's gradient reads the input: without it neither the map nor its codes are kept, and it may change."""
    x, w = torch.randn(2, 6, 3, 5), torch.randn(4, 6)
    for i, t in enumerate((x, torch.randn(4), torch.randn(2, 4, 3, 5))):   # the gradient of the input, the bias, the residual
        kept = []
        args = [x.clone(), w, torch.randn(4), torch.randn(2, 4, 3, 5)]
        args[(0, 2, 3)[i]] = t.clone().requires_grad_(True)
        if i == 0:
            args[0] = args[0] * 1.0   # (a result, that may change in place)
        with torch.autograd.graph.saved_tensors_hooks(lambda v: kept.append(v) or v, lambda v: v):
            y = tvdcn.pointwise_conv(*args, act, keep)
        assert not any(v.shape == x.shape or v.dtype in (torch.int8, torch.uint8) for v in kept)
        if i:
            args[0].add_(1)
        y.sum().backward()
    # the operator asks for an input where the weight's gradient is asked for
    g = torch.randn(2, 4, 3, 5)
    dx, dw, db = OPS._pointwise_conv_backward(g, None, None, None, w, None, 0, [True, False, True])
    assert dx.shape == x.shape and dw is None and db.shape == (4,)
    with pytest.raises(RuntimeError, match="expected the input"):
        OPS._pointwise_conv_backward(g, None, None, None, w, None, 0, [True, True, True])


def test_results_are_channels_last():
    for shape in ((2, 6, 4, 5), (2, 6, 4), (2, 6, 3, 4, 5), (3, 6)):
        for device in ("cpu", "meta"):
            x = torch.zeros(shape, device=device, requires_grad=True)
            w = torch.zeros(4, 6, device=device, requires_grad=True)
            n = tvdcn.group_norm_act(x, 2)
            y = tvdcn.pointwise_conv(n, w, None, None, "gelu")
            for t in (n, y):
                assert t.movedim(1, -1).is_contiguous()
            assert y.shape == (shape[0], 4, *shape[2:])
            y.backward(torch.zeros_like(y))
            assert x.grad.shape == x.shape and w.grad.shape == w.shape
            q, e = tvdcn.compress_activation(n.detach())
            assert q.movedim(1, -1).is_contiguous() and e.shape == (shape[0], 1, *shape[2:])
            assert tvdcn.expand_activation(q, e, torch.float32).shape == shape


@pytest.mark.parametrize("keep", [False, True])
def test_modules_script_and_compile(keep):
    class Block(torch.nn.Module):
        def __init__(self):
            super().__init__()
            self.norm = tvdcn.GroupNormAct(2, 6, activation="silu", keep_int8=keep)
            self.conv = tvdcn.PointwiseConv(6, 6, activation="gelu", keep_int8=keep)

        def forward(self, x):
            return self.conv(self.norm(x), x)

    m, x = Block(), torch.randn(2, 6, 4, 3)
    assert m.norm.weight.shape == (6,) and m.conv.weight.shape == (6, 6)
    y = m(x)
    assert torch.equal(torch.jit.script(m)(x), y)
    y.sum().backward()
    assert all(p.grad is not None for p in m.parameters())
    meta = Block().to("meta")
    out = torch.compile(meta, backend="aot_eager", fullgraph=True)(torch.randn(2, 6, 4, 3, device="meta"))
    assert out.shape == x.shape
    assert "activation=silu" in repr(m) and "activation=gelu" in repr(m) and ("keep_int8" in repr(m)) == keep
    assert tvdcn.GroupNormAct(2, 6, affine=False).weight is None and tvdcn.PointwiseConv(6, 4, bias=False).bias is None
    conv = torch.nn.Conv2d(6, 4, 1)
    assert torch.allclose(tvdcn.pointwise_conv(x, conv.weight, conv.bias), conv(x), atol=1e-5)


@pytest.mark.parametrize("dtype", DTYPES)
def test_shapes_without_data_have_the_layouts_of_the_results(dtype):
    """What compilation plans with: sizes, strides and types of the Meta kernels are the host kernels'."""
    for shape, groups, out in LAYOUT_SHAPES:
        assert layouts("meta", dtype, shape, groups, out) == layouts("cpu", dtype, shape, groups, out), shape


def test_empty_maps():
    for shape in ((0, 6, 4), (2, 6, 0)):
        x, w = torch.zeros(shape, requires_grad=True), torch.zeros(4, 6, requires_grad=True)
        g = torch.ones(6, requires_grad=True)
        tvdcn.pointwise_conv(tvdcn.group_norm_act(x, 2, g), w).sum().backward()
        assert not w.grad.any() and not g.grad.any() and x.grad.shape == shape


def test_inline_assembly_declares_the_registers_it_names():
    """A scalar register that an asm statement writes by name stands in its list of clobbers."""
    folder = os.path.join(os.path.dirname(tvdcn.extension.HIP_LIB_PATH), "csrc", "hip")
    seen = 0
    for name in sorted(os.listdir(folder)):
        with open(os.path.join(folder, name)) as f:
            source = f.read()
        for text in re.findall(r"\basm\s*(?:volatile)?\s*\((.*?)\);", source, re.S):
            for register in re.findall(r"s_mov_b32 (m0|vcc_lo|exec_lo|s\d+)\b", text):
                seen += 1
                assert '"%s"' % register in text, (name, text)
    assert seen > 0


# ---- C ABI ----

class NormDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("activation", ctypes.c_int32), ("batch", ctypes.c_int64),
                ("pixels", ctypes.c_int64), ("channels", ctypes.c_int64), ("groups", ctypes.c_int64), ("eps", ctypes.c_double)]


class PointDesc(ctypes.Structure):
    _fields_ = [("dtype", ctypes.c_int32), ("activation", ctypes.c_int32), ("rows", ctypes.c_int64),
                ("in_channels", ctypes.c_int64), ("out_channels", ctypes.c_int64)]


SUCCESS, INVALID, SMALL, UNSUPPORTED = 0, 1, 2, 3
P, SIZE, I32, I64 = ctypes.c_void_p, ctypes.c_size_t, ctypes.c_int32, ctypes.c_int64


@pytest.fixture(scope="module")
def lib():
    l = ctypes.CDLL(tvdcn.extension.HIP_LIB_PATH)
    l.tvdcn_last_error.restype = ctypes.c_char_p
    for n in ("group_norm_act_forward", "group_norm_act_backward", "pointwise_conv_forward", "pointwise_conv_backward"):
        getattr(l, "tvdcn_%s_workspace_size" % n).restype = SIZE
    l.tvdcn_group_norm_act_forward.argtypes = [P] * 8 + [SIZE, P]
    l.tvdcn_group_norm_act_backward.argtypes = [P] * 13 + [SIZE, P]
    l.tvdcn_pointwise_conv_forward.argtypes = [P] * 8 + [SIZE, P]
    l.tvdcn_pointwise_conv_backward.argtypes = [P] * 11 + [SIZE, P]
    l.tvdcn_compress_activation.argtypes = [I32, I64, I64, P, P, P, P]
    l.tvdcn_expand_activation.argtypes = [I32, I64, I64, P, P, P, P]
    return l


def norm_desc(**kw):
    d = dict(dtype=0, activation=0, batch=2, pixels=9, channels=8, groups=2, eps=1e-5)
    d.update(kw)
    return NormDesc(**d)


def point_desc(**kw):
    d = dict(dtype=0, activation=0, rows=9, in_channels=8, out_channels=16)
    d.update(kw)
    return PointDesc(**d)


BAD_NORM = [(dict(dtype=4), INVALID), (dict(dtype=1), UNSUPPORTED), (dict(activation=4), INVALID), (dict(batch=-1), INVALID),
            (dict(pixels=-1), INVALID), (dict(channels=0), INVALID), (dict(groups=3), INVALID), (dict(groups=0), INVALID),
            (dict(eps=-1.0), INVALID), (dict(eps=float("inf")), INVALID), (dict(channels=1 << 21, groups=1), UNSUPPORTED),
            (dict(batch=1 << 40, pixels=1 << 40), UNSUPPORTED)]
BAD_POINT = [(dict(dtype=-1), INVALID), (dict(dtype=1), UNSUPPORTED), (dict(activation=-1), INVALID), (dict(rows=-1), INVALID),
             (dict(in_channels=0), INVALID), (dict(out_channels=-3), INVALID), (dict(in_channels=1 << 21), UNSUPPORTED),
             (dict(in_channels=1 << 20, out_channels=1 << 20), UNSUPPORTED), (dict(rows=1 << 62), UNSUPPORTED)]


def test_c_abi_refuses_descriptors(lib):
    p, big = P(4096), 1 << 40
    for kw, status in BAD_NORM:
        d = ctypes.byref(norm_desc(**kw))
        assert lib.tvdcn_group_norm_act_forward_workspace_size(d) == 0
        assert lib.tvdcn_group_norm_act_backward_workspace_size(d) == 0
        assert lib.tvdcn_group_norm_act_forward(d, p, p, p, p, p, p, p, big, None) == status, kw
        assert lib.tvdcn_group_norm_act_backward(d, p, p, None, None, p, p, p, p, p, p, p, p, big, None) == status, kw
        assert lib.tvdcn_last_error()
    for kw, status in BAD_POINT:
        d = ctypes.byref(point_desc(**kw))
        assert lib.tvdcn_pointwise_conv_forward_workspace_size(d) == 0
        assert lib.tvdcn_pointwise_conv_backward_workspace_size(d, 1) == 0
        assert lib.tvdcn_pointwise_conv_forward(d, p, p, p, p, p, p, p, big, None) == status, kw
        assert lib.tvdcn_pointwise_conv_backward(d, p, p, None, None, p, p, p, p, p, p, big, None) == status, kw
    for f in (lib.tvdcn_compress_activation, lib.tvdcn_expand_activation):
        for dtype, rows, c, status in ((1, 2, 8, UNSUPPORTED), (7, 2, 8, INVALID), (0, -1, 8, INVALID), (0, 2, 0, INVALID),
                                       (0, 2, 1 << 21, UNSUPPORTED), (0, 1 << 60, 8, UNSUPPORTED)):
            assert f(dtype, rows, c, p, p, p, None) == status
        assert f(0, 2, 8, p, None, p, None) == INVALID and f(0, 2, 8, p, p, P(4100), None) == INVALID
        assert f(0, 0, 8, None, None, None, None) == SUCCESS


def test_c_abi_refuses_pointers_and_workspaces(lib):
    p, odd, big = P(4096), P(4104), 1 << 40
    d = ctypes.byref(norm_desc(pixels=1 << 20))   # (groups that a workgroup holds need no workspace forward)
    f, b = lib.tvdcn_group_norm_act_forward, lib.tvdcn_group_norm_act_backward
    assert f(None, p, p, p, p, p, p, p, big, None) == INVALID
    assert f(d, None, p, p, p, p, p, p, big, None) == INVALID and f(d, p, p, p, None, p, p, p, big, None) == INVALID
    assert f(d, p, odd, p, p, p, p, p, big, None) == INVALID and f(d, p, p, p, p, p, p, odd, big, None) == INVALID
    need = lib.tvdcn_group_norm_act_forward_workspace_size(d)
    assert need > 0 and f(d, p, p, p, p, p, p, p, need - 1, None) == SMALL and f(d, p, p, p, p, p, p, None, big, None) == SMALL
    need = lib.tvdcn_group_norm_act_backward_workspace_size(d)
    assert b(d, p, p, None, None, p, p, p, p, p, p, p, p, need - 1, None) == SMALL
    assert b(d, p, None, None, None, p, p, p, p, p, p, p, p, big, None) == INVALID    # neither input nor codes
    assert b(d, p, p, p, p, p, p, p, p, p, p, p, p, big, None) == INVALID             # both
    assert b(d, p, None, p, None, p, p, p, p, p, p, p, p, big, None) == INVALID       # codes alone
    assert b(d, None, p, None, None, p, p, p, p, p, p, p, p, big, None) == INVALID
    assert b(d, p, p, None, None, p, p, p, p, None, None, None, p, big, None) == SUCCESS   # nothing asked for
    d = ctypes.byref(point_desc(dtype=2, activation=2, in_channels=9))   # (channels in eights, or float32: none)
    f, b = lib.tvdcn_pointwise_conv_forward, lib.tvdcn_pointwise_conv_backward
    assert f(d, None, p, p, p, p, p, p, big, None) == INVALID and f(d, p, p, p, p, None, p, p, big, None) == INVALID
    assert f(d, p, p, odd, p, p, p, p, big, None) == INVALID
    need = lib.tvdcn_pointwise_conv_forward_workspace_size(d)
    assert need > 0 and f(d, p, p, p, p, p, p, p, need - 1, None) == SMALL
    need = lib.tvdcn_pointwise_conv_backward_workspace_size(d, 0)
    assert b(d, p, p, None, None, p, p, p, p, p, p, need - 1, None) == SMALL
    assert b(d, p, p, None, None, p, None, p, p, p, p, big, None) == INVALID          # the activation's argument
    assert b(d, p, p, p, p, p, p, p, p, p, p, big, None) == INVALID
    assert b(d, p, None, None, None, p, p, p, p, p, p, big, None) == INVALID
    assert b(d, p, p, None, None, None, p, p, p, p, p, big, None) == INVALID
    assert lib.tvdcn_group_norm_act_forward_workspace_size(ctypes.byref(norm_desc())) == 0
    # 16-bit maps of whole eights of channels are multiplied where they lie, and so are float32 ones of small products
    assert lib.tvdcn_pointwise_conv_forward_workspace_size(ctypes.byref(point_desc(dtype=0, in_channels=9))) == 0
    large = dict(rows=1 << 20, in_channels=512, out_channels=512)
    assert lib.tvdcn_pointwise_conv_forward_workspace_size(ctypes.byref(point_desc(**large))) > 0
    assert lib.tvdcn_pointwise_conv_forward_workspace_size(ctypes.byref(point_desc(dtype=3))) == 0
    # rows of none: nothing to do, no pointers needed
    assert f(ctypes.byref(point_desc(rows=0)), None, None, None, None, None, None, None, 0, None) == SUCCESS
    assert lib.tvdcn_group_norm_act_forward(ctypes.byref(norm_desc(batch=0)), None, None, None, None, None, None, None, 0, None) == SUCCESS


def test_c_abi_statistics_are_single_floats(lib):
    p, big, d = P(4096), 1 << 40, ctypes.byref(norm_desc(pixels=1 << 20))
    f, b = lib.tvdcn_group_norm_act_forward, lib.tvdcn_group_norm_act_backward
    assert b(d, p, p, None, None, p, p, P(4100), P(4116), None, None, None, p, big, None) == SUCCESS   # (nothing asked for)
    assert b(d, p, p, None, None, p, p, P(4098), p, None, None, None, p, big, None) == INVALID
    assert b(d, p, p, None, None, p, p, p, None, p, p, p, p, big, None) == INVALID
    assert f(d, p, p, p, p, P(4098), p, p, big, None) == INVALID and f(d, p, p, p, p, p, None, p, big, None) == INVALID
