"""What the operators that treat a pixel's channels as one vector (a token) are measured by.

Every case is one pass as a program makes it: without gradients for inference, the forward and all gradients
for training. A feature map is (batch, channels, *size) with its channels contiguous in memory (torch's
``channels_last`` in two dimensions), or (batch, channels) where it has no grid.

* ``norm``: root-mean-square normalisation of every pixel, of the map or of its sum with a shortcut, which is a
  result too,
* ``norm8``: the same for inference, its result in 8 bits, and the values these stand for,
* ``quantize``: a map to 8 bits and back,
* ``product8``: the pointwise convolution of an 8-bit map with 8-bit weights,
* ``dropout``: values zeroed at random, added to a shortcut; the mask is made again in the backward.

In 8 bits a pixel (or an output channel of a weight) has one scale, ``max(max |x| / 127, 2^-126)`` rounded to
float32, and the codes ``x / scale`` rounded to whole numbers, ties to the even one; they stand for ``code * scale``.

The mask comes from Philox4x32-10 (Salmon et al., "Parallel random numbers: as easy as 1, 2, 3"): the key is the
seed, the counter the number of a group of eight values, in the order of their channels-last memory. A value has
16 of the 128 bits and is dropped where they are less than ``round(65536 p)``.
"""
import math

import numpy
import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_EPS = 1e-6
_LEAST_SCALE = 2.0 ** -126


def _norm(name, batch, channels, size, **kw):
    return dict(dict(name=name, op="norm", batch=batch, channels=channels, size=size, residual=True, dtype="bf16",
                     train=True), **kw)


def _norm8(name, batch, channels, size, **kw):
    return dict(dict(name=name, op="norm8", batch=batch, channels=channels, size=size, residual=True, dtype="bf16"), **kw)


def _quantize(name, batch, channels, size, dtype):
    return dict(name=name, op="quantize", batch=batch, channels=channels, size=size, dtype=dtype)


def _product8(name, batch, channels, out, size, **kw):
    return dict(dict(name=name, op="product8", batch=batch, channels=channels, out=out, size=size, activation="none",
                     residual=False, dtype="bf16"), **kw)


def _dropout(name, batch, channels, size, p, **kw):
    return dict(dict(name=name, op="dropout", batch=batch, channels=channels, size=size, p=p, residual=True,
                     dtype="bf16"), **kw)


def listed():
    return [
        # one pixel, or one token, of a served model: latency
        _norm("norm_pixel_infer", 1, 256, "", train=False),
        # channels that divide by nothing useful on a ragged grid, in float32
        _norm("norm_ragged_train_f32", 3, 71, "61x47", dtype="f32"),
        # in front of the long sequence layer of bench.py's suite
        _norm("norm_sequence_train_f16", 16, 512, "4096", dtype="f16"),
        # one image at a coarse level of a feature pyramid, served in 8 bits
        _norm8("norm8_image", 1, 256, "25x38"),
        # long sequences served in 8 bits
        _norm8("norm8_sequence_f16", 16, 512, "4096", dtype="f16"),
        # a small float32 map
        _quantize("quantize_ragged_f32", 3, 71, "61x47", "f32"),
        # what the narrowing layer of a block reads, widened fourfold from the long sequence layer
        _quantize("quantize_wide_sequence", 16, 2048, "4096", "bf16"),
        # one pixel, or one token, of a served model: its widening layer
        _product8("product8_pixel", 1, 256, 1024, "", activation="gelu"),
        # channels that divide by nothing useful, added to a shortcut
        _product8("product8_ragged_f16", 3, 71, 101, "61x47", activation="relu", residual=True, dtype="f16"),
        # the narrowing layer of long sequences, added to its shortcut: the most work
        _product8("product8_sequence", 16, 2048, 512, "4096", residual=True),
        # a small float32 map in training
        _dropout("dropout_ragged_train_f32", 3, 71, "61x47", 0.2, dtype="f32"),
        # the branch of a block over long sequences, in training
        _dropout("dropout_sequence_train", 16, 512, "4096", 0.1),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A pass of the same kinds: every operator, direction and type, 1 to 16 images, grids of none to three axes, from
    single pixels to the listed ones, channel counts of any kind."""
    op = rng.choice(("norm", "norm", "norm8", "quantize", "product8", "product8", "dropout"))
    batch = _log_int(rng, 1, 16)
    dim = rng.choice((0, 1, 2, 2, 3))
    size = "x".join(str(_log_int(rng, 1, {1: 4096, 2: 64, 3: 16}[dim])) for _ in range(dim))
    if dim == 0:
        batch = _log_int(rng, 1, 4096)

    def width(lo, hi):
        n = _log_int(rng, lo, hi)
        return max(8, n // 8 * 8) if rng.random() < 0.6 else n

    dtype, residual = rng.choice(("f32", "f16", "bf16")), rng.random() < 0.5
    # of the gradient of a vector of two or three values, its direction taken out, next to nothing is left
    channels = width(8 if op == "norm" else 3, 512 if op in ("norm", "norm8", "dropout") else 2048)
    if op == "norm":
        case = _norm("", batch, channels, size, residual=residual, dtype=dtype, train=rng.random() < 0.6)
    elif op == "norm8":
        # (a float32 result next to a rounding border falls to either side by its last bit: 8-bit serving is of 16-bit maps)
        case = _norm8("", batch, channels, size, residual=residual, dtype=rng.choice(("f16", "bf16")))
    elif op == "quantize":
        case = _quantize("", batch, channels, size, dtype)
    elif op == "product8":
        case = _product8("", batch, channels, width(3, 2048 * 512 // max(channels, 512)), size, residual=residual,
                         activation=rng.choice(("none", "relu", "silu", "gelu")), dtype=dtype)
    else:
        case = _dropout("", batch, channels, size, rng.choice((0.05, 0.1, 0.2, 0.5)), residual=residual, dtype=dtype)
    del case["name"]
    return case


def _size(case):
    return [int(s) for s in case["size"].split("x")] if case["size"] else []


def _rows(case):
    return case["batch"] * math.prod(_size(case))


def _map(gen, case, channels, spread=None, shift=None):
    """A (batch, channels, *size) map in channels-last memory."""
    x = torch.randn([case["batch"], *_size(case), channels], generator=gen, device="cuda")
    if spread is not None:
        x = x * spread
    if shift is not None:
        x = x + shift
    return x.to(_DTYPES[case["dtype"]]).movedim(-1, 1)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed * 6151 + 29)
    op, dtype, c = case["op"], _DTYPES[case["dtype"]], case["channels"]
    # a layer's outputs: channels of unlike spread and mean
    spread = torch.exp(0.4 * torch.randn(c, generator=gen, device="cuda"))
    shift = 0.5 * torch.randn(c, generator=gen, device="cuda")
    x = _map(gen, case, c, spread, shift)
    state = dict(case=case, residual=None)
    if op == "product8":
        # what a served model holds: the layer's input and its weights in 8 bits
        codes, scales = _in_8_bits(x.movedim(1, -1).float())
        state.update(codes=codes.to(torch.int8).movedim(-1, 1), scales=scales)
        codes, scales = _in_8_bits(torch.randn(case["out"], c, generator=gen, device="cuda") / math.sqrt(c))
        state.update(weight_codes=codes.to(torch.int8), weight_scales=scales)
        state["bias"] = (0.2 * torch.randn(case["out"], generator=gen, device="cuda")).to(dtype)
        if case["residual"]:
            state["residual"] = _map(gen, case, case["out"])
        return state
    state["x"] = x
    if op != "quantize" and case["residual"]:
        state["residual"] = _map(gen, case, c)
    if op in ("norm", "norm8"):
        state["weight"] = (1 + 0.2 * torch.randn(c, generator=gen, device="cuda")).to(dtype)
    if op == "dropout":
        state["seed"] = torch.randint(2 ** 62, (1,), generator=gen, device="cuda")
    if op == "dropout" or case.get("train"):
        state["grad"] = _map(gen, case, c)
        if op == "norm" and case["residual"]:
            state["grad_sum"] = _map(gen, case, c)
        for name in ("x", "residual", "weight"):
            if state.get(name) is not None:
                state[name].requires_grad_(True)
    return state


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "norm8": _plain_norm8, "quantize": _plain_quantize, "product8": _plain_product8,
                "dropout": _plain_dropout}[state["case"]["op"]](state)


def _run_own(state):
    import tvdcn
    case, residual = state["case"], state["residual"]
    op = case["op"]
    if op == "product8":
        with torch.no_grad():
            return tvdcn.pointwise_conv_int8(state["codes"], state["scales"], state["weight_codes"],
                                             state["weight_scales"], state["bias"], residual, case["activation"],
                                             dtype=_DTYPES[case["dtype"]])
    x = state["x"]
    if op == "quantize":
        codes, scales = tvdcn.quantize_int8(x)
        return [tvdcn.dequantize_int8(codes, scales, x.dtype), scales]
    weight = state.get("weight")
    if op == "norm8":
        with torch.no_grad():
            if residual is None:
                codes, scales = tvdcn.rms_norm_int8(x, weight, _EPS)
                return [tvdcn.dequantize_int8(codes, scales, x.dtype), scales]
            codes, scales, total = tvdcn.add_rms_norm_int8(x, residual, weight, _EPS)
            return [tvdcn.dequantize_int8(codes, scales, x.dtype), scales, total]
    if op == "dropout":
        y = tvdcn.seeded_dropout(x, case["p"], state["seed"], residual)
        inputs = [x] if residual is None else [x, residual]
        return [y.detach(), *torch.autograd.grad(y, inputs, state["grad"])]
    with torch.set_grad_enabled(case["train"]):
        results = [tvdcn.rms_norm(x, weight, _EPS)] if residual is None else tvdcn.add_rms_norm(x, residual, weight, _EPS)
    if not case["train"]:
        return list(results)
    grads = [state["grad"]] if residual is None else [state["grad"], state["grad_sum"]]
    inputs = [t for t in (x, residual, weight) if t is not None]
    return [*[y.detach() for y in results], *torch.autograd.grad(results, inputs, grads)]


# ---- plain forms, in 32 bits ----

def _in_8_bits(rows, border=False):
    """Codes (whole numbers) and scales of (..., channels) float32 rows. border: the quotients in 64 bits, since in 32 some
    fall to the other side of a rounding border, which float32 results show."""
    scales = (rows.abs().amax(-1) / 127).clamp(min=_LEAST_SCALE)
    if border:
        return torch.round(rows.double() / scales.double().unsqueeze(-1)).float(), scales
    return torch.round(rows / scales.unsqueeze(-1)), scales


def _plain_values(rows, dtype):
    codes, scales = _in_8_bits(rows, border=dtype == torch.float32)
    return [(codes * scales.unsqueeze(-1)).to(dtype).movedim(-1, 1), scales]


def _plain_total(state):
    """The rows that are normalised, and the sum as a result."""
    x, dtype = state["x"].movedim(1, -1), state["x"].dtype
    if state["residual"] is None:
        return x.float(), []
    total = (x.float() + state["residual"].movedim(1, -1).float()).to(dtype)
    return total.float(), [total.movedim(-1, 1)]


def _plain_norm(state):
    dtype, weight = state["x"].dtype, state["weight"].float()
    rows, total = _plain_total(state)
    rstd = torch.rsqrt(rows.square().mean(-1, keepdim=True) + _EPS)
    normal = rows * rstd
    results = [(normal * weight).to(dtype).movedim(-1, 1), *total]
    if not state["case"]["train"]:
        return results
    grad = state["grad"].movedim(1, -1).float()
    slope = grad * weight
    dx = rstd * (slope - normal * (slope * normal).mean(-1, keepdim=True))
    if total:
        dx = dx + state["grad_sum"].movedim(1, -1).float()
    dx = dx.to(dtype).movedim(-1, 1)
    dweight = (grad * normal).reshape(-1, weight.numel()).sum(0).to(dtype)
    return [*results, dx, *([dx] if total else []), dweight]


def _plain_norm8(state):
    rows, total = _plain_total(state)
    normal = rows * torch.rsqrt(rows.square().mean(-1, keepdim=True) + _EPS)
    return [*_plain_values(normal * state["weight"].float(), state["x"].dtype), *total]


def _plain_quantize(state):
    return _plain_values(state["x"].movedim(1, -1).float(), state["x"].dtype)


def _act(z, activation):
    if activation == "relu":
        return z.clamp(min=0)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _plain_product8(state):
    case = state["case"]
    codes = state["codes"].movedim(1, -1)
    z = codes.reshape(-1, case["channels"]).float() @ state["weight_codes"].float().t()
    z = z * state["scales"].reshape(-1, 1) * state["weight_scales"] + state["bias"].float()
    y = _act(z, case["activation"]).view(*codes.shape[:-1], case["out"])
    if state["residual"] is not None:
        y = y + state["residual"].movedim(1, -1).float()
    return y.to(_DTYPES[case["dtype"]]).movedim(-1, 1)


_LOW = 0xFFFFFFFF


def _kept(seed, count, p):
    """Which of `count` values are kept: Philox4x32-10 in 64-bit whole numbers, whose products wrap."""
    group = torch.arange((count + 7) // 8, device=seed.device)
    c0, c1, c2, c3 = group & _LOW, group >> 32, torch.zeros_like(group), torch.zeros_like(group)
    k0, k1 = seed & _LOW, (seed >> 32) & _LOW
    for _ in range(10):
        a, b = c0 * 0xD2511F53, c2 * 0xCD9E8D57
        c0, c1, c2, c3 = ((b >> 32) & _LOW) ^ c1 ^ k0, b & _LOW, ((a >> 32) & _LOW) ^ c3 ^ k1, a & _LOW
        k0, k1 = (k0 + 0x9E3779B9) & _LOW, (k1 + 0xBB67AE85) & _LOW
    words = torch.stack([c0, c1, c2, c3], -1)
    bits = torch.stack([words & 0xFFFF, words >> 16], -1).view(-1)[:count]
    return bits >= round(65536 * p)


def _plain_dropout(state):
    case, dtype = state["case"], state["x"].dtype
    rows = state["x"].movedim(1, -1)
    kept = _kept(state["seed"], rows.numel(), case["p"]).view(rows.shape)
    scale = 65536 / (65536 - round(65536 * case["p"]))

    def drop(v):
        return torch.where(kept, v.movedim(1, -1).float() * scale, 0.0)

    y = drop(state["x"])
    if state["residual"] is not None:
        y = y + state["residual"].movedim(1, -1).float()
    dx = drop(state["grad"]).to(dtype).movedim(-1, 1)
    return [y.to(dtype).movedim(-1, 1), dx, *([] if state["residual"] is None else [state["grad"]])]


# ---- the operators' definitions, in 64 bits ----

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        return {"norm": _exact_norm, "norm8": _exact_norm8, "quantize": _exact_quantize, "product8": _exact_product8,
                "dropout": _exact_dropout}[case["op"]](case, state)


def _exact_8_bits(x):
    step = x.abs().max(1)[0].div(127).clamp(min=_LEAST_SCALE).float().double()
    return [torch.round(x / step[:, None]) * step[:, None], step]


def _exact_total(state):
    x = state["x"].double()
    if state["residual"] is None:
        return x, []
    x = (x + state["residual"].double()).to(state["x"].dtype).double()   # the sum is held in the map's type
    return x, [x]


def _exact_unit(x):
    """x over the root of the mean of its squares, and that root."""
    root = torch.sqrt((x * x).sum(1, keepdim=True) / x.shape[1] + _EPS)
    return x / root, root


def _channels(v, like):
    return v.double().view(1, -1, *[1] * (like.dim() - 2))


def _exact_norm(case, state):
    x, total = _exact_total(state)
    unit, root = _exact_unit(x)
    weight = _channels(state["weight"], x)
    results = [unit * weight, *total]
    if not case["train"]:
        return results
    grad = state["grad"].double()
    back = grad * weight
    dx = (back - unit * (back * unit).sum(1, keepdim=True) / x.shape[1]) / root
    if total:
        dx = dx + state["grad_sum"].double()
    others = [d for d in range(x.dim()) if d != 1]
    return [*results, dx, *([dx] if total else []), (grad * unit).sum(others)]


def _exact_norm8(case, state):
    x, total = _exact_total(state)
    return [*_exact_8_bits(_exact_unit(x)[0] * _channels(state["weight"], x)), *total]


def _exact_quantize(case, state):
    return _exact_8_bits(state["x"].double())


def _exact_product8(case, state):
    x = state["codes"].double() * state["scales"].double()[:, None]
    weight = state["weight_codes"].double() * state["weight_scales"].double()[:, None]
    x = x.flatten(2).transpose(1, 2).reshape(-1, case["channels"]) if x.dim() > 2 else x
    z = torch.addmm(state["bias"].double(), x, weight.t())
    y = {"none": lambda: z, "relu": lambda: torch.relu(z), "silu": lambda: z * torch.sigmoid(z),
         "gelu": lambda: z * torch.special.ndtr(z)}[case["activation"]]()
    y = y.view(case["batch"], -1, case["out"]).transpose(1, 2).reshape(case["batch"], case["out"], *_size(case))
    return y if state["residual"] is None else y + state["residual"].double()


def _exact_mask(seed, count, p):
    """The kept values by Philox4x32-10, on the host."""
    u = numpy.uint64
    low, half = u(0xFFFFFFFF), u(32)
    group = numpy.arange(-(-count // 8), dtype=u)
    words = [group & low, group >> half, numpy.zeros_like(group), numpy.zeros_like(group)]
    keys = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        first, second = words[0] * u(0xD2511F53), words[2] * u(0xCD9E8D57)
        words = [(second >> half) ^ words[1] ^ u(keys[0]), second & low, (first >> half) ^ words[3] ^ u(keys[1]), first & low]
        keys = [(keys[0] + 0x9E3779B9) % 2 ** 32, (keys[1] + 0xBB67AE85) % 2 ** 32]
    bits = numpy.stack(words, 1).astype("<u4").view("<u2").reshape(-1)[:count]
    return torch.from_numpy(bits >= round(65536 * p))


def _exact_dropout(case, state):
    shape = [case["batch"], *_size(case), case["channels"]]
    mask = _exact_mask(int(state["seed"]), math.prod(shape), case["p"]).view(shape).movedim(-1, 1).cuda()
    factor = mask.double() / (1 - round(65536 * case["p"]) / 65536)
    y, grad = state["x"].double() * factor, state["grad"].double()
    if state["residual"] is None:
        return [y, grad * factor]
    return [y + state["residual"].double(), grad * factor, grad]


def work(case):
    e = {"f32": 4}.get(case["dtype"], 2)
    rows, c = _rows(case), case["channels"]
    entries, op = rows * c, case["op"]
    if op == "product8":
        out = case["out"]
        return {"bytes": entries + out * c + 4 * (rows + out) + e * (out + rows * out * (2 if case["residual"] else 1)),
                "flops": 2 * entries * out}
    if op == "quantize":
        # |x|, the largest, the scaling and the rounding; and back
        return {"bytes": 2 * e * entries + 4 * rows, "flops": 5 * entries}
    if op == "dropout":
        # x to y, with the shortcut; the incoming gradient to x's (the shortcut's is the incoming one). Ten rounds of two
        # products for eight values, each time
        return {"bytes": e * entries * (5 if case["residual"] else 4), "flops": 2 * entries * 4}
    added = case["residual"]
    maps = 3 if added else 1   # x, the shortcut and the sum
    if op == "norm8":
        return {"bytes": e * ((maps + 1) * entries + c) + 4 * rows, "flops": 9 * entries}
    # the result; backward: the gradients of both results and what was normalised in, that of x (and the shortcut) and of the
    # weight out
    maps += 1 + ((4 if added else 3) if case["train"] else 0)
    return {"bytes": e * (maps * entries + (2 if case["train"] else 1) * c), "flops": (14 if case["train"] else 4) * entries}
