"""What the channels-last operators next to the convolutions are measured by.

Every case is one pass as a program makes it: the forward under ``no_grad`` for inference, the forward
and all gradients for training. A feature map is (batch, channels, *size) with its channels contiguous in
memory (torch's ``channels_last`` in two dimensions), or (batch, channels) where it has no grid.

* ``norm``: group normalisation, affine map and activation,
* ``pointwise``: ``activation(x W^T + bias) + residual`` over the channels of every pixel,
* ``round_trip``: a feature map kept in 8 bits and read back; with ``kept8`` the two others keep their
  input for the backward pass so.

An 8-bit map holds, for every 32 channels of a pixel, one exponent k, the least (and at least -126) with
``max |x| <= 127 * 2^k``, and the codes ``q = x / 2^k`` rounded to whole numbers, ties to the even one.
It stands for ``q * 2^k``.
"""
import math

import torch

own = False

_DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
_BLOCK = 32
_EPS = 1e-5


def _norm(name, batch, channels, size, groups, **kw):
    case = dict(name=name, op="norm", batch=batch, channels=channels, size=size, groups=groups, activation="silu",
                dtype="bf16", train=True, kept8=False)
    case.update(kw)
    return case


def _pointwise(name, batch, channels, out, size, **kw):
    case = dict(name=name, op="pointwise", batch=batch, channels=channels, out=out, size=size, activation="none",
                residual=False, dtype="bf16", train=True, kept8=False)
    case.update(kw)
    return case


def _round_trip(name, batch, channels, size, dtype):
    return dict(name=name, op="round_trip", batch=batch, channels=channels, size=size, dtype=dtype)


def listed():
    return [
        # one image of a toy model: launches and host time
        _norm("norm_tiny_infer", 1, 32, "10x10", 8, train=False),
        # behind the backbone layer of bench.py's metric line, in a bfloat16 model
        _norm("norm_layer_train", 8, 256, "64x64", 32),
        # groups of nine channels on a grid that divides by nothing useful, in float32
        _norm("norm_ragged_train_f32", 3, 63, "61x47", 7, activation="relu", dtype="f32"),
        # behind the long sequence layer of bench.py's suite, its input kept in 8 bits
        _norm("norm_sequence_train_kept8", 16, 512, "4096", 32, activation="gelu", dtype="f16", kept8=True),
        # one pixel, or one token, of a served model: latency
        _pointwise("pointwise_pixel_infer", 1, 256, 1024, "", activation="gelu", train=False),
        # one image at a coarse level of a feature pyramid, served, added to its shortcut
        _pointwise("pointwise_image_infer_f16", 1, 256, 256, "25x38", activation="relu", residual=True, dtype="f16",
                   train=False),
        # the widening layer of a block behind the backbone layer
        _pointwise("pointwise_layer_train", 8, 256, 1024, "64x64", activation="gelu"),
        # channels that divide by nothing useful, float32, added to a shortcut
        _pointwise("pointwise_ragged_train_f32", 3, 71, 101, "61x47", activation="relu", residual=True, dtype="f32"),
        # the backbone layer's projection in float32
        _pointwise("pointwise_layer_train_f32", 8, 256, 256, "64x64", dtype="f32"),
        # widening of long sequences, its input kept in 8 bits: the most work
        _pointwise("pointwise_sequence_train_kept8", 16, 512, 2048, "4096", activation="silu", dtype="f16", kept8=True),
        # a small float32 map to 8 bits and back, its last block of channels short
        _round_trip("round_trip_ragged_f32", 3, 72, "61x47", "f32"),
        # the long sequence layer's activations to 8 bits and back
        _round_trip("round_trip_sequence", 16, 512, "4096", "bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    """A pass of the same kinds: every operator, direction, type and activation, 1 to 16 images, grids of
    none to three axes, from single pixels to the listed ones, channel counts of any kind."""
    while True:
        op = rng.choice(("norm", "norm", "pointwise", "pointwise", "round_trip"))
        batch = _log_int(rng, 1, 16)
        dim = rng.choice((0, 1, 2, 2, 3))
        hi = {1: 4096, 2: 72, 3: 18}
        size = "x".join(str(_log_int(rng, 1 if op != "norm" else 3, hi[dim])) for _ in range(dim))
        if dim == 0:
            batch = _log_int(rng, 1, 4096)
        channels = _log_int(rng, 3, 512)
        if rng.random() < 0.6:
            channels = max(8, channels // 8 * 8)
        dtype, train, kept8 = rng.choice(("f32", "f16", "bf16")), rng.random() < 0.7, rng.random() < 0.3
        activation = rng.choice(("none", "relu", "silu", "gelu"))
        if op == "round_trip":
            case = _round_trip("", batch, channels, size, dtype)
        elif op == "norm":
            groups = rng.choice([g for g in range(1, min(channels, 64) + 1) if channels % g == 0])
            case = _norm("", batch, channels, size, groups, activation=activation, dtype=dtype, train=train,
                         kept8=kept8 and train)
            # of the gradient of a few values, mean and spread taken out, next to nothing is left
            if _pixels(case) * (channels // groups) < 16:
                continue
        else:
            out = _log_int(rng, 3, 2048)
            if rng.random() < 0.6:
                out = max(8, out // 8 * 8)
            case = _pointwise("", batch, channels, out, size, activation=activation, residual=rng.random() < 0.4,
                              dtype=dtype, train=train, kept8=kept8 and train)
        del case["name"]
        return case


def _size(case):
    return [int(s) for s in case["size"].split("x")] if case["size"] else []


def _pixels(case):
    return math.prod(_size(case))


def _map(gen, case, channels, spread=None, shift=None):
    """A (batch, channels, *size) map in channels-last memory."""
    x = torch.randn([case["batch"], *_size(case), channels], generator=gen, device="cuda")
    if spread is not None:
        x = x * spread
    if shift is not None:
        x = x + shift
    return x.to(_DTYPES[case["dtype"]]).movedim(-1, 1)


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed * 7919 + 17)
    dtype, c = _DTYPES[case["dtype"]], case["channels"]

    def vector(n, scale=1.0, shift=0.0):
        return (torch.randn(n, generator=gen, device="cuda") * scale + shift).to(dtype)

    # a layer's outputs: channels of unlike spread and mean
    spread = torch.exp(0.4 * torch.randn(c, generator=gen, device="cuda"))
    shift = 0.5 * torch.randn(c, generator=gen, device="cuda")
    state = dict(case=case, x=_map(gen, case, c, spread, shift))
    if case["op"] == "norm":
        state.update(weight=vector(c, 0.2, 1.0), bias=vector(c, 0.2))
        if case["train"]:
            state["grad"] = _map(gen, case, c)
    elif case["op"] == "pointwise":
        weight = torch.randn(case["out"], c, generator=gen, device="cuda") / math.sqrt(c)
        state.update(weight=weight.to(dtype), bias=vector(case["out"], 0.2))
        state["residual"] = _map(gen, case, case["out"]) if case["residual"] else None
        if case["train"]:
            state["grad"] = _map(gen, case, case["out"])
    if case.get("train"):
        for name in ("x", "weight", "bias", "residual"):
            if state.get(name) is not None:
                state[name].requires_grad_(True)
    return state


def run(state):
    if own:
        return _run_own(state)
    with torch.no_grad():
        return {"norm": _plain_norm, "pointwise": _plain_pointwise, "round_trip": _plain_round_trip}[
            state["case"]["op"]](state)


def _run_own(state):
    import tvdcn
    case = state["case"]
    if case["op"] == "round_trip":
        codes, exponents = tvdcn.compress_activation(state["x"])
        return tvdcn.expand_activation(codes, exponents, state["x"].dtype)

    def forward():
        if case["op"] == "norm":
            return tvdcn.group_norm_act(state["x"], case["groups"], state["weight"], state["bias"], _EPS,
                                        case["activation"], keep_int8=case["kept8"])
        return tvdcn.pointwise_conv(state["x"], state["weight"], state["bias"], state["residual"],
                                    case["activation"], keep_int8=case["kept8"])

    if not case["train"]:
        with torch.no_grad():
            return forward()
    y = forward()
    inputs = [state[n] for n in ("x", "weight", "bias", "residual") if state.get(n) is not None]
    return [y.detach(), *torch.autograd.grad(y, inputs, state["grad"])]


# ---- plain forms, in 32 bits ----

def _act(z, activation):
    if activation == "relu":
        return z.clamp(min=0)
    if activation == "silu":
        return z / (1 + torch.exp(-z))
    if activation == "gelu":
        return 0.5 * z * (1 + torch.erf(z * math.sqrt(0.5)))
    return z


def _act_slope(z, activation):
    if activation == "relu":
        return (z > 0).to(z.dtype)
    if activation == "silu":
        s = 1 / (1 + torch.exp(-z))
        return s * (1 + z * (1 - s))
    if activation == "gelu":
        return 0.5 * (1 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    return torch.ones_like(z)


def _in_8_bits(x):
    """The values that the 8-bit form of a (..., channels) map stands for. All steps are exact but the rounding."""
    c, most = x.shape[-1], torch.finfo(x.dtype).max
    blocks = torch.nn.functional.pad(x.float(), (0, -c % _BLOCK)).unflatten(-1, (-1, _BLOCK))
    part, power = torch.frexp(blocks.abs().amax(-1, keepdim=True))
    k = torch.where(part > 127 / 128, power - 6, power - 7).clamp(min=-126)
    return torch.ldexp(torch.round(torch.ldexp(blocks, -k)), k).flatten(-2)[..., :c].clamp(-most, most)


def _plain_norm(state):
    case, dtype = state["case"], state["x"].dtype
    b, c, g, p = case["batch"], case["channels"], case["groups"], _pixels(case)
    rows = state["x"].movedim(1, -1)
    x = rows.float().reshape(b, p, g, c // g)
    weight, bias = (state[n].float().view(g, c // g) for n in ("weight", "bias"))
    mean = x.mean((1, 3), keepdim=True)
    rstd = torch.rsqrt((x - mean).square().mean((1, 3), keepdim=True) + _EPS)
    y = _act((x - mean) * rstd * weight + bias, case["activation"])
    y = y.to(dtype).view(rows.shape).movedim(-1, 1)
    if not case["train"]:
        return y
    if case["kept8"]:
        x = _in_8_bits(rows).reshape(b, p, g, c // g)
    normal = (x - mean) * rstd
    dz = state["grad"].movedim(1, -1).float().reshape(b, p, g, c // g)
    dz = dz * _act_slope(normal * weight + bias, case["activation"])
    dn = dz * weight
    dx = rstd * (dn - dn.mean((1, 3), keepdim=True) - normal * (dn * normal).mean((1, 3), keepdim=True))
    return [y, dx.to(dtype).view(rows.shape).movedim(-1, 1), (dz * normal).sum((0, 1)).view(c).to(dtype),
            dz.sum((0, 1)).view(c).to(dtype)]


def _plain_pointwise(state):
    case, dtype, weight = state["case"], state["x"].dtype, state["weight"].float()
    rows = state["x"].movedim(1, -1)
    shape = [*rows.shape[:-1], case["out"]]
    x = rows.float().reshape(-1, case["channels"])
    z = x @ weight.t() + state["bias"].float()
    y = _act(z, case["activation"])
    if case["residual"]:
        y = y + state["residual"].movedim(1, -1).float().reshape(y.shape)
    y = y.to(dtype).view(shape).movedim(-1, 1)
    if not case["train"]:
        return y
    if case["kept8"]:
        x = _in_8_bits(rows).reshape(x.shape)
    dz = state["grad"].movedim(1, -1).float().reshape(z.shape) * _act_slope(z, case["activation"])
    grads = [(dz @ weight).to(dtype).view(rows.shape).movedim(-1, 1), (dz.t() @ x).to(dtype), dz.sum(0).to(dtype)]
    return [y, *grads, *([state["grad"]] if case["residual"] else [])]


def _plain_round_trip(state):
    return _in_8_bits(state["x"].movedim(1, -1)).to(state["x"].dtype).movedim(-1, 1)


# ---- the operators' definitions, in 64 bits ----

def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        x = state["x"].double()
        if case["op"] == "round_trip":
            return _exact_8_bits(x, state["x"].dtype)
        f, df = _exact_activation(case["activation"])
        if case["op"] == "norm":
            return _exact_norm(case, state, x, f, df)
        return _exact_pointwise(case, state, x, f, df)


def _exact_8_bits(x, dtype):
    out = torch.empty_like(x)
    for first in range(0, x.shape[1], _BLOCK):
        block = x[:, first:first + _BLOCK]
        step = torch.exp2(torch.ceil(torch.log2(block.abs().amax(1, keepdim=True) / 127)).clamp(min=-126))
        out[:, first:first + _BLOCK] = torch.round(block / step) * step
    most = torch.finfo(dtype).max
    return out.clamp(-most, most)


def _exact_activation(name):
    if name == "none":
        return (lambda z: z), torch.ones_like
    if name == "relu":
        return torch.relu, (lambda z: torch.heaviside(z, torch.zeros_like(z)))
    if name == "silu":
        return (lambda z: z * torch.sigmoid(z)), (
            lambda z: torch.sigmoid(z) + z * torch.sigmoid(z) * torch.sigmoid(-z))
    cdf = torch.special.ndtr
    return (lambda z: z * cdf(z)), (lambda z: cdf(z) + z * torch.exp(-z.square() / 2) / math.sqrt(2 * math.pi))


def _exact_norm(case, state, x, f, df):
    b, c, g = case["batch"], case["channels"], case["groups"]
    x = x.reshape(b, g, c // g, -1)
    count = x[0, 0].numel()
    mean = x.sum((2, 3), keepdim=True) / count
    scale = 1 / torch.sqrt(((x - mean) ** 2).sum((2, 3), keepdim=True) / count + _EPS)
    weight, bias = (state[n].double().view(1, g, c // g, 1) for n in ("weight", "bias"))
    y = f(scale * (x - mean) * weight + bias).view(state["x"].shape)
    if not case["train"]:
        return y
    if case["kept8"]:
        x = _exact_8_bits(state["x"].double(), state["x"].dtype).reshape(x.shape)
    h = scale * (x - mean)
    dz = state["grad"].double().reshape(h.shape) * df(h * weight + bias)
    dh = dz * weight
    along = (dh.sum((2, 3), keepdim=True) + h * (dh * h).sum((2, 3), keepdim=True)) / count
    return [y, (scale * (dh - along)).view(state["x"].shape), (dz * h).sum((0, 3)).view(c), dz.sum((0, 3)).view(c)]


def _exact_pointwise(case, state, x, f, df):
    def as_rows(v):
        return v.flatten(2).transpose(1, 2).reshape(-1, v.shape[1]) if v.dim() > 2 else v

    def as_map(v):
        return v.view(case["batch"], -1, v.shape[-1]).transpose(1, 2).reshape(case["batch"], v.shape[-1], *_size(case))

    weight, bias = state["weight"].double(), state["bias"].double()
    z = torch.addmm(bias, as_rows(x), weight.t())
    y = as_map(f(z))
    if case["residual"]:
        y = y + state["residual"].double()
    if not case["train"]:
        return y
    if case["kept8"]:
        x = _exact_8_bits(x, state["x"].dtype)
    dz = as_rows(state["grad"].double()) * df(z)
    grads = [as_map(dz.mm(weight)), dz.t().mm(as_rows(x)), dz.sum(0)]
    return [y, *grads, *([state["grad"].double()] if case["residual"] else [])]


def work(case):
    e = {"f32": 4}.get(case["dtype"], 2)
    rows = case["batch"] * _pixels(case)
    entries = rows * case["channels"]
    if case["op"] == "round_trip":
        # |x|, maximum, scaling, rounding; and back
        return {"bytes": 2 * entries * e, "flops": 5 * entries}
    if case["op"] == "norm":
        # x to y; with the gradients, the incoming one to the outgoing one
        maps = 4 if case["train"] else 2
        return {"bytes": maps * entries * e + maps * case["channels"] * e, "flops": maps * 6 * entries}
    out = rows * case["out"]
    weights = case["channels"] * case["out"] + case["out"]
    forward = entries + out + weights + (out if case["residual"] else 0)
    # backward: the incoming gradient in, those of x, the weight and the bias out (the shortcut's is the incoming one)
    backward = entries + out + weights
    return {"bytes": e * (forward + (backward if case["train"] else 0)),
            "flops": (3 if case["train"] else 1) * 2 * rows * case["channels"] * case["out"]}
