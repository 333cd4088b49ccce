// Operators on channels-last maps: group_norm_act, pointwise_conv, compress_activation and expand_activation,
// registered in the `tvdcn` namespace with CUDA (= HIP), CPU, Meta, Autograd and Autocast kernels. No counterpart in
// the reference. A map is a (batch, channels, *size) tensor, or (rows, channels); it is laid out channels-last (a map
// that is not comes in as a copy) and every result is a channels-last map. The CUDA kernels check, allocate results
// and workspace from the caching allocator and call the C ABI on the current stream; the CPU kernels compute the same
// definitions with ATen in float32 (float64 for float64 maps).
#include <array>
#include <cmath>
#include <tuple>

#include "map_tensors.h"

namespace tvdcn_amd {
namespace {

constexpr int64_t kBlock = 32;   // channels of an 8-bit map that share an exponent

// ---------------------------------------------------------------------------
// compress_activation / expand_activation
// ---------------------------------------------------------------------------
const char *COMPRESS = "compress_activation", *EXPAND = "expand_activation";

int64_t blocks_of(int64_t channels) { return (channels + kBlock - 1) / kBlock; }

void check_compress(const Tensor &x) {
    check_map(x, COMPRESS);
    TORCH_CHECK(x.scalar_type() != at::kDouble, COMPRESS, ": float32, float16 and bfloat16 maps only");
}
void check_kept(const Tensor &codes, const Tensor &exponents, const char *name) {
    TORCH_CHECK(codes.dim() >= 2 && codes.scalar_type() == at::kChar && codes.size(1) > 0, name,
                ": expected int8 codes of shape (batch, channels, *size)");
    TORCH_CHECK(exponents.scalar_type() == at::kByte && exponents.sizes() == map_shape(codes, blocks_of(codes.size(1))), name,
                ": expected uint8 exponents of shape ", map_shape(codes, blocks_of(codes.size(1))), ", got ",
                exponents.scalar_type(), " ", exponents.sizes());
    TORCH_CHECK(codes.device() == exponents.device(), name, ": expected all tensors on ", codes.device(),
                ", but exponents is on ", exponents.device());
}
void check_expand(const Tensor &codes, const Tensor &exponents, at::ScalarType dtype) {
    check_kept(codes, exponents, EXPAND);
    TORCH_CHECK(dtype == at::kFloat || dtype == at::kHalf || dtype == at::kBFloat16, EXPAND,
                ": float32, float16 and bfloat16 maps only, got ", dtype);
}

Two compress_hip(const Tensor &x) {
    check_compress(x);
    c10::DeviceGuard guard(x.device());
    const Tensor r = rows_of(x);
    const int64_t C = x.size(1);
    Tensor codes = new_map(x.sizes(), x.options().dtype(at::kChar));
    Tensor exps = new_map(map_shape(x, blocks_of(C)), x.options().dtype(at::kByte));
    check_status(tvdcn_compress_activation(map_dtype(x.scalar_type(), COMPRESS), x.size(0) * pixels_of(x), C, ptr(r),
                                           (int8_t *)ptr(codes), (uint8_t *)ptr(exps), stream_of(x)),
                 COMPRESS);
    return {codes, exps};
}
Tensor expand_hip(const Tensor &codes, const Tensor &exponents, at::ScalarType dtype) {
    check_expand(codes, exponents, dtype);
    c10::DeviceGuard guard(codes.device());
    const Tensor q = rows_of(codes), e = rows_of(exponents);
    const int64_t C = codes.size(1);
    Tensor y = new_map(codes.sizes(), codes.options().dtype(dtype));
    check_status(tvdcn_expand_activation(map_dtype(dtype, EXPAND), codes.size(0) * pixels_of(codes), C, (const int8_t *)ptr(q),
                                         (const uint8_t *)ptr(e), ptr(y), stream_of(codes)),
                 EXPAND);
    return y;
}

Two compress_meta(const Tensor &x) {
    check_compress(x);
    const int64_t C = x.size(1);
    return {new_map(x.sizes(), x.options().dtype(at::kChar)), new_map(map_shape(x, blocks_of(C)), x.options().dtype(at::kByte))};
}
Tensor expand_meta(const Tensor &codes, const Tensor &exponents, at::ScalarType dtype) {
    check_expand(codes, exponents, dtype);
    return new_map(codes.sizes(), codes.options().dtype(dtype));
}

Two compress_cpu(const Tensor &x) {
    if (x.numel() == 0) return compress_meta(x);   // (empty tensors of x's device)
    check_compress(x);
    const int64_t C = x.size(1), B = blocks_of(C);
    // in float64 the scaling is exact for every float32
    Tensor r = at::constant_pad_nd(to_rows(x).to(at::kDouble), {0, B * kBlock - C});
    r = r.unflatten(-1, {B, kBlock});
    const Tensor big = r.abs().amax(-1, true), bad = big.isfinite().logical_not();
    Tensor part, power;
    std::tie(part, power) = at::frexp(big.masked_fill(bad, 0.0));
    const Tensor k = at::where(part > 127.0 / 128.0, power - 6, power - 7).clamp_min(-126).masked_fill(part == 0.0, -126);
    const Tensor q = at::round(at::ldexp(r, -k)).masked_fill(bad, 0.0).to(at::kChar);
    const Tensor e = (k + 127).masked_fill(bad, 255).to(at::kByte);
    return {to_map(q.flatten(-2).narrow(-1, 0, C).contiguous()), to_map(e.squeeze(-1).contiguous())};
}
// the values as [..., channels] float64
Tensor expand_rows(const Tensor &codes, const Tensor &exponents, at::ScalarType dtype) {
    const int64_t C = codes.size(1);
    const Tensor q = to_rows(codes).to(at::kDouble), e = to_rows(exponents).to(at::kInt);
    const Tensor wide = e.repeat_interleave(kBlock, -1).narrow(-1, 0, C);
    const double most = dtype == at::kHalf ? 65504.0 : dtype == at::kFloat ? 3.4028234663852886e38 : 3.3895313892515355e38;
    return at::ldexp(q, wide - 127).clamp(-most, most).masked_fill(wide == 255, NAN);
}
Tensor expand_cpu(const Tensor &codes, const Tensor &exponents, at::ScalarType dtype) {
    check_expand(codes, exponents, dtype);
    return to_map(expand_rows(codes, exponents, dtype).to(dtype));
}

// ---------------------------------------------------------------------------
// group_norm_act
// ---------------------------------------------------------------------------
const char *NORM = "group_norm_act";

void check_norm(const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias, double eps, int64_t activation) {
    check_map(x, NORM);
    TORCH_CHECK(groups > 0 && x.size(1) % groups == 0, NORM, ": expected the number of channels to be divisible by "
                "num_groups, got ", x.size(1), " channels and num_groups=", groups);
    TORCH_CHECK(std::isfinite(eps) && eps >= 0.0, NORM, ": eps must be finite and not negative, got ", eps);
    check_activation(activation, NORM);
    check_like(x, weight, "weight", {x.size(1)}, NORM);
    check_like(x, bias, "bias", {x.size(1)}, NORM);
}
// The backward's input: the map, or its 8-bit form, of the gradient's shape; needed: not to be left out
void check_source(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents, int64_t channels,
                  const char *name, bool needed) {
    TORCH_CHECK(!(has(input) && has(codes)) && (has(input) || has(codes) || !needed) && has(codes) == has(exponents), name,
                " backward: expected the input, or its codes and exponents");
    check_like(grad, input, "input", map_shape(grad, channels), name);
    if (has(codes)) {
        check_kept(*codes, *exponents, name);
        TORCH_CHECK(codes->sizes() == map_shape(grad, channels) && codes->device() == grad.device(), name,
                    " backward: the codes do not match the gradient");
        TORCH_CHECK(grad.scalar_type() != at::kDouble, name, ": 8-bit maps of float64 are not supported");
    }
}
void check_norm_backward(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents,
                         MaybeTensor weight, MaybeTensor bias, const Tensor &stats, int64_t activation) {
    check_map(grad, NORM);
    check_activation(activation, NORM);
    check_source(grad, input, codes, exponents, grad.size(1), NORM, true);
    check_like(grad, weight, "weight", {grad.size(1)}, NORM);
    check_like(grad, bias, "bias", {grad.size(1)}, NORM);
    TORCH_CHECK(stats.dim() == 3 && stats.size(0) == 2 && stats.size(1) == grad.size(0) && stats.size(2) > 0 &&
                    grad.size(1) % stats.size(2) == 0 &&
                    stats.scalar_type() == (grad.scalar_type() == at::kDouble ? at::kDouble : at::kFloat) &&
                    stats.device() == grad.device(),
                NORM, " backward: the statistics are not those of the forward");
}

// y and the statistics (2, batch, groups): means, reciprocal deviations
Two norm_forward_hip(const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias, double eps, int64_t act) {
    check_norm(x, groups, weight, bias, eps, act);
    c10::DeviceGuard guard(x.device());
    const Tensor r = rows_of(x), w = flat(weight), b = flat(bias);
    const tvdcn_norm_desc d{map_dtype(x.scalar_type(), NORM), (int32_t)act, x.size(0), pixels_of(x), x.size(1), groups, eps};
    Tensor y = new_map(x.sizes(), x.options());
    Tensor stats = at::empty({2, x.size(0), groups}, x.options().dtype(at::kFloat));
    if (x.numel() == 0) return {y, stats.zero_()};
    const size_t n = tvdcn_group_norm_act_forward_workspace_size(&d);
    const Tensor work = n ? bytes(x, n) : Tensor();
    float *mean = (float *)ptr(stats);
    check_status(tvdcn_group_norm_act_forward(&d, ptr(r), ptr(w), ptr(b), ptr(y), mean, mean + x.size(0) * groups, ptr(work), n, stream_of(x)), NORM);
    return {y, stats};
}
Three norm_backward_hip(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents, MaybeTensor weight,
                        MaybeTensor bias, const Tensor &stats_, int64_t act, std::array<bool, 3> want) {
    check_norm_backward(grad, input, codes, exponents, weight, bias, stats_, act);
    c10::DeviceGuard guard(grad.device());
    const Tensor g = rows_of(grad), r = rows_of(input), q = rows_of(codes), e = rows_of(exponents);
    const Tensor w = flat(weight), b = flat(bias);
    const int64_t C = grad.size(1), groups = stats_.size(2);
    const Tensor stats = stats_.contiguous();
    const float *mean = (const float *)ptr(stats);
    const tvdcn_norm_desc d{map_dtype(grad.scalar_type(), NORM), (int32_t)act, grad.size(0), pixels_of(grad), C, groups, 0.0};
    Tensor dx, dw, db;
    if (want[0]) dx = new_map(grad.sizes(), grad.options());
    if (want[1]) dw = at::empty({C}, grad.options());
    if (want[2]) db = at::empty({C}, grad.options());
    const size_t n = tvdcn_group_norm_act_backward_workspace_size(&d);
    const Tensor work = n ? bytes(grad, n) : Tensor();
    check_status(tvdcn_group_norm_act_backward(&d, ptr(g), ptr(r), (const int8_t *)ptr(q), (const uint8_t *)ptr(e), ptr(w), ptr(b),
                                               mean, mean ? mean + grad.size(0) * groups : nullptr, ptr(dx), ptr(dw), ptr(db),
                                               ptr(work), n, stream_of(grad)),
                 "group_norm_act backward");
    return {dx, dw, db};
}

Two norm_forward_meta(const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias, double eps, int64_t act) {
    check_norm(x, groups, weight, bias, eps, act);
    const auto o = x.options().dtype(x.scalar_type() == at::kDouble ? at::kDouble : at::kFloat);
    return {new_map(x.sizes(), x.options()), at::empty({2, x.size(0), groups}, o)};
}
Three norm_backward_meta(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents, MaybeTensor weight,
                         MaybeTensor bias, const Tensor &stats, int64_t act, std::array<bool, 3> want) {
    check_norm_backward(grad, input, codes, exponents, weight, bias, stats, act);
    const int64_t C = grad.size(1);
    return {want[0] ? new_map(grad.sizes(), grad.options()) : Tensor(), want[1] ? at::empty({C}, grad.options()) : Tensor(),
            want[2] ? at::empty({C}, grad.options()) : Tensor()};
}

// d act'(z); zero where a rectifier is shut, also of a gradient that is not finite
Tensor act_slopes(const Tensor &d, const Tensor &z, int64_t act) {
    if (act == TVDCN_ACT_RELU) return d.masked_fill(z <= 0, 0.0);
    if (act == TVDCN_ACT_SILU) {
        const Tensor s = at::sigmoid(z);
        return d * (s * (1 + z * (1 - s)));
    }
    if (act == TVDCN_ACT_GELU)
        return d * (at::erfc(z * -M_SQRT1_2) * 0.5 + z * at::exp(z.square() * -0.5) * (0.5 * M_2_SQRTPI * M_SQRT1_2));
    return d;
}

struct NormRows {   // [batch, pixels, groups, channels per group] and parameters that broadcast over it
    Tensor x, w, b;
};
NormRows norm_rows(const Tensor &map, int64_t groups, MaybeTensor weight, MaybeTensor bias) {
    const int64_t Cg = map.size(-1) / groups;
    const auto t = wide_type(map);
    auto param = [&](MaybeTensor p, double none) {
        return has(p) ? p->to(t).reshape({groups, Cg}) : at::full({groups, Cg}, none, map.options().dtype(t));
    };
    return {map.to(t).reshape({map.size(0), -1, groups, Cg}), param(weight, 1.0), param(bias, 0.0)};
}

Two norm_forward_cpu(const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias, double eps, int64_t act) {
    check_norm(x, groups, weight, bias, eps, act);
    if (x.numel() == 0) return {new_map(x.sizes(), x.options()), at::zeros({2, x.size(0), groups}, x.options().dtype(wide_type(x)))};
    const Tensor rows = to_rows(x);
    const NormRows n = norm_rows(rows, groups, weight, bias);
    const Tensor mean = n.x.mean(at::IntArrayRef({1, 3}), true), d = n.x - mean;
    const Tensor rstd = at::rsqrt(d.square().mean(at::IntArrayRef({1, 3}), true) + eps);
    const Tensor y = act_value(d * rstd * n.w + n.b, act).to(x.scalar_type()).reshape(rows.sizes());
    return {to_map(y), at::stack({mean.reshape({x.size(0), groups}), rstd.reshape({x.size(0), groups})})};
}
Three norm_backward_cpu(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents, MaybeTensor weight,
                        MaybeTensor bias, const Tensor &stats, int64_t act, std::array<bool, 3> want) {
    check_norm_backward(grad, input, codes, exponents, weight, bias, stats, act);
    const int64_t C = grad.size(1), groups = stats.size(2);
    const auto t = grad.scalar_type();
    if (grad.numel() == 0)
        return {want[0] ? new_map(grad.sizes(), grad.options()) : Tensor(), want[1] ? at::zeros({C}, grad.options()) : Tensor(),
                want[2] ? at::zeros({C}, grad.options()) : Tensor()};
    const Tensor rows = to_rows(grad);
    const Tensor src = has(input) ? to_rows(*input) : expand_rows(*codes, *exponents, t).to(at::kFloat);
    const NormRows n = norm_rows(src, groups, weight, bias);
    const Tensor rs = stats[1].reshape({-1, 1, groups, 1}), h = (n.x - stats[0].reshape({-1, 1, groups, 1})) * rs;
    const Tensor dz = act_slopes(rows.to(wide_type(grad)).reshape(n.x.sizes()), h * n.w + n.b, act), dn = dz * n.w;
    Tensor dx, dw, db;
    if (want[0]) dx = to_map((rs * (dn - dn.mean(at::IntArrayRef({1, 3}), true) - h * (dn * h).mean(at::IntArrayRef({1, 3}), true))).to(t).reshape(rows.sizes()));
    if (want[1]) dw = (dz * h).sum(at::IntArrayRef({0, 1})).reshape({C}).to(t);
    if (want[2]) db = dz.sum(at::IntArrayRef({0, 1})).reshape({C}).to(t);
    return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// pointwise_conv
// ---------------------------------------------------------------------------
const char *POINT = "pointwise_conv";

void check_weight(const Tensor &x, const Tensor &weight, int64_t channels, int at) {
    TORCH_CHECK(weight.dim() == 2 && weight.size(0) > 0 && weight.size(1) > 0, POINT,
                ": expected a weight of shape (out_channels, in_channels), got ", weight.sizes());
    TORCH_CHECK(weight.size(at) == channels, POINT, ": expected a weight for ", channels, at ? " input" : " output",
                " channels, got ", weight.sizes());
    check_like(x, weight, "weight", weight.sizes(), POINT);
}
void check_pointwise(const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual, int64_t activation) {
    check_map(x, POINT);
    check_weight(x, weight, x.size(1), 1);
    check_activation(activation, POINT);
    check_like(x, bias, "bias", {weight.size(0)}, POINT);
    check_like(x, residual, "residual", map_shape(x, weight.size(0)), POINT);
}
// What the activation's argument is kept in: the map's type, but float16 for a silu or gelu of a bfloat16 map
at::ScalarType argument_type(const Tensor &x, int64_t act) {
    return x.scalar_type() == at::kBFloat16 && (act == TVDCN_ACT_SILU || act == TVDCN_ACT_GELU) ? at::kHalf : x.scalar_type();
}
void check_pointwise_backward(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents,
                              const Tensor &weight, MaybeTensor pre, int64_t activation, bool weight_grad) {
    check_map(grad, POINT);
    check_weight(grad, weight, grad.size(1), 0);
    check_activation(activation, POINT);
    check_source(grad, input, codes, exponents, weight.size(1), POINT, weight_grad);   // (only the weight's gradient reads it)
    TORCH_CHECK(activation == TVDCN_ACT_NONE || has(pre), POINT, " backward: the activation's argument is missing");
    if (activation != TVDCN_ACT_NONE)
        TORCH_CHECK(pre->sizes() == grad.sizes() && pre->scalar_type() == argument_type(grad, activation) &&
                        pre->device() == grad.device(),
                    POINT, " backward: the activation's argument is not that of the forward");
}

Two point_forward_hip(const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual, int64_t act,
                      bool save_pre) {
    check_pointwise(x, weight, bias, residual, act);
    c10::DeviceGuard guard(x.device());
    const Tensor r = rows_of(x), w = flat(maybe(weight)), b = flat(bias), res = rows_of(residual);
    const int64_t N = weight.size(0);
    const tvdcn_pointwise_desc d{map_dtype(x.scalar_type(), POINT), (int32_t)act, x.size(0) * pixels_of(x), x.size(1), N};
    Tensor y = new_map(map_shape(x, N), x.options());
    Tensor pre = save_pre ? new_map(y.sizes(), x.options().dtype(argument_type(x, act))) : Tensor();
    const size_t n = tvdcn_pointwise_conv_forward_workspace_size(&d);
    const Tensor work = n ? bytes(x, n) : Tensor();
    check_status(tvdcn_pointwise_conv_forward(&d, ptr(r), ptr(w), ptr(b), ptr(res), ptr(y), ptr(pre),
                                              ptr(work), n, stream_of(x)),
                 POINT);
    return {y, pre};
}
Three point_backward_hip(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents, const Tensor &weight,
                         MaybeTensor pre, int64_t act, std::array<bool, 3> want) {
    check_pointwise_backward(grad, input, codes, exponents, weight, pre, act, want[1]);
    c10::DeviceGuard guard(grad.device());
    const Tensor g = rows_of(grad), r = rows_of(input), q = rows_of(codes), e = rows_of(exponents), p = rows_of(pre);
    const Tensor w = flat(maybe(weight));
    const int64_t N = weight.size(0), K = weight.size(1);
    const tvdcn_pointwise_desc d{map_dtype(grad.scalar_type(), POINT), (int32_t)act, grad.size(0) * pixels_of(grad), K, N};
    Tensor dx, dw, db;
    if (want[0]) dx = new_map(map_shape(grad, K), grad.options());
    if (want[1]) dw = at::empty({N, K}, grad.options());
    if (want[2]) db = at::empty({N}, grad.options());
    const size_t n = tvdcn_pointwise_conv_backward_workspace_size(&d, has(codes));
    const Tensor work = n ? bytes(grad, n) : Tensor();
    check_status(tvdcn_pointwise_conv_backward(&d, ptr(g), ptr(r), (const int8_t *)ptr(q), (const uint8_t *)ptr(e), ptr(w), ptr(p),
                                               ptr(dx), ptr(dw), ptr(db), ptr(work), n, stream_of(grad)),
                 "pointwise_conv backward");
    return {dx, dw, db};
}

Two point_forward_meta(const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual, int64_t act,
                       bool save_pre) {
    check_pointwise(x, weight, bias, residual, act);
    const auto shape = map_shape(x, weight.size(0));
    return {new_map(shape, x.options()), save_pre ? new_map(shape, x.options().dtype(argument_type(x, act))) : Tensor()};
}
Three point_backward_meta(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents,
                          const Tensor &weight, MaybeTensor pre, int64_t act, std::array<bool, 3> want) {
    check_pointwise_backward(grad, input, codes, exponents, weight, pre, act, want[1]);
    const auto o = grad.options();
    return {want[0] ? new_map(map_shape(grad, weight.size(1)), o) : Tensor(), want[1] ? at::empty(weight.sizes(), o) : Tensor(),
            want[2] ? at::empty({weight.size(0)}, o) : Tensor()};
}

// the activation's argument from what is kept: one beyond float16 is its largest value
Tensor argument(const Tensor &pre, at::ScalarType t) {
    return pre.scalar_type() == at::kHalf ? pre.to(t).clamp(-65504.0, 65504.0) : pre.to(t);
}

Two point_forward_cpu(const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual, int64_t act,
                      bool save_pre) {
    check_pointwise(x, weight, bias, residual, act);
    const auto t = wide_type(x);
    const Tensor y = new_rows(x, weight.size(0), x.options());
    const Tensor rows = to_rows(x).to(t).reshape({-1, x.size(1)});
    Tensor z = rows.mm(weight.to(t).t());
    if (has(bias)) z = z + bias->to(t);
    Tensor v = act_value(z, act);
    if (has(residual)) v = v + to_rows(*residual).to(t).reshape(v.sizes());
    return {to_map(v.to(x.scalar_type()).reshape(y.sizes())),
            save_pre ? to_map(z.to(argument_type(x, act)).reshape(y.sizes())) : Tensor()};
}
Three point_backward_cpu(const Tensor &grad, MaybeTensor input, MaybeTensor codes, MaybeTensor exponents, const Tensor &weight,
                         MaybeTensor pre, int64_t act, std::array<bool, 3> want) {
    check_pointwise_backward(grad, input, codes, exponents, weight, pre, act, want[1]);
    const auto t = wide_type(grad), out = grad.scalar_type();
    const int64_t N = weight.size(0), K = weight.size(1);
    Tensor dz = to_rows(grad).to(t).reshape({-1, N});
    if (act != TVDCN_ACT_NONE) dz = act_slopes(dz, argument(to_rows(*pre), t).reshape({-1, N}), act);
    Tensor dx, dw, db;
    if (want[0]) dx = to_map(dz.mm(weight.to(t)).to(out).reshape(new_rows(grad, K, grad.options()).sizes()));
    if (want[1]) {
        const Tensor x = has(input) ? to_rows(*input) : expand_rows(*codes, *exponents, out);
        dw = dz.t().mm(x.to(t).reshape({-1, K})).to(out);
    }
    if (want[2]) db = dz.sum(0).to(out);
    return {dx, dw, db};
}

// ---------------------------------------------------------------------------
// dispatch, autograd, autocast
// ---------------------------------------------------------------------------
using NormFwd = Two(const Tensor &, int64_t, MaybeTensor, MaybeTensor, double, int64_t);
using NormBwd = Three(const Tensor &, MaybeTensor, MaybeTensor, MaybeTensor, MaybeTensor, MaybeTensor, const Tensor &,
                      int64_t, std::array<bool, 3>);
using PointFwd = Two(const Tensor &, const Tensor &, MaybeTensor, MaybeTensor, int64_t, bool);
using PointBwd = Three(const Tensor &, MaybeTensor, MaybeTensor, MaybeTensor, const Tensor &, MaybeTensor, int64_t,
                       std::array<bool, 3>);

auto &norm_fwd() { static auto op = op_of<NormFwd>("tvdcn::_group_norm_act_forward"); return op; }
auto &norm_bwd() { static auto op = op_of<NormBwd>("tvdcn::_group_norm_act_backward"); return op; }
auto &point_fwd() { static auto op = op_of<PointFwd>("tvdcn::_pointwise_conv_forward"); return op; }
auto &point_bwd() { static auto op = op_of<PointBwd>("tvdcn::_pointwise_conv_backward"); return op; }
auto &compress_op() { static auto op = op_of<Two(const Tensor &)>("tvdcn::compress_activation"); return op; }

class NormFunction : public torch::autograd::Function<NormFunction> {
   public:
    static Tensor forward(AutogradContext *ctx, const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias,
                          double eps, int64_t act, bool keep_int8) {
        at::AutoDispatchBelowADInplaceOrView guard;
        Two r = norm_fwd().call(x, groups, weight, bias, eps, act);
        Tensor input = x, codes, exps;
        if (keep_int8) {
            std::tie(codes, exps) = compress_op().call(x);
            input = Tensor();
        }
        ctx->save_for_backward({input, codes, exps, get(weight), get(bias), std::get<1>(r)});
        ctx->saved_data["act"] = act;
        ctx->saved_data["weight"] = (int64_t)(has(weight) ? 1 : -1);
        ctx->saved_data["bias"] = (int64_t)(has(bias) ? 1 + has(weight) : -1);
        return std::get<0>(r);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g) {
        check_no_tangents(NORM, {g[0]});
        const auto s = ctx->get_saved_variables();
        const std::array<bool, 3> want{ctx->needs_input_grad(0), wanted(ctx, "weight"), wanted(ctx, "bias")};
        Three r;
        {
            at::AutoDispatchBelowADInplaceOrView guard;
            r = norm_bwd().call(g[0], maybe(s[0]), maybe(s[1]), maybe(s[2]), maybe(s[3]), maybe(s[4]), s[5],
                                ctx->saved_data["act"].toInt(), want);
        }
        const variable_list d = with_node(r, {g[0], s[0], s[3], s[4]}, NORM);
        return {d[0], Tensor(), d[1], d[2], Tensor(), Tensor(), Tensor()};
    }
};

class PointFunction : public torch::autograd::Function<PointFunction> {
   public:
    static Tensor forward(AutogradContext *ctx, const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual,
                          int64_t act, bool keep_int8) {
        at::AutoDispatchBelowADInplaceOrView guard;
        // the activation's argument; where y is positive exactly where it is, y serves
        const bool by_y = act == TVDCN_ACT_RELU && !has(residual);
        const bool slope = act != TVDCN_ACT_NONE && (needs(x) || needs(weight) || needs(bias));
        Two r = point_fwd().call(x, weight, bias, residual, act, slope && !by_y);
        const Tensor y = std::get<0>(r), pre = !slope ? Tensor() : by_y ? y : std::get<1>(r);
        Tensor input, codes, exps;   // (only the weight's gradient reads them)
        if (needs(weight)) {
            if (keep_int8) std::tie(codes, exps) = compress_op().call(x);
            else input = x;
        }
        ctx->save_for_backward({input, codes, exps, weight, pre});
        ctx->saved_data["act"] = act;
        ctx->saved_data["bias"] = (int64_t)(has(bias) ? 2 : -1);
        ctx->saved_data["residual"] = (int64_t)(has(residual) ? 2 + has(bias) : -1);
        return y;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g) {
        check_no_tangents(POINT, {g[0]});
        const auto s = ctx->get_saved_variables();
        const std::array<bool, 3> want{ctx->needs_input_grad(0), ctx->needs_input_grad(1), wanted(ctx, "bias")};
        Three r;
        if (want[0] || want[1] || want[2]) {
            at::AutoDispatchBelowADInplaceOrView guard;
            r = point_bwd().call(g[0], maybe(s[0]), maybe(s[1]), maybe(s[2]), s[3], maybe(s[4]),
                                 ctx->saved_data["act"].toInt(), want);
        }
        const variable_list d = with_node(r, {g[0], s[0], s[3], s[4]}, POINT);
        return {d[0], d[1], d[2], wanted(ctx, "residual") ? g[0] : Tensor(), Tensor(), Tensor()};
    }
};

Tensor norm_autograd(const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias, double eps, int64_t act,
                     bool keep_int8) {
    check_no_tangents(NORM, {x, get(weight), get(bias)});
    if (any_grad({x, get(weight), get(bias)})) {
        if (keep_int8)
            TORCH_CHECK(x.scalar_type() != at::kDouble, NORM, ": 8-bit maps of float64 are not supported");
        return NormFunction::apply(x, groups, weight, bias, eps, act, keep_int8);
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    return std::get<0>(norm_fwd().call(x, groups, weight, bias, eps, act));
}
Tensor norm_direct(const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias, double eps, int64_t act, bool) {
    return std::get<0>(norm_fwd().call(x, groups, weight, bias, eps, act));
}
Tensor point_autograd(const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual, int64_t act,
                      bool keep_int8) {
    check_no_tangents(POINT, {x, weight, get(bias), get(residual)});
    if (any_grad({x, weight, get(bias), get(residual)})) {
        if (keep_int8)
            TORCH_CHECK(x.scalar_type() != at::kDouble, POINT, ": 8-bit maps of float64 are not supported");
        return PointFunction::apply(x, weight, bias, residual, act, keep_int8);
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    return std::get<0>(point_fwd().call(x, weight, bias, residual, act, false));
}
Tensor point_direct(const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual, int64_t act, bool) {
    return std::get<0>(point_fwd().call(x, weight, bias, residual, act, false));
}

// autocast: the normalisation keeps the map's type (its sums are float32 whatever that is) and takes its parameters in
// it, rounded where that has 16 bits, as a matrix product's weights are there: parameters have the map's type everywhere. The
// pointwise convolution runs in the autocast type, as torch's matrix products do

Tensor norm_autocast(const Tensor &x, int64_t groups, MaybeTensor weight, MaybeTensor bias, double eps, int64_t act,
                     bool keep_int8) {
    static auto op = op_of<Tensor(const Tensor &, int64_t, MaybeTensor, MaybeTensor, double, int64_t, bool)>("tvdcn::group_norm_act");
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    return op.call(x, groups, cast(x.scalar_type(), weight), cast(x.scalar_type(), bias), eps, act, keep_int8);
}
Tensor point_autocast(const Tensor &x, const Tensor &weight, MaybeTensor bias, MaybeTensor residual, int64_t act,
                      bool keep_int8) {
    static auto op = op_of<Tensor(const Tensor &, const Tensor &, MaybeTensor, MaybeTensor, int64_t, bool)>("tvdcn::pointwise_conv");
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    const auto t = at::autocast::get_autocast_dtype(c10::DeviceType::CUDA);
    return op.call(cast(t, x), cast(t, weight), cast(t, bias), cast(t, residual), act, keep_int8);
}

}  // namespace
}  // namespace tvdcn_amd

TORCH_LIBRARY_FRAGMENT(tvdcn, m) {
    m.def("compress_activation(Tensor input) -> (Tensor, Tensor)");
    m.def("expand_activation(Tensor codes, Tensor exponents, ScalarType dtype) -> Tensor");
    m.def("group_norm_act(Tensor input, int num_groups, Tensor? weight=None, Tensor? bias=None, float eps=1e-05, "
          "int activation=0, bool keep_int8=False) -> Tensor");
    m.def("_group_norm_act_forward(Tensor input, int num_groups, Tensor? weight, Tensor? bias, float eps, "
          "int activation) -> (Tensor, Tensor)");
    m.def("_group_norm_act_backward(Tensor grad, Tensor? input, Tensor? codes, Tensor? exponents, Tensor? weight, "
          "Tensor? bias, Tensor stats, int activation, bool[3] output_mask) -> (Tensor, Tensor, Tensor)");
    m.def("pointwise_conv(Tensor input, Tensor weight, Tensor? bias=None, Tensor? residual=None, int activation=0, "
          "bool keep_int8=False) -> Tensor");
    m.def("_pointwise_conv_forward(Tensor input, Tensor weight, Tensor? bias, Tensor? residual, int activation, "
          "bool save_pre) -> (Tensor, Tensor)");
    m.def("_pointwise_conv_backward(Tensor grad, Tensor? input, Tensor? codes, Tensor? exponents, Tensor weight, "
          "Tensor? pre, int activation, bool[3] output_mask) -> (Tensor, Tensor, Tensor)");
}

#define TVDCN_MAP_IMPLS(SUFFIX)                                                          \
    m.impl("compress_activation", TORCH_FN(tvdcn_amd::compress_##SUFFIX));               \
    m.impl("expand_activation", TORCH_FN(tvdcn_amd::expand_##SUFFIX));                   \
    m.impl("group_norm_act", TORCH_FN(tvdcn_amd::norm_direct));                          \
    m.impl("_group_norm_act_forward", TORCH_FN(tvdcn_amd::norm_forward_##SUFFIX));       \
    m.impl("_group_norm_act_backward", TORCH_FN(tvdcn_amd::norm_backward_##SUFFIX));     \
    m.impl("pointwise_conv", TORCH_FN(tvdcn_amd::point_direct));                         \
    m.impl("_pointwise_conv_forward", TORCH_FN(tvdcn_amd::point_forward_##SUFFIX));      \
    m.impl("_pointwise_conv_backward", TORCH_FN(tvdcn_amd::point_backward_##SUFFIX));

TORCH_LIBRARY_IMPL(tvdcn, CUDA, m) { TVDCN_MAP_IMPLS(hip) }
TORCH_LIBRARY_IMPL(tvdcn, CPU, m) { TVDCN_MAP_IMPLS(cpu) }
TORCH_LIBRARY_IMPL(tvdcn, Meta, m) { TVDCN_MAP_IMPLS(meta) }
TORCH_LIBRARY_IMPL(tvdcn, Autograd, m) {
    m.impl("group_norm_act", TORCH_FN(tvdcn_amd::norm_autograd));
    m.impl("pointwise_conv", TORCH_FN(tvdcn_amd::point_autograd));
}
TORCH_LIBRARY_IMPL(tvdcn, Autocast, m) {
    m.impl("group_norm_act", TORCH_FN(tvdcn_amd::norm_autocast));
    m.impl("pointwise_conv", TORCH_FN(tvdcn_amd::point_autocast));
}
