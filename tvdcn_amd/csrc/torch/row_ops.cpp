// Operators that take the channels of a pixel as one vector: rms_norm, add_rms_norm, their 8-bit forms, quantize_int8,
// dequantize_int8, pointwise_conv_int8 and seeded_dropout, registered in the `tvdcn` namespace with CUDA (= HIP), CPU, Meta,
// Autograd and Autocast kernels, on the maps of map_ops.cpp and by its rules. No counterpart in the reference.
#include <array>
#include <cmath>
#include <tuple>

#include "map_tensors.h"

namespace tvdcn_amd {
namespace {

const char *RMS = "rms_norm", *RMS8 = "rms_norm_int8", *QUANTIZE = "quantize_int8", *DEQUANTIZE = "dequantize_int8",
           *POINT8 = "pointwise_conv_int8", *DROPOUT = "seeded_dropout";
constexpr int64_t kMostSum = 131071;   // channels whose products of codes 32 bits hold the sum of
const double kLeastScale = std::ldexp(1.0, -126), kMostScale = 2.6793883890187504e+36;   // (127 of the latter are finite)
const double kFarScale = std::ldexp(1.0, 96);

// (batch, *size): one value per pixel
std::vector<int64_t> pixel_shape(const Tensor &x) {
    std::vector<int64_t> s{x.size(0)};
    for (int64_t i = 2; i < x.dim(); ++i) s.push_back(x.size(i));
    return s;
}
int64_t rows_in(const Tensor &x) { return x.size(0) * pixels_of(x); }
Tensor floats(const Tensor &t) { return t.defined() ? t.contiguous() : t; }   // (a float's alignment will do)

// ---------------------------------------------------------------------------
// rms_norm, add_rms_norm, and their 8-bit forms
// ---------------------------------------------------------------------------
void check_rms(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps, const char *name) {
    check_map(x, name);
    const float e = (float)eps;
    TORCH_CHECK(std::isnormal(e) && e > 0.f, name, ": eps must be a normal float32 above zero, got ", eps);
    check_like(x, residual, "residual", x.sizes(), name);
    check_like(x, weight, "weight", {x.size(1)}, name);
}
void check_rms8(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps) {
    check_rms(x, residual, weight, eps, RMS8);
    TORCH_CHECK(x.scalar_type() != at::kDouble, RMS8, ": float32, float16 and bfloat16 maps only");
}
void check_rms_backward(const Tensor &grad, MaybeTensor grad_sum, const Tensor &normalised, const Tensor &rstd, MaybeTensor weight) {
    check_map(grad, RMS);
    check_like(grad, maybe(normalised), "normalised rows", grad.sizes(), RMS);
    check_like(grad, grad_sum, "sum's gradient", grad.sizes(), RMS);
    check_like(grad, weight, "weight", {grad.size(1)}, RMS);
    TORCH_CHECK(rstd.sizes() == pixel_shape(grad) && rstd.scalar_type() == wide_type(grad) && rstd.device() == grad.device(), RMS,
                " backward: the statistics are not those of the forward");
}
tvdcn_rms_norm_desc rms_desc(const Tensor &x, double eps, const char *name) {
    return {map_dtype(x.scalar_type(), name), rows_in(x), x.size(1), eps};
}

// y, the sum (where there is a residual) and the reciprocal roots (where asked for)
Three rms_forward_hip(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps, bool save) {
    check_rms(x, residual, weight, eps, RMS);
    c10::DeviceGuard guard(x.device());
    const auto d = rms_desc(x, eps, RMS);
    const Tensor r = rows_of(x), res = rows_of(residual), w = flat(weight);
    Tensor y = new_map(x.sizes(), x.options());
    Tensor sum = has(residual) ? new_map(x.sizes(), x.options()) : Tensor();
    Tensor rstd = save ? new_flat(pixel_shape(x), x.options().dtype(at::kFloat)) : Tensor();
    check_status(tvdcn_rms_norm_forward(&d, ptr(r), ptr(res), ptr(w), ptr(sum), ptr(y), (float *)ptr(rstd), stream_of(x)), RMS);
    return {y, sum, rstd};
}
Two rms_backward_hip(const Tensor &grad, MaybeTensor grad_sum, const Tensor &normalised, const Tensor &rstd, MaybeTensor weight,
                     std::array<bool, 2> want) {
    check_rms_backward(grad, grad_sum, normalised, rstd, weight);
    c10::DeviceGuard guard(grad.device());
    const auto d = rms_desc(grad, 1.0, RMS);
    const Tensor g = rows_of(grad), gs = rows_of(grad_sum), x = rows_of(normalised), w = flat(weight), st = floats(rstd);
    Tensor dx, dw;
    if (want[0]) dx = new_map(grad.sizes(), grad.options());
    if (want[1]) dw = new_flat({grad.size(1)}, grad.options());
    const size_t n = want[1] ? tvdcn_rms_norm_backward_workspace_size(&d) : 0;
    const Tensor work = n ? bytes(grad, n) : Tensor();
    check_status(tvdcn_rms_norm_backward(&d, ptr(g), ptr(gs), ptr(x), (const float *)ptr(st), ptr(w), ptr(dx), ptr(dw), ptr(work), n,
                                         stream_of(grad)),
                 "rms_norm backward");
    return {dx, dw};
}
// codes, scales, the sum
Three rms8_hip(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps) {
    check_rms8(x, residual, weight, eps);
    c10::DeviceGuard guard(x.device());
    const auto d = rms_desc(x, eps, RMS8);
    const Tensor r = rows_of(x), res = rows_of(residual), w = flat(weight);
    Tensor codes = new_map(x.sizes(), x.options().dtype(at::kChar));
    Tensor scales = new_flat(pixel_shape(x), x.options().dtype(at::kFloat));
    Tensor sum = has(residual) ? new_map(x.sizes(), x.options()) : Tensor();
    check_status(tvdcn_rms_norm_int8(&d, ptr(r), ptr(res), ptr(w), ptr(sum), (int8_t *)ptr(codes), (float *)ptr(scales), stream_of(x)),
                 RMS8);
    return {codes, scales, sum};
}

Three rms_forward_meta(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps, bool save) {
    check_rms(x, residual, weight, eps, RMS);
    return {new_map(x.sizes(), x.options()), has(residual) ? new_map(x.sizes(), x.options()) : Tensor(),
            save ? at::empty(pixel_shape(x), x.options().dtype(wide_type(x))) : Tensor()};
}
Two rms_backward_meta(const Tensor &grad, MaybeTensor grad_sum, const Tensor &normalised, const Tensor &rstd, MaybeTensor weight,
                      std::array<bool, 2> want) {
    check_rms_backward(grad, grad_sum, normalised, rstd, weight);
    return {want[0] ? new_map(grad.sizes(), grad.options()) : Tensor(), want[1] ? at::empty({grad.size(1)}, grad.options()) : Tensor()};
}
Three rms8_meta(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps) {
    check_rms8(x, residual, weight, eps);
    return {new_map(x.sizes(), x.options().dtype(at::kChar)), at::empty(pixel_shape(x), x.options().dtype(at::kFloat)),
            has(residual) ? new_map(x.sizes(), x.options()) : Tensor()};
}

// ---- host kernels: [rows, channels] in float32 (float64 for float64 maps) ----
Tensor rows_matrix(const Tensor &x, at::ScalarType t) { return to_rows(x).to(t).reshape({-1, x.size(1)}); }
Tensor rows_to_map(const Tensor &rows, const Tensor &like) { return to_map(rows.reshape(new_rows(like, rows.size(1), rows.options()).sizes())); }
Tensor parameter(MaybeTensor w, int64_t n, const at::TensorOptions &o) { return has(w) ? w->to(o.dtype()) : at::ones({n}, o); }

struct Rms {
    Tensor sum, rows, rstd;   // the map x + residual, its rows, their reciprocal roots [rows, 1]
};
Rms rms_of(const Tensor &x, MaybeTensor residual, double eps) {
    const auto t = wide_type(x);
    Rms k;
    if (has(residual)) {
        const Tensor s = (rows_matrix(x, t) + rows_matrix(*residual, t)).to(x.scalar_type());
        k.sum = rows_to_map(s, x);
        k.rows = s.to(t);
    } else {
        k.rows = rows_matrix(x, t);
    }
    // (squares beyond float32 fit float64)
    k.rstd = at::rsqrt(k.rows.to(at::kDouble).square().mean(at::IntArrayRef({1}), true) + eps).to(t);
    return k;
}
Three rms_forward_cpu(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps, bool save) {
    check_rms(x, residual, weight, eps, RMS);
    if (x.numel() == 0) return rms_forward_meta(x, residual, weight, eps, save);   // (empty tensors of x's device)
    const Rms k = rms_of(x, residual, eps);
    const Tensor y = (k.rows * k.rstd * parameter(weight, x.size(1), k.rows.options())).to(x.scalar_type());
    return {rows_to_map(y, x), k.sum, save ? k.rstd.reshape(pixel_shape(x)) : Tensor()};
}
Two rms_backward_cpu(const Tensor &grad, MaybeTensor grad_sum, const Tensor &normalised, const Tensor &rstd, MaybeTensor weight,
                     std::array<bool, 2> want) {
    check_rms_backward(grad, grad_sum, normalised, rstd, weight);
    const auto t = wide_type(grad), out = grad.scalar_type();
    const int64_t C = grad.size(1);
    if (grad.numel() == 0)
        return {want[0] ? new_map(grad.sizes(), grad.options()) : Tensor(), want[1] ? at::zeros({C}, grad.options()) : Tensor()};
    const Tensor dy = rows_matrix(grad, t), rs = rstd.reshape({-1, 1}), h = rows_matrix(normalised, t) * rs;
    Tensor dx, dw;
    if (want[0]) {
        const Tensor dh = dy * parameter(weight, C, dy.options());
        Tensor d = rs * (dh - h * (dh * h).mean(at::IntArrayRef({1}), true));
        if (has(grad_sum)) d = d + rows_matrix(*grad_sum, t);
        dx = rows_to_map(d.to(out), grad);
    }
    if (want[1]) dw = (dy * h).sum(0).to(out);
    return {dx, dw};
}

// codes [rows, channels] and scales [rows] of float32 rows
Two codes_of(const Tensor &rows) {
    const Tensor big = rows.abs().amax(1), bad = big.isfinite().logical_not();
    // (the scale is a float32; the quotients, in float64, are rounded as exact ones would be)
    const Tensor scales = (big * (1.0f / 127.0f)).clamp(kLeastScale, kMostScale).masked_fill(bad, 1.0);
    const Tensor q = at::round(rows.to(at::kDouble) / scales.to(at::kDouble).unsqueeze(1)).masked_fill(bad.unsqueeze(1), 0.0);
    return {q.to(at::kChar), scales.masked_fill(bad, NAN)};
}
Three rms8_cpu(const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps) {
    check_rms8(x, residual, weight, eps);
    if (x.numel() == 0) return rms8_meta(x, residual, weight, eps);
    const Rms k = rms_of(x, residual, eps);
    const Two q = codes_of(k.rows * k.rstd * parameter(weight, x.size(1), k.rows.options()));
    return {rows_to_map(std::get<0>(q), x), std::get<1>(q).reshape(pixel_shape(x)), k.sum};
}

// ---------------------------------------------------------------------------
// quantize_int8 / dequantize_int8
// ---------------------------------------------------------------------------
void check_quantize(const Tensor &x) {
    check_map(x, QUANTIZE);
    TORCH_CHECK(x.scalar_type() != at::kDouble, QUANTIZE, ": float32, float16 and bfloat16 maps only");
}
void check_codes(const Tensor &codes, const Tensor &scales, const char *name, const char *what = "") {
    TORCH_CHECK(codes.dim() >= 2 && codes.scalar_type() == at::kChar && codes.size(1) > 0, name, ": expected int8 ", what,
                "codes of shape (batch, channels, *size), got ", codes.scalar_type(), " ", codes.sizes());
    TORCH_CHECK(scales.scalar_type() == at::kFloat && scales.sizes() == pixel_shape(codes), name, ": expected float32 ", what,
                "scales of shape ", pixel_shape(codes), ", got ", scales.scalar_type(), " ", scales.sizes());
    TORCH_CHECK(codes.device() == scales.device(), name, ": expected all tensors on ", codes.device(), ", but ", what,
                "scales is on ", scales.device());
}
void check_out_type(at::ScalarType dtype, const char *name) {
    TORCH_CHECK(dtype == at::kFloat || dtype == at::kHalf || dtype == at::kBFloat16, name,
                ": float32, float16 and bfloat16 maps only, got ", dtype);
}
void check_dequantize(const Tensor &codes, const Tensor &scales, at::ScalarType dtype) {
    check_codes(codes, scales, DEQUANTIZE);
    check_out_type(dtype, DEQUANTIZE);
}

Two quantize_hip(const Tensor &x) {
    check_quantize(x);
    c10::DeviceGuard guard(x.device());
    const Tensor r = rows_of(x);
    Tensor codes = new_map(x.sizes(), x.options().dtype(at::kChar));
    Tensor scales = new_flat(pixel_shape(x), x.options().dtype(at::kFloat));
    check_status(tvdcn_quantize_int8(map_dtype(x.scalar_type(), QUANTIZE), rows_in(x), x.size(1), ptr(r), (int8_t *)ptr(codes),
                                     (float *)ptr(scales), stream_of(x)),
                 QUANTIZE);
    return {codes, scales};
}
Tensor dequantize_hip(const Tensor &codes, const Tensor &scales, at::ScalarType dtype) {
    check_dequantize(codes, scales, dtype);
    c10::DeviceGuard guard(codes.device());
    const Tensor q = rows_of(codes), s = floats(scales);
    Tensor y = new_map(codes.sizes(), codes.options().dtype(dtype));
    check_status(tvdcn_dequantize_int8(map_dtype(dtype, DEQUANTIZE), rows_in(codes), codes.size(1), (const int8_t *)ptr(q),
                                       (const float *)ptr(s), ptr(y), stream_of(codes)),
                 DEQUANTIZE);
    return y;
}
Two quantize_meta(const Tensor &x) {
    check_quantize(x);
    return {new_map(x.sizes(), x.options().dtype(at::kChar)), at::empty(pixel_shape(x), x.options().dtype(at::kFloat))};
}
Tensor dequantize_meta(const Tensor &codes, const Tensor &scales, at::ScalarType dtype) {
    check_dequantize(codes, scales, dtype);
    return new_map(codes.sizes(), codes.options().dtype(dtype));
}
Two quantize_cpu(const Tensor &x) {
    if (x.numel() == 0) return quantize_meta(x);
    check_quantize(x);
    const Two q = codes_of(rows_matrix(x, at::kFloat));
    return {rows_to_map(std::get<0>(q), x), std::get<1>(q).reshape(pixel_shape(x))};
}
Tensor dequantize_cpu(const Tensor &codes, const Tensor &scales, at::ScalarType dtype) {
    if (codes.numel() == 0) return dequantize_meta(codes, scales, dtype);
    check_dequantize(codes, scales, dtype);
    return rows_to_map((rows_matrix(codes, at::kFloat) * scales.reshape({-1, 1})).to(dtype), codes);
}

// ---------------------------------------------------------------------------
// pointwise_conv_int8
// ---------------------------------------------------------------------------
void check_point8(const Tensor &codes, const Tensor &scales, const Tensor &wcodes, const Tensor &wscales, MaybeTensor bias,
                  MaybeTensor residual, int64_t activation, at::ScalarType dtype) {
    check_codes(codes, scales, POINT8);
    TORCH_CHECK(wcodes.dim() == 2 && wcodes.size(0) > 0, POINT8, ": expected weight codes of shape (out_channels, in_channels), got ",
                wcodes.sizes());
    check_codes(wcodes, wscales, POINT8, "weight ");
    TORCH_CHECK(wcodes.size(1) == codes.size(1), POINT8, ": expected a weight for ", codes.size(1), " input channels, got ", wcodes.sizes());
    TORCH_CHECK(wcodes.device() == codes.device(), POINT8, ": expected all tensors on ", codes.device(), ", but weight codes is on ",
                wcodes.device());
    TORCH_CHECK(codes.size(1) <= kMostSum, POINT8, ": more than ", kMostSum, " input channels");
    check_activation(activation, POINT8);
    check_out_type(dtype, POINT8);
    auto check_as_out = [&](MaybeTensor t, const char *what, at::IntArrayRef sizes) {
        if (!has(t)) return;
        TORCH_CHECK(t->sizes() == sizes, POINT8, ": expected ", what, " of shape ", sizes, ", got ", t->sizes());
        TORCH_CHECK(t->scalar_type() == dtype, POINT8, ": expected ", what, " of dtype ", dtype, ", got ", t->scalar_type());
        TORCH_CHECK(t->device() == codes.device(), POINT8, ": expected all tensors on ", codes.device(), ", but ", what, " is on ",
                    t->device());
    };
    check_as_out(bias, "bias", {wcodes.size(0)});
    check_as_out(residual, "residual", map_shape(codes, wcodes.size(0)));
}

Tensor point8_hip(const Tensor &codes, const Tensor &scales, const Tensor &wcodes, const Tensor &wscales, MaybeTensor bias,
                  MaybeTensor residual, int64_t act, at::ScalarType dtype) {
    check_point8(codes, scales, wcodes, wscales, bias, residual, act, dtype);
    c10::DeviceGuard guard(codes.device());
    const Tensor q = rows_of(codes), s = floats(scales), wq = flat(maybe(wcodes)), ws = floats(wscales), b = flat(bias), r = rows_of(residual);
    const int64_t N = wcodes.size(0);
    const tvdcn_pointwise_desc d{map_dtype(dtype, POINT8), (int32_t)act, rows_in(codes), codes.size(1), N};
    Tensor y = new_map(map_shape(codes, N), codes.options().dtype(dtype));
    const size_t n = tvdcn_pointwise_conv_int8_workspace_size(&d);
    const Tensor work = n ? bytes(codes, n) : Tensor();
    check_status(tvdcn_pointwise_conv_int8(&d, (const int8_t *)ptr(q), (const float *)ptr(s), (const int8_t *)ptr(wq),
                                           (const float *)ptr(ws), ptr(b), ptr(r), ptr(y), ptr(work), n, stream_of(codes)),
                 POINT8);
    return y;
}
Tensor point8_meta(const Tensor &codes, const Tensor &scales, const Tensor &wcodes, const Tensor &wscales, MaybeTensor bias,
                   MaybeTensor residual, int64_t act, at::ScalarType dtype) {
    check_point8(codes, scales, wcodes, wscales, bias, residual, act, dtype);
    return new_map(map_shape(codes, wcodes.size(0)), codes.options().dtype(dtype));
}
Tensor point8_cpu(const Tensor &codes, const Tensor &scales, const Tensor &wcodes, const Tensor &wscales, MaybeTensor bias,
                  MaybeTensor residual, int64_t act, at::ScalarType dtype) {
    check_point8(codes, scales, wcodes, wscales, bias, residual, act, dtype);
    if (codes.numel() == 0) return point8_meta(codes, scales, wcodes, wscales, bias, residual, act, dtype);
    // (the whole sums are exact in float64)
    const Tensor sums = rows_matrix(codes, at::kDouble).mm(wcodes.to(at::kDouble).t()).to(at::kFloat);
    // (a row's scale beyond 2^96 comes last: up to that its product with the sum, below 2^31, is a float32)
    const Tensor sr = scales.reshape({-1, 1}), far = sr.abs() > kFarScale;
    Tensor z = far.any().item<bool>() ? at::where(far, sums * wscales * sr, sums * sr * wscales) : sums * sr * wscales;
    if (has(bias)) z = z + bias->to(at::kFloat);
    z = act_value(z, act);
    if (has(residual)) z = z + rows_matrix(*residual, at::kFloat);
    return rows_to_map(z.to(dtype), codes);
}

// ---------------------------------------------------------------------------
// seeded_dropout
// ---------------------------------------------------------------------------
void check_dropout(const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) {
    check_map(x, DROPOUT);
    TORCH_CHECK(p >= 0.0 && p <= 1.0, DROPOUT, ": p must be in [0, 1], got ", p);
    TORCH_CHECK(seed.scalar_type() == at::kLong && seed.numel() == 1, DROPOUT, ": expected an int64 seed of one element, got ",
                seed.scalar_type(), " ", seed.sizes());
    TORCH_CHECK(seed.device() == x.device(), DROPOUT, ": expected all tensors on ", x.device(), ", but seed is on ", seed.device());
    check_like(x, residual, "residual", x.sizes(), DROPOUT);
}
Tensor dropout_hip(const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) {
    check_dropout(x, p, seed, residual);
    c10::DeviceGuard guard(x.device());
    const Tensor r = rows_of(x), res = rows_of(residual);
    Tensor y = new_map(x.sizes(), x.options());
    check_status(tvdcn_seeded_dropout(map_dtype(x.scalar_type(), DROPOUT), x.numel(), p, seed.data_ptr<int64_t>(), ptr(r), ptr(res),
                                      ptr(y), stream_of(x)),
                 DROPOUT);
    return y;
}
Tensor dropout_meta(const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) {
    check_dropout(x, p, seed, residual);
    return new_map(x.sizes(), x.options());
}
// The four words of Philox4x32-10 at a counter of 64 bits
std::array<uint32_t, 4> philox(uint64_t counter, uint64_t seed) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0, k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
    for (int i = 0; i < 10; ++i, k0 += 0x9E3779B9u, k1 += 0xBB67AE85u) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0, c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1, c3 = (uint32_t)a;
    }
    return {c0, c1, c2, c3};
}
Tensor dropout_cpu(const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) {
    check_dropout(x, p, seed, residual);
    if (x.numel() == 0) return dropout_meta(x, p, seed, residual);
    const auto t = wide_type(x);
    const Tensor rows = to_rows(x);
    const int64_t n = x.numel();
    const uint64_t key = (uint64_t)seed.reshape({-1}).data_ptr<int64_t>()[0];
    const uint32_t drop = (uint32_t)std::nearbyint(p * 65536.0);
    Tensor kept = at::empty(rows.sizes(), rows.options().dtype(at::kBool));
    bool *k = kept.data_ptr<bool>();
    for (int64_t g = 0; g * 8 < n; ++g) {
        const auto words = philox((uint64_t)g, key);
        for (int64_t e = 0; e < 8 && g * 8 + e < n; ++e) k[g * 8 + e] = (words[e / 2] >> (16 * (e % 2)) & 0xffffu) >= drop;
    }
    const double scale = drop < 65536 ? 65536.0 / (65536 - drop) : 0.0;
    Tensor v = (rows.to(t) * scale).masked_fill(kept.logical_not(), 0.0);
    if (has(residual)) v = v + to_rows(*residual).to(t);
    return to_map(v.to(x.scalar_type()));
}

// ---------------------------------------------------------------------------
// dispatch, autograd, autocast
// ---------------------------------------------------------------------------
using RmsFwd = Three(const Tensor &, MaybeTensor, MaybeTensor, double, bool);
using RmsBwd = Two(const Tensor &, MaybeTensor, const Tensor &, const Tensor &, MaybeTensor, std::array<bool, 2>);
using Rms8 = Three(const Tensor &, MaybeTensor, MaybeTensor, double);
using Point8 = Tensor(const Tensor &, const Tensor &, const Tensor &, const Tensor &, MaybeTensor, MaybeTensor, int64_t, at::ScalarType);
using Dropout = Tensor(const Tensor &, double, const Tensor &, MaybeTensor);

auto &rms_fwd() { static auto op = op_of<RmsFwd>("tvdcn::_rms_norm_forward"); return op; }
auto &rms_bwd() { static auto op = op_of<RmsBwd>("tvdcn::_rms_norm_backward"); return op; }
auto &rms8_op() { static auto op = op_of<Rms8>("tvdcn::_rms_norm_int8"); return op; }
auto &quantize_op() { static auto op = op_of<Two(const Tensor &)>("tvdcn::quantize_int8"); return op; }
auto &dequantize_op() { static auto op = op_of<Tensor(const Tensor &, const Tensor &, at::ScalarType)>("tvdcn::dequantize_int8"); return op; }
auto &point8_op() { static auto op = op_of<Point8>("tvdcn::pointwise_conv_int8"); return op; }
auto &dropout_op() { static auto op = op_of<Dropout>("tvdcn::_seeded_dropout"); return op; }

class RmsFunction : public torch::autograd::Function<RmsFunction> {
   public:
    static variable_list forward(AutogradContext *ctx, const Tensor &x, MaybeTensor residual, MaybeTensor weight, double eps) {
        at::AutoDispatchBelowADInplaceOrView guard;
        const Three r = rms_fwd().call(x, residual, weight, eps, true);
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({has(residual) ? std::get<1>(r) : x, std::get<2>(r), get(weight)});
        ctx->saved_data["residual"] = (int64_t)(has(residual) ? 1 : -1);
        ctx->saved_data["weight"] = (int64_t)(has(weight) ? 1 + has(residual) : -1);
        if (!has(residual)) return {std::get<0>(r)};
        if (!needs(x) && !needs(residual)) ctx->mark_non_differentiable({std::get<1>(r)});   // (the sum does not know the weight)
        return {std::get<0>(r), std::get<1>(r)};
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &g) {
        const Tensor gy = g[0], gs = g.size() > 1 ? g[1] : Tensor();
        check_no_tangents(RMS, {gy, gs});
        const auto s = ctx->get_saved_variables();
        const bool added = ctx->saved_data["residual"].toInt() >= 0;
        const std::array<bool, 2> want{ctx->needs_input_grad(0) || wanted(ctx, "residual"), wanted(ctx, "weight")};
        Tensor dx = gs, dw;   // (a gradient of the sum alone goes through)
        if (gy.defined() && (want[0] || want[1])) {
            Two r;
            {
                at::AutoDispatchBelowADInplaceOrView guard;
                r = rms_bwd().call(gy, maybe(gs), s[0], s[1], maybe(s[2]), want);
            }
            const variable_list d = with_node({std::get<0>(r), std::get<1>(r), Tensor()}, {gy, gs, s[0], s[2]}, RMS);
            dx = d[0], dw = d[1];
        }
        const Tensor none;
        return {ctx->needs_input_grad(0) ? dx : none, added && wanted(ctx, "residual") ? dx : none, dw, none};
    }
};

class DropoutFunction : public torch::autograd::Function<DropoutFunction> {
   public:
    static Tensor forward(AutogradContext *ctx, const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) {
        at::AutoDispatchBelowADInplaceOrView guard;
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({seed});
        ctx->saved_data["p"] = p;
        ctx->saved_data["residual"] = (int64_t)(has(residual) ? 2 : -1);
        return dropout_op().call(x, p, seed, residual);
    }
    // linear in the gradient: the operator itself, differentiable again
    static variable_list backward(AutogradContext *ctx, const variable_list &g) {
        check_no_tangents(DROPOUT, {g[0]});
        const Tensor none;
        if (!g[0].defined()) return {none, none, none, none};
        Tensor dx;
        if (ctx->needs_input_grad(0)) {
            const auto s = ctx->get_saved_variables();
            const double p = ctx->saved_data["p"].toDouble();
            if (any_grad({g[0]})) {   // (a graph of the backward is made)
                static auto op = op_of<Dropout>("tvdcn::seeded_dropout");
                dx = op.call(g[0], p, s[0], {});
            } else {
                at::AutoDispatchBelowADInplaceOrView guard;
                dx = dropout_op().call(g[0], p, s[0], {});
            }
        }
        return {dx, none, none, wanted(ctx, "residual") ? g[0] : none};
    }
};

Tensor rms_autograd(const Tensor &x, MaybeTensor weight, double eps) {
    check_no_tangents(RMS, {x, get(weight)});
    if (any_grad({x, get(weight)})) return RmsFunction::apply(x, optional<Tensor>(), weight, eps)[0];
    at::AutoDispatchBelowADInplaceOrView guard;
    return std::get<0>(rms_fwd().call(x, {}, weight, eps, false));
}
Two add_rms_autograd(const Tensor &x, const Tensor &residual, MaybeTensor weight, double eps) {
    check_no_tangents(RMS, {x, residual, get(weight)});
    if (any_grad({x, residual, get(weight)})) {
        const variable_list r = RmsFunction::apply(x, optional<Tensor>(residual), weight, eps);
        return {r[0], r[1]};
    }
    at::AutoDispatchBelowADInplaceOrView guard;
    const Three r = rms_fwd().call(x, residual, weight, eps, false);
    return {std::get<0>(r), std::get<1>(r)};
}
Tensor rms_direct(const Tensor &x, MaybeTensor weight, double eps) { return std::get<0>(rms_fwd().call(x, {}, weight, eps, false)); }
Two add_rms_direct(const Tensor &x, const Tensor &residual, MaybeTensor weight, double eps) {
    const Three r = rms_fwd().call(x, residual, weight, eps, false);
    return {std::get<0>(r), std::get<1>(r)};
}
Two rms8_direct(const Tensor &x, MaybeTensor weight, double eps) {
    const Three r = rms8_op().call(x, {}, weight, eps);
    return {std::get<0>(r), std::get<1>(r)};
}
Three add_rms8_direct(const Tensor &x, const Tensor &residual, MaybeTensor weight, double eps) {
    return rms8_op().call(x, residual, weight, eps);
}
Tensor dropout_autograd(const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) {
    check_no_tangents(DROPOUT, {x, get(residual)});
    if (any_grad({x, get(residual)})) return DropoutFunction::apply(x, p, seed, residual);
    at::AutoDispatchBelowADInplaceOrView guard;
    return dropout_op().call(x, p, seed, residual);
}
Tensor dropout_direct(const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) { return dropout_op().call(x, p, seed, residual); }

// Rounding to 8 bits has no gradient: a call that would lose one is refused
void check_no_grad(const char *name, std::initializer_list<Tensor> ts) {
    check_no_tangents(name, ts);
    TORCH_CHECK(!any_grad(ts), name, ": has no gradient; call it under torch.no_grad() or with inputs that require none");
}
Two rms8_autograd(const Tensor &x, MaybeTensor weight, double eps) {
    check_no_grad(RMS8, {x, get(weight)});
    at::AutoDispatchBelowADInplaceOrView guard;
    return rms8_direct(x, weight, eps);
}
Three add_rms8_autograd(const Tensor &x, const Tensor &residual, MaybeTensor weight, double eps) {
    check_no_grad(RMS8, {x, residual, get(weight)});
    at::AutoDispatchBelowADInplaceOrView guard;
    return add_rms8_direct(x, residual, weight, eps);
}
Two quantize_autograd(const Tensor &x) {
    check_no_grad(QUANTIZE, {x});
    at::AutoDispatchBelowADInplaceOrView guard;
    return quantize_op().call(x);
}
Tensor dequantize_autograd(const Tensor &codes, const Tensor &scales, at::ScalarType dtype) {
    check_no_grad(DEQUANTIZE, {scales});
    at::AutoDispatchBelowADInplaceOrView guard;
    return dequantize_op().call(codes, scales, dtype);
}
Tensor point8_autograd(const Tensor &codes, const Tensor &scales, const Tensor &wcodes, const Tensor &wscales, MaybeTensor bias,
                       MaybeTensor residual, int64_t act, at::ScalarType dtype) {
    check_no_grad(POINT8, {scales, wscales, get(bias), get(residual)});
    at::AutoDispatchBelowADInplaceOrView guard;
    return point8_op().call(codes, scales, wcodes, wscales, bias, residual, act, dtype);
}

// autocast: a map and its shortcut in the wider type of the two, as torch's sums take theirs; parameters in that, as the other
// normalisation's; what goes into an 8-bit product's result in that result's type
at::ScalarType wider(const Tensor &x, MaybeTensor r) { return has(r) ? at::promote_types(x.scalar_type(), r->scalar_type()) : x.scalar_type(); }

Tensor rms_autocast(const Tensor &x, MaybeTensor weight, double eps) {
    static auto op = op_of<Tensor(const Tensor &, MaybeTensor, double)>("tvdcn::rms_norm");
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    return op.call(x, cast(x.scalar_type(), weight), eps);
}
Two add_rms_autocast(const Tensor &x, const Tensor &residual, MaybeTensor weight, double eps) {
    static auto op = op_of<Two(const Tensor &, const Tensor &, MaybeTensor, double)>("tvdcn::add_rms_norm");
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    const auto t = wider(x, residual);
    return op.call(cast(t, x), cast(t, residual), cast(t, weight), eps);
}
Two rms8_autocast(const Tensor &x, MaybeTensor weight, double eps) {
    static auto op = op_of<Two(const Tensor &, MaybeTensor, double)>("tvdcn::rms_norm_int8");
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    return op.call(x, cast(x.scalar_type(), weight), eps);
}
Three add_rms8_autocast(const Tensor &x, const Tensor &residual, MaybeTensor weight, double eps) {
    static auto op = op_of<Three(const Tensor &, const Tensor &, MaybeTensor, double)>("tvdcn::add_rms_norm_int8");
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    const auto t = wider(x, residual);
    return op.call(cast(t, x), cast(t, residual), cast(t, weight), eps);
}
Tensor point8_autocast(const Tensor &codes, const Tensor &scales, const Tensor &wcodes, const Tensor &wscales, MaybeTensor bias,
                       MaybeTensor residual, int64_t act, at::ScalarType dtype) {
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    return point8_op().call(codes, scales, wcodes, wscales, cast(dtype, bias), cast(dtype, residual), act, dtype);
}
Tensor dropout_autocast(const Tensor &x, double p, const Tensor &seed, MaybeTensor residual) {
    static auto op = op_of<Dropout>("tvdcn::seeded_dropout");
    c10::impl::ExcludeDispatchKeyGuard no_autocast(c10::DispatchKey::Autocast);
    const auto t = wider(x, residual);
    return op.call(cast(t, x), p, seed, cast(t, residual));
}

}  // namespace
}  // namespace tvdcn_amd

TORCH_LIBRARY_FRAGMENT(tvdcn, m) {
    m.def("rms_norm(Tensor input, Tensor? weight=None, float eps=1e-06) -> Tensor");
    m.def("add_rms_norm(Tensor input, Tensor residual, Tensor? weight=None, float eps=1e-06) -> (Tensor, Tensor)");
    m.def("_rms_norm_forward(Tensor input, Tensor? residual, Tensor? weight, float eps, bool save_rstd) -> (Tensor, Tensor, Tensor)");
    m.def("_rms_norm_backward(Tensor grad, Tensor? grad_sum, Tensor normalised, Tensor rstd, Tensor? weight, bool[2] output_mask) "
          "-> (Tensor, Tensor)");
    m.def("rms_norm_int8(Tensor input, Tensor? weight=None, float eps=1e-06) -> (Tensor, Tensor)");
    m.def("add_rms_norm_int8(Tensor input, Tensor residual, Tensor? weight=None, float eps=1e-06) -> (Tensor, Tensor, Tensor)");
    m.def("_rms_norm_int8(Tensor input, Tensor? residual, Tensor? weight, float eps) -> (Tensor, Tensor, Tensor)");
    m.def("quantize_int8(Tensor input) -> (Tensor, Tensor)");
    m.def("dequantize_int8(Tensor codes, Tensor scales, ScalarType dtype) -> Tensor");
    m.def("pointwise_conv_int8(Tensor codes, Tensor scales, Tensor weight_codes, Tensor weight_scales, Tensor? bias, "
          "Tensor? residual, int activation, ScalarType dtype) -> Tensor");
    m.def("seeded_dropout(Tensor input, float p, Tensor seed, Tensor? residual=None) -> Tensor");
    m.def("_seeded_dropout(Tensor input, float p, Tensor seed, Tensor? residual) -> Tensor");
}

#define TVDCN_ROW_IMPLS(SUFFIX)                                                  \
    m.impl("rms_norm", TORCH_FN(tvdcn_amd::rms_direct));                         \
    m.impl("add_rms_norm", TORCH_FN(tvdcn_amd::add_rms_direct));                 \
    m.impl("_rms_norm_forward", TORCH_FN(tvdcn_amd::rms_forward_##SUFFIX));      \
    m.impl("_rms_norm_backward", TORCH_FN(tvdcn_amd::rms_backward_##SUFFIX));    \
    m.impl("rms_norm_int8", TORCH_FN(tvdcn_amd::rms8_direct));                   \
    m.impl("add_rms_norm_int8", TORCH_FN(tvdcn_amd::add_rms8_direct));           \
    m.impl("_rms_norm_int8", TORCH_FN(tvdcn_amd::rms8_##SUFFIX));                \
    m.impl("quantize_int8", TORCH_FN(tvdcn_amd::quantize_##SUFFIX));             \
    m.impl("dequantize_int8", TORCH_FN(tvdcn_amd::dequantize_##SUFFIX));         \
    m.impl("pointwise_conv_int8", TORCH_FN(tvdcn_amd::point8_##SUFFIX));         \
    m.impl("seeded_dropout", TORCH_FN(tvdcn_amd::dropout_direct));               \
    m.impl("_seeded_dropout", TORCH_FN(tvdcn_amd::dropout_##SUFFIX));

TORCH_LIBRARY_IMPL(tvdcn, CUDA, m) { TVDCN_ROW_IMPLS(hip) }
TORCH_LIBRARY_IMPL(tvdcn, CPU, m) { TVDCN_ROW_IMPLS(cpu) }
TORCH_LIBRARY_IMPL(tvdcn, Meta, m) { TVDCN_ROW_IMPLS(meta) }
TORCH_LIBRARY_IMPL(tvdcn, Autograd, m) {
    m.impl("rms_norm", TORCH_FN(tvdcn_amd::rms_autograd));
    m.impl("add_rms_norm", TORCH_FN(tvdcn_amd::add_rms_autograd));
    m.impl("rms_norm_int8", TORCH_FN(tvdcn_amd::rms8_autograd));
    m.impl("add_rms_norm_int8", TORCH_FN(tvdcn_amd::add_rms8_autograd));
    m.impl("quantize_int8", TORCH_FN(tvdcn_amd::quantize_autograd));
    m.impl("dequantize_int8", TORCH_FN(tvdcn_amd::dequantize_autograd));
    m.impl("pointwise_conv_int8", TORCH_FN(tvdcn_amd::point8_autograd));
    m.impl("seeded_dropout", TORCH_FN(tvdcn_amd::dropout_autograd));
}
TORCH_LIBRARY_IMPL(tvdcn, Autocast, m) {
    m.impl("rms_norm", TORCH_FN(tvdcn_amd::rms_autocast));
    m.impl("add_rms_norm", TORCH_FN(tvdcn_amd::add_rms_autocast));
    m.impl("rms_norm_int8", TORCH_FN(tvdcn_amd::rms8_autocast));
    m.impl("add_rms_norm_int8", TORCH_FN(tvdcn_amd::add_rms8_autocast));
    m.impl("pointwise_conv_int8", TORCH_FN(tvdcn_amd::point8_autocast));
    m.impl("seeded_dropout", TORCH_FN(tvdcn_amd::dropout_autocast));
}
