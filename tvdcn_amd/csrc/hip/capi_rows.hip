// C ABI of the operators that take a row as one vector (declared in include/tvdcn_hip.h): checks of the arguments, the
// workspace, and the launches on the caller's stream. Host-side only: no allocation, no synchronisation.
#include <climits>
#include <cmath>

#include "capi_checks.h"
#include "rows.h"

using namespace tvdcn_hip;

namespace {

constexpr const char *NORM = "rms_norm", *NORM8 = "rms_norm_int8", *QUANTIZE = "quantize_int8", *DEQUANTIZE = "dequantize_int8",
                     *POINT8 = "pointwise_conv_int8", *DROPOUT = "seeded_dropout";
constexpr int64_t MOST_SUM = 131071;   // products of 8-bit codes whose sum fits 32 bits

tvdcn_status norm_args(const char *what, const tvdcn_rms_norm_desc *d) {
    if (!d) return invalid("null descriptor");
    RETURN_IF(check_type(what, d->dtype));
    RETURN_IF(check_map(what, d->rows, d->channels));
    const float eps = (float)d->eps;
    if (!std::isnormal(eps) || eps < 0.f) return invalid(std::string(what) + ": eps must be a normal float32 above zero");
    return TVDCN_STATUS_SUCCESS;
}

tvdcn_status point_args(const tvdcn_pointwise_desc *d, Int8ProductArgs &a) {
    if (!d) return invalid("null descriptor");
    RETURN_IF(check_type(POINT8, d->dtype, d->activation));
    RETURN_IF(check_map(POINT8, d->rows, d->in_channels));
    RETURN_IF(check_map(POINT8, d->rows, d->out_channels));
    if (d->in_channels > MOST_SUM) return api_fail(TVDCN_STATUS_NOT_SUPPORTED, "pointwise_conv_int8: more than 131071 input channels");
    if (d->in_channels * d->out_channels > INT_MAX) return api_fail(TVDCN_STATUS_NOT_SUPPORTED, "pointwise_conv_int8: weight too large");
    a = Int8ProductArgs{};
    a.dtype = d->dtype;
    a.act = d->activation;
    a.rows = d->rows;
    a.in = (int)d->in_channels;
    a.out = (int)d->out_channels;
    return TVDCN_STATUS_SUCCESS;
}

RowArgs row_args(int32_t dtype, int64_t rows, int64_t channels) {
    RowArgs a{};
    a.dtype = dtype;
    a.rows = rows;
    a.channels = (int)channels;
    return a;
}

}  // namespace

extern "C" {

tvdcn_status tvdcn_rms_norm_forward(const tvdcn_rms_norm_desc *desc, const void *input, const void *residual,
                                    const void *weight, void *sum, void *output, float *rstd, void *stream) {
    RETURN_IF(norm_args(NORM, desc));
    api_clear_error();
    if (desc->rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(NORM, {input, output}, {residual, weight, sum}));
    RETURN_IF(check_floats({rstd}));
    if ((residual != nullptr) != (sum != nullptr)) return invalid("rms_norm: a residual and its sum go together");
    RowArgs a = row_args(desc->dtype, desc->rows, desc->channels);
    a.eps = (float)desc->eps;
    a.x = input;
    a.residual = residual;
    a.weight = weight;
    a.sum = sum;
    a.y = output;
    a.rstd = rstd;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_RMS_NORM, s, [&] { return launch_rms_norm(a, s); });
}

tvdcn_status tvdcn_rms_norm_int8(const tvdcn_rms_norm_desc *desc, const void *input, const void *residual,
                                 const void *weight, void *sum, int8_t *codes, float *scales, void *stream) {
    RETURN_IF(norm_args(NORM8, desc));
    api_clear_error();
    if (desc->rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(NORM8, {input, codes}, {residual, weight, sum}));
    if (!scales) return invalid("rms_norm_int8: null tensor");
    RETURN_IF(check_floats({scales}));
    if ((residual != nullptr) != (sum != nullptr)) return invalid("rms_norm_int8: a residual and its sum go together");
    RowArgs a = row_args(desc->dtype, desc->rows, desc->channels);
    a.eps = (float)desc->eps;
    a.x = input;
    a.residual = residual;
    a.weight = weight;
    a.sum = sum;
    a.codes = codes;
    a.scales = scales;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_RMS_NORM, s, [&] { return launch_rms_norm_int8(a, s); });
}

size_t tvdcn_rms_norm_backward_workspace_size(const tvdcn_rms_norm_desc *desc) {
    if (norm_args(NORM, desc)) return 0;
    RowGradArgs a{};
    a.dtype = desc->dtype;
    a.rows = desc->rows;
    a.channels = (int)desc->channels;
    return (size_t)rms_norm_part_floats(a) * 4;
}

tvdcn_status tvdcn_rms_norm_backward(const tvdcn_rms_norm_desc *desc, const void *grad_out, const void *grad_sum,
                                     const void *normalised, const float *rstd, const void *weight, void *grad_input,
                                     void *grad_weight, void *workspace, size_t workspace_bytes, void *stream) {
    RETURN_IF(norm_args(NORM, desc));
    api_clear_error();
    RETURN_IF(check_pointers(NORM, {}, {grad_out, grad_sum, normalised, weight, grad_input, grad_weight}));
    RETURN_IF(check_floats({rstd}));
    if (!grad_input && !grad_weight) return TVDCN_STATUS_SUCCESS;
    RowGradArgs a{};
    a.dtype = desc->dtype;
    a.rows = desc->rows;
    a.channels = (int)desc->channels;
    if (a.rows > 0) {
        RETURN_IF(check_pointers(NORM, {normalised, grad_out}, {}));
        if (!rstd) return invalid("rms_norm: null tensor");
        if (grad_weight) RETURN_IF(check_workspace(workspace, workspace_bytes, (size_t)rms_norm_part_floats(a) * 4));
    }
    a.dy = grad_out;
    a.dsum = grad_sum;
    a.x = normalised;
    a.rstd = rstd;
    a.weight = weight;
    a.dx = grad_input;
    a.dweight = grad_weight;
    a.part = static_cast<float *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_RMS_NORM, s, [&] { return launch_rms_norm_backward(a, s); });
}

tvdcn_status tvdcn_quantize_int8(int32_t dtype, int64_t rows, int64_t channels, const void *input, int8_t *codes,
                                 float *scales, void *stream) {
    RETURN_IF(check_type(QUANTIZE, dtype));
    RETURN_IF(check_map(QUANTIZE, rows, channels));
    api_clear_error();
    if (rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(QUANTIZE, {input, codes}, {}));
    if (!scales) return invalid("quantize_int8: null tensor");
    RETURN_IF(check_floats({scales}));
    RowArgs a = row_args(dtype, rows, channels);
    a.x = input;
    a.codes = codes;
    a.scales = scales;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_INT8_MAP, s, [&] { return launch_quantize(a, s); });
}

tvdcn_status tvdcn_dequantize_int8(int32_t dtype, int64_t rows, int64_t channels, const int8_t *codes,
                                   const float *scales, void *output, void *stream) {
    RETURN_IF(check_type(DEQUANTIZE, dtype));
    RETURN_IF(check_map(DEQUANTIZE, rows, channels));
    api_clear_error();
    if (rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(DEQUANTIZE, {codes, output}, {}));
    if (!scales) return invalid("dequantize_int8: null tensor");
    RETURN_IF(check_floats({scales}));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_INT8_MAP, s,
                      [&] { return launch_dequantize(dtype, rows, (int)channels, codes, scales, output, s); });
}

size_t tvdcn_pointwise_conv_int8_workspace_size(const tvdcn_pointwise_desc *desc) {
    Int8ProductArgs a;
    return point_args(desc, a) ? 0 : pointwise_int8_bytes(a);
}

tvdcn_status tvdcn_pointwise_conv_int8(const tvdcn_pointwise_desc *desc, const int8_t *codes, const float *scales,
                                       const int8_t *weight_codes, const float *weight_scales, const void *bias,
                                       const void *residual, void *output, void *workspace, size_t workspace_bytes,
                                       void *stream) {
    Int8ProductArgs a;
    RETURN_IF(point_args(desc, a));
    api_clear_error();
    if (a.rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(POINT8, {codes, weight_codes, output}, {bias, residual}));
    if (!scales || !weight_scales) return invalid("pointwise_conv_int8: null tensor");
    RETURN_IF(check_floats({scales, weight_scales}));
    RETURN_IF(check_workspace(workspace, workspace_bytes, pointwise_int8_bytes(a)));
    a.codes = codes;
    a.scales = scales;
    a.weight_codes = weight_codes;
    a.weight_scales = weight_scales;
    a.bias = bias;
    a.residual = residual;
    a.y = output;
    a.work = static_cast<char *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_POINTWISE_INT8, s, [&] { return launch_pointwise_int8(a, s); });
}

tvdcn_status tvdcn_seeded_dropout(int32_t dtype, int64_t n, double p, const int64_t *seed, const void *input,
                                  const void *residual, void *output, void *stream) {
    RETURN_IF(check_type(DROPOUT, dtype));
    RETURN_IF(check_map(DROPOUT, n, 1));
    if (!(p >= 0.0 && p <= 1.0)) return invalid("seeded_dropout: p must be in [0, 1]");
    api_clear_error();
    if (n == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(DROPOUT, {input, output}, {residual}));
    if (!seed || (reinterpret_cast<uintptr_t>(seed) & 7)) return invalid("seeded_dropout: the seed must be there, 8-byte aligned");
    const int drop = (int)std::nearbyint(p * 65536.0);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_DROPOUT, s, [&] { return launch_dropout(dtype, n, drop, seed, input, residual, output, s); });
}

}  // extern "C"
