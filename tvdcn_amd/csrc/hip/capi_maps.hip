// C ABI of the operators on channels-last maps (declared in include/tvdcn_hip.h): checks of the arguments, the
// workspace, and the launches on the caller's stream. Host-side only: no allocation, no synchronisation.
#include <climits>
#include <cmath>
#include <initializer_list>
#include <string>

#include "capi.h"
#include "maps.h"

using namespace tvdcn_hip;

namespace {

constexpr int64_t MOST_CHANNELS = 1 << 20;
constexpr int64_t MOST_ELEMENTS = (int64_t)1 << 40;   // of a map: its bytes, and its workspace's, fit 64 bits

tvdcn_status invalid(const std::string &msg) { return api_fail(TVDCN_STATUS_INVALID_ARGUMENT, msg); }

tvdcn_status check_type(const char *what, int32_t dtype, int32_t activation = TVDCN_ACT_NONE) {
    if (dtype < 0 || dtype > 3) return invalid(std::string(what) + ": unknown dtype");
    if (dtype == TVDCN_DTYPE_FLOAT64)
        return api_fail(TVDCN_STATUS_NOT_SUPPORTED, std::string(what) + ": float32, float16 and bfloat16 only");
    if (activation < TVDCN_ACT_NONE || activation > TVDCN_ACT_GELU) return invalid(std::string(what) + ": unknown activation");
    return TVDCN_STATUS_SUCCESS;
}

tvdcn_status check_map(const char *what, int64_t rows, int64_t channels) {
    if (rows < 0) return invalid(std::string(what) + ": negative size");
    if (channels <= 0) return invalid(std::string(what) + ": channels must be positive");
    if (channels > MOST_CHANNELS)
        return api_fail(TVDCN_STATUS_NOT_SUPPORTED, std::string(what) + ": more than 2^20 channels");
    if (rows > MOST_ELEMENTS / channels) return api_fail(TVDCN_STATUS_NOT_SUPPORTED, std::string(what) + ": map too large");
    return TVDCN_STATUS_SUCCESS;
}

tvdcn_status check_pointers(const char *what, std::initializer_list<const void *> needed,
                            std::initializer_list<const void *> optional) {
    for (const void *p : needed)
        if (!p) return invalid(std::string(what) + ": null tensor");
    for (auto list : {needed, optional})
        for (const void *p : list)
            if (reinterpret_cast<uintptr_t>(p) & 15) return invalid("tensor pointers must be 16-byte aligned");
    return TVDCN_STATUS_SUCCESS;
}

// statistics: single floats
tvdcn_status check_floats(std::initializer_list<const void *> pointers) {
    for (const void *p : pointers)
        if (reinterpret_cast<uintptr_t>(p) & 3) return invalid("statistics must be 4-byte aligned");
    return TVDCN_STATUS_SUCCESS;
}

tvdcn_status check_workspace(const void *workspace, size_t have, size_t need) {
    if (have < need || (need > 0 && !workspace))
        return api_fail(TVDCN_STATUS_WORKSPACE_TOO_SMALL, "workspace too small: " + std::to_string(have) + " bytes, " +
                                                              std::to_string(need) + " needed");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return invalid("workspace must be 16-byte aligned");
    return TVDCN_STATUS_SUCCESS;
}

#define RETURN_IF(expr) \
    if (const tvdcn_status st_ = (expr)) return st_

constexpr const char *NORM = "group_norm_act", *POINT = "pointwise_conv";

tvdcn_status norm_args(const tvdcn_norm_desc *d, NormArgs &a) {
    if (!d) return invalid("null descriptor");
    RETURN_IF(check_type(NORM, d->dtype, d->activation));
    if (d->batch < 0 || d->pixels < 0) return invalid("group_norm_act: negative size");
    if (d->pixels > 0 && d->batch > MOST_ELEMENTS / d->pixels)
        return api_fail(TVDCN_STATUS_NOT_SUPPORTED, "group_norm_act: map too large");
    RETURN_IF(check_map(NORM, d->batch * d->pixels, d->channels));
    RETURN_IF(check_map(NORM, d->batch, d->channels));
    if (d->groups <= 0 || d->channels % d->groups) return invalid("group_norm_act: channels must be divisible by groups");
    if (!(d->eps >= 0.0) || !std::isfinite(d->eps)) return invalid("group_norm_act: eps must be finite and not negative");
    a = NormArgs{};
    a.dtype = d->dtype;
    a.act = d->activation;
    a.batch = d->batch;
    a.pixels = d->pixels;
    a.channels = (int)d->channels;
    a.groups = (int)d->groups;
    a.eps = (float)d->eps;
    return TVDCN_STATUS_SUCCESS;
}

size_t norm_bytes(const NormArgs &a, bool backward) {
    return a.batch == 0 || a.pixels == 0 ? 0 : (size_t)norm_part_floats(a, backward) * 4;
}

tvdcn_status point_args(const tvdcn_pointwise_desc *d, PointwiseArgs &a) {
    if (!d) return invalid("null descriptor");
    RETURN_IF(check_type(POINT, d->dtype, d->activation));
    RETURN_IF(check_map(POINT, d->rows, d->in_channels));
    RETURN_IF(check_map(POINT, d->rows, d->out_channels));
    if (d->in_channels * d->out_channels > INT_MAX) return api_fail(TVDCN_STATUS_NOT_SUPPORTED, "pointwise_conv: weight too large");
    a = PointwiseArgs{};
    a.dtype = d->dtype;
    a.act = d->activation;
    a.rows = d->rows;
    a.in = (int)d->in_channels;
    a.out = (int)d->out_channels;
    return TVDCN_STATUS_SUCCESS;
}

const int8_t *const KEPT = reinterpret_cast<const int8_t *>(16);   // in a workspace query: an 8-bit input

tvdcn_status check_source(const char *what, const void *input, const int8_t *codes, const uint8_t *exponents) {
    if ((input != nullptr) == (codes != nullptr) || (codes != nullptr) != (exponents != nullptr))
        return invalid(std::string(what) + " backward: the input, or its codes and exponents");
    return TVDCN_STATUS_SUCCESS;
}

}  // namespace

extern "C" {

tvdcn_status tvdcn_compress_activation(int32_t dtype, int64_t rows, int64_t channels, const void *input, int8_t *codes,
                                       uint8_t *exponents, void *stream) {
    RETURN_IF(check_type("compress_activation", dtype));
    RETURN_IF(check_map("compress_activation", rows, channels));
    api_clear_error();
    if (rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers("compress_activation", {input, codes, exponents}, {}));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_INT8_MAP, s,
                      [&] { return launch_compress(dtype, rows, (int)channels, input, codes, exponents, s); });
}

tvdcn_status tvdcn_expand_activation(int32_t dtype, int64_t rows, int64_t channels, const int8_t *codes,
                                     const uint8_t *exponents, void *output, void *stream) {
    RETURN_IF(check_type("expand_activation", dtype));
    RETURN_IF(check_map("expand_activation", rows, channels));
    api_clear_error();
    if (rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers("expand_activation", {codes, exponents, output}, {}));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_INT8_MAP, s, [&] {
        return launch_expand(dtype, false, rows, (int)channels, channels, codes, exponents, output, s);
    });
}

size_t tvdcn_group_norm_act_forward_workspace_size(const tvdcn_norm_desc *desc) {
    NormArgs a;
    return norm_args(desc, a) ? 0 : norm_bytes(a, false);
}

size_t tvdcn_group_norm_act_backward_workspace_size(const tvdcn_norm_desc *desc) {
    NormArgs a;
    return norm_args(desc, a) ? 0 : norm_bytes(a, true);
}

tvdcn_status tvdcn_group_norm_act_forward(const tvdcn_norm_desc *desc, const void *input, const void *weight,
                                          const void *bias, void *output, float *mean, float *rstd, void *workspace,
                                          size_t workspace_bytes, void *stream) {
    NormArgs a;
    RETURN_IF(norm_args(desc, a));
    api_clear_error();
    if (a.batch == 0 || a.pixels == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(NORM, {input, output}, {weight, bias}));
    if (!mean || !rstd) return invalid("group_norm_act: null tensor");
    RETURN_IF(check_floats({mean, rstd}));
    RETURN_IF(check_workspace(workspace, workspace_bytes, norm_bytes(a, false)));
    a.x = input;
    a.weight = weight;
    a.bias = bias;
    a.y = output;
    a.mean = mean;
    a.rstd = rstd;
    a.part = static_cast<float *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_GROUP_NORM, s, [&] { return launch_norm_forward(a, s); });
}

tvdcn_status tvdcn_group_norm_act_backward(const tvdcn_norm_desc *desc, const void *grad_out, const void *input,
                                           const int8_t *codes, const uint8_t *exponents, const void *weight,
                                           const void *bias, const float *mean, const float *rstd, void *grad_input,
                                           void *grad_weight, void *grad_bias, void *workspace, size_t workspace_bytes,
                                           void *stream) {
    NormArgs a;
    RETURN_IF(norm_args(desc, a));
    api_clear_error();
    RETURN_IF(check_pointers(NORM, {}, {grad_out, input, codes, exponents, weight, bias, grad_input, grad_weight, grad_bias}));
    RETURN_IF(check_floats({mean, rstd}));
    if (a.batch > 0 && a.pixels > 0) {
        RETURN_IF(check_source(NORM, input, codes, exponents));
        RETURN_IF(check_pointers(NORM, {grad_out}, {}));
        if (!mean || !rstd) return invalid("group_norm_act: null tensor");
        RETURN_IF(check_workspace(workspace, workspace_bytes, norm_bytes(a, true)));
    }
    if (!grad_input && !grad_weight && !grad_bias) return TVDCN_STATUS_SUCCESS;
    a.x = input;
    a.codes = codes;
    a.exps = exponents;
    a.weight = weight;
    a.bias = bias;
    a.mean = const_cast<float *>(mean);
    a.rstd = const_cast<float *>(rstd);
    a.dy = grad_out;
    a.dx = grad_input;
    a.dweight = grad_weight;
    a.dbias = grad_bias;
    a.part = static_cast<float *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_GROUP_NORM, s, [&] { return launch_norm_backward(a, s); });
}

size_t tvdcn_pointwise_conv_forward_workspace_size(const tvdcn_pointwise_desc *desc) {
    PointwiseArgs a;
    return point_args(desc, a) ? 0 : pointwise_forward_bytes(a);
}

size_t tvdcn_pointwise_conv_backward_workspace_size(const tvdcn_pointwise_desc *desc, int32_t kept_int8) {
    PointwiseArgs a;
    if (point_args(desc, a)) return 0;
    a.codes = kept_int8 ? KEPT : nullptr;
    return pointwise_backward_bytes(a);
}

tvdcn_status tvdcn_pointwise_conv_forward(const tvdcn_pointwise_desc *desc, const void *input, const void *weight,
                                          const void *bias, const void *residual, void *output, void *pre,
                                          void *workspace, size_t workspace_bytes, void *stream) {
    PointwiseArgs a;
    RETURN_IF(point_args(desc, a));
    api_clear_error();
    if (a.rows == 0) return TVDCN_STATUS_SUCCESS;
    RETURN_IF(check_pointers(POINT, {input, weight, output}, {bias, residual, pre}));
    RETURN_IF(check_workspace(workspace, workspace_bytes, pointwise_forward_bytes(a)));
    a.x = input;
    a.weight = weight;
    a.bias = bias;
    a.residual = residual;
    a.y = output;
    a.pre = pre;
    a.work = static_cast<char *>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_POINTWISE, s, [&] { return launch_pointwise_forward(a, s); });
}

tvdcn_status tvdcn_pointwise_conv_backward(const tvdcn_pointwise_desc *desc, const void *grad_out, const void *input,
                                           const int8_t *codes, const uint8_t *exponents, const void *weight,
                                           const void *pre, void *grad_input, void *grad_weight, void *grad_bias,
                                           void *workspace, size_t workspace_bytes, void *stream) {
    PointwiseArgs a;
    RETURN_IF(point_args(desc, a));
    api_clear_error();
    RETURN_IF(check_pointers(POINT, {}, {grad_out, input, codes, exponents, weight, pre, grad_input, grad_weight, grad_bias}));
    if (!grad_input && !grad_weight && !grad_bias) return TVDCN_STATUS_SUCCESS;
    if (a.rows > 0) {
        RETURN_IF(check_pointers(POINT, {grad_out}, {}));
        if (grad_weight) RETURN_IF(check_source(POINT, input, codes, exponents));
        if (grad_input && !weight) return invalid("pointwise_conv: null tensor");
        if (a.act != TVDCN_ACT_NONE && !pre) return invalid("pointwise_conv backward: the activation's argument is missing");
    }
    a.x = input;
    a.codes = codes;
    a.exps = exponents;
    a.weight = weight;
    a.pre = const_cast<void *>(pre);
    a.dy = grad_out;
    a.dx = grad_input;
    a.dweight = grad_weight;
    a.dbias = grad_bias;
    a.work = static_cast<char *>(workspace);
    RETURN_IF(check_workspace(workspace, workspace_bytes, pointwise_backward_bytes(a)));
    hipStream_t s = static_cast<hipStream_t>(stream);
    return api_launch(TVDCN_KERNEL_POINTWISE, s, [&] { return launch_pointwise_backward(a, s); });
}

}  // extern "C"
