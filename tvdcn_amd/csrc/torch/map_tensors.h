// What the operators on channels-last maps share (map_ops.cpp, row_ops.cpp): checks of their arguments, the maps' memory, the
// current stream, and their nodes in autograd's graph.
#pragma once

#include <ATen/ATen.h>
#include <ATen/autocast_mode.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/autograd.h>
#include <torch/library.h>

#include <cmath>
#include <tuple>
#include <vector>

#include "tvdcn_hip.h"

namespace tvdcn_amd {
namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
typedef std::tuple<Tensor, Tensor> Two;
typedef std::tuple<Tensor, Tensor, Tensor> Three;
typedef const optional<Tensor> &MaybeTensor;

inline bool has(MaybeTensor t) { return t.has_value() && t->defined(); }
inline Tensor get(MaybeTensor t) { return has(t) ? *t : Tensor(); }
inline optional<Tensor> maybe(const Tensor &t) { return t.defined() ? optional<Tensor>(t) : optional<Tensor>(); }

inline int32_t map_dtype(at::ScalarType t, const char *name) {
    switch (t) {
        case at::kFloat: return TVDCN_DTYPE_FLOAT32;
        case at::kHalf: return TVDCN_DTYPE_FLOAT16;
        case at::kBFloat16: return TVDCN_DTYPE_BFLOAT16;
        default: TORCH_CHECK(false, name, ": unsupported dtype ", t, " on the GPU (expected float32, float16 or bfloat16)");
    }
    return -1;
}

inline void check_map(const Tensor &x, const char *name) {
    TORCH_CHECK(x.dim() >= 2, name, ": expected a (batch, channels, *size) input, got ", x.dim(), " dimensions");
    TORCH_CHECK(x.size(1) > 0, name, ": the input needs channels");
    const auto t = x.scalar_type();
    TORCH_CHECK(t == at::kFloat || t == at::kDouble || t == at::kHalf || t == at::kBFloat16, name, ": unsupported dtype ", t,
                " (expected float32/64, float16, bfloat16)");
}

inline void check_like(const Tensor &x, MaybeTensor t, const char *what, at::IntArrayRef sizes, const char *name) {
    if (!has(t)) return;
    TORCH_CHECK(t->sizes() == sizes, name, ": expected ", what, " of shape ", sizes, ", got ", t->sizes());
    TORCH_CHECK(t->scalar_type() == x.scalar_type(), name, ": expected ", what, " of dtype ", x.scalar_type(), ", got ",
                t->scalar_type());
    TORCH_CHECK(t->device() == x.device(), name, ": expected all tensors on ", x.device(), ", but ", what, " is on ",
                t->device());
}

inline void check_activation(int64_t activation, const char *name) {
    TORCH_CHECK(activation >= TVDCN_ACT_NONE && activation <= TVDCN_ACT_GELU, name, ": unknown activation ", activation);
}

// Dense channels-last memory: the last axes' strides under a channel stride of one
inline bool is_rows(const Tensor &x) {
    const auto sizes = x.sizes(), strides = x.strides();
    const int64_t n = x.dim();
    int64_t run = sizes[1];
    if (sizes[1] > 1 && strides[1] != 1) return false;
    for (int64_t i = n - 1; i >= 2; --i) {
        if (sizes[i] > 1 && strides[i] != run) return false;
        run *= sizes[i];
    }
    return sizes[0] <= 1 || strides[0] == run || x.numel() == 0;
}
inline bool is_aligned(const Tensor &x) { return x.is_meta() || (reinterpret_cast<uintptr_t>(x.data_ptr()) & 15) == 0; }
// an empty map of these sizes in channels-last memory
inline Tensor new_map(at::IntArrayRef sizes, const at::TensorOptions &options) {
    const size_t n = sizes.size();
    c10::SmallVector<int64_t, 6> strides(n);
    int64_t run = 1;
    strides[1] = run, run *= std::max<int64_t>(sizes[1], 1);
    for (size_t i = n - 1; i >= 2; --i) strides[i] = run, run *= std::max<int64_t>(sizes[i], 1);
    strides[0] = run;
    // (on the GPU without the dispatcher: 0.3 us of a call's 6)
    if (options.device().is_cuda()) return Tensor(at::detail::empty_strided_cuda(sizes, strides, options));
    return at::empty_strided(sizes, strides, options);
}
// the map with its channels contiguous per pixel, 16-byte aligned: itself, or a copy
inline Tensor rows_of(const Tensor &x) {
    if (is_rows(x) && is_aligned(x)) return x;
    return new_map(x.sizes(), x.options()).copy_(x);
}
inline Tensor rows_of(MaybeTensor x) { return has(x) ? rows_of(*x) : Tensor(); }
// [batch, *size, channels] (host kernels)
inline Tensor to_rows(const Tensor &x) { return x.dim() == 2 ? x.contiguous() : x.movedim(1, -1).contiguous(); }
inline Tensor flat(MaybeTensor v) {   // a parameter, contiguous and 16-byte aligned
    if (!has(v)) return Tensor();
    Tensor r = v->contiguous();
    return (reinterpret_cast<uintptr_t>(r.data_ptr()) & 15) == 0 ? r : r.clone();
}
// an empty channels-last map of x's batch and size with `channels` channels, as rows
inline Tensor new_rows(const Tensor &x, int64_t channels, at::TensorOptions options) {
    std::vector<int64_t> s{x.size(0)};
    for (int64_t i = 2; i < x.dim(); ++i) s.push_back(x.size(i));
    s.push_back(channels);
    return at::empty(s, options);
}
inline Tensor to_map(const Tensor &rows) { return rows.dim() == 2 ? rows : rows.movedim(-1, 1); }
inline std::vector<int64_t> map_shape(const Tensor &x, int64_t channels) {
    std::vector<int64_t> s = x.sizes().vec();
    s[1] = channels;
    return s;
}
inline int64_t pixels_of(const Tensor &x) {
    int64_t n = 1;
    for (int64_t i = 2; i < x.dim(); ++i) n *= x.size(i);
    return n;
}

inline void check_status(tvdcn_status st, const char *what) {
    TORCH_CHECK(st == TVDCN_STATUS_SUCCESS, what, " failed (status ", (int)st, "): ", tvdcn_last_error());
}
inline void *stream_of(const Tensor &t) { return (void *)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
inline void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
// (on the GPU; see new_map)
inline Tensor new_flat(at::IntArrayRef sizes, const at::TensorOptions &options) { return Tensor(at::detail::empty_cuda(sizes, options)); }
inline Tensor bytes(const Tensor &x, size_t n) { return new_flat({(int64_t)n}, x.options().dtype(at::kByte)); }

inline at::ScalarType wide_type(const Tensor &t) { return t.scalar_type() == at::kDouble ? at::kDouble : at::kFloat; }

inline Tensor act_value(const Tensor &z, int64_t act) {
    if (act == TVDCN_ACT_RELU) return at::relu(z);
    if (act == TVDCN_ACT_SILU) return z * at::sigmoid(z);
    if (act == TVDCN_ACT_GELU) return z * at::erfc(z * -M_SQRT1_2) * 0.5;
    return z;
}
template <typename Sig> c10::TypedOperatorHandle<Sig> op_of(const char *name) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").template typed<Sig>();
}
// A node that raises where a second derivative is asked for. all: the n gradients, then the tensors that they depend on.
class NoSecondDerivative : public torch::autograd::Function<NoSecondDerivative> {
   public:
    static variable_list forward(AutogradContext *ctx, at::TensorList all, int64_t n, const std::string &name) {
        at::AutoDispatchBelowADInplaceOrView guard;
        ctx->saved_data["name"] = name;
        variable_list out;
        for (int64_t i = 0; i < n; ++i) out.push_back(all[i].alias());
        return out;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &) {
        TORCH_CHECK(false, "double backwards on ", ctx->saved_data["name"].toStringRef(), " not supported");
        return {};
    }
};

// Which gradients are asked for: the node's edges are those of the tensors that were given
inline bool wanted(AutogradContext *ctx, const char *edge) {
    const int64_t i = ctx->saved_data[edge].toInt();
    return i >= 0 && ctx->needs_input_grad(i);
}

// Forward-mode derivatives have no formula here: a tangent that an input brings is refused, not dropped
inline void check_no_tangents(const char *name, std::initializer_list<Tensor> ts) {
    for (const Tensor &t : ts)
        TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(0).defined(), name, ": forward-mode derivatives (jvp) are not supported");
}

inline bool needs(const Tensor &t) { return t.defined() && t.requires_grad(); }
inline bool needs(MaybeTensor t) { return has(t) && t->requires_grad(); }

// The gradients (undefined where not wanted), with the raising node where a graph of the backward is made
inline variable_list with_node(const Three &g, const variable_list &used, const char *name) {
    variable_list r{std::get<0>(g), std::get<1>(g), std::get<2>(g)};
    bool graph = false;
    if (at::GradMode::is_enabled())
        for (const Tensor &t : used) graph = graph || needs(t);
    if (!graph) return r;
    variable_list there, in;
    for (const Tensor &t : r)
        if (t.defined()) there.push_back(t);
    for (const Tensor &t : used)
        if (t.defined()) in.push_back(t);
    if (there.empty()) return r;
    const size_t n = there.size();
    there.insert(there.end(), in.begin(), in.end());
    const variable_list made = NoSecondDerivative::apply(at::TensorList(there), (int64_t)n, std::string(name));
    size_t at = 0;
    for (Tensor &t : r)
        if (t.defined()) t = made[at++];
    return r;
}

inline bool any_grad(std::initializer_list<Tensor> ts) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor &t : ts)
        if (needs(t)) return true;
    return false;
}

inline Tensor cast(at::ScalarType t, const Tensor &x) { return at::autocast::cached_cast(t, x, c10::DeviceType::CUDA); }
inline optional<Tensor> cast(at::ScalarType t, MaybeTensor x) { return has(x) ? optional<Tensor>(cast(t, *x)) : optional<Tensor>(); }

}  // namespace
}  // namespace tvdcn_amd
