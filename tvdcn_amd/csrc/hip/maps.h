// Operators on channels-last maps, [rows][channels] with rows = batch x pixels: group normalisation with
// activation, the pointwise convolution and 8-bit activations. Shared host and device definitions.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "../../../include/tvdcn_hip.h"

namespace tvdcn_hip {

typedef float fvec4 __attribute__((ext_vector_type(4)));

// 8-bit maps: channels per block of one exponent, its bias in the stored byte, and the byte of a block that held a
// value that is not finite
constexpr int kKeptBlock = 32;
constexpr int kKeptBias = 127;
constexpr int kKeptNaN = 255;

inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }
inline int64_t round_up(int64_t a, int64_t b) { return ceil_div(a, b) * b; }

// ---- launchers (group_norm.hip, kept_maps.hip, pointwise.hip): asynchronous on `s`, nothing allocated ----

struct NormArgs {
    int dtype, act;
    int64_t batch, pixels;   // pixels per image
    int channels, groups;
    float eps;
    const void *x;           // [batch][pixels][channels], or null where the 8-bit form stands in for it
    const int8_t *codes;
    const uint8_t *exps;
    const void *weight, *bias;   // [channels] or null
    void *y;
    float *mean, *rstd;          // [batch][groups]
    const void *dy;
    void *dx, *dweight, *dbias;
    float *part;                 // workspace
};
int64_t norm_part_floats(const NormArgs &a, bool backward);
hipError_t launch_norm_forward(const NormArgs &a, hipStream_t s);
hipError_t launch_norm_backward(const NormArgs &a, hipStream_t s);

hipError_t launch_compress(int dtype, int64_t rows, int channels, const void *x, int8_t *codes, uint8_t *exps,
                           hipStream_t s);
// the values into rows of `pitch` elements, zero beyond the channels; as_bf16: bfloat16 whatever the map's type
hipError_t launch_expand(int dtype, bool as_bf16, int64_t rows, int channels, int64_t pitch, const int8_t *codes,
                         const uint8_t *exps, void *y, hipStream_t s);

struct PointwiseArgs {
    int dtype, act;
    int64_t rows;
    int in, out;
    const void *x, *weight, *bias, *residual;
    void *y, *pre;               // pre: the activation's argument, kept for the backward (or null)
    const void *dy;
    const int8_t *codes;
    const uint8_t *exps;
    void *dx, *dweight, *dbias;
    char *work;
};
size_t pointwise_forward_bytes(const PointwiseArgs &a);
size_t pointwise_backward_bytes(const PointwiseArgs &a);
hipError_t launch_pointwise_forward(const PointwiseArgs &a, hipStream_t s);
hipError_t launch_pointwise_backward(const PointwiseArgs &a, hipStream_t s);

// ---- device helpers ----

typedef __bf16 bf16;
typedef _Float16 f16;

// N elements in one access (in 16-byte ones where they are more)
template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack {
    T v[N];
};

// Activations. The argument is float32; ERF32: the error function to float32's last bits, otherwise erfc(u) =
// e^(-u^2) (a1 t + ... + a6 t^6), t = 1 / (1 + p u), at a third of the instructions. p and the a, of sum 1, are the least-maximum
// fit of e^(u^2) erfc(u) in that form: the distribution function is within 1.5e-7 of its value, and 3e-5 relative in the left
// tail, where gelu's results are z times it: a sixteenth of float16's half step. (A form that is close in absolute terms alone
// is off by steps there. Here u = |z| / sqrt(2), and the result halved: in the constants.)
__device__ __forceinline__ float normal_cdf_poly(float z, float gauss) {   // gauss = e^(-z^2/2)
    const float t = __builtin_amdgcn_rcpf(fmaf(fabsf(z), 0.4177f * 0.70710678118654752f, 1.f));
    const float poly =
        t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, 0.5f * -0.16677121f, 0.5f * 0.49751058f), 0.5f * -0.10272032f), 0.5f * 0.31840753f),
                         0.5f * 0.21653781f),
                 0.5f * 0.23703562f);
    const float tail = gauss * poly;
    return z < 0.f ? tail : 1.f - tail;
}
// e^(-z^2/2)
template <bool PRECISE> __device__ __forceinline__ float gauss_of(float z) {
    return PRECISE ? expf(-0.5f * z * z) : __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);   // (log2(e) / 2)
}
template <bool ERF32> __device__ __forceinline__ float normal_cdf(float z, float gauss) {
    return ERF32 ? 0.5f * erfcf(-z * 0.70710678118654752f) : normal_cdf_poly(z, gauss);
}
template <bool PRECISE> __device__ __forceinline__ float exp32(float v) { return PRECISE ? expf(v) : __expf(v); }
// a / b: for the 16-bit types by the reciprocal instruction (a last bit of float32 off, at a tenth of the instructions)
template <bool PRECISE> __device__ __forceinline__ float quotient(float a, float b) {
    return PRECISE ? a / b : a * __builtin_amdgcn_rcpf(b);
}

// (silu below about -87: e^-z is no float32, or its reciprocal none of full precision; results of under 2e-36 are 0)
template <bool PRECISE> __device__ __forceinline__ float act_value(float z, int act) {
    switch (act) {
        case TVDCN_ACT_RELU: return z < 0.f ? 0.f : z;   // (a NaN stays one)
        case TVDCN_ACT_SILU: return quotient<PRECISE>(z, 1.f + exp32<PRECISE>(-z));
        case TVDCN_ACT_GELU: return z * normal_cdf<PRECISE>(z, gauss_of<PRECISE>(z));
        default: return z;
    }
}
// N values at once: the (uniform) choice is made once for them
template <bool PRECISE, int N> __device__ __forceinline__ void act_values(float *z, int act) {
    if (act == TVDCN_ACT_NONE) return;
    if (act == TVDCN_ACT_RELU) {
#pragma unroll
        for (int v = 0; v < N; ++v) z[v] = act_value<PRECISE>(z[v], TVDCN_ACT_RELU);
    } else if (act == TVDCN_ACT_SILU) {
#pragma unroll
        for (int v = 0; v < N; ++v) z[v] = act_value<PRECISE>(z[v], TVDCN_ACT_SILU);
    } else {
#pragma unroll
        for (int v = 0; v < N; ++v) z[v] = act_value<PRECISE>(z[v], TVDCN_ACT_GELU);
    }
}
template <bool PRECISE> __device__ __forceinline__ float act_slope(float z, int act) {
    switch (act) {
        case TVDCN_ACT_SILU: {
            const float s = quotient<PRECISE>(1.f, 1.f + exp32<PRECISE>(-z));
            return s * (1.f + z * (1.f - s));
        }
        case TVDCN_ACT_GELU: {
            const float gauss = gauss_of<PRECISE>(z);
            return fmaf(z * gauss, 0.39894228040143268f, normal_cdf<PRECISE>(z, gauss));
        }
        default: return 1.f;
    }
}

// d *= slope(z)
template <bool PRECISE, int N> __device__ __forceinline__ void act_slopes(float *d, const float *z, int act) {
    if (act == TVDCN_ACT_NONE) return;
    if (act == TVDCN_ACT_RELU) {
#pragma unroll
        for (int v = 0; v < N; ++v) d[v] = z[v] <= 0.f ? 0.f : d[v];   // (also of a gradient that is not finite)
    } else if (act == TVDCN_ACT_SILU) {
#pragma unroll
        for (int v = 0; v < N; ++v) d[v] *= act_slope<PRECISE>(z[v], TVDCN_ACT_SILU);
    } else {
#pragma unroll
        for (int v = 0; v < N; ++v) d[v] *= act_slope<PRECISE>(z[v], TVDCN_ACT_GELU);
    }
}

template <typename T> constexpr bool is_f32() { return sizeof(T) == 4; }
template <typename T> __device__ __forceinline__ float most() { return 0.f; }
template <> __device__ __forceinline__ float most<float>() { return 3.402823466e38f; }
template <> __device__ __forceinline__ float most<f16>() { return 65504.f; }
template <> __device__ __forceinline__ float most<bf16>() { return 3.389531390e38f; }

// The activation's argument as it is kept for the backward: in the map's type, but for a silu or gelu of a bfloat16 map as float16
// in the same 16 bits. Its slopes need the argument's last bits where it is of the order of 1, not its range: three bits more there
// take the argument out of the gradients' error, which falls from 1.5 roundings of the map's type to 1.4. One beyond float16 is
// read as its largest value, at which the slopes are what they are further out (0 or 1; at an infinity they would be NaN).
template <typename T> struct Argument {   // silu and gelu
    typedef T type;
};
template <> struct Argument<bf16> {
    typedef f16 type;
};
template <typename T, int N> __device__ __forceinline__ void kept_arguments(const float *z, T *o, int act) {
    if constexpr (is_f32<T>()) {
#pragma unroll
        for (int v = 0; v < N; ++v) o[v] = z[v];
    } else if (std::is_same<T, bf16>::value && act != TVDCN_ACT_SILU && act != TVDCN_ACT_GELU) {
#pragma unroll
        for (int v = 0; v < N; ++v) o[v] = (T)z[v];
    } else {
#pragma unroll
        for (int v = 0; v < N; ++v) o[v] = __builtin_bit_cast(T, (f16)z[v]);
    }
}
template <typename Z, int N> __device__ __forceinline__ void argument_values(float *z) {
    if constexpr (std::is_same<Z, f16>::value)
#pragma unroll
        for (int v = 0; v < N; ++v) z[v] = fabsf(z[v]) == __builtin_inff() ? copysignf(most<f16>(), z[v]) : z[v];
}

// What code q of exponent byte e stands for: q * 2^(e - bias) clamped to T's finite values, NaN for a block that held a value
// that is not finite. The scaling is exact; only 64 and more steps of the largest exponent of all pass the finite values.
template <typename T> __device__ __forceinline__ float kept_scale(uint8_t e) {
    return e == kKeptNaN ? __builtin_nanf("") : __uint_as_float((uint32_t)e << 23);
}
template <typename T> __device__ __forceinline__ float most_scale() { return 5.316911983e36f; }   // 2^122
template <> __device__ __forceinline__ float most_scale<f16>() { return 1024.f; }
template <typename T, int N> __device__ __forceinline__ void kept_values(const int8_t *q, uint8_t e, float *f) {
    const float scale = kept_scale<T>(e);
#pragma unroll
    for (int v = 0; v < N; ++v) f[v] = (float)q[v] * scale;
    if (scale >= most_scale<T>())
#pragma unroll
        for (int v = 0; v < N; ++v) f[v] = fminf(fmaxf(f[v], -most<T>()), most<T>());
}

}  // namespace tvdcn_hip
