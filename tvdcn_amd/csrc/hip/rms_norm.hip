// Root-mean-square normalisation of every row [channels] of a channels-last map, of the map or of its sum with a shortcut, with
// its result in the map's type or in 8 bits, its gradients, and maps in 8 bits and back:
//
//   s = x + r (in the map's type),  rstd = (avg(s^2) + eps)^-1/2,  y = w s rstd
//   dh = w dy,  h = s rstd,  dx = rstd (dh - h avg(dh h)) + ds,  dw = sum over rows of dy h
//   scale = max(max |v| (1 / 127), 2^-126),  code = v / scale rounded, ties to even
//
// Bound by memory: a row stays in registers between the sums over it and its results, so every value is read once and written
// once. Rows are laid over as few lanes as hold them (a power of two, up to a wave, N accesses of 16 bytes each: several short
// rows to a wave), rows beyond a wave's registers over a workgroup, rows beyond that are read twice. Rows whose size is no
// multiple of 16 bytes are read and written by the same accesses, unaligned, and by single values at their ends.
//
// Sums are float32, in a fixed order. Squares beyond float32 are summed again at 2^-140 of their size.
#include <algorithm>

#include "rows.h"

namespace tvdcn_hip {
namespace {

constexpr int TB = 256;
constexpr int HELD = 4;         // accesses of a lane that holds its part of a long row
constexpr int MOST_TB = 1024;
constexpr int GRAD_TB = 512;    // backward: three maps and the weight's gradient are held (at 1024 lanes they do not fit)
constexpr float LEAST_SCALE = 1.1754943508222875e-38f;   // 2^-126
constexpr float MOST_SCALE = 2.6793883890187504e+36f;     // 127 of it are finite

template <typename T> constexpr int vec() { return 16 / (int)sizeof(T); }

// N elements at any address that their type allows
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};

// VEC elements of a row, of which `left` are in it: WHOLE rows are made of whole accesses
template <typename T, int VEC, bool WHOLE> __device__ __forceinline__ void load(const T *p, int left, T *o) {
    if constexpr (WHOLE) {
        Pack<T, VEC> k{};
        if (left > 0) k = *reinterpret_cast<const Pack<T, VEC> *>(p);
#pragma unroll
        for (int v = 0; v < VEC; ++v) o[v] = k.v[v];
    } else if (left >= VEC) {
        const Loose<T, VEC> k = *reinterpret_cast<const Loose<T, VEC> *>(p);
#pragma unroll
        for (int v = 0; v < VEC; ++v) o[v] = k.v[v];
    } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v) o[v] = v < left ? p[v] : (T)0;
    }
}
template <typename T, int VEC, bool WHOLE> __device__ __forceinline__ void store(T *p, int left, const T *o) {
    if constexpr (WHOLE) {
        Pack<T, VEC> k;
#pragma unroll
        for (int v = 0; v < VEC; ++v) k.v[v] = o[v];
        if (left > 0) *reinterpret_cast<Pack<T, VEC> *>(p) = k;
    } else if (left >= VEC) {
        Loose<T, VEC> k;
#pragma unroll
        for (int v = 0; v < VEC; ++v) k.v[v] = o[v];
        *reinterpret_cast<Loose<T, VEC> *>(p) = k;
    } else {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            if (v < left) p[v] = o[v];
    }
}
template <typename T, int VEC> __device__ __forceinline__ void widen(const T *o, float *f) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) f[v] = (float)o[v];
}
template <typename T, int VEC> __device__ __forceinline__ void narrow(const float *f, T *o) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) o[v] = (T)f[v];
}

// The lanes of a row: 2^log2 of a wave, or a whole workgroup (`red`: a word per wave)
struct Add {
    static __device__ __forceinline__ float of(float a, float b) { return a + b; }
};
struct Most {   // of magnitudes, as bits: a NaN's are above an infinity's
    static __device__ __forceinline__ float of(float a, float b) {
        return __uint_as_float(max(__float_as_uint(a), __float_as_uint(b)));
    }
};
template <typename Op, bool BLOCK> __device__ __forceinline__ float over_row(float v, int log2, float *red) {
#pragma unroll
    for (int m = 0; m < 6; ++m)
        if (BLOCK || m < log2) v = Op::of(v, __shfl_xor(v, 1 << m));
    if constexpr (BLOCK) {
        const int waves = (int)blockDim.x >> 6, wave = threadIdx.x >> 6;
        __syncthreads();   // what was read of `red` before is over
        if ((threadIdx.x & 63) == 0) red[wave] = v;
        __syncthreads();
        v = red[0];
        for (int w = 1; w < waves; ++w) v = Op::of(v, red[w]);
    }
    return v;
}

constexpr float DOWN = 8.470329472543003e-22f, DOWN2 = DOWN * DOWN;   // 2^-70
static_assert(DOWN * 1180591620717411303424.f == 1.f && DOWN2 > 0, "");

__device__ __forceinline__ bool is_infinite(float v) { return v == __builtin_inff(); }

// Codes of VEC values: v / scale rounded to the nearest, ties to even, as if the quotient were exact. v inv is within 2^-16 of it
// (|v / scale| <= 127), so the rounding is settled unless it comes that close to a border; there v - code scale, which is exact,
// says which side.
template <int VEC> __device__ __forceinline__ void codes_of(const float *v, float scale, int8_t *o) {
    const float inv = 1.f / scale;
    float q[VEC], near = 0.f;
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
        const float t = v[e] * inv;
        q[e] = rintf(t);
        near = fmaxf(near, fabsf(t - q[e]));
    }
    if (near > 0.49996f)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float rest = 2.f * fmaf(-q[e], scale, v[e]);
            if (fabsf(rest) > scale || (fabsf(rest) == scale && ((int)q[e] & 1))) q[e] += copysignf(1.f, rest);
        }
#pragma unroll
    for (int e = 0; e < VEC; ++e) o[e] = (int8_t)(int)q[e];
}
// the scale of a row whose largest magnitude is `big`: NaN where that is not finite (the row then stands for NaN)
__device__ __forceinline__ float scale_of(float big) {
    return big < __builtin_inff() ? fminf(fmaxf(big * (1.f / 127.f), LEAST_SCALE), MOST_SCALE) : __builtin_nanf("");
}

enum Mode { NORM, NORM8, QUANTIZE };

struct RowKernelArgs {
    int64_t rows;
    int channels, log2;
    float inv_channels, eps;
    const void *x, *residual, *weight;
    void *sum, *y;
    float *rstd, *scales;
    int8_t *codes;
};

template <typename T, int VEC> __device__ __forceinline__ void add_in_type(float *f, const T *r, T *sum) {
#pragma unroll
    for (int v = 0; v < VEC; ++v) {
        sum[v] = (T)(f[v] + (float)r[v]);
        f[v] = (float)sum[v];
    }
}

// A lane has N accesses of a row, LANES apart. BLOCK: a workgroup's lanes, otherwise 2^log2 of a wave.
template <typename T, int N, bool WHOLE, int MODE, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? MOST_TB : TB) row_kernel(RowKernelArgs a) {
    constexpr int VEC = vec<T>();
    __shared__ float red[BLOCK ? MOST_TB / 64 : 1];
    const int t = threadIdx.x, C = a.channels;
    const int lanes = BLOCK ? (int)blockDim.x : 1 << a.log2, l = t & (lanes - 1);
    const int per = BLOCK ? 1 : TB >> a.log2;   // rows of a workgroup
    float w[N][VEC];
    if constexpr (MODE != QUANTIZE)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * lanes + l) * VEC;
            if (a.weight) {
                T o[VEC];
                load<T, VEC, WHOLE>((const T *)a.weight + c, C - c, o);
                widen<T, VEC>(o, w[n]);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) w[n][v] = 1.f;
            }
        }
    for (int64_t row = (int64_t)blockIdx.x * per + (BLOCK ? 0 : t >> a.log2); row < a.rows; row += (int64_t)gridDim.x * per) {
        const int64_t at = row * C;
        T x[N][VEC], r[N][VEC];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * lanes + l) * VEC;
            load<T, VEC, WHOLE>((const T *)a.x + at + c, C - c, x[n]);
        }
        if (MODE != QUANTIZE && a.residual)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = (n * lanes + l) * VEC;
                load<T, VEC, WHOLE>((const T *)a.residual + at + c, C - c, r[n]);
            }
        float f[N][VEC];
#pragma unroll
        for (int n = 0; n < N; ++n) widen<T, VEC>(x[n], f[n]);
        if constexpr (MODE != QUANTIZE) {
            if (a.residual)
#pragma unroll
                for (int n = 0; n < N; ++n) {
                    const int c = (n * lanes + l) * VEC;
                    add_in_type<T, VEC>(f[n], r[n], x[n]);
                    store<T, VEC, WHOLE>((T *)a.sum + at + c, C - c, x[n]);
                }
            float ss = 0.f;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int v = 0; v < VEC; ++v) ss = fmaf(f[n][v], f[n][v], ss);
            ss = over_row<Add, BLOCK>(ss, a.log2, red);
            float rstd = 1.f / sqrtf(fmaf(ss, a.inv_channels, a.eps));
            if (is_infinite(ss)) {   // (the same for all lanes of the row)
                ss = 0.f;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) ss = fmaf(f[n][v] * DOWN, f[n][v] * DOWN, ss);
                ss = over_row<Add, BLOCK>(ss, a.log2, red);
                rstd = DOWN / sqrtf(fmaf(ss, a.inv_channels, a.eps * DOWN2));
            }
            if (a.rstd && l == 0) a.rstd[row] = rstd;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[n][v] = f[n][v] * rstd * w[n][v];
        }
        if constexpr (MODE == NORM) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = (n * lanes + l) * VEC;
                T o[VEC];
                narrow<T, VEC>(f[n], o);
                store<T, VEC, WHOLE>((T *)a.y + at + c, C - c, o);
            }
        } else {
            float big = 0.f;   // (beyond the row's end: zeros)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int v = 0; v < VEC; ++v) big = Most::of(big, (n * lanes + l) * VEC + v < C ? fabsf(f[n][v]) : 0.f);
            const float scale = scale_of(over_row<Most, BLOCK>(big, a.log2, red));
            if (l == 0) a.scales[row] = scale;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = (n * lanes + l) * VEC;
                int8_t q[VEC] = {};
                if (scale == scale) codes_of<VEC>(f[n], scale, q);
                store<int8_t, VEC, WHOLE>(a.codes + at + c, C - c, q);
            }
        }
    }
}

// Rows beyond a workgroup's registers: read once for the sums (and written as the sum), once more for each result that needs them
template <typename T, bool WHOLE, int MODE> __global__ void __launch_bounds__(MOST_TB) long_row_kernel(RowKernelArgs a) {
    constexpr int VEC = vec<T>();
    __shared__ float red[MOST_TB / 64];
    const int t = threadIdx.x, C = a.channels;
    const bool added = MODE != QUANTIZE && a.residual;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = row * C;
        auto values = [&](int c, float *f, bool write) {
            T x[VEC], r[VEC];
            load<T, VEC, WHOLE>((const T *)a.x + at + c, C - c, x);
            widen<T, VEC>(x, f);
            if (!added) return;
            load<T, VEC, WHOLE>((const T *)a.residual + at + c, C - c, r);
            add_in_type<T, VEC>(f, r, x);
            if (write) store<T, VEC, WHOLE>((T *)a.sum + at + c, C - c, x);
        };
        float rstd = 1.f;
        if constexpr (MODE != QUANTIZE) {
            float ss = 0.f;
            for (int c = t * VEC; c < C; c += MOST_TB * VEC) {
                float f[VEC];
                values(c, f, true);
#pragma unroll
                for (int v = 0; v < VEC; ++v) ss = fmaf(f[v], f[v], ss);
            }
            ss = over_row<Add, true>(ss, 6, red);
            rstd = 1.f / sqrtf(fmaf(ss, a.inv_channels, a.eps));
            if (is_infinite(ss)) {
                ss = 0.f;
                for (int c = t * VEC; c < C; c += MOST_TB * VEC) {
                    float f[VEC];
                    values(c, f, false);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) ss = fmaf(f[v] * DOWN, f[v] * DOWN, ss);
                }
                ss = over_row<Add, true>(ss, 6, red);
                rstd = DOWN / sqrtf(fmaf(ss, a.inv_channels, a.eps * DOWN2));
            }
            if (a.rstd && t == 0) a.rstd[row] = rstd;
        }
        auto result = [&](int c, float *f) {
            values(c, f, false);
            if constexpr (MODE != QUANTIZE) {
                T o[VEC];
                if (a.weight) load<T, VEC, WHOLE>((const T *)a.weight + c, C - c, o);
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[v] = f[v] * rstd * (a.weight ? (float)o[v] : 1.f);
            }
        };
        if constexpr (MODE == NORM) {
            for (int c = t * VEC; c < C; c += MOST_TB * VEC) {
                float f[VEC];
                T o[VEC];
                result(c, f);
                narrow<T, VEC>(f, o);
                store<T, VEC, WHOLE>((T *)a.y + at + c, C - c, o);
            }
        } else {
            float big = 0.f;
            for (int c = t * VEC; c < C; c += MOST_TB * VEC) {
                float f[VEC];
                result(c, f);
#pragma unroll
                for (int v = 0; v < VEC; ++v) big = Most::of(big, c + v < C ? fabsf(f[v]) : 0.f);
            }
            const float scale = scale_of(over_row<Most, true>(big, 6, red));
            if (t == 0) a.scales[row] = scale;
            for (int c = t * VEC; c < C; c += MOST_TB * VEC) {
                float f[VEC];
                int8_t q[VEC] = {};
                result(c, f);
                if (scale == scale) codes_of<VEC>(f, scale, q);
                store<int8_t, VEC, WHOLE>(a.codes + at + c, C - c, q);
            }
        }
    }
}

template <typename T, bool WHOLE>
__global__ void __launch_bounds__(TB) dequantize_kernel(int64_t rows, int C, int log2, const int8_t *__restrict__ codes,
                                                        const float *__restrict__ scales, T *__restrict__ y) {
    constexpr int VEC = vec<T>();
    const int lanes = 1 << log2, l = threadIdx.x & (lanes - 1), per = TB >> log2;
    for (int64_t row = (int64_t)blockIdx.x * per + (threadIdx.x >> log2); row < rows; row += (int64_t)gridDim.x * per) {
        const float scale = scales[row];
        for (int c = l * VEC; c < C; c += lanes * VEC) {
            int8_t q[VEC];
            T o[VEC];
            load<int8_t, VEC, WHOLE>(codes + row * C + c, C - c, q);
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] = (T)((float)q[v] * scale);
            store<T, VEC, WHOLE>(y + row * C + c, C - c, o);
        }
    }
}

// ---- backward ----

struct RowGradKernelArgs {
    int64_t rows;
    int channels, log2;
    float inv_channels;
    const void *dy, *dsum, *x, *weight;
    const float *rstd;
    void *dx;
    float *part;   // [workgroups][channels], or null
};

template <typename T, int N, bool WHOLE, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? GRAD_TB : TB) row_grad_kernel(RowGradKernelArgs a) {
    constexpr int VEC = vec<T>();
    extern __shared__ float shared[];   // BLOCK: a word per wave; otherwise [waves][lanes * N * VEC]
    const int t = threadIdx.x, C = a.channels;
    const int lanes = BLOCK ? (int)blockDim.x : 1 << a.log2, l = t & (lanes - 1);
    const int per = BLOCK ? 1 : TB >> a.log2;
    float w[N][VEC], dw[N][VEC];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        const int c = (n * lanes + l) * VEC;
        T o[VEC];
        if (a.weight) load<T, VEC, WHOLE>((const T *)a.weight + c, C - c, o);
#pragma unroll
        for (int v = 0; v < VEC; ++v) w[n][v] = a.weight ? (float)o[v] : 1.f, dw[n][v] = 0.f;
    }
    for (int64_t row = (int64_t)blockIdx.x * per + (BLOCK ? 0 : t >> a.log2); row < a.rows; row += (int64_t)gridDim.x * per) {
        const int64_t at = row * C;
        T x[N][VEC], dy[N][VEC], ds[N][VEC];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * lanes + l) * VEC;
            load<T, VEC, WHOLE>((const T *)a.x + at + c, C - c, x[n]);
            load<T, VEC, WHOLE>((const T *)a.dy + at + c, C - c, dy[n]);
        }
        if (a.dsum)
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = (n * lanes + l) * VEC;
                load<T, VEC, WHOLE>((const T *)a.dsum + at + c, C - c, ds[n]);
            }
        const float rstd = a.rstd[row];
        float h[N][VEC], dh[N][VEC], dot = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float d = (float)dy[n][v];
                h[n][v] = (float)x[n][v] * rstd;
                dh[n][v] = d * w[n][v];
                dw[n][v] = fmaf(d, h[n][v], dw[n][v]);
                dot = fmaf(dh[n][v], h[n][v], dot);
            }
        if (a.dx) {
            dot = over_row<Add, BLOCK>(dot, a.log2, shared) * a.inv_channels;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                const int c = (n * lanes + l) * VEC;
                T o[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v)
                    o[v] = (T)fmaf(rstd, fmaf(-h[n][v], dot, dh[n][v]), a.dsum ? (float)ds[n][v] : 0.f);
                store<T, VEC, WHOLE>((T *)a.dx + at + c, C - c, o);
            }
        }
    }
    if (!a.part) return;
    float *part = a.part + (int64_t)blockIdx.x * C;
    if constexpr (BLOCK) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int c = (n * lanes + l) * VEC;
            store<float, VEC, false>(part + c, C - c, dw[n]);
        }
    } else {
        // the rows that share a wave, then the waves
        const int width = lanes * N * VEC, wave = t >> 6;
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                float s = dw[n][v];
#pragma unroll
                for (int m = 0; m < 6; ++m)
                    if (m >= a.log2) s += __shfl_xor(s, 1 << m);
                if ((t & 63) < lanes) shared[wave * width + (n * lanes + l) * VEC + v] = s;
            }
        __syncthreads();
        for (int c = t; c < C; c += TB) {
            float s = shared[c];
#pragma unroll
            for (int k = 1; k < TB / 64; ++k) s += shared[k * width + c];
            part[c] = s;
        }
    }
}

// Rows beyond a workgroup's registers: dx row by row in two readings, the weight's gradient column by column
template <typename T, bool WHOLE> __global__ void __launch_bounds__(MOST_TB) long_row_grad_kernel(RowGradKernelArgs a) {
    constexpr int VEC = vec<T>();
    __shared__ float red[MOST_TB / 64];
    const int t = threadIdx.x, C = a.channels;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = row * C;
        const float rstd = a.rstd[row];
        float dot = 0.f;
        auto read = [&](int c, float *h, float *dh) {
            T x[VEC], dy[VEC], w[VEC];
            load<T, VEC, WHOLE>((const T *)a.x + at + c, C - c, x);
            load<T, VEC, WHOLE>((const T *)a.dy + at + c, C - c, dy);
            if (a.weight) load<T, VEC, WHOLE>((const T *)a.weight + c, C - c, w);
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] = (float)x[v] * rstd, dh[v] = (float)dy[v] * (a.weight ? (float)w[v] : 1.f);
        };
        for (int c = t * VEC; c < C; c += MOST_TB * VEC) {
            float h[VEC], dh[VEC];
            read(c, h, dh);
#pragma unroll
            for (int v = 0; v < VEC; ++v) dot = fmaf(dh[v], h[v], dot);
        }
        dot = over_row<Add, true>(dot, 6, red) * a.inv_channels;
        for (int c = t * VEC; c < C; c += MOST_TB * VEC) {
            float h[VEC], dh[VEC];
            T ds[VEC] = {}, o[VEC];
            read(c, h, dh);
            if (a.dsum) load<T, VEC, WHOLE>((const T *)a.dsum + at + c, C - c, ds);
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] = (T)fmaf(rstd, fmaf(-h[v], dot, dh[v]), (float)ds[v]);
            store<T, VEC, WHOLE>((T *)a.dx + at + c, C - c, o);
        }
    }
}
template <typename T> __global__ void __launch_bounds__(TB) long_weight_grad_kernel(RowGradKernelArgs a, int64_t chunk) {
    const int c = blockIdx.x * TB + threadIdx.x, C = a.channels;
    if (c >= C) return;
    const int64_t first = blockIdx.y * chunk, last = first + chunk < a.rows ? first + chunk : a.rows;
    float s = 0.f;
    for (int64_t row = first; row < last; ++row)
        s = fmaf((float)((const T *)a.dy)[row * C + c], (float)((const T *)a.x)[row * C + c] * a.rstd[row], s);
    a.part[(int64_t)blockIdx.y * C + c] = s;
}

// dw = the sum of its parts: 16 channels per workgroup, 64 lanes along the parts, four loads of a lane in flight
constexpr int FIN = 1024;
template <typename T>
__global__ void __launch_bounds__(FIN) row_finish_kernel(const float *__restrict__ part, T *__restrict__ dw, int C, int parts) {
    __shared__ float red[FIN];
    const int t = threadIdx.x, c = (int)blockIdx.x * 16 + (t & 15);
    float s = 0.f;
    if (c < C)
        for (int u = t >> 4; u < parts; u += 4 * (FIN / 16)) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = u + k * (FIN / 16) < parts ? part[(int64_t)(u + k * (FIN / 16)) * C + c] : 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) s += v[k];
        }
    red[t] = s;
    __syncthreads();
    if (t < 64) {   // four lanes a channel, 16 parts each
        for (int k = 64; k < FIN; k += 64) s += red[t + k];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        if (t < 16 && c < C) dw[c] = (T)s;
    }
}

// ---- host ----

// How rows lie over lanes: 2^log2 of a wave with N accesses each, a workgroup of `threads`, or (threads = 0) read in turn
struct RowShape {
    int log2, n, threads;
    bool block;
};
RowShape row_shape(int channels, int vec, int most) {
    const int packs = (int)ceil_div(channels, vec);
    RowShape k{0, 1, 0, false};
    if (packs <= 64 * HELD) {
        while (k.log2 < 6 && 1 << k.log2 < packs) ++k.log2;
        while (k.n << k.log2 < packs) k.n *= 2;
        return k;
    }
    k.block = true;
    k.n = HELD;
    for (k.threads = 128; k.threads < most && k.threads * HELD < packs;) k.threads *= 2;
    if (k.threads * HELD < packs) k.threads = 0;
    return k;
}

unsigned row_grid(int64_t units, int64_t most) { return (unsigned)std::min(units, most); }

template <typename T, bool WHOLE, int MODE> hipError_t launch_rows(const RowArgs &a, hipStream_t s) {
    const RowShape k = row_shape(a.channels, vec<T>(), MOST_TB);
    const RowKernelArgs p{a.rows, a.channels, k.log2, (float)(1.0 / a.channels), a.eps, a.x, a.residual, a.weight,
                          a.sum, a.y, a.rstd, a.scales, a.codes};
    if (k.block) {
        if (k.threads) row_kernel<T, HELD, WHOLE, MODE, true><<<row_grid(a.rows, 4096), k.threads, 0, s>>>(p);
        else long_row_kernel<T, WHOLE, MODE><<<row_grid(a.rows, 1024), MOST_TB, 0, s>>>(p);
        return hipGetLastError();
    }
    const unsigned grid = row_grid(ceil_div(a.rows, TB >> k.log2), 4096);
    if (k.n == 1) row_kernel<T, 1, WHOLE, MODE, false><<<grid, TB, 0, s>>>(p);
    else if (k.n == 2) row_kernel<T, 2, WHOLE, MODE, false><<<grid, TB, 0, s>>>(p);
    else row_kernel<T, HELD, WHOLE, MODE, false><<<grid, TB, 0, s>>>(p);
    return hipGetLastError();
}
template <typename T, int MODE> hipError_t launch_rows(const RowArgs &a, hipStream_t s) {
    return a.channels % vec<T>() == 0 ? launch_rows<T, true, MODE>(a, s) : launch_rows<T, false, MODE>(a, s);
}
template <int MODE> hipError_t launch_rows(const RowArgs &a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return launch_rows<float, MODE>(a, s);
        case TVDCN_DTYPE_FLOAT16: return launch_rows<f16, MODE>(a, s);
        default: return launch_rows<bf16, MODE>(a, s);
    }
}

template <typename T> hipError_t dequantize(int64_t rows, int channels, const int8_t *codes, const float *scales, T *y, hipStream_t s) {
    int log2 = 0;
    while (log2 < 8 && vec<T>() << log2 < channels) ++log2;
    const unsigned grid = row_grid(ceil_div(rows, TB >> log2), 16384);
    if (channels % vec<T>() == 0) dequantize_kernel<T, true><<<grid, TB, 0, s>>>(rows, channels, log2, codes, scales, y);
    else dequantize_kernel<T, false><<<grid, TB, 0, s>>>(rows, channels, log2, codes, scales, y);
    return hipGetLastError();
}

// Workgroups of the backward: each keeps a part of the weight's gradient
int64_t grad_parts(const RowGradArgs &a) {
    const RowShape k = row_shape(a.channels, a.dtype == TVDCN_DTYPE_FLOAT32 ? 4 : 8, GRAD_TB);
    if (k.block && !k.threads) return std::min<int64_t>(a.rows, 256);
    return k.block ? std::min<int64_t>(a.rows, 1024) : std::min<int64_t>(ceil_div(a.rows, TB >> k.log2), 1024);
}

template <typename T, int N, bool WHOLE> hipError_t launch_held_grad(const RowGradKernelArgs &p, unsigned grid, hipStream_t s) {
    row_grad_kernel<T, N, WHOLE, false><<<grid, TB, (TB / 64) * (N << p.log2) * vec<T>() * 4, s>>>(p);
    return hipGetLastError();
}

template <typename T, bool WHOLE> hipError_t launch_grad(const RowGradArgs &a, hipStream_t s) {
    const RowShape k = row_shape(a.channels, vec<T>(), GRAD_TB);
    RowGradKernelArgs p{a.rows, a.channels, k.log2, (float)(1.0 / a.channels), a.dy, a.dsum, a.x, a.weight, a.rstd, a.dx,
                        a.dweight ? a.part : nullptr};
    const int64_t parts = grad_parts(a);
    hipError_t e = hipSuccess;
    if (a.rows == 0) {
    } else if (k.block && !k.threads) {
        if (a.dx) long_row_grad_kernel<T, WHOLE><<<row_grid(a.rows, 1024), MOST_TB, 0, s>>>(p);
        if (e = hipGetLastError(); e != hipSuccess) return e;
        if (a.dweight) {
            const int64_t chunk = ceil_div(a.rows, parts);
            // (fewer chunks than parts where they do not divide: the rest stand for no rows and are zeros)
            long_weight_grad_kernel<T><<<dim3((unsigned)ceil_div(a.channels, TB), (unsigned)parts), TB, 0, s>>>(p, chunk);
        }
        e = hipGetLastError();
    } else if (k.block) {
        row_grad_kernel<T, HELD, WHOLE, true><<<(unsigned)parts, k.threads, GRAD_TB / 64 * 4, s>>>(p);
        e = hipGetLastError();
    } else {
        e = k.n == 1   ? launch_held_grad<T, 1, WHOLE>(p, (unsigned)parts, s)
            : k.n == 2 ? launch_held_grad<T, 2, WHOLE>(p, (unsigned)parts, s)
                       : launch_held_grad<T, HELD, WHOLE>(p, (unsigned)parts, s);
    }
    if (e != hipSuccess || !a.dweight) return e;
    row_finish_kernel<T><<<(unsigned)ceil_div(a.channels, 16), FIN, 0, s>>>(a.part, (T *)a.dweight, a.channels, (int)parts);
    return hipGetLastError();
}
template <typename T> hipError_t launch_grad(const RowGradArgs &a, hipStream_t s) {
    return a.channels % vec<T>() == 0 ? launch_grad<T, true>(a, s) : launch_grad<T, false>(a, s);
}

}  // namespace

hipError_t launch_rms_norm(const RowArgs &a, hipStream_t s) { return launch_rows<NORM>(a, s); }
hipError_t launch_rms_norm_int8(const RowArgs &a, hipStream_t s) { return launch_rows<NORM8>(a, s); }
hipError_t launch_quantize(const RowArgs &a, hipStream_t s) { return launch_rows<QUANTIZE>(a, s); }

hipError_t launch_dequantize(int dtype, int64_t rows, int channels, const int8_t *codes, const float *scales, void *y, hipStream_t s) {
    if (rows == 0) return hipSuccess;
    switch (dtype) {
        case TVDCN_DTYPE_FLOAT32: return dequantize(rows, channels, codes, scales, (float *)y, s);
        case TVDCN_DTYPE_FLOAT16: return dequantize(rows, channels, codes, scales, (f16 *)y, s);
        default: return dequantize(rows, channels, codes, scales, (bf16 *)y, s);
    }
}

int64_t rms_norm_part_floats(const RowGradArgs &a) { return grad_parts(a) * a.channels; }

hipError_t launch_rms_norm_backward(const RowGradArgs &a, hipStream_t s) {
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return launch_grad<float>(a, s);
        case TVDCN_DTYPE_FLOAT16: return launch_grad<f16>(a, s);
        default: return launch_grad<bf16>(a, s);
    }
}

}  // namespace tvdcn_hip
