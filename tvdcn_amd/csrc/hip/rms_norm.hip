// Root-mean-square normalisation of every row [channels] of a channels-last map, of the map or of its sum with a shortcut, with
// its result in the map's type or in 8 bits, its gradients, and maps in 8 bits and back:
//
//   s = x + r (in the map's type),  rstd = (avg(s^2) + eps)^-1/2,  y = w s rstd
//   dh = w dy,  h = s rstd,  dx = rstd (dh - h avg(dh h)) + ds,  dw = sum over rows of dy h
//   scale = max(max |v| (1 / 127), 2^-126),  code = v / scale rounded, ties to even
//
// Bound by memory: a row stays in registers between the sums over it and its results, so every value is read once and written
// once. Rows are laid over as few lanes as hold them (a power of two, up to a wave, N accesses of 16 bytes each: several short
// rows to a wave), rows beyond a wave's registers over a workgroup. Rows beyond that are read again for each result that needs the
// whole row first: x (and r) twice for y, twice for the codes of a map, three times for those of a normalised row; backward x
// and dy twice for dx and once more for dw. (Rows that end within an access: Fit, below.)
//
// Sums are float32, in a fixed order. A mean beyond float32 is taken again of squares at 2^-160 of their size.
#include <algorithm>
#include <type_traits>

#include "rows.h"

namespace tvdcn_hip {
namespace {

constexpr int TB = 256;
constexpr int HELD = 4;         // accesses of a lane that holds its part of a long row
constexpr int HELD_TB = 512;    // lanes that hold a long row (at 1024 there are registers for less than their accesses)
constexpr int LONG_TB = 1024;   // lanes that read a longer one in turn
constexpr float LEAST_SCALE = 1.1754943508222875e-38f;   // 2^-126
constexpr float MOST_SCALE = 2.6793883890187504e+36f;     // 127 of it are finite

template <typename T> constexpr int vec() { return 16 / (int)sizeof(T); }

// How a row's accesses of VEC = 16 / sizeof(T) elements lie: WHOLE rows are made of whole ones, aligned; a LOOSE row's last one ends
// with the row and repeats elements of the one before it, which count once in the row's sums and are stored twice, the same
// (unaligned); TINY rows are shorter than one, and read and written by single elements.
enum Fit { WHOLE, LOOSE, TINY };

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
template <typename T, int N> struct __attribute__((packed, aligned(sizeof(T)))) Unaligned {
    T v[N];
};
template <typename T> struct Values {
    T v[vec<T>()];
};

// A lane's access i of a row: its first element, how many of its elements are another access's, whether it has any of its own
template <typename T, int FIT> struct Place {
    int c, over;
    bool on;
    __device__ __forceinline__ Place(int i, int C) {
        constexpr int VEC = vec<T>();
        const int at = i * VEC;
        on = at < C;
        c = FIT == LOOSE ? min(at, C - VEC) : at;
        over = FIT == LOOSE ? at - c : 0;
    }
    __device__ __forceinline__ bool own(int v) const { return FIT != LOOSE || v >= over; }
};

// (outside the row: zeros, or what another access has)
template <typename T, int FIT> __device__ __forceinline__ u32x4 load(const T *row, const Place<T, FIT> &k, int C) {
    if constexpr (FIT == WHOLE) {
        return k.on ? *reinterpret_cast<const u32x4 *>(row + k.c) : u32x4{0, 0, 0, 0};
    } else if constexpr (FIT == LOOSE) {
        return __builtin_bit_cast(u32x4, *reinterpret_cast<const Unaligned<T, vec<T>()> *>(row + k.c));
    } else {
        Values<T> o{};
#pragma unroll
        for (int v = 0; v < vec<T>() - 1; ++v)
            if (k.c + v < C) o.v[v] = row[k.c + v];
        return __builtin_bit_cast(u32x4, o);
    }
}
template <typename T, int FIT, typename D> __device__ __forceinline__ void store(D *row, const Place<T, FIT> &k, int C, const D *o) {
    constexpr int VEC = vec<T>();
    if (!k.on) return;
    if constexpr (FIT == WHOLE) {
        Pack<D, VEC> p;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.v[v] = o[v];
        *reinterpret_cast<Pack<D, VEC> *>(row + k.c) = p;
    } else if constexpr (FIT == LOOSE) {
        Unaligned<D, VEC> p;
#pragma unroll
        for (int v = 0; v < VEC; ++v) p.v[v] = o[v];
        *reinterpret_cast<Unaligned<D, VEC> *>(row + k.c) = p;
    } else {
#pragma unroll
        for (int v = 0; v < VEC - 1; ++v)
            if (k.c + v < C) row[k.c + v] = o[v];
    }
}
template <typename T> __device__ __forceinline__ void widen(const u32x4 &raw, float *f) {
    const Values<T> o = __builtin_bit_cast(Values<T>, raw);
#pragma unroll
    for (int v = 0; v < vec<T>(); ++v) f[v] = (float)o.v[v];
}
template <typename T> __device__ __forceinline__ void narrow(const float *f, T *o) {
#pragma unroll
    for (int v = 0; v < vec<T>(); ++v) o[v] = (T)f[v];
}
// x as it is now: what is made of it from here on is made again, not kept from before
__device__ __forceinline__ void anew(u32x4 &x) { asm volatile("" : "+v"(x)); }

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

// The reciprocal root of a row whose squares `squares(f)` sums, of its values times f. Where the mean is no float32, the values are taken at
// 2^-80 of their size: the largest square is then 2^96, 2^20 channels of them 2^116, and what made the mean infinite (a sum of 2^128,
// or eps) is 2^-52 at least, beside which what vanishes below float32 does not count. (2^-160 itself is no float32: eps takes 2^-80
// twice.) The mean is the same for all lanes of the row, and so is the way taken.
constexpr float DOWN = 8.271806125530277e-25f;   // 2^-80
static_assert(DOWN * 1099511627776.f * 1099511627776.f == 1.f, "");
template <typename F> __device__ __forceinline__ float reciprocal_root(F &&squares, float inv_channels, float eps) {
    const float mean = fmaf(squares(1.f), inv_channels, eps);
    if (mean != __builtin_inff()) return 1.f / sqrtf(mean);
    return DOWN / sqrtf(fmaf(squares(DOWN), inv_channels, eps * DOWN * DOWN));
}

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

// f += r, rounded to the type, which `sum` receives
template <typename T> __device__ __forceinline__ void add_in_type(float *f, const u32x4 &r, T *sum) {
    float g[vec<T>()];
    widen<T>(r, g);
#pragma unroll
    for (int v = 0; v < vec<T>(); ++v) {
        sum[v] = (T)(f[v] + g[v]);
        f[v] = (float)sum[v];
    }
}

// A lane has N accesses of a row. BLOCK: a row is a workgroup's, otherwise 2^log2 lanes of a wave's. The next row's loads are on
// their way while a row is worked on.
template <typename T, int N, int FIT, int MODE, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? HELD_TB : TB) row_kernel(RowKernelArgs a) {
    constexpr int VEC = vec<T>();
    __shared__ float red[BLOCK ? HELD_TB / 64 : 1];
    const int t = threadIdx.x, C = a.channels;
    const int lanes = BLOCK ? (int)blockDim.x : 1 << a.log2, l = t & (lanes - 1);
    const int per = BLOCK ? 1 : TB >> a.log2;   // rows of a workgroup
    const bool added = MODE != QUANTIZE && a.residual;
    auto place = [&](int n) { return Place<T, FIT>(n * lanes + l, C); };
    float w[N][VEC];
    if constexpr (MODE != QUANTIZE)
#pragma unroll
        for (int n = 0; n < N; ++n) {
            if (a.weight) {
                widen<T>(load<T, FIT>((const T *)a.weight, place(n), C), w[n]);
            } else {
#pragma unroll
                for (int v = 0; v < VEC; ++v) w[n][v] = 1.f;
            }
        }
    u32x4 x[N], r[N];
    auto fetch = [&](int64_t row) {
#pragma unroll
        for (int n = 0; n < N; ++n) x[n] = load<T, FIT>((const T *)a.x + row * C, place(n), C);
        if (added)
#pragma unroll
            for (int n = 0; n < N; ++n) r[n] = load<T, FIT>((const T *)a.residual + row * C, place(n), C);
    };
    const int64_t stride = (int64_t)gridDim.x * per;
    int64_t row = (int64_t)blockIdx.x * per + (BLOCK ? 0 : t >> a.log2);
    if (row < a.rows) fetch(row);
    for (; row < a.rows; row += stride) {
        const int64_t at = row * C;
        float f[N][VEC];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            widen<T>(x[n], f[n]);
            if (added) {
                T sum[VEC];
                add_in_type<T>(f[n], r[n], sum);
                store<T, FIT>((T *)a.sum + at, place(n), C, sum);
            }
        }
        if (row + stride < a.rows) fetch(row + stride);
        if constexpr (MODE != QUANTIZE) {
            auto squares = [&](float down) {
                float ss = 0.f;
#pragma unroll
                for (int n = 0; n < N; ++n)
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const float s = place(n).own(v) ? f[n][v] * down : 0.f;
                        ss = fmaf(s, s, ss);
                    }
                return over_row<Add, BLOCK>(ss, a.log2, red);
            };
            const float rstd = reciprocal_root(squares, a.inv_channels, a.eps);
            if (a.rstd && l == 0) a.rstd[row] = rstd;
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[n][v] = f[n][v] * rstd * w[n][v];
        }
        if constexpr (MODE == NORM) {
#pragma unroll
            for (int n = 0; n < N; ++n) {
                T o[VEC];
                narrow<T>(f[n], o);
                store<T, FIT>((T *)a.y + at, place(n), C, o);
            }
        } else {
            float big = 0.f;   // (outside the row: zeros, another access's values, or NaN as all of the row)
#pragma unroll
            for (int n = 0; n < N; ++n)
#pragma unroll
                for (int v = 0; v < VEC; ++v) big = Most::of(big, fabsf(f[n][v]));
            const float scale = scale_of(over_row<Most, BLOCK>(big, a.log2, red));
            if (l == 0) a.scales[row] = scale;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                int8_t q[VEC] = {};
                if (scale == scale) codes_of<VEC>(f[n], scale, q);
                store<T, FIT>(a.codes + at, place(n), C, q);
            }
        }
    }
}

// Rows beyond a workgroup's registers: read for the sum of squares (and written as the sum with the shortcut), for the largest magnitude where
// there are codes, and for the results (2048 x 32768 bfloat16 with the sum: 8 bits 141-151 us)
template <typename T, int FIT, int MODE> __global__ void __launch_bounds__(LONG_TB) long_row_kernel(RowKernelArgs a) {
    constexpr int VEC = vec<T>();
    __shared__ float red[LONG_TB / 64];
    const int t = threadIdx.x, C = a.channels;
    const bool added = MODE != QUANTIZE && a.residual;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = row * C;
        auto values = [&](const Place<T, FIT> &k, float *f, bool write) {
            widen<T>(load<T, FIT>((const T *)a.x + at, k, C), f);
            if (!added) return;
            T sum[VEC];
            add_in_type<T>(f, load<T, FIT>((const T *)a.residual + at, k, C), sum);
            if (write) store<T, FIT>((T *)a.sum + at, k, C, sum);
        };
        float rstd = 1.f;
        if constexpr (MODE != QUANTIZE) {
            auto squares = [&](float down) {
                float ss = 0.f;
                for (int i = t; i * VEC < C; i += LONG_TB) {
                    const Place<T, FIT> k(i, C);
                    float f[VEC];
                    values(k, f, down == 1.f);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const float s = k.own(v) ? f[v] * down : 0.f;
                        ss = fmaf(s, s, ss);
                    }
                }
                return over_row<Add, true>(ss, 6, red);
            };
            rstd = reciprocal_root(squares, a.inv_channels, a.eps);
            if (a.rstd && t == 0) a.rstd[row] = rstd;
        }
        auto result = [&](const Place<T, FIT> &k, float *f) {
            values(k, f, false);
            if constexpr (MODE != QUANTIZE) {
                float w[VEC];
                if (a.weight) widen<T>(load<T, FIT>((const T *)a.weight, k, C), w);
#pragma unroll
                for (int v = 0; v < VEC; ++v) f[v] = f[v] * rstd * (a.weight ? w[v] : 1.f);
            }
        };
        if constexpr (MODE == NORM) {
            for (int i = t; i * VEC < C; i += LONG_TB) {
                const Place<T, FIT> k(i, C);
                float f[VEC];
                T o[VEC];
                result(k, f);
                narrow<T>(f, o);
                store<T, FIT>((T *)a.y + at, k, C, o);
            }
        } else {
            float big = 0.f;
            for (int i = t; i * VEC < C; i += LONG_TB) {
                float f[VEC];
                result(Place<T, FIT>(i, C), f);
#pragma unroll
                for (int v = 0; v < VEC; ++v) big = Most::of(big, fabsf(f[v]));
            }
            const float scale = scale_of(over_row<Most, true>(big, 6, red));
            if (t == 0) a.scales[row] = scale;
            for (int i = t; i * VEC < C; i += LONG_TB) {
                const Place<T, FIT> k(i, C);
                float f[VEC];
                int8_t q[VEC] = {};
                result(k, f);
                if (scale == scale) codes_of<VEC>(f, scale, q);
                store<T, FIT>(a.codes + at, k, C, q);
            }
        }
    }
}

template <typename T, int FIT>
__global__ void __launch_bounds__(TB) dequantize_kernel(int64_t rows, int C, int log2, const int8_t *__restrict__ codes,
                                                        const float *__restrict__ scales, T *__restrict__ y) {
    constexpr int VEC = vec<T>();
    const int lanes = 1 << log2, l = threadIdx.x & (lanes - 1), per = TB >> log2;
    for (int64_t row = (int64_t)blockIdx.x * per + (threadIdx.x >> log2); row < rows; row += (int64_t)gridDim.x * per) {
        const float scale = scales[row];
        const int8_t *from = codes + row * C;
        for (int i = l; i * VEC < C; i += lanes) {
            const Place<T, FIT> k(i, C);
            Unaligned<int8_t, VEC> q{};
            if constexpr (FIT == WHOLE) {
                const Pack<int8_t, VEC> p = *reinterpret_cast<const Pack<int8_t, VEC> *>(from + k.c);
#pragma unroll
                for (int v = 0; v < VEC; ++v) q.v[v] = p.v[v];
            } else if constexpr (FIT == LOOSE) {
                q = *reinterpret_cast<const Unaligned<int8_t, VEC> *>(from + k.c);
            } else {
#pragma unroll
                for (int v = 0; v < VEC - 1; ++v)
                    if (k.c + v < C) q.v[v] = from[k.c + v];
            }
            T o[VEC];
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] = (T)((float)q.v[v] * scale);
            store<T, FIT>(y + row * C, k, C, o);
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
    float *part;     // [workgroups][channels], or null
    void *dweight;   // the weight's gradient itself, where one workgroup has all rows; or null
};

// Maps stay as they were read, in the map's type: the second use widens them again, since as float32 a long row of a 16-bit map
// would fill the registers (65536 x 2048: 292 us so, two waves to a SIMD).
template <typename T, int N, int FIT, bool BLOCK>
__global__ void __launch_bounds__(BLOCK ? HELD_TB : TB) row_grad_kernel(RowGradKernelArgs a) {
    constexpr int VEC = vec<T>();
    extern __shared__ float shared[];   // BLOCK: a word per wave; otherwise [waves][lanes * N * VEC]
    const int t = threadIdx.x, C = a.channels;
    const int lanes = BLOCK ? (int)blockDim.x : 1 << a.log2, l = t & (lanes - 1);
    const int per = BLOCK ? 1 : TB >> a.log2;
    auto place = [&](int n) { return Place<T, FIT>(n * lanes + l, C); };
    u32x4 w[N];
    float dw[N][VEC];
#pragma unroll
    for (int n = 0; n < N; ++n) {
        if (a.weight) w[n] = load<T, FIT>((const T *)a.weight, place(n), C);
#pragma unroll
        for (int v = 0; v < VEC; ++v) dw[n][v] = 0.f;
    }
    auto weights = [&](int n, float *f) {
        if (a.weight) {
            widen<T>(w[n], f);
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) f[v] = 1.f;
        }
    };
    for (int64_t row = (int64_t)blockIdx.x * per + (BLOCK ? 0 : t >> a.log2); row < a.rows; row += (int64_t)gridDim.x * per) {
        const int64_t at = row * C;
        u32x4 x[N], dy[N], ds[N];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            x[n] = load<T, FIT>((const T *)a.x + at, place(n), C);
            dy[n] = load<T, FIT>((const T *)a.dy + at, place(n), C);
        }
        if (a.dsum)
#pragma unroll
            for (int n = 0; n < N; ++n) ds[n] = load<T, FIT>((const T *)a.dsum + at, place(n), C);
        const float rstd = a.rstd[row];
        float dot = 0.f;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            float fx[VEC], fd[VEC], fw[VEC];
            widen<T>(x[n], fx), widen<T>(dy[n], fd), weights(n, fw);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float h = fx[v] * rstd;
                dw[n][v] = fmaf(fd[v], h, dw[n][v]);
                dot = fmaf(place(n).own(v) ? fd[v] * fw[v] : 0.f, h, dot);
            }
        }
        if (a.dx) {
            dot = over_row<Add, BLOCK>(dot, a.log2, shared) * a.inv_channels;
#pragma unroll
            for (int n = 0; n < N; ++n) {
                if constexpr (N > 1) anew(x[n]), anew(dy[n]), anew(w[n]);
                float fx[VEC], fd[VEC], fw[VEC], fs[VEC] = {};
                widen<T>(x[n], fx), widen<T>(dy[n], fd), weights(n, fw);
                if (a.dsum) widen<T>(ds[n], fs);
                T o[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) o[v] = (T)fmaf(rstd, fmaf(-(fx[v] * rstd), dot, fd[v] * fw[v]), fs[v]);
                store<T, FIT>((T *)a.dx + at, place(n), C, o);
            }
        }
    }
    if (!a.part && !a.dweight) return;
    auto put = [&](int c, float v) {
        if (a.dweight) ((T *)a.dweight)[c] = (T)v;
        else a.part[(int64_t)blockIdx.x * C + c] = v;
    };
    if constexpr (BLOCK) {
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int v = 0; v < VEC; ++v)
                if (place(n).on && place(n).c + v < C) put(place(n).c + v, dw[n][v]);
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
                if ((t & 63) < lanes && place(n).on) shared[wave * width + place(n).c + v] = s;
            }
        __syncthreads();
        for (int c = t; c < C; c += TB) {
            float s = shared[c];
#pragma unroll
            for (int k = 1; k < TB / 64; ++k) s += shared[k * width + c];
            put(c, s);
        }
    }
}

// Rows beyond a workgroup's registers: dx row by row in two readings, the weight's gradient column by column
template <typename T, int FIT> __global__ void __launch_bounds__(LONG_TB) long_row_grad_kernel(RowGradKernelArgs a) {
    constexpr int VEC = vec<T>();
    __shared__ float red[LONG_TB / 64];
    const int t = threadIdx.x, C = a.channels;
    for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const int64_t at = row * C;
        const float rstd = a.rstd[row];
        auto read = [&](const Place<T, FIT> &k, float *h, float *dh) {
            float w[VEC];
            widen<T>(load<T, FIT>((const T *)a.x + at, k, C), h);
            widen<T>(load<T, FIT>((const T *)a.dy + at, k, C), dh);
            if (a.weight) widen<T>(load<T, FIT>((const T *)a.weight, k, C), w);
#pragma unroll
            for (int v = 0; v < VEC; ++v) h[v] *= rstd, dh[v] *= a.weight ? w[v] : 1.f;
        };
        float dot = 0.f;
        for (int i = t; i * VEC < C; i += LONG_TB) {
            const Place<T, FIT> k(i, C);
            float h[VEC], dh[VEC];
            read(k, h, dh);
#pragma unroll
            for (int v = 0; v < VEC; ++v) dot = fmaf(k.own(v) ? dh[v] : 0.f, h[v], dot);
        }
        dot = over_row<Add, true>(dot, 6, red) * a.inv_channels;
        for (int i = t; i * VEC < C; i += LONG_TB) {
            const Place<T, FIT> k(i, C);
            float h[VEC], dh[VEC], ds[VEC] = {};
            T o[VEC];
            read(k, h, dh);
            if (a.dsum) widen<T>(load<T, FIT>((const T *)a.dsum + at, k, C), ds);
#pragma unroll
            for (int v = 0; v < VEC; ++v) o[v] = (T)fmaf(rstd, fmaf(-h[v], dot, dh[v]), ds[v]);
            store<T, FIT>((T *)a.dx + at, k, C, o);
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
// grad: two accesses of more lanes, where there are as many, leave registers for twice the waves
RowShape row_shape(int channels, int vec, bool grad) {
    const int packs = (int)ceil_div(channels, vec);
    RowShape k{0, 1, 0, false};
    if (packs <= 64 * HELD) {
        while (k.log2 < 6 && 1 << k.log2 < packs) ++k.log2;
        while (k.n << k.log2 < packs) k.n *= 2;
        return k;
    }
    k.block = true;
    k.n = grad && packs <= 2 * HELD_TB ? 2 : HELD;
    for (k.threads = 128; k.threads < HELD_TB && k.threads * k.n < packs;) k.threads *= 2;
    if (k.threads * k.n < packs) k.threads = 0;
    return k;
}

// Workgroups of the forward: eight times what is there at once, so that the quick ones go on (65536 x 2048 bfloat16 into 8 bits:
// 1024 / 2048 / 4096 / 8192 workgroups take 84 / 84 / 80 / 77 us; 131072 x 71 12.5 / 11.8 / 11.6 / 13.2 normalised)
constexpr int64_t MOST_GROUPS = 8192;
unsigned row_grid(int64_t units, int64_t most) { return (unsigned)std::min(units, most); }

// calls f with the Fit of rows of this type and length as a constant
template <typename T, typename F> hipError_t with_fit(int channels, F &&f) {
    if (channels % vec<T>() == 0) return f(std::integral_constant<int, WHOLE>());
    if (channels > vec<T>()) return f(std::integral_constant<int, LOOSE>());
    return f(std::integral_constant<int, TINY>());
}

template <typename T, int MODE> hipError_t launch_rows(const RowArgs &a, hipStream_t s) {
    const RowShape k = row_shape(a.channels, vec<T>(), false);
    const RowKernelArgs p{a.rows, a.channels, k.log2, (float)(1.0 / a.channels), a.eps, a.x, a.residual, a.weight,
                          a.sum, a.y, a.rstd, a.scales, a.codes};
    return with_fit<T>(a.channels, [&](auto fit) {
        constexpr int FIT = decltype(fit)::value;
        const unsigned grid = row_grid(ceil_div(a.rows, TB >> k.log2), MOST_GROUPS);
        if constexpr (FIT == TINY) {
            row_kernel<T, 1, FIT, MODE, false><<<grid, TB, 0, s>>>(p);
        } else if (k.block) {
            if (k.threads) row_kernel<T, HELD, FIT, MODE, true><<<row_grid(a.rows, MOST_GROUPS), k.threads, 0, s>>>(p);
            else long_row_kernel<T, FIT, MODE><<<row_grid(a.rows, 1024), LONG_TB, 0, s>>>(p);
        } else if (k.n == 1) {
            row_kernel<T, 1, FIT, MODE, false><<<grid, TB, 0, s>>>(p);
        } else if (k.n == 2) {
            row_kernel<T, 2, FIT, MODE, false><<<grid, TB, 0, s>>>(p);
        } else {
            row_kernel<T, HELD, FIT, MODE, false><<<grid, TB, 0, s>>>(p);
        }
        return hipGetLastError();
    });
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
    return with_fit<T>(channels, [&](auto fit) {
        dequantize_kernel<T, decltype(fit)::value><<<grid, TB, 0, s>>>(rows, channels, log2, codes, scales, y);
        return hipGetLastError();
    });
}

// Workgroups of the backward: each keeps a part of the weight's gradient. One alone writes the gradient itself: where it has up to
// four rounds of rows, which take less than the launch that would add up the parts.
int64_t grad_parts(const RowGradArgs &a) {
    const RowShape k = row_shape(a.channels, a.dtype == TVDCN_DTYPE_FLOAT32 ? 4 : 8, true);
    if (k.block && !k.threads) return std::min<int64_t>(a.rows, 256);
    const int64_t units = k.block ? a.rows : ceil_div(a.rows, TB >> k.log2);
    // (long rows: the parts of 1024 would be a quarter of what 4096 x 8192 reads and writes)
    return units > 0 && units <= 4 ? 1 : std::min<int64_t>(units, k.block ? 512 : 1024);
}

template <typename T> hipError_t launch_grad(const RowGradArgs &a, hipStream_t s) {
    const RowShape k = row_shape(a.channels, vec<T>(), true);
    const int64_t parts = grad_parts(a);
    const bool in_turn = k.block && !k.threads, alone = parts == 1 && !in_turn;
    RowGradKernelArgs p{a.rows, a.channels, k.log2, (float)(1.0 / a.channels), a.dy, a.dsum, a.x, a.weight, a.rstd, a.dx,
                        a.dweight && !alone ? a.part : nullptr, alone ? a.dweight : nullptr};
    const hipError_t e = a.rows == 0 ? hipSuccess : with_fit<T>(a.channels, [&](auto fit) {
        constexpr int FIT = decltype(fit)::value;
        const unsigned grid = (unsigned)parts, bytes = (TB / 64) * (k.n << k.log2) * vec<T>() * 4;
        if constexpr (FIT == TINY) {
            row_grad_kernel<T, 1, FIT, false><<<grid, TB, bytes, s>>>(p);
        } else if (in_turn) {
            if (a.dx) long_row_grad_kernel<T, FIT><<<row_grid(a.rows, 1024), LONG_TB, 0, s>>>(p);
            if (hipError_t e = hipGetLastError()) return e;
            // (fewer chunks than parts where they do not divide: the rest stand for no rows and are zeros)
            if (a.dweight)
                long_weight_grad_kernel<T><<<dim3((unsigned)ceil_div(a.channels, TB), grid), TB, 0, s>>>(p, ceil_div(a.rows, parts));
        } else if (k.block) {
            const auto kernel = k.n == 2 ? row_grad_kernel<T, 2, FIT, true> : row_grad_kernel<T, HELD, FIT, true>;
            kernel<<<grid, k.threads, HELD_TB / 64 * 4, s>>>(p);
        } else if (k.n == 1) {
            row_grad_kernel<T, 1, FIT, false><<<grid, TB, bytes, s>>>(p);
        } else if (k.n == 2) {
            row_grad_kernel<T, 2, FIT, false><<<grid, TB, bytes, s>>>(p);
        } else {
            row_grad_kernel<T, HELD, FIT, false><<<grid, TB, bytes, s>>>(p);
        }
        return hipGetLastError();
    });
    if (e != hipSuccess || !a.dweight || alone) return e;
    row_finish_kernel<T><<<(unsigned)ceil_div(a.channels, 16), FIN, 0, s>>>(a.part, (T *)a.dweight, a.channels, (int)parts);
    return hipGetLastError();
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
