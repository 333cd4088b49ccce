// Dropout whose mask is never stored: y = (kept ? x / (1 - p) : 0) + r, where what is kept follows from the seed and a value's
// place in the channels-last map alone, so the backward makes the same mask again (the same kernel on the gradient).
//
// Random bits: Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", 2011). Key: the seed's two
// halves; counter: the number of a group of eight values, in the map's memory order. Value j of the group has the low (j even) or high
// half of word j / 2, and is dropped where that is below `drop`: 16 bits a value take a quarter of the multiplications that
// 64 would, and make p a multiple of 2^-16 (the scale is that p's).
//
// Bound by memory: 16 bytes a lane, the ten rounds (20 products of 32 x 32 bits for eight values) beside them.
#include "rows.h"

namespace tvdcn_hip {
namespace {

constexpr int TB = 256, GROUP = 8;

__device__ __forceinline__ void philox(uint64_t counter, uint32_t k0, uint32_t k1, uint32_t *o) {
    uint32_t c0 = (uint32_t)counter, c1 = (uint32_t)(counter >> 32), c2 = 0, c3 = 0;
#pragma unroll
    for (int i = 0; i < 10; ++i) {
        const uint64_t a = (uint64_t)c0 * 0xD2511F53u, b = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(b >> 32) ^ c1 ^ k0, c1 = (uint32_t)b;
        c2 = (uint32_t)(a >> 32) ^ c3 ^ k1, c3 = (uint32_t)a;
        k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
    }
    o[0] = c0, o[1] = c1, o[2] = c2, o[3] = c3;
}

template <typename T>
__global__ void __launch_bounds__(TB) dropout_kernel(const T *__restrict__ x, const T *__restrict__ residual, T *__restrict__ y,
                                                     const int64_t *__restrict__ seed, int64_t n, uint32_t drop, float scale) {
    const uint64_t key = (uint64_t)*seed;
    typedef Pack<T, GROUP> P;
    for (int64_t g = (int64_t)blockIdx.x * TB + threadIdx.x; g * GROUP < n; g += (int64_t)gridDim.x * TB) {
        const int64_t at = g * GROUP;
        const bool whole = at + GROUP <= n;
        P v{}, r{}, o;
        if (whole) {
            v = *reinterpret_cast<const P *>(x + at);
            if (residual) r = *reinterpret_cast<const P *>(residual + at);
        } else {
#pragma unroll
            for (int e = 0; e < GROUP; ++e)
                if (at + e < n) {
                    v.v[e] = x[at + e];
                    if (residual) r.v[e] = residual[at + e];
                }
        }
        uint32_t bits[4];
        philox((uint64_t)g, (uint32_t)key, (uint32_t)(key >> 32), bits);
#pragma unroll
        for (int e = 0; e < GROUP; ++e) {
            const uint32_t u = e % 2 ? bits[e / 2] >> 16 : bits[e / 2] & 0xffffu;
            // (a dropped value is none, whatever it holds; without a shortcut nothing is added: -0 stays -0)
            const float f = u >= drop ? (float)v.v[e] * scale : 0.f;
            o.v[e] = (T)(residual ? f + (float)r.v[e] : f);
        }
        if (whole) {
            *reinterpret_cast<P *>(y + at) = o;
        } else {
#pragma unroll
            for (int e = 0; e < GROUP; ++e)
                if (at + e < n) y[at + e] = o.v[e];
        }
    }
}

template <typename T>
hipError_t dropout(int64_t n, int drop, const int64_t *seed, const void *x, const void *residual, void *y, hipStream_t s) {
    const int64_t blocks = ceil_div(ceil_div(n, GROUP), TB);
    const float scale = drop < 65536 ? (float)(65536.0 / (65536 - drop)) : 0.f;
    dropout_kernel<T><<<(unsigned)(blocks < 16384 ? blocks : 16384), TB, 0, s>>>((const T *)x, (const T *)residual, (T *)y, seed, n,
                                                                                 (uint32_t)drop, scale);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_dropout(int dtype, int64_t n, int drop, const int64_t *seed, const void *x, const void *residual, void *y,
                          hipStream_t s) {
    if (n == 0) return hipSuccess;
    switch (dtype) {
        case TVDCN_DTYPE_FLOAT32: return dropout<float>(n, drop, seed, x, residual, y, s);
        case TVDCN_DTYPE_FLOAT16: return dropout<f16>(n, drop, seed, x, residual, y, s);
        default: return dropout<bf16>(n, drop, seed, x, residual, y, s);
    }
}

}  // namespace tvdcn_hip
