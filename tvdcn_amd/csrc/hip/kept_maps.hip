// 8-bit activations. A map [rows][channels] is kept as one int8 code per value and one exponent per block of 32
// channels of a row: k is the least exponent (at least -126) with max |x| <= 127 * 2^k, q = x / 2^k rounded to the
// nearest, ties to even. A power of two as the scale makes the scaling exact, so the code has one rounding, of at most
// half a step, 2^(k-1) <= max |x| / 127, and is the same however it is computed; values come back exactly representable
// in any of the map types. A block that holds an infinity or a NaN comes back as NaN: a fault in the forward is not
// hidden from the backward.
//
// Bound by memory: each value is read once, with 16-byte loads where the rows allow them; the lanes that share a block
// reduce its maximum by shuffles.
#include "maps.h"

namespace tvdcn_hip {
namespace {

constexpr int TB = 256;

// k + bias of a block whose largest magnitude has these bits: max = m 2^e with m in [1/2, 1), k = e - 7 where
// m <= 127/128, else e - 6
__device__ __forceinline__ int kept_exponent(uint32_t bits) {
    if (bits >= 0x7f800000u) return kKeptNaN;
    const int e = (int)(bits >> 23) - 126;                 // (a subnormal's is too low: the bound below holds it)
    const int k = (bits & 0x7fffffu) > 0x7e0000u ? e - 6 : e - 7;
    return max(k, -126) + kKeptBias;
}

// A lane holds VEC neighbouring channels, 32 / VEC lanes a block. Lanes of a row: a whole number of blocks.
template <typename T, int VEC>
__global__ void __launch_bounds__(TB) compress_kernel(const T *__restrict__ x, int8_t *__restrict__ codes,
                                                      uint8_t *__restrict__ exps, int64_t lanes, int C, int blocks) {
    constexpr int LPB = kKeptBlock / VEC;
    const int lanes_row = blocks * LPB;
    for (int64_t i = (int64_t)blockIdx.x * TB + threadIdx.x; i < lanes; i += (int64_t)gridDim.x * TB) {
        // lanes is a multiple of LPB and so is the stride: the lanes of a block run together
        const int64_t row = i / lanes_row;
        const int j = (int)(i - row * lanes_row), c = j * VEC;
        const bool in = c < C;   // (with VEC > 1 the channels are a multiple of VEC)
        Pack<T, VEC> p{};
        if (in) p = *reinterpret_cast<const Pack<T, VEC> *>(x + row * C + c);
        uint32_t big = 0;
#pragma unroll
        for (int v = 0; v < VEC; ++v) big = max(big, __float_as_uint((float)p.v[v]) & 0x7fffffffu);
#pragma unroll
        for (int m = 1; m < LPB; m <<= 1) big = max(big, (uint32_t)__shfl_xor((int)big, m));
        const int e = kept_exponent(big);
        // 2^-k: a normal float32 for every k from -126 to 122
        const float inv = __uint_as_float((uint32_t)(254 - (e == kKeptNaN ? 127 : e)) << 23);
        Pack<int8_t, VEC> q;
#pragma unroll
        for (int v = 0; v < VEC; ++v) q.v[v] = e == kKeptNaN ? (int8_t)0 : (int8_t)(int)rintf((float)p.v[v] * inv);
        if (in) {
            *reinterpret_cast<Pack<int8_t, VEC> *>(codes + row * C + c) = q;
            if (j % LPB == 0) exps[row * blocks + j / LPB] = (uint8_t)e;
        }
    }
}

// T: the type whose values the codes stand for (the clamp); D: the type written
template <typename T, typename D, int VEC>
__global__ void __launch_bounds__(TB) expand_kernel(const int8_t *__restrict__ codes, const uint8_t *__restrict__ exps,
                                                    D *__restrict__ y, int64_t lanes, int C, int lanes_row,
                                                    int64_t pitch) {
    const int blocks = (C + kKeptBlock - 1) / kKeptBlock;
    for (int64_t i = (int64_t)blockIdx.x * TB + threadIdx.x; i < lanes; i += (int64_t)gridDim.x * TB) {
        const int64_t row = i / lanes_row;
        const int c = (int)(i - row * lanes_row) * VEC;
        Pack<D, VEC> p{};
        if (c < C) {
            const Pack<int8_t, VEC> q = *reinterpret_cast<const Pack<int8_t, VEC> *>(codes + row * C + c);
            float f[VEC];
            kept_values<T, VEC>(q.v, exps[row * blocks + c / kKeptBlock], f);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                // (the one value beyond bfloat16 that a float32 block can stand for is the clamp itself)
                if (sizeof(D) < sizeof(T) && f[v] == f[v]) f[v] = fminf(fmaxf(f[v], -most<D>()), most<D>());
                p.v[v] = (D)f[v];
            }
        }
        *reinterpret_cast<Pack<D, VEC> *>(y + row * pitch + c) = p;
    }
}

unsigned grid_of(int64_t lanes) {
    const int64_t b = ceil_div(lanes, TB);
    return (unsigned)(b < 16384 ? b : 16384);   // 64 waves of 256 threads per CU in turn; the rest by the stride
}

template <typename T> hipError_t compress(int64_t rows, int C, const void *x, int8_t *codes, uint8_t *exps, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    const int blocks = (int)ceil_div(C, kKeptBlock);
    if (C % V == 0) {
        const int64_t lanes = rows * blocks * (kKeptBlock / V);
        compress_kernel<T, V><<<grid_of(lanes), TB, 0, s>>>((const T *)x, codes, exps, lanes, C, blocks);
    } else {
        const int64_t lanes = rows * blocks * kKeptBlock;
        compress_kernel<T, 1><<<grid_of(lanes), TB, 0, s>>>((const T *)x, codes, exps, lanes, C, blocks);
    }
    return hipGetLastError();
}

template <typename T, typename D>
hipError_t expand(int64_t rows, int C, int64_t pitch, const int8_t *codes, const uint8_t *exps, void *y, hipStream_t s) {
    constexpr int V = 16 / sizeof(D);
    if (C % V == 0 && pitch % V == 0) {
        const int64_t lanes = rows * (pitch / V);
        expand_kernel<T, D, V><<<grid_of(lanes), TB, 0, s>>>(codes, exps, (D *)y, lanes, C, (int)(pitch / V), pitch);
    } else {
        const int64_t lanes = rows * pitch;
        expand_kernel<T, D, 1><<<grid_of(lanes), TB, 0, s>>>(codes, exps, (D *)y, lanes, C, (int)pitch, pitch);
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_compress(int dtype, int64_t rows, int channels, const void *x, int8_t *codes, uint8_t *exps,
                           hipStream_t s) {
    if (rows == 0) return hipSuccess;
    switch (dtype) {
        case TVDCN_DTYPE_FLOAT32: return compress<float>(rows, channels, x, codes, exps, s);
        case TVDCN_DTYPE_FLOAT16: return compress<f16>(rows, channels, x, codes, exps, s);
        default: return compress<bf16>(rows, channels, x, codes, exps, s);
    }
}

hipError_t launch_expand(int dtype, bool as_bf16, int64_t rows, int channels, int64_t pitch, const int8_t *codes,
                         const uint8_t *exps, void *y, hipStream_t s) {
    if (rows == 0) return hipSuccess;
    switch (dtype) {
        case TVDCN_DTYPE_FLOAT32:
            return as_bf16 ? expand<float, bf16>(rows, channels, pitch, codes, exps, y, s)
                           : expand<float, float>(rows, channels, pitch, codes, exps, y, s);
        case TVDCN_DTYPE_FLOAT16: return expand<f16, f16>(rows, channels, pitch, codes, exps, y, s);
        default: return expand<bf16, bf16>(rows, channels, pitch, codes, exps, y, s);
    }
}

}  // namespace tvdcn_hip
