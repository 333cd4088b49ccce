// The pointwise convolution of an 8-bit map with 8-bit weights: y = act(sx sw sum(q qw) + b) + r, with a scale sx per row and sw per
// output channel. The sums are whole numbers, exact in 32 bits up to 131071 channels (2^17 products of at most 2^14).
//
// The kernels are those of product_kernels.h on 16x16x64 MFMAs: twice the products per instruction and byte of the 16-bit ones.
// Channels that are no multiple of 16 are copied to rows that are, with zeros behind them.
#include "product_kernels.h"
#include "rows.h"

namespace tvdcn_hip {
namespace {

constexpr int TB = 256;

// Rows of C bytes to rows of 16 lanes_row bytes, zeros behind them; both operands in one launch
struct CodeCopy {
    const int8_t *from;
    int8_t *to;
    int64_t rows;
};
__global__ void __launch_bounds__(TB) pad_codes_kernel(CodeCopy first, CodeCopy second, int C, int lanes_row, int64_t lanes_first, int64_t lanes) {
    for (int64_t n = (int64_t)blockIdx.x * TB + threadIdx.x; n < lanes; n += (int64_t)gridDim.x * TB) {
        const CodeCopy &m = n < lanes_first ? first : second;
        const int64_t i = n < lanes_first ? n : n - lanes_first, row = i / lanes_row;
        const int c = (int)(i - row * lanes_row) * 16;
        const int8_t *p = m.from + row * C + c;
        Pack<int8_t, 16> o{};
        if (c + 16 <= C) {
            __builtin_memcpy(&o, p, 16);
        } else {
#pragma unroll
            for (int v = 0; v < 15; ++v)
                if (c + v < C) o.v[v] = p[v];
        }
        *reinterpret_cast<Pack<int8_t, 16> *>(m.to + i * 16) = o;
    }
}

struct Plan {
    int64_t pitch;
    bool copies;
    size_t w_at, x_at, bytes;
};
Plan plan(const Int8ProductArgs &a) {
    Plan k{};
    k.pitch = round_up(a.in, 16);
    k.copies = a.in % 16 != 0;
    if (k.copies) {
        k.x_at = round_up(a.out * k.pitch, 256);
        k.bytes = k.x_at + a.rows * k.pitch;
    }
    return k;
}

template <typename T> hipError_t product(const Int8ProductArgs &a, hipStream_t s) {
    const Plan k = plan(a);
    const int8_t *x = a.codes, *w = a.weight_codes;
    if (k.copies) {
        const int lanes_row = (int)(k.pitch / 16);
        CodeCopy first{x, (int8_t *)a.work + k.x_at, a.rows}, second{w, (int8_t *)a.work, a.out};
        const int64_t lanes = (a.rows + a.out) * lanes_row, blocks = ceil_div(lanes, TB);
        pad_codes_kernel<<<(unsigned)(blocks < 16384 ? blocks : 16384), TB, 0, s>>>(first, second, a.in, lanes_row, a.rows * lanes_row, lanes);
        if (hipError_t e = hipGetLastError()) return e;
        x = first.to, w = second.to;
    }
    const int64_t half = k.pitch / 2;   // in elements of two codes
    Product p{};
    p.C = {w, half, a.out * half, half, a.out};
    p.cols = a.out;
    p.splits = 1;
    p.share = half;
    p.bias = a.bias;
    p.act = a.act;
    p.scale_c = a.weight_scales;
    // rows in runs whose workgroups HIP takes in one launch
    const int64_t run = (int64_t)(1 << 22) / ceil_div(a.out, 64) * 64;
    for (int64_t first = 0; first < a.rows; first += run) {
        p.rows = (int)std::min(a.rows - first, run);
        p.R = {x + first * k.pitch, half, p.rows * half, half, p.rows};
        p.out = (T *)a.y + first * a.out;
        p.residual = a.residual ? (const T *)a.residual + first * a.out : nullptr;
        p.scale_r = a.scales + first;
        const double steps = (double)ceil_div(half, 64);
        auto tiles = [&](int r, int c) { return ceil_div(p.rows, r) * ceil_div(p.cols, c); };
        hipError_t e;
        (void)steps;
        if (p.cols % 8 == 0 && tiles(256, 256) >= 256) e = launch_wide<T, false, false, 4, Codes>(p, s);
        else if (p.cols % 8 == 0 && tiles(256, 128) >= 256) e = launch_wide<T, false, false, 2, Codes>(p, s);
        else if (tiles(128, 128) >= 512) e = launch_tiles<T, false, false, 2, 2, 4, 4, 2, 2, Codes>(p, s);
        else e = launch_tiles<T, false, false, 2, 2, 2, 2, 3, 2, Codes>(p, s);
        if (e) return e;
    }
    return hipSuccess;
}

}  // namespace

size_t pointwise_int8_bytes(const Int8ProductArgs &a) { return a.rows == 0 ? 0 : plan(a).bytes; }

hipError_t launch_pointwise_int8(const Int8ProductArgs &a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return product<float>(a, s);
        case TVDCN_DTYPE_FLOAT16: return product<f16>(a, s);
        default: return product<bf16>(a, s);
    }
}

}  // namespace tvdcn_hip
