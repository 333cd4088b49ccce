// The pointwise convolution of an 8-bit map with 8-bit weights: y = act(sx sw sum(q qw) + b) + r, with a scale sx per row and sw per
// output channel. The sums are whole numbers, exact in 32 bits up to 131071 channels (2^17 products of at most 2^14).
//
// Large products take the tiles of product_kernels.h on 16x16x64 MFMAs: twice the products per instruction and byte of the 16-bit
// ones. Channels that are no multiple of 16 are copied to rows that are, with zeros behind them. Small products have a kernel of
// their own, without copies.
//
// 8192 x 8192 to 8192 runs at 2590 to 2680 TOP/s (a plain library product of 8-bit integers: 2150). With few channels the results bound
// it. 65536 x 2048 to 512, 64 us of products at the library's rate: 66-68 us, 71-76 with a residual, 75-78 with gelu; float32 results
// 77 and 105-108 with a residual (80 of reading and writing). 65536 x 512 to 2048, the same products: 100-104, 137-140 and 141-149;
// float32 151-156, 258 with a residual (220 of reading and writing), 255-261 with gelu. A tile's stores come from all CUs at about the same
// time, and only the next tile's first stage overlaps them (none where a float32 residual is read, whose loads are not counted): two
// workgroups of 256 x 128 to a CU, one storing while the other multiplies, ran at 1920 TOP/s and were slower throughout. Rows that are no
// whole 16 bytes are copied first: 65536 x 2040 to 512 takes 118-123 us, 65536 x 520 to 2048 135 and 186 with gelu. A reduction is not split
// over workgroups: 1, 16, 64, 256 and 1024 x 4096 to 4096 take 5, 7, 12, 16 and 43 us, of which 3, 3, 4, 4 and 16 are memory and products.
#include <cmath>

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

// Small products, straight from memory (the caches) to the MFMAs: a lane's 16 bytes along the reduction are 16 bytes of a row, at
// any alignment, so neither LDS stages nor copies are needed, and there are workgroups enough where 64 x 64 tiles leave most of the
// chip idle: 1 x 2048 to 512 takes 3.8 us (64 x 64 tiles 8.4), 256 x 512 to 2048 5.5 (5.8), 2048 x 71 to 101 3.8 (7.7 with its copy).
// A workgroup has 16 columns of 16 MF rows; its four waves take 64 bytes of the reduction in turn and add up through LDS.
//
// WHOLE: rows of whole 16 bytes. Otherwise (at least 16 bytes a row) the 16 bytes at a row's end are read and shifted down, which
// leaves zeros behind it.
template <bool WHOLE> __device__ __forceinline__ i32x4 load_codes(const int8_t *row, int k, int K) {
    if constexpr (WHOLE) {
        return k < K ? *reinterpret_cast<const i32x4 *>(row + k) : i32x4{0, 0, 0, 0};
    } else {
        if (k >= K) return i32x4{0, 0, 0, 0};
        const int over = max(k + 16 - K, 0);   // bytes past the row's end
        uint32_t v[4];
        __builtin_memcpy(v, row + (k - over), 16);
        if (over) {
            if (over & 8) v[0] = v[2], v[1] = v[3], v[2] = v[3] = 0;
            if (over & 4) v[0] = v[1], v[1] = v[2], v[2] = v[3], v[3] = 0;
            const int bits = (over & 3) * 8;
            v[0] = __builtin_amdgcn_alignbit(v[1], v[0], bits), v[1] = __builtin_amdgcn_alignbit(v[2], v[1], bits);
            v[2] = __builtin_amdgcn_alignbit(v[3], v[2], bits), v[3] >>= bits;
        }
        return i32x4{(int)v[0], (int)v[1], (int)v[2], (int)v[3]};
    }
}

template <typename T, int MF, bool WHOLE>
__global__ void __launch_bounds__(TB) direct_product_kernel(Product p, const int8_t *__restrict__ x, const int8_t *__restrict__ w, int K) {
    constexpr int WAVES = TB / 64, STEP = WAVES * 64;
    constexpr int AHEAD = MF == 1 ? 8 : 4;   // steps whose loads are in flight together
    static_assert(MF <= WAVES, "");
    __shared__ i32x4 red[WAVES][MF][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), q = lane >> 4, r = lane & 15;
    const int total = p.tiles_r * p.tiles_c, id = blockIdx.x, per = total / 8, extra = total % 8, xcd = id % 8;
    const int tile = xcd * per + min(xcd, extra) + id / 8;   // an XCD has neighbouring tiles, columns first
    const int row0 = tile / p.tiles_c * (16 * MF), col0 = tile % p.tiles_c * 16;
    // (rows and columns beyond the edge repeat the last ones: their results are not stored)
    const int8_t *from_w = w + (int64_t)min(col0 + r, p.cols - 1) * K, *from_x[MF];
#pragma unroll
    for (int j = 0; j < MF; ++j) from_x[j] = x + (int64_t)min(row0 + j * 16 + r, p.rows - 1) * K;
    i32x4 acc[MF];
#pragma unroll
    for (int j = 0; j < MF; ++j) acc[j] = i32x4{0, 0, 0, 0};
    for (int k0 = wave * 64; k0 < K; k0 += AHEAD * STEP) {
        i32x4 a[AHEAD], b[AHEAD][MF];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int k = k0 + u * STEP + q * 16;
            if (u && k0 + u * STEP >= K) break;   // (uniform)
            a[u] = load_codes<WHOLE>(from_w, k, K);
#pragma unroll
            for (int j = 0; j < MF; ++j) b[u][j] = load_codes<WHOLE>(from_x[j], k, K);
        }
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (u && k0 + u * STEP >= K) break;
#pragma unroll
            for (int j = 0; j < MF; ++j) acc[j] = mfma(a[u], b[u][j], acc[j]);
        }
    }
#pragma unroll
    for (int j = 0; j < MF; ++j) red[wave][j][lane] = acc[j];
    __syncthreads();
    if (wave >= MF) return;
    // wave j stores fragment j: a lane has four columns of a row
    i32x4 sum = red[0][wave][lane];
#pragma unroll
    for (int k = 1; k < WAVES; ++k) sum += red[k][wave][lane];
    const int row = row0 + wave * 16 + r, col = col0 + q * 4;
    if (row >= p.rows) return;
    const float sr = p.scale_r[row];
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = scaled((float)sum[e], sr, p.scale_c[min(col + e, p.cols - 1)]);
    emit<T, 4>(p, 0, row, col, v);
}

// ---- host ----

// Which kernel a product takes: the least of what they are measured to take, in microseconds. A launch, with the loads and results that
// nothing overlaps, and so much per 128 bytes of the reduction; then the rounds after the first of a full chip (for the direct
// kernel, the workgroups after the first 256). Tiles along the reduction are rows of 16 bytes: others are copied first. The
// 256-wide tiles write whole eights of columns.
//                         direct  64 x 64  128 x 128  256 x 128  256 x 256   (measured; us)
//   64 x 512 to 512          4.0      5.5      10.3       9.8       13.3
//   950 x 256 to 256         3.7      5.0      10.4       8.4       11.5
//   4096 x 512 to 512       13.9      7.3      12.2      10.8       14.7
//   4096 x 333 to 264       13.5      9.5      14.6      13.0       16.4
//   8601 x 2048 to 512      78       23.0      23.3      22.8       31.0
//   32768 x 256 to 256      34       15.5      14.1      11.4       14.3
//   32768 x 512 to 2048    339      101        88        66         54
//   32768 x 2048 to 2048  1133      287       202       170        133
enum Kernel { DIRECT, SMALL, BIG, HALF, WIDE };
double kernel_cost(Kernel k, int64_t rows, int64_t cols, int64_t in) {
    auto tiles = [&](int r, int c) { return (double)ceil_div(rows, r) * ceil_div(cols, c); };
    auto later = [&](int r, int c, int slots) { return std::ceil(tiles(r, c) / slots) - 1; };
    auto filled = [&](int r, int c, int slots) { return std::min(1.0, tiles(r, c) / slots); };
    const double steps = (double)ceil_div(in, 128), copy = in % 16 ? 2.5 + (rows + cols) * in * 0.45e-6 : 0;
    switch (k) {
        case DIRECT: return 2.8 + 2.3e-3 * in + std::max(0.0, tiles(rows <= 16 ? 16 : 64, 16) - 256) * (1.7e-3 + 8e-6 * in) * (in % 16 ? 1.9 : 1);
        case SMALL: return copy + 4.2 + 0.33 * steps + later(64, 64, 512) * (1.6 + 0.41 * steps);
        case BIG: return copy + 8.8 + 0.67 * steps + 4.5 * filled(128, 128, 512) + later(128, 128, 512) * (6 + 1.25 * steps);
        case HALF: return copy + 6.5 + 0.87 * steps + 3.5 * filled(256, 128, 256) + later(256, 128, 256) * (4 + 0.93 * steps);
        default: return copy + 8.4 + 1.26 * steps + 5 * filled(256, 256, 256) + later(256, 256, 256) * (5 + 1.7 * steps);
    }
}
Kernel choose(const Int8ProductArgs &a) {
    Kernel best = SMALL;
    for (Kernel k : {DIRECT, BIG, HALF, WIDE}) {
        if (k == DIRECT ? a.in < 16 : k >= HALF && a.out % 8 != 0) continue;
        if (kernel_cost(k, a.rows, a.out, a.in) < kernel_cost(best, a.rows, a.out, a.in)) best = k;
    }
    return best;
}

struct Plan {
    Kernel kernel;
    int64_t pitch;
    bool copies;
    size_t x_at, bytes;
};
Plan plan(const Int8ProductArgs &a) {
    Plan k{};
    k.kernel = choose(a);
    k.copies = a.in % 16 != 0 && k.kernel != DIRECT;
    k.pitch = k.copies ? round_up(a.in, 16) : a.in;
    if (k.copies) {
        k.x_at = round_up(a.out * k.pitch, 256);
        k.bytes = k.x_at + a.rows * k.pitch;
    }
    return k;
}

template <typename T, int MF> hipError_t launch_direct(Product &p, const int8_t *x, const int8_t *w, int K, hipStream_t s) {
    p.tiles_r = (int)ceil_div(p.rows, 16 * MF);
    p.tiles_c = (int)ceil_div(p.cols, 16);
    const auto kernel = K % 16 == 0 ? direct_product_kernel<T, MF, true> : direct_product_kernel<T, MF, false>;
    kernel<<<(unsigned)(p.tiles_r * p.tiles_c), TB, 0, s>>>(p, x, w, K);
    return hipGetLastError();
}

template <typename T> hipError_t launch_one(Kernel kernel, Product &p, const int8_t *x, const int8_t *w, int K, hipStream_t s) {
    if constexpr (!is_f32<T>()) {
        if (p.residual && kernel == WIDE) return launch_wide<T, false, false, 4, Codes, true>(p, s);
        if (p.residual && kernel == HALF) return launch_wide<T, false, false, 2, Codes, true>(p, s);
    }
    switch (kernel) {
        case WIDE: return launch_wide<T, false, false, 4, Codes>(p, s);
        case HALF: return launch_wide<T, false, false, 2, Codes>(p, s);
        case BIG: return launch_tiles<T, false, false, 2, 2, 4, 4, 2, 2, Codes>(p, s);
        case SMALL: return launch_tiles<T, false, false, 2, 2, 2, 2, 3, 2, Codes>(p, s);
        default: return p.rows <= 16 ? launch_direct<T, 1>(p, x, w, K, s) : launch_direct<T, 4>(p, x, w, K, s);
    }
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
    const int64_t run = (int64_t)(1 << 21) / ceil_div(a.out, 64) * 64;
    for (int64_t first = 0; first < a.rows; first += run) {
        p.rows = (int)std::min(a.rows - first, run);
        p.R = {x + first * k.pitch, half, p.rows * half, half, p.rows};
        p.out = (T *)a.y + first * a.out;
        p.residual = a.residual ? (const T *)a.residual + first * a.out : nullptr;
        p.scale_r = a.scales + first;
        if (hipError_t e = launch_one<T>(k.kernel, p, x + first * k.pitch, w, (int)k.pitch, s)) return e;
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
