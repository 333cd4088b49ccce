// Matrix product kernels on channels-last maps, out[r][c] = sum_t R(r, t) C(c, t): of 16-bit, float32 and 8-bit operands (the
// pointwise convolution's three contractions, and its 8-bit form). Included by the files that launch them.
//
// An operand is either t-contiguous ([r][t]: x, W and dz in y and dx) or t-major ([t][r]: W in dx, dz and x in dW); a
// t-major tile goes through LDS as it lies in memory and its fragments are transposed by the LDS read
// (ds_read_b64_tr_b16), so no operand is ever transposed in memory. The operand of the output's contiguous side takes
// the MFMA's row side: a lane then holds neighbouring output channels of one pixel and stores them together, with bias,
// activation and residual applied on the way.
//
// Tiles of 64 along t are staged by direct-to-LDS loads into two or three buffers: the next tiles' loads are in flight while
// the current one is multiplied. LDS chunks of 16 bytes are swizzled (on the global side of the load, since the LDS side is
// fixed by the lane) so that the lanes of a read fall into different banks. Values beyond an operand's edge are read as
// zeros by the buffer's own bounds check.
//
// 8-bit operands (t-contiguous) go through the same staging two codes to a 16-bit element: the 16 bytes that a lane has of a
// 16x16x32 MFMA's 16-bit operand are those of a 16x16x64 one's 8-bit operand. Their sums are whole numbers, scaled by row and
// column as they are stored.
#pragma once

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "kernels.h"
#include "maps.h"

namespace tvdcn_hip {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int BK = 64;      // of the reduction in a tile of product_kernel

__device__ __forceinline__ fvec4 mfma(const bf16x8 &a, const bf16x8 &b, const fvec4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ fvec4 mfma(const f16x8 &a, const f16x8 &b, const fvec4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
// MFMA m of a fragment: all of a 16-bit one, or of a float32 one the lanes' m-th values along t
template <typename F> __device__ __forceinline__ fvec4 mfma_part(const F &a, const F &b, const fvec4 &c, int) { return mfma(a, b, c); }
__device__ __forceinline__ fvec4 mfma_part(const fvec4 &a, const fvec4 &b, const fvec4 &c, int m) {
    return __builtin_amdgcn_mfma_f32_16x16x4f32(a[m], b[m], c, 0, 0, 0);
}
// two codes of an 8-bit operand
struct Codes {
    int8_t v[2];
};
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ i32x4 mfma(const i32x4 &a, const i32x4 &b, const i32x4 &c) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ i32x4 mfma_part(const i32x4 &a, const i32x4 &b, const i32x4 &c, int) { return mfma(a, b, c); }

template <typename E> struct Frag;
template <> struct Frag<bf16> { typedef bf16x8 type; };
template <> struct Frag<f16> { typedef f16x8 type; };
template <> struct Frag<float> { typedef fvec4 type; };   // along t
template <> struct Frag<Codes> { typedef i32x4 type; };
// sums of an MFMA
template <typename E> struct Sums { typedef fvec4 type; };
template <> struct Sums<Codes> { typedef i32x4 type; };

// A matrix of 16-bit elements. t-contiguous: `width` rows of `lim` elements; t-major: `lim` rows of `width` elements.
// Rows are `ld` apart, a multiple of 8; so are lim (t-contiguous) and width (t-major). Pieces are `plane` apart.
struct Operand {
    const void *p;
    int64_t ld, plane, lim, width;
};

struct Product {
    Operand R, C;
    int pieces_c;             // float32 in pieces: of a value of C (of R: 3)
    int rows, cols;           // of the output
    int64_t share;            // reduction per workgroup (a multiple of SHARE, or all of it)
    int tiles_r, tiles_c, splits;
    void *out;                // [rows][cols]; float32 sums [splits][rows][cols] where sums
    const void *bias, *residual;
    void *pre;
    int act;
    bool sums;
    const float *scale_r, *scale_c;   // 8-bit operands: of a row's and a column's codes
};

// 64 lanes x 16 bytes from a buffer into 1 KB of LDS at `lds` (uniform). m0 is declared as written: the compiler allocates it to
// nothing, which it warns of, but may keep it set from one of its own uses to the next.
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_to_lds(const u32x4 &rsrc, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(offset), "s"(rsrc)
                 : "memory", "m0");
}
// 64 lanes x 4 bytes, into 256 bytes of LDS
__device__ __forceinline__ void load_words_to_lds(const u32x4 &rsrc, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(offset), "s"(rsrc)
                 : "memory", "m0");
}
#pragma clang diagnostic pop

template <int N> constexpr int log2_of() { return N <= 1 ? 0 : 1 + log2_of<N / 2>(); }

// Stages tiles of an operand: B rows (columns of the output, or rows) x BK = 64. The NW waves issue B BK / 512 loads of 1 KB.
//  t-contiguous: LDS row of BK elements per output index; chunk j of row n at j ^ swz(n)
//  t-major:      LDS row of B elements per t; chunk j of row t at j ^ 2 swz(t)
template <bool TM, bool PERM, int B, int F, int NW> struct Stager {
    static constexpr int LOADS = B * BK / 512 / NW, CH = (TM ? B : BK) / 8;   // chunks of an LDS row
    static_assert(LOADS * 512 * NW == B * BK, "");
    uint32_t off[LOADS];
    bool in[LOADS];          // t-contiguous: the row exists; t-major: the columns do
    int at[LOADS];           // first reduction index of the lane's chunk

    // Which chunk positions a row is turned by. t-contiguous: the 16 rows of one fragment read fall into different chunks
    // of an LDS pass of 256 bytes (two rows); t-major: so do the eight rows of half a transposed read.
    static __device__ __forceinline__ int swz(int n) {
        if (TM) return (n & 3) | ((n >> 3) & 1) << 2;
        if (PERM) return ((n >> 1) & 1) | ((n >> log2_of<4 * F>()) & 3) << 1;
        return (n >> 1) & 7;
    }
    __device__ __forceinline__ void init(const Operand &o, int64_t first, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int e = (wave * LOADS + i) * 512 + lane * 8, row = e / (CH * 8), slot = e % (CH * 8) / 8;
            if (TM) {
                const int chunk = slot ^ ((2 * swz(row)) & (CH - 1));
                off[i] = (uint32_t)(row * (int)o.ld + chunk * 8) * 2u;
                in[i] = first + chunk * 8 < o.width;
                at[i] = row;
            } else {
                const int chunk = slot ^ swz(row);
                off[i] = (uint32_t)(row * (int)o.ld + chunk * 8) * 2u;
                in[i] = first + row < o.width;
                at[i] = chunk * 8;
            }
        }
    }
    __device__ __forceinline__ void load(const Operand &o, int64_t first, int64_t k0, int64_t kend, uint32_t lds,
                                         int wave) const {
        const int64_t lim = kend < o.lim ? kend : o.lim;
        const int left = (int)(lim - k0 < BK ? lim - k0 : BK);
        const uint64_t base = (uint64_t)o.p + 2 * (uint64_t)(TM ? k0 * o.ld + first : first * o.ld + k0);
        const u32x4 rsrc = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
#pragma unroll
        for (int i = 0; i < LOADS; ++i)
            load_to_lds(rsrc, in[i] && at[i] < left ? off[i] : 0x80000000u, lds + (uint32_t)(wave * LOADS + i) * 1024u);
    }
    // the fragment of 16 output indexes, reduction kk * 32 + (lane / 16) * 8 + 0..7
    template <typename E>
    static __device__ __forceinline__ typename Frag<E>::type frag(const char *tile, int origin, int i, int kk, int lane) {
        const int q = lane >> 4, r = lane & 15;
        if constexpr (TM) {
            union {
                s16x4 h[2];
                typename Frag<E>::type f;
            } u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                // 16 lanes read four rows t of 16 columns; the read hands lane r the column r of the four
                const int t = kk * 32 + q * 8 + h * 4 + r / 4, c = origin + i * 16 + (r & 3) * 4;
                const char *p = tile + t * (B * 2) + (((c >> 3) ^ ((2 * swz(t)) & (CH - 1))) << 4) + (c & 7) * 2;
                typedef __attribute__((address_space(3))) s16x4 *lds_t;
                u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
            }
            return u.f;
        } else {
            // PERM: the MFMA's row r is output index (r / 4) 4F + 4i + r % 4, so that a lane's F fragments are 4F
            // neighbouring indexes
            const int n = origin + (PERM ? (r >> 2) * (4 * F) + i * 4 + (r & 3) : i * 16 + r);
            return *reinterpret_cast<const typename Frag<E>::type *>(tile + n * (BK * 2) + (((kk * 4 + q) ^ swz(n)) << 4));
        }
    }
};

// A sum of products of codes (below 2^31), times the scales of its row and column: the row's first, which a float32 holds up to 2^96, and
// a larger one last, so that an infinity stands only for a result that is one. (Scales of 2^-126 and more lose nothing either way.) Such
// rows are rare: a wave without one (`far`) does not choose for every value, which would take two instructions each.
constexpr float FAR_SCALE = 7.922816251426434e+28f;   // 2^96
__device__ __forceinline__ bool is_far(float scale_r) { return fabsf(scale_r) > FAR_SCALE; }
__device__ __forceinline__ float scaled(float sum, float scale_r, float scale_c) {
    return is_far(scale_r) ? sum * scale_c * scale_r : sum * scale_r * scale_c;
}
__device__ __forceinline__ float scaled(float sum, float scale_r, float scale_c, float bias) {
    return is_far(scale_r) ? fmaf(sum * scale_c, scale_r, bias) : fmaf(sum * scale_r, scale_c, bias);
}

// RUN neighbouring outputs of one row
template <typename T, int RUN>
__device__ __forceinline__ void emit(const Product &p, int split, int row, int col, const float *acc) {
    if (col >= p.cols) return;
    const int64_t at = (int64_t)row * p.cols + col;
    if (p.sums) {
        float *o = (float *)p.out + (int64_t)split * p.rows * p.cols + at;
        if (p.cols % 4 == 0) {
#pragma unroll
            for (int v = 0; v < RUN; v += 4)
                if (col + v < p.cols) *reinterpret_cast<fvec4 *>(o + v) = fvec4{acc[v], acc[v + 1], acc[v + 2], acc[v + 3]};
        } else {
#pragma unroll
            for (int v = 0; v < RUN; ++v)
                if (col + v < p.cols) o[v] = acc[v];
        }
        return;
    }
    float z[RUN], r[RUN];
    if (p.cols % RUN == 0) {
        typedef Pack<T, RUN> P;
#pragma unroll
        for (int v = 0; v < RUN; ++v) z[v] = acc[v], r[v] = 0.f;
        if (p.bias) {
            const P b = *reinterpret_cast<const P *>((const T *)p.bias + col);
#pragma unroll
            for (int v = 0; v < RUN; ++v) z[v] += (float)b.v[v];
        }
        if (p.residual) {
            const P b = *reinterpret_cast<const P *>((const T *)p.residual + at);
#pragma unroll
            for (int v = 0; v < RUN; ++v) r[v] = (float)b.v[v];
        }
        P o;
        if (p.pre) {
            kept_arguments<T, RUN>(z, o.v, p.act);
            *reinterpret_cast<P *>((T *)p.pre + at) = o;
        }
#pragma unroll
        for (int v = 0; v < RUN; ++v) o.v[v] = (T)(act_value<is_f32<T>()>(z[v], p.act) + r[v]);
        *reinterpret_cast<P *>((T *)p.out + at) = o;
    } else {
        // (loads that stay in the row, all on their way at once)
        const int last = p.cols - 1 - col;
#pragma unroll
        for (int v = 0; v < RUN; ++v) z[v] = r[v] = 0.f;
        if (p.bias)
#pragma unroll
            for (int v = 0; v < RUN; ++v) z[v] = (float)((const T *)p.bias)[col + (v < last ? v : last)];
        if (p.residual)
#pragma unroll
            for (int v = 0; v < RUN; ++v) r[v] = (float)((const T *)p.residual)[at + (v < last ? v : last)];
#pragma unroll
        for (int v = 0; v < RUN; ++v) z[v] += acc[v];
        if (p.pre) {
            T o[RUN];
            kept_arguments<T, RUN>(z, o, p.act);
#pragma unroll
            for (int v = 0; v < RUN; ++v)
                if (v <= last) ((T *)p.pre)[at + v] = o[v];
        }
        act_values<is_f32<T>(), RUN>(z, p.act);
#pragma unroll
        for (int v = 0; v < RUN; ++v)
            if (v <= last) ((T *)p.out)[at + v] = (T)(z[v] + r[v]);
    }
}

// WR x WC waves, each FR x FC fragments of 16 x 16; STAGES tiles of BK along the reduction in LDS. T: the results' type, E the
// operands'
template <typename T, bool RT, bool CT, int WR, int WC, int FR, int FC, int STAGES, int BLOCKS, typename E = T>
__global__ void __launch_bounds__(WR * WC * 64, BLOCKS * WR * WC / 4) product_kernel(Product p) {
    constexpr int NW = WR * WC, BR = WR * 16 * FR, BC = WC * 16 * FC, TILE = (BR + BC) * BK * 2;
    extern __shared__ __align__(1024) char smem[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Workgroups go to the 8 XCDs in turn; each XCD takes a run of neighbouring tiles, columns first, so that the
    // operand of the rows is read into one L2 only
    const int total = p.tiles_r * p.tiles_c * p.splits, id = blockIdx.x;
    const int per = total / 8, extra = total % 8, xcd = id % 8;
    const int tile = xcd * per + min(xcd, extra) + id / 8;
    const int split = tile / (p.tiles_r * p.tiles_c), in_split = tile - split * (p.tiles_r * p.tiles_c);
    const int row0 = in_split / p.tiles_c * BR, col0 = in_split % p.tiles_c * BC;
    const int64_t kall = p.R.lim > p.C.lim ? p.R.lim : p.C.lim;
    const int64_t kbeg = split * p.share, kend = kbeg + p.share < kall ? kbeg + p.share : kall;
    const int iters = (int)((kend - kbeg + BK - 1) / BK);

    typedef Stager<RT, false, BR, FR, NW> SR;
    typedef Stager<CT, !CT, BC, FC, NW> SC;
    constexpr int LOADS = SR::LOADS + SC::LOADS;
    SR sr;
    SC sc;
    sr.init(p.R, row0, wave, lane);
    sc.init(p.C, col0, wave, lane);
    typedef __attribute__((address_space(3))) char *lds_t;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_t)smem;
    const int wr = wave / WC, wc = wave % WC;

    typedef typename Sums<E>::type Sum;
    Sum acc[FC][FR];
#pragma unroll
    for (int i = 0; i < FC; ++i)
#pragma unroll
        for (int j = 0; j < FR; ++j) acc[i][j] = Sum{0, 0, 0, 0};

    int step = 0, to = 0, at = 0;   // the next tile to stage and its buffer; the buffer to read
    auto stage = [&]() {
        const int64_t k0 = kbeg + (int64_t)step * BK;
        sr.load(p.R, row0, k0, kend, lds + to * TILE, wave);
        sc.load(p.C, col0, k0, kend, lds + to * TILE + BR * BK * 2, wave);
        ++step;
        if (++to == STAGES) to = 0;
    };
    for (int it = 0; it < STAGES - 1 && it < iters; ++it) stage();
    for (int it = 0; it < iters; ++it) {
        // this tile's loads have landed (those of the STAGES - 2 after it may be on their way), and every wave has read
        // the tile before it
        if (it + STAGES - 1 <= iters)
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LOADS * (STAGES - 2)) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (it + STAGES - 1 < iters) stage();
        const char *tr = smem + at * TILE, *tc = tr + BR * BK * 2;
        if (++at == STAGES) at = 0;
#pragma unroll
        for (int kk = 0; kk < BK / 32; ++kk) {
            typename Frag<E>::type a[FC], b[FR];
#pragma unroll
            for (int i = 0; i < FC; ++i) a[i] = SC::template frag<E>(tc, wc * 16 * FC, i, kk, lane);
#pragma unroll
            for (int j = 0; j < FR; ++j) b[j] = SR::template frag<E>(tr, wr * 16 * FR, j, kk, lane);
#pragma unroll
            for (int i = 0; i < FC; ++i)
#pragma unroll
                for (int j = 0; j < FR; ++j) acc[i][j] = mfma(a[i], b[j], acc[i][j]);
        }
    }

    const int q = lane >> 4;
    constexpr bool CODES = std::is_same<E, Codes>::value;
    float scale[CODES ? FC : 1][4];   // of this lane's columns
    if constexpr (CODES)
#pragma unroll
        for (int i = 0; i < FC; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int col = col0 + wc * 16 * FC + q * 4 * FC + i * 4 + e;
                scale[i][e] = p.scale_c[col < p.cols ? col : 0];
            }
#pragma unroll
    for (int j = 0; j < FR; ++j) {
        const int row = row0 + wr * 16 * FR + j * 16 + (lane & 15);
        if (row >= p.rows) continue;
        if constexpr (!CT) {
#pragma unroll
            for (int i = 0; i < FC; i += 2) {
                float v[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e], v[4 + e] = acc[i + 1][j][e];
                if constexpr (CODES) {
                    const float sr = p.scale_r[row];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = scaled(v[e], sr, scale[i + e / 4][e % 4]);
                }
                emit<T, 8>(p, split, row, col0 + wc * 16 * FC + q * 4 * FC + i * 4, v);
            }
        } else {
#pragma unroll
            for (int i = 0; i < FC; ++i) {
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e];
                emit<T, 4>(p, split, row, col0 + wc * 16 * FC + i * 16 + q * 4, v);
            }
        }
    }
}

// The product in tiles of 256 x 256 (or 256 x 128), for outputs that fill the chip with them: half the operand traffic of 128 x
// 128 tiles (three quarters), and that traffic, not the MFMAs, bounds those.
//
// Eight waves, 2 along the rows x 4 along the columns, 128 x 64 each (128 x 32: FC = 2 column fragments instead of 4). A stage
// of 64 along the reduction is cut into sub-tiles of 8 KB (64 output indexes each), loaded by one 1 KB load per wave; LDS holds
// two stages. A stage is worked off in four phases of 4 FC MFMAs: phase p takes two row fragments (rows 64 p .. 64 p + 63 of the
// tile, those of both wave rows) against the column fragments, which phase 0 reads and keeps in registers. A phase is a memory half (LDS reads, two
// loads) and an MFMA half, a barrier behind each; the second wave row runs one half behind the first, so that each SIMD has
// one wave multiplying while its other one reads.
//
// The loads of a stage are issued as soon as the phases that read the sub-tile's place are over, up to seven phases ahead:
//   phase 1, 2 of stage i: columns of stage i + 2 (FC = 2: all in phase 1);  phase 3: rows 0..127 of stage i + 2;
//   phase 0 of stage i + 1: rows 128..255 of stage i + 2
// (both wave rows have then read the place: the one behind ends its reads a half before). At the end of phase 3's memory
// half the loads issued after columns and rows 0..127 of the next stage are 4 + FC (rows 128..255 of it; columns and rows 0..127
// of the one behind it), at the end of phase 1's those after this stage's rows 128..255 are 6 + FC (the next stage's FC + 4, and
// two columns): vmcnt to those counts, a barrier before the first read.
//
// Workgroups are persistent: a tile's stages follow the last one's, the first loads of the next tile are under way while the
// results are stored.
//
// float32 on its own MFMAs (FC = 2) goes the same way in stages of 32, the same bytes: a lane's four values along the reduction
// serve four MFMAs, quarter q of a wave holds t = 4 q + m in MFMA m, of both operands. 143 TFLOP/s along the reduction (the MFMAs'
// own rate is 157); 32768 x 256 from 256 takes 49 us with launch, first loads and results, a plain library product 42.
template <bool TM, bool PERM, int ES> struct SubTile {
    // the turn of an LDS row (128 bytes, 8 chunks): 16 rows of a fragment read, or the eight rows of half a transposed
    // read, fall into different places of an LDS pass of 256 bytes. float32, t-major: rows of 256 bytes, of which the four
    // quarters of a wave read 64 bytes each of rows four apart
    static __device__ __forceinline__ int swz(int n) {
        if (TM && ES == 4) return ((n >> 2) & 3) << 2;
        if (TM) return (((n >> 1) & 1) | ((n >> 3) & 1) << 1) << 1;
        if (PERM) return ((n >> 1) & 1) | ((n >> 3) & 3) << 1;
        return (n >> 1) & 7;
    }
    // the byte offset of a lane's 16 bytes from the sub-tile's first element; `at`: its first reduction index
    static __device__ __forceinline__ uint32_t offset(const Operand &o, int wave, int lane, int &at) {
        constexpr int CH = TM && ES == 4 ? 16 : 8, N = 16 / ES;   // chunks of an LDS row, elements of a chunk
        const int row = wave * (64 / CH) + lane / CH, chunk = (lane & (CH - 1)) ^ swz(row);
        at = TM ? 0 : chunk * N;
        return (uint32_t)(row * (int)o.ld + chunk * N) * (uint32_t)ES;
    }
    // 16 output indexes from `first`, reduction kk * 32 + (lane / 16) * 8 + 0..7 (float32: half of these). PERM: fragments 2i and
    // 2i + 1 share 32, the MFMA's row r is (r / 4) 8 + r % 4 (+ 4): a lane then holds eight neighbouring indexes of theirs, four lanes 64 bytes of a
    // 16-bit row
    template <typename E>
    static __device__ __forceinline__ typename Frag<E>::type frag(const char *tile, int first, int kk, int lane) {
        const int q = lane >> 4, r = lane & 15;
        if constexpr (TM && ES == 4) {   // (t = kk * 16 + 4 q + 0..3)
            fvec4 f;
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int t = kk * 16 + q * 4 + m, c = first + r;
                f[m] = *reinterpret_cast<const float *>(tile + t * 256 + (((c >> 2) ^ swz(t)) << 4) + (c & 3) * 4);
            }
            return f;
        } else if constexpr (TM) {
            union {
                s16x4 h[2];
                typename Frag<E>::type f;
            } u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = kk * 32 + q * 8 + h * 4 + r / 4, c = first + (r & 3) * 4;
                const char *p = tile + t * 128 + (((c >> 3) ^ swz(t)) << 4) + (c & 7) * 2;
                typedef __attribute__((address_space(3))) s16x4 *lds_t;
                u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
            }
            return u.f;
        } else {
            const int n = PERM ? (first & ~31) + (r >> 2) * 8 + (first & 16) / 4 + (r & 3) : first + r;
            return *reinterpret_cast<const typename Frag<E>::type *>(tile + n * 128 + (((kk * 4 + q) ^ swz(n)) << 4));
        }
    }
};

// The results of a tile of 256 rows: acc[i][j] are the fragments of columns i and rows j, `first` + 32 j this lane's rows, col0 its
// wave's first column, q its quarter of a fragment's columns.
template <typename T, bool CT, int FC>
__device__ __forceinline__ void store_results(const Product &p, const fvec4 (&acc)[FC][8], int split, int first, int col0, int q) {
            // Results: a lane's columns are the same in all its rows. What is read on the way comes ahead of its use: the bias once,
            // the residual a row ahead of the stores.
            constexpr int RUN = CT ? 4 : 8, RUNS = 4 * FC / RUN;
            typedef Pack<T, RUN> Run;
            const int colbase = col0 + q * RUN;
            auto col_of = [&](int r) { return colbase + r * 4 * RUN; };
            Run bias[RUNS] = {}, ahead_r[RUNS] = {};
            auto residual = [&](int row) {
#pragma unroll
                for (int r = 0; r < RUNS; ++r)
                    if (row < p.rows && col_of(r) < p.cols)
                        ahead_r[r] = *reinterpret_cast<const Run *>((const T *)p.residual + (int64_t)row * p.cols + col_of(r));
            };
            if (p.bias)
#pragma unroll
                for (int r = 0; r < RUNS; ++r)
                    if (col_of(r) < p.cols) bias[r] = *reinterpret_cast<const Run *>((const T *)p.bias + col_of(r));
            if (p.residual) residual(first);
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int row = first + j * 32;
                Run res[RUNS];
#pragma unroll
                for (int r = 0; r < RUNS; ++r) res[r] = ahead_r[r];
                if (p.residual && j < 7) residual(row + 32);
#pragma unroll
                for (int r = 0; r < RUNS; ++r) {
                    const int col = col_of(r);
                    float v[RUN];
#pragma unroll
                    for (int e = 0; e < RUN; ++e) v[e] = CT ? acc[r][j][e] : acc[r * 2 + e / 4][j][e % 4];
                    if (row >= p.rows || col >= p.cols) continue;
                    const int64_t at_o = (int64_t)row * p.cols + col;
                    if (p.sums) {
                        float *o = (float *)p.out + (int64_t)split * p.rows * p.cols + at_o;
#pragma unroll
                        for (int e = 0; e < RUN; e += 4) *reinterpret_cast<fvec4 *>(o + e) = fvec4{v[e], v[e + 1], v[e + 2], v[e + 3]};
                        continue;
                    }
                    Run o;
                    if (p.bias)
#pragma unroll
                        for (int e = 0; e < RUN; ++e) v[e] += (float)bias[r].v[e];
                    if (p.pre) {
                        kept_arguments<T, RUN>(v, o.v, p.act);
                        *reinterpret_cast<Run *>((T *)p.pre + at_o) = o;
                    }
                    act_values<is_f32<T>(), RUN>(v, p.act);
                    if (p.residual)
#pragma unroll
                        for (int e = 0; e < RUN; ++e) v[e] += (float)res[r].v[e];
#pragma unroll
                    for (int e = 0; e < RUN; ++e) o.v[e] = (T)v[e];
                    *reinterpret_cast<Run *>((T *)p.out + at_o) = o;
                }
            }
}

// What a tile's scaled results need, in LDS: scales of the columns and of the rows, and the bias (zeros where there is none), 1 KB
// each. A wave loads at most two runs of 256 bytes of them.
template <typename T> struct TileScales {
    static constexpr int BIAS = 2048, BYTES = BIAS + 1024;
    static __device__ __forceinline__ void stage(const Product &p, int row0, int col0, uint32_t lds, int wave, int lane) {
        auto scalar = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
        auto load = [&](const void *from, int first, int left, uint32_t size, int part, uint32_t to) {
            const uint64_t base = (uint64_t)from + size * (uint64_t)(uint32_t)first;
            const uint32_t bytes = from ? (uint32_t)min(left, 256) * size : 0u;
            load_words_to_lds(u32x4{scalar((uint32_t)base), scalar((uint32_t)(base >> 32)), scalar(bytes), 0x00020000u},
                              (uint32_t)(part * 256 + lane * 4), scalar(to + part * 256));
        };
        if (wave < 4) load(p.scale_c, col0, p.cols - col0, 4, wave, lds);
        else load(p.scale_r, row0, p.rows - row0, 4, wave - 4, lds + 1024);
        if (wave < (int)sizeof(T)) load(p.bias, col0, p.cols - col0, sizeof(T), wave, lds + BIAS);
    }
};

// Results of 8-bit operands, scaled by row and column, of rows 32 FIRST .. 32 (FIRST + ROWS) - 1 of the tile. Their products take half the
// time, so what is read on the way weighs twice: scales and bias lie in LDS (`scales`), and so does a residual of 16 bits (STAGED:
// `staged`, the lane's first value of row 32 FIRST at `place`; rows of 128 FC bytes); one of float32 is read AHEAD rows before its use.
// row0, col0: the tile's (uniform) first row and column; lane_row, lane_col: from there to the lane's first.
template <typename T, int FC, int FIRST, int ROWS, bool STAGED>
__device__ __forceinline__ void store_scaled(const Product &p, const i32x4 (&acc)[FC][8], int row0, int col0, int lane_row, int lane_col,
                                             const char *scales, const char *staged = nullptr, uint32_t place = 0) {
    constexpr int RUN = 8, RUNS = FC / 2, AHEAD = FC == 4 ? 1 : 2;   // (as registers allow)
    constexpr bool READ = !STAGED && is_f32<T>();   // (a residual of 16 bits is staged)
    typedef Pack<T, RUN> Run;
    typedef Pack<float, RUN> Scales;
    const int rows = p.rows - row0 - lane_row, cols = p.cols - col0 - lane_col;   // from the lane's first to the edge
    const uint32_t off = (uint32_t)lane_row * (uint32_t)p.cols + (uint32_t)lane_col;
    const int64_t origin = (int64_t)row0 * p.cols + col0;
    Run bias[RUNS], ahead[READ ? AHEAD : 1][RUNS] = {};
    Scales scale[RUNS];
    float scale_r[ROWS];
    auto residual = [&](int j) {
        const T *from = (const T *)p.residual + origin + (int64_t)j * 32 * p.cols;
#pragma unroll
        for (int r = 0; r < RUNS; ++r)
            if (j * 32 < rows && r * 32 < cols) ahead[j % AHEAD][r] = *reinterpret_cast<const Run *>(from + (off + r * 32));
    };
#pragma unroll
    for (int j = 0; j < ROWS; ++j) scale_r[j] = *reinterpret_cast<const float *>(scales + 1024 + (lane_row + (FIRST + j) * 32) * 4);
    bool far = false;
#pragma unroll
    for (int j = 0; j < ROWS; ++j) far = far || is_far(scale_r[j]);
    far = __any(far);
#pragma unroll
    for (int r = 0; r < RUNS; ++r) {
        scale[r] = *reinterpret_cast<const Scales *>(scales + (lane_col + r * 32) * 4);
        bias[r] = *reinterpret_cast<const Run *>(scales + TileScales<T>::BIAS + (lane_col + r * 32) * sizeof(T));
    }
    if constexpr (READ)
        if (p.residual)
#pragma unroll
            for (int j = 0; j < AHEAD; ++j) residual(FIRST + j);
#pragma unroll
    for (int j = FIRST; j < FIRST + ROWS; ++j) {
        T *to = (T *)p.out + origin + (int64_t)j * 32 * p.cols;
        Run res[RUNS] = {};
#pragma unroll
        for (int r = 0; r < RUNS; ++r) {
            // (chunks of 16 bytes lie turned by their row: the run 32 columns on is four chunks away either way)
            if constexpr (STAGED) res[r] = *reinterpret_cast<const Run *>(staged + (place ^ (r * 64u)) + (j - FIRST) * 32 * 128 * FC);
            if constexpr (READ) res[r] = ahead[j % AHEAD][r];
        }
        if constexpr (READ)
            if (p.residual && j + AHEAD < FIRST + ROWS) residual(j + AHEAD);
#pragma unroll
        for (int r = 0; r < RUNS; ++r) {
            float v[RUN];
            if (far) {
#pragma unroll
                for (int e = 0; e < RUN; ++e) v[e] = scaled((float)acc[r * 2 + e / 4][j][e % 4], scale_r[j - FIRST], scale[r].v[e], (float)bias[r].v[e]);
            } else {
#pragma unroll
                for (int e = 0; e < RUN; ++e) v[e] = fmaf((float)acc[r * 2 + e / 4][j][e % 4] * scale_r[j - FIRST], scale[r].v[e], (float)bias[r].v[e]);
            }
            act_values<is_f32<T>(), RUN>(v, p.act);
            if constexpr (STAGED || READ)
#pragma unroll
                for (int e = 0; e < RUN; ++e) v[e] += (float)res[r].v[e];
            Run o;
#pragma unroll
            for (int e = 0; e < RUN; ++e) o.v[e] = (T)v[e];
            if (j * 32 < rows && r * 32 < cols) *reinterpret_cast<Run *>(to + (off + r * 32)) = o;
        }
        __builtin_amdgcn_sched_barrier(0);   // (a row's values at a time: more at once do not fit the registers)
    }
}

// A workgroup's tiles: the XCD's run of neighbouring ones (columns first), its workgroups in turn
struct WideTiles {
    int first, step, count;
    __device__ __forceinline__ WideTiles(const Product &p) {
        const int total = p.tiles_r * p.tiles_c * p.splits, xcd = blockIdx.x % 8, slot = blockIdx.x / 8;
        const int per = total / 8, extra = total % 8, run = per + (xcd < extra);
        step = (gridDim.x + 7 - xcd) / 8;
        first = xcd * per + min(xcd, extra) + slot;
        count = run > slot ? (run - slot + step - 1) / step : 0;
    }
};
// Tiles go through eight columns of them at a time, rows behind: a run of 32 (an XCD's workgroups) is then about as wide as it
// is high, and shares most of what it reads.
template <int BC, int STEP = 64> struct WideTile {
    int split, row0, col0, nk;
    int64_t kbeg;
    __device__ __forceinline__ WideTile(const Product &p, int tile) {
        const int plane = p.tiles_r * p.tiles_c;
        split = tile / plane;
        int t = tile - split * plane;
        const int band = t / (p.tiles_r * 8), wide = min(8, p.tiles_c - band * 8);
        t -= band * p.tiles_r * 8;
        row0 = t / wide * 256, col0 = (band * 8 + t % wide) * BC;
        const int64_t kall = p.R.lim > p.C.lim ? p.R.lim : p.C.lim;
        kbeg = split * p.share;
        const int64_t kend = kbeg + p.share < kall ? kbeg + p.share : kall;
        nk = (int)((kend - kbeg + STEP - 1) / STEP);
    }
};

// Where a workgroup's loads of one operand are: the stage's base, and how many bytes from a sub-tile's first element on are
// its own (rows, or columns of the last t, behind the edge are then read as zeros)
// ANY: sub-tiles of `unit` output indexes instead of 64, which may be set to lie anywhere.
template <bool TM, int B, int STEP = 64, int ES = 2, bool ANY = false> struct WideSource {
    uint64_t base, step;     // of a stage; from sub-tile to sub-tile
    int inside;              // output indexes from the tile's first one on
    uint32_t rows;           // t-major: the bytes of the stage's t before the last one
    uint32_t pitch;          // bytes
    uint32_t off;            // the lane's offset, past the end where its reduction indexes are
    int stages, tail;        // from this one to the operand's end, and the length of the last of them
    int unit_;
    __device__ __forceinline__ int unit() const { return ANY ? unit_ : 64; }
    __device__ __forceinline__ void set(uint64_t from, uint32_t row_bytes, int indexes, int unit, uint32_t lane_off) {
        base = from, pitch = row_bytes, step = (uint64_t)(uint32_t)unit * row_bytes, inside = indexes, unit_ = unit, off = lane_off;
    }
    __device__ __forceinline__ int left() const { return stages > 1 ? STEP : tail; }
    __device__ __forceinline__ void trim(uint32_t lane_off, int lane_at) {
        if (TM) rows = (uint32_t)(left() - 1) * pitch, off = lane_off;
        else off = lane_at < left() ? lane_off : 0x80000000u;
    }
    __device__ __forceinline__ void enter(const Operand &o, int first, int64_t k0, uint32_t lane_off, int lane_at) {
        base = (uint64_t)o.p + ES * (uint64_t)(TM ? k0 * o.ld + first : first * o.ld + k0);
        inside = __builtin_amdgcn_readfirstlane((int)(o.width - first < B ? o.width - first : B));
        pitch = (uint32_t)ES * (uint32_t)o.ld;
        step = TM ? 64 * ES : 64 * (uint64_t)pitch;
        if (ANY) unit_ = 64;
        const int64_t t = o.lim - k0, n = (t + STEP - 1) / STEP;
        stages = __builtin_amdgcn_readfirstlane((int)(n < (1 << 30) ? n : 1 << 30));
        tail = (((int)t - 1) & (STEP - 1)) + 1;
        trim(lane_off, lane_at);
    }
    __device__ __forceinline__ void advance(uint32_t lane_off, int lane_at) {
        base += TM ? STEP * (uint64_t)pitch : ES * STEP;
        --stages;
        trim(lane_off, lane_at);
    }
    __device__ __forceinline__ u32x4 descriptor(int q, uint64_t beyond = 0) const {
        const uint64_t b = base + q * step + beyond;
        const int n = min(max(inside - unit() * q, 0), unit());
        const uint32_t bytes = TM ? (n ? rows + (uint32_t)ES * n : 0u) : (uint32_t)n * pitch;
        // (uniform, which the compiler does not always see)
        auto scalar = [](uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); };
        return u32x4{scalar((uint32_t)b), scalar((uint32_t)(b >> 32)), scalar(bytes), 0x00020000u};
    }
};

//
// 8-bit operands: what the results read comes through LDS, so that no load waits behind those of the next stages, and a tile's
// stores are not waited for: the counts of the next tile's first stage allow for them. 65536 x 512 to 2048 takes 103 us (110 with
// scales read and stores waited for as the results are made, 134 with the scales row by row), with gelu 146 (159).
//
// STAGED: their results of 16 bits with a residual. The residual's tile goes through LDS as two more stages behind the tile's own, rows
// 0..127 and 128..255: its loads are under way during the last products, all of them at once, where a lane's registers hold two
// rows' (65536 x 512 to 2048: 137 us instead of 177, 65536 x 2048 to 512 77 instead of 89). The next tile's first loads are issued as
// the halves are done with.
template <int FC> struct StagedResidual {
    static constexpr int LANES = 8 * FC, ROWS = 64 / FC;   // to a row of 128 FC bytes; rows of a sub-tile of 8 KB
    // the lane's row of a sub-tile and its chunk of 16 bytes: chunk c of row n lies at c ^ n % 16, so that a read of 16 rows
    // falls into different banks
    int row, chunk;
    uint32_t off;
    __device__ __forceinline__ StagedResidual(const Product &p, int wave, int lane) {
        row = wave * (ROWS / 8) + lane / LANES;
        chunk = (lane & (LANES - 1)) ^ (row & 15);
        off = (uint32_t)row * (uint32_t)p.cols * 2u + (uint32_t)chunk * 16u;
    }
    // the next stage's loads are of a half of the tile at row0, col0: from the rows' places and, FC = 4, the columns'
    template <typename R, typename C>
    __device__ __forceinline__ void aim(const Product &p, int row0, int col0, int half, bool any, R &rows, C &cols) const {
        const int first = row0 + half * 128, inside = any ? min(max(p.rows - first, 0), 128) : 0;
        const uint64_t base = (uint64_t)p.residual + 2 * ((uint64_t)(uint32_t)first * (uint32_t)p.cols + (uint32_t)col0);
        const uint32_t pitch = (uint32_t)p.cols * 2u, at = chunk * 8 < p.cols - col0 ? off : 0x80000000u;
        rows.set(base, pitch, inside, ROWS, at);
        cols.set(base + 4 * ROWS * (uint64_t)pitch, pitch, FC == 4 ? inside - 4 * ROWS : 0, ROWS, at);
    }
};

template <typename T, bool RT, bool CT, int FC, typename E = T, bool STAGED = false>
__global__ void __launch_bounds__(512, 2) wide_product_kernel(Product p) {
    constexpr int BC = 64 * FC, COLS = 32768, STAGE = COLS + BC * 128;   // bytes; the columns' sub-tiles follow the rows'
    constexpr int ES = sizeof(E), STEP = 128 / ES;                       // of the reduction in a stage
    constexpr int PARTS = ES == 4 ? 4 : 1;                               // MFMAs of a fragment
    extern __shared__ __align__(1024) char smem[];
    typedef SubTile<RT, false, ES> SR;
    typedef SubTile<CT, !CT, ES> SC;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    const WideTiles tiles(p);
    if (tiles.count == 0) return;
    typedef __attribute__((address_space(3))) char *lds_t;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_t)smem + (uint32_t)wave * 1024u;

    int at_r, at_c;
    const uint32_t off_r = SR::offset(p.R, wave, lane, at_r), off_c = SC::offset(p.C, wave, lane, at_c);

    // the stage to load next
    int tile_n = 0, step = 0, buf = 0;
    WideTile<BC, STEP> ahead(p, tiles.first);
    WideSource<RT, 256, STEP, ES, STAGED> rows;
    WideSource<CT, BC, STEP, ES, STAGED> cols;
    const StagedResidual<FC> residual(p, wave, lane);
    auto enter = [&]() {
        const int64_t k0 = ahead.kbeg + (int64_t)step * STEP;
        rows.enter(p.R, ahead.row0, k0, off_r, at_r);
        cols.enter(p.C, ahead.col0, k0, off_c, at_c);
        if (tile_n >= tiles.count) rows.inside = cols.inside = 0;   // past the last tile: loads that fetch nothing
    };
    auto next = [&]() {
        buf ^= 1;
        if (++step < ahead.nk) {
            rows.advance(off_r, at_r);
            cols.advance(off_c, at_c);
            return;
        }
        if constexpr (STAGED)
            if (step < ahead.nk + 2) {
                residual.aim(p, ahead.row0, ahead.col0, step - ahead.nk, tile_n < tiles.count, rows, cols);
                return;
            }
        step = 0;
        if (++tile_n < tiles.count) ahead = WideTile<BC, STEP>(p, tiles.first + tile_n * tiles.step);
        enter();
    };
    // two sub-tiles' loads, their descriptors made ahead (beside the MFMAs)
    u32x4 d0, d1;
    uint32_t to, off;
    auto aim_rows = [&](int q) { d0 = rows.descriptor(q), d1 = rows.descriptor(q + 1), off = rows.off, to = lds + buf * STAGE + q * 8192; };
    auto aim_cols = [&](int q) { d0 = cols.descriptor(q), d1 = cols.descriptor(q + 1), off = cols.off, to = lds + buf * STAGE + COLS + q * 8192; };
    auto load = [&]() { load_to_lds(d0, off, to), load_to_lds(d1, off, to + 8192); };

    enter();
    aim_cols(0), load();
    if (FC == 4) aim_cols(2), load();
    aim_rows(0), load();
    aim_rows(2), load();
    next();
    aim_cols(0), load();
    if (FC == 4) aim_cols(2), load();
    aim_rows(0), load();
    aim_rows(2);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 + FC) : "memory");

    constexpr bool CODES = std::is_same<E, Codes>::value;
    constexpr int SCALES = 2 * STAGE, STORES = 8 * (FC / 2) * (sizeof(T) / 2);   // stores of a lane's results, 16 bytes each
    bool stored = false;   // CODES: the last tile's stores may be under way, STORES of them behind its last loads (STAGED: half of them)
    int at = 0;
    for (int n = 0; n < tiles.count; ++n) {
        const WideTile<BC, STEP> tile(p, tiles.first + n * tiles.step);
        if constexpr (CODES) TileScales<T>::stage(p, tile.row0, tile.col0, lds - wave * 1024u + SCALES + (n & 1) * TileScales<T>::BYTES, wave, lane);
        typedef typename Sums<E>::type Sum;
        Sum acc[FC][8];
#pragma unroll
        for (int i = 0; i < FC; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] = Sum{0, 0, 0, 0};
        if (wr) asm volatile("s_barrier" ::: "memory");   // one half behind
        for (int it = 0; it < tile.nk; ++it) {
            const char *tr = smem + at * STAGE, *tc = tr + COLS + wc * FC / 4 * 8192;
            at ^= 1;
            typename Frag<E>::type a[2][FC];
            auto phase = [&](auto number) {
                constexpr int ph = decltype(number)::value;
                typename Frag<E>::type b[2][2];
#pragma unroll
                for (int kk = 0; kk < 2; ++kk) {
                    if constexpr (ph == 0) {
#pragma unroll
                        for (int i = 0; i < FC; ++i) a[kk][i] = SC::template frag<E>(tc, wc * FC % 4 * 16 + i * 16, kk, lane);
                    }
#pragma unroll
                    for (int j = 0; j < 2; ++j) b[kk][j] = SR::template frag<E>(tr + ph * 8192, j * 32 + wr * 16, kk, lane);
                }
                if constexpr (FC == 4 || ph != 2) load();
                if (CODES && ph == 1 && it == 0 && stored)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"((FC == 4 ? 10 : 8) + (STAGED ? STORES / 2 : STORES)) : "memory");
                else if (CODES && ph == 3 && it == 0 && stored && !STAGED)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(4 + FC + STORES) : "memory");
                else if constexpr (ph == 1)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(FC == 4 ? 10 : 8) : "memory");
                else if constexpr (ph == 3)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(4 + FC) : "memory");
                else
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_s_setprio(1);
                if constexpr (ph == 0) next();
#pragma unroll
                for (int kk = 0; kk < 2; ++kk)
#pragma unroll
                    for (int m = 0; m < PARTS; ++m)
#pragma unroll
                        for (int i = 0; i < FC; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j) acc[i][ph * 2 + j] = mfma_part(a[kk][i], b[kk][j], acc[i][ph * 2 + j], m);
                if constexpr (ph == 0) aim_cols(0);
                if constexpr (ph == 1 && FC == 4) aim_cols(2);
                if constexpr (ph == 2) aim_rows(0);
                if constexpr (ph == 3) aim_rows(2);
#pragma unroll
                for (int m = 0; m < 4 * FC * PARTS; ++m) {   // scalar work between the MFMAs
                    __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x4, 3, 0);
                }
                __builtin_amdgcn_s_setprio(0);
                asm volatile("s_barrier" ::: "memory");
            };
            phase(std::integral_constant<int, 0>());
            phase(std::integral_constant<int, 1>());
            phase(std::integral_constant<int, 2>());
            phase(std::integral_constant<int, 3>());
        }
        if (!wr) asm volatile("s_barrier" ::: "memory");   // level again
        if constexpr (CODES) {
            // A whole tile's stores are counted, STORES a lane; at an edge some lanes have none, and all are waited for. So are they
            // where a tile has one stage alone, since that one's waits are for its scales too.
            const bool whole = tile.row0 + 256 <= p.rows && tile.col0 + BC <= p.cols && tile.nk > 1;
            const int lane_row = wr * 16 + (lane & 15), lane_col = wc * 16 * FC + (lane >> 4) * 8;
            const char *scales = smem + SCALES + (n & 1) * TileScales<T>::BYTES;
            if constexpr (STAGED) {
                // Every wave has read the last stage: the last loads of the residual's second half. Its first half has landed when
                // those of the second are the only ones left.
                const uint32_t place = lane_row * 128 * FC + (((lane_col >> 3) ^ (lane & 15)) << 4);
                load();
                asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 + FC) : "memory");
                next();
                store_scaled<T, FC, 0, 4, true>(p, acc, tile.row0, tile.col0, lane_row, lane_col, scales, smem + at * STAGE, place);
                if (whole) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(STORES / 2) : "memory");
                else asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
                aim_cols(0), load();
                if (FC == 4) aim_cols(2), load();
                aim_rows(0), load();
                aim_rows(2), load();
                next();
                store_scaled<T, FC, 4, 4, true>(p, acc, tile.row0, tile.col0, lane_row, lane_col, scales, smem + (at ^ 1) * STAGE, place);
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                aim_cols(0), load();
                if (FC == 4) aim_cols(2), load();
                aim_rows(0), load();
                aim_rows(2);
                if (whole) asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 + FC + STORES / 2) : "memory");
                else asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(4 + FC) : "memory");
                stored = whole;
            } else {
                store_scaled<T, FC, 0, 8, false>(p, acc, tile.row0, tile.col0, lane_row, lane_col, scales);
                stored = whole && !(is_f32<T>() && p.residual);
                if (stored) asm volatile("s_barrier" ::: "memory");
                else asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
            }
        } else {
            store_results<T, CT, FC>(p, acc, tile.split, tile.row0 + wr * 16 + (lane & 15), tile.col0 + wc * 16 * FC, lane >> 4);
            // the loads' counts above are of loads alone
            asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
        }
    }
    // (no load to LDS outlives the workgroup)
    if constexpr (CODES) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

// ---- host ----

template <typename T, bool RT, bool CT, int WR, int WC, int FR, int FC, int STAGES, int BLOCKS, typename E = T>
hipError_t launch_tiles(Product &p, hipStream_t s) {
    constexpr int BR = WR * 16 * FR, BC = WC * 16 * FC, LDS = STAGES * (BR + BC) * BK * 2;
    static std::atomic<unsigned long long> done{0};
    const auto kernel = product_kernel<T, RT, CT, WR, WC, FR, FC, STAGES, BLOCKS, E>;
    if (hipError_t e = raise_lds_limit((const void *)kernel, done)) return e;
    p.tiles_r = (int)ceil_div(p.rows, BR);
    p.tiles_c = (int)ceil_div(p.cols, BC);
    kernel<<<(unsigned)(p.tiles_r * p.tiles_c * p.splits), WR * WC * 64, LDS, s>>>(p);
    return hipGetLastError();
}

// the persistent kernels: a workgroup per CU
template <typename K> hipError_t launch_persistent(K kernel, std::atomic<unsigned long long> &done, Product &p, int cols, int lds, hipStream_t s) {
    if (hipError_t e = raise_lds_limit((const void *)kernel, done)) return e;
    p.tiles_r = (int)ceil_div(p.rows, 256);
    p.tiles_c = (int)ceil_div(p.cols, cols);
    const int64_t tiles = (int64_t)p.tiles_r * p.tiles_c * p.splits;
    kernel<<<(unsigned)(tiles < 256 ? tiles : 256), 512, lds, s>>>(p);
    return hipGetLastError();
}
template <typename T, bool RT, bool CT, int FC, typename E = T, bool STAGED = false> hipError_t launch_wide(Product &p, hipStream_t s) {
    static std::atomic<unsigned long long> done{0};
    return launch_persistent(wide_product_kernel<T, RT, CT, FC, E, STAGED>, done, p, 64 * FC,
                             2 * (32768 + 64 * FC * 128) + (std::is_same<E, Codes>::value ? 2 * TileScales<T>::BYTES : 0), s);
}

}  // namespace
}  // namespace tvdcn_hip
