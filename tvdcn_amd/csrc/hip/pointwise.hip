// The pointwise convolution over channels-last maps: y = act(x W^T + b) + r, and its gradients
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum dz.
//
// The three contractions are the matrix products of product_kernels.h, on 16x16x32 MFMAs.
//
// float32 maps are multiplied on the float32 MFMAs as they lie, or, where the products are large, as three bfloat16 pieces
// per value (exact) by the six products of pieces that reach float32's precision: 2^-24 relative to the operands' products, at
// a sixth of the 16-bit rate (2.6 times the rate of the float32 MFMAs). An infinite operand may turn into a NaN there where
// float32 would keep an infinity.
#include <algorithm>
#include <atomic>
#include <tuple>
#include <type_traits>

#include "product_kernels.h"

namespace tvdcn_hip {
namespace {

constexpr int TB = 256;
constexpr int SHARE = 64;   // rows of the weight gradient's shares come in multiples of this

// float32: the three pieces of both operands (or of the rows' alone: PC = 1 piece of the columns', values that bfloat16 holds) in
// one stage of 32 along the reduction, multiplied there in all their pairs: half the loads and LDS reads of going through the
// pieces' products one after another. Tiles of 256 x 128, waves and phases as above: a phase has 24 MFMAs (12).
//
// A block of 64 output indexes x 32 x one piece is 4 KB, four loads. Three loads per wave are the columns of a stage (PC = 1: one),
// three rows 0..127, three rows 128..255: issued in phase 1 of stage i for stage i + 2, in phase 3 for it, and in phase 0 of stage
// i + 1 for stage i + 2. At the end of phase 3's memory half 6 + PC are younger than what the next stage starts with, at the end
// of phase 1's 6 + 2 PC younger than its rows 128..255.
template <bool TM, bool PERM> struct Block32 {
    static __device__ __forceinline__ int swz(int n) {
        if (TM) return (((n >> 1) & 1) | ((n >> 3) & 1) << 1) << 1;   // LDS rows of 64 indexes, two to a pass of 256 bytes
        return (PERM ? n >> 3 : n >> 2) & 3;                          // LDS rows of 32 along t, four to a pass
    }
    // load `part` of a block: the lane's offset, and its first reduction index
    static __device__ __forceinline__ uint32_t offset(const Operand &o, int part, int lane, int &at) {
        const int row = TM ? part * 8 + lane / 8 : part * 16 + lane / 4;
        const int chunk = TM ? (lane & 7) ^ swz(row) : (lane & 3) ^ swz(row);
        at = TM ? 0 : chunk * 8;
        return (uint32_t)(row * (int)o.ld + chunk * 8) * 2u;
    }
    static __device__ __forceinline__ bf16x8 frag(const char *block, int first, int lane) {
        const int q = lane >> 4, r = lane & 15;
        if constexpr (TM) {
            union {
                s16x4 h[2];
                bf16x8 f;
            } u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int t = q * 8 + h * 4 + r / 4, c = first + (r & 3) * 4;
                const char *p = block + t * 128 + (((c >> 3) ^ swz(t)) << 4) + (c & 7) * 2;
                typedef __attribute__((address_space(3))) s16x4 *lds_t;
                u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
            }
            return u.f;
        } else {
            const int n = PERM ? (first & ~31) + (r >> 2) * 8 + (first & 16) / 4 + (r & 3) : first + r;
            return *reinterpret_cast<const bf16x8 *>(block + n * 64 + ((q ^ swz(n)) << 4));
        }
    }
};

template <bool RT, bool CT, int PC> __global__ void __launch_bounds__(512, 2) pieces_product_kernel(Product p) {
    constexpr int BC = 128, COLS = 4 * 3 * 4096, STAGE = COLS + 2 * PC * 4096;
    extern __shared__ __align__(1024) char smem[];
    typedef Block32<RT, false> SR;
    typedef Block32<CT, !CT> SC;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wave >> 2, wc = wave & 3;
    const WideTiles tiles(p);
    if (tiles.count == 0) return;
    typedef __attribute__((address_space(3))) char *lds_t;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_t)smem;

    // load l of the wave: part (3 wave + l) % 4 of block (3 wave + l) / 4 of two rows' quarters (block: 3 quarter + piece), and the
    // same of the columns' halves
    uint32_t off_r[3], off_c[PC];
    int at_r[3], at_c[PC];
#pragma unroll
    for (int l = 0; l < 3; ++l) off_r[l] = SR::offset(p.R, (wave * 3 + l) & 3, lane, at_r[l]);
#pragma unroll
    for (int l = 0; l < PC; ++l) off_c[l] = SC::offset(p.C, (wave * PC + l) & 3, lane, at_c[l]);

    int tile_n = 0, step = 0, buf = 0;
    WideTile<BC, 32> ahead(p, tiles.first);
    WideSource<RT, 256, 32> rows;
    WideSource<CT, BC, 32> cols;
    auto enter = [&]() {
        const int64_t k0 = ahead.kbeg + (int64_t)step * 32;
        rows.enter(p.R, ahead.row0, k0, 0, 0);
        cols.enter(p.C, ahead.col0, k0, 0, 0);
        if (tile_n >= tiles.count) rows.inside = cols.inside = 0;   // past the last tile: loads that fetch nothing
    };
    auto next = [&]() {
        buf ^= 1;
        if (++step < ahead.nk) {
            rows.advance(0, 0);
            cols.advance(0, 0);
            return;
        }
        step = 0;
        if (++tile_n < tiles.count) ahead = WideTile<BC, 32>(p, tiles.first + tile_n * tiles.step);
        enter();
    };
    u32x4 d[3];
    uint32_t off[3], to = 0;
    const uint64_t plane_r = 2 * (uint64_t)p.R.plane, plane_c = 2 * (uint64_t)p.C.plane;
    auto aim_rows = [&](int q) {
#pragma unroll
        for (int l = 0; l < 3; ++l) {
            const int block = (wave * 3 + l) >> 2;
            d[l] = rows.descriptor(q + block / 3, block % 3 * plane_r);
            off[l] = RT || at_r[l] < rows.left() ? off_r[l] : 0x80000000u;
        }
        to = lds + buf * STAGE + q * 12288 + wave * (3 * 1024);
    };
    auto aim_cols = [&]() {
#pragma unroll
        for (int l = 0; l < PC; ++l) {
            const int block = (wave * PC + l) >> 2;
            d[l] = cols.descriptor(block / PC, block % PC * plane_c);
            off[l] = CT || at_c[l] < cols.left() ? off_c[l] : 0x80000000u;
        }
        to = lds + buf * STAGE + COLS + wave * PC * 1024;
    };
    auto load = [&](auto count) {
#pragma unroll
        for (int l = 0; l < decltype(count)::value; ++l) load_to_lds(d[l], off[l], to + l * 1024);
    };
    typedef std::integral_constant<int, 3> Rows;
    typedef std::integral_constant<int, PC> Cols;

    enter();
    aim_cols(), load(Cols());
    aim_rows(0), load(Rows());
    aim_rows(2), load(Rows());
    next();
    aim_cols(), load(Cols());
    aim_rows(0), load(Rows());
    aim_rows(2);
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(6 + PC) : "memory");

    int at = 0;
    for (int n = 0; n < tiles.count; ++n) {
        const WideTile<BC, 32> tile(p, tiles.first + n * tiles.step);
        fvec4 acc[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[i][j] = fvec4{0.f, 0.f, 0.f, 0.f};
        if (wr) asm volatile("s_barrier" ::: "memory");   // one half behind
        for (int it = 0; it < tile.nk; ++it) {
            const char *tr = smem + at * STAGE, *tc = tr + COLS + wc / 2 * PC * 4096;
            at ^= 1;
            bf16x8 a[PC][2];
            auto phase = [&](auto number) {
                constexpr int ph = decltype(number)::value;
                bf16x8 b[3][2];
                if constexpr (ph == 0)
#pragma unroll
                    for (int k = 0; k < PC; ++k)
#pragma unroll
                        for (int i = 0; i < 2; ++i) a[k][i] = SC::frag(tc + k * 4096, wc % 2 * 32 + i * 16, lane);
#pragma unroll
                for (int k = 0; k < 3; ++k)
#pragma unroll
                    for (int j = 0; j < 2; ++j) b[k][j] = SR::frag(tr + (ph * 3 + k) * 4096, j * 32 + wr * 16, lane);
                if constexpr (ph == 0 || ph == 3) load(Rows());
                if constexpr (ph == 1) load(Cols());
                if constexpr (ph == 1)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(6 + 2 * PC) : "memory");
                else if constexpr (ph == 3)
                    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(6 + PC) : "memory");
                else
                    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
                __builtin_amdgcn_s_setprio(1);
                if constexpr (ph == 0) next();
                // the smallest products first: pieces of the rows x of the columns
#pragma unroll
                for (int sum = 2; sum >= 0; --sum)
#pragma unroll
                    for (int k = sum; k >= 0; --k)
                        if (sum - k < PC)
#pragma unroll
                            for (int i = 0; i < 2; ++i)
#pragma unroll
                                for (int j = 0; j < 2; ++j)
                                    acc[i][ph * 2 + j] = mfma(a[(sum - k) % PC][i], b[k][j], acc[i][ph * 2 + j]);
                if constexpr (ph == 0) aim_cols();
                if constexpr (ph == 2) aim_rows(0);
                if constexpr (ph == 3) aim_rows(2);
#pragma unroll
                for (int m = 0; m < (PC == 3 ? 24 : 12); ++m) {   // scalar work between the MFMAs
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
        store_results<float, CT, 2>(p, acc, tile.split, tile.row0 + wr * 16 + (lane & 15), tile.col0 + wc * 32, lane >> 4);
        // the loads' counts above are of loads alone
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");
    }
}

// float32 as it lies, on the float32 MFMAs (16x16x4): no pieces, no copies of the operands, any pitch. Waves 2 x 2 of 2 x 2
// fragments, tiles of 64 x 64 (128 x 128 ones are 2% faster to 8% slower); a step is 16 along the reduction, staged through
// registers (16-byte loads where the rows allow them), double-buffered in LDS. A lane's four values along the reduction serve
// four MFMAs: quarter q of a wave holds t = 4 q + m in MFMA m, of both operands. t-contiguous tiles lie in rows of 16 (a wave
// reads 1 KB in a row), t-major ones in rows of B + 4, so that the four quarters' rows, four apart, fall into different banks.
// Bound by the MFMAs (157 TFLOP/s) and the steps' barriers: 87 TFLOP/s at 32768 x 256 from 256 with silu and residual, 105 at
// 4096 x 2048 from 2048.
template <bool TM, int B> struct FloatStage {
    static constexpr int N = B / 64, LD = TM ? B + 4 : 16, BYTES = (TM ? 16 : B) * LD * 4;   // accesses of 16 bytes per thread
    fvec4 v[N];
    const float *p[N];   // where the next step's lie
    int64_t pace;
    int at[N], more;     // the access's first t of a step; t-major, its columns up to the edge
    // (outputs beyond the edge are not stored: what they are made of is any value that may be read)
    __device__ __forceinline__ void init(const Operand &o, int64_t first, int64_t k0, int t) {
        more = (int)(o.width - first < B ? o.width - first : B);
        pace = TM ? 16 * o.ld : 16;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = t + i * 256, n = TM ? id % (B / 4) * 4 : id / 4;
            at[i] = TM ? id / (B / 4) : id % 4 * 4;
            p[i] = (const float *)o.p + (TM ? (k0 + at[i]) * o.ld + first + (n < more ? n : 0) : (first + (n < more ? n : 0)) * o.ld + k0 + at[i]);
            if (TM) at[i] |= (n < more ? n : 0) << 8;
        }
    }
    // a step of which `left` along t remain
    __device__ __forceinline__ void load(bool vec, int left) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int k = TM ? at[i] & 255 : at[i];
            if (TM) {
                const int cols = more - (at[i] >> 8);   // (at least one)
                if (k >= left) {
                    v[i] = fvec4{0.f, 0.f, 0.f, 0.f};
                } else if (vec) {
                    v[i] = *reinterpret_cast<const fvec4 *>(p[i]);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[i][e] = p[i][e < cols ? e : 0];
                }
            } else if (vec && left >= 16) {
                v[i] = *reinterpret_cast<const fvec4 *>(p[i]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i][e] = p[i][k + e < left ? e : -k];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (k + e >= left) v[i][e] = 0.f;
            }
            p[i] += pace;
        }
    }
    __device__ __forceinline__ void store(float *tile, int t) const {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int id = t + i * 256;
            *reinterpret_cast<fvec4 *>(TM ? tile + id / (B / 4) * LD + id % (B / 4) * 4 : tile + id * 4) = v[i];
        }
    }
    static __device__ __forceinline__ fvec4 frag(const float *tile, int first, int lane) {
        const int q = lane >> 4, n = first + (lane & 15);
        if constexpr (TM) {
            fvec4 f;
#pragma unroll
            for (int m = 0; m < 4; ++m) f[m] = tile[(q * 4 + m) * LD + n];
            return f;
        } else {
            return *reinterpret_cast<const fvec4 *>(tile + n * LD + q * 4);
        }
    }
};

template <bool RT, bool CT> __global__ void __launch_bounds__(256) float_product_kernel(Product p, bool vec_r, bool vec_c) {
    constexpr int F = 2, B = 32 * F;
    typedef FloatStage<RT, B> SR;
    typedef FloatStage<CT, B> SC;
    __shared__ __align__(16) char smem[2 * (SR::BYTES + SC::BYTES)];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, wr = wave >> 1, wc = wave & 1;
    const int total = p.tiles_r * p.tiles_c * p.splits, id = blockIdx.x;
    const int per = total / 8, extra = total % 8, xcd = id % 8;
    const int tile = xcd * per + min(xcd, extra) + id / 8;
    const int split = tile / (p.tiles_r * p.tiles_c), in_split = tile - split * (p.tiles_r * p.tiles_c);
    const int row0 = in_split / p.tiles_c * B, col0 = in_split % p.tiles_c * B;
    const int64_t kbeg = split * p.share, kend = kbeg + p.share < p.R.lim ? kbeg + p.share : p.R.lim;
    fvec4 acc[F][F];
#pragma unroll
    for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j] = fvec4{0.f, 0.f, 0.f, 0.f};
    SR sr;
    SC sc;
    sr.init(p.R, row0, kbeg, t);
    sc.init(p.C, col0, kbeg, t);
    auto left = [&](int64_t k0) { return (int)(kend - k0 < 16 ? kend - k0 : 16); };
    sr.load(vec_r, left(kbeg));
    sc.load(vec_c, left(kbeg));
    int buf = 0;
    for (int64_t k0 = kbeg; k0 < kend; k0 += 16, buf ^= 1) {
        float *tr = (float *)(smem + buf * (SR::BYTES + SC::BYTES)), *tc = (float *)((char *)tr + SR::BYTES);
        sr.store(tr, t);
        sc.store(tc, t);
        __syncthreads();   // (a wave that stores into the other buffer has passed this: every read of that one is over)
        if (k0 + 16 < kend) {
            sr.load(vec_r, left(k0 + 16));
            sc.load(vec_c, left(k0 + 16));
        }
        fvec4 a[F], b[F];
#pragma unroll
        for (int i = 0; i < F; ++i) a[i] = SC::frag(tc, wc * 16 * F + i * 16, lane);
#pragma unroll
        for (int j = 0; j < F; ++j) b[j] = SR::frag(tr, wr * 16 * F + j * 16, lane);
#pragma unroll
        for (int m = 0; m < 4; ++m)
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < F; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i][m], b[j][m], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int j = 0; j < F; ++j) {
        const int row = row0 + wr * 16 * F + j * 16 + (lane & 15);
        if (row >= p.rows) continue;
#pragma unroll
        for (int i = 0; i < F; ++i) {
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = acc[i][j][e];
            emit<float, 4>(p, split, row, col0 + wc * 16 * F + i * 16 + (lane >> 4) * 4, v);
        }
    }
}

// ---- operands laid out for the product: rows of a multiple of 8 elements, zeros behind the channels ----

// float32 as three bfloat16 pieces, each the rest rounded to the nearest: hi + mid + lo = x exactly (hi leaves at most 16
// bits, mid at most 7), and mid <= 2^-8 |x|, lo <= 2^-17 |x|, so the products left out are under 2^-24 of the operands'.
// A finite value beyond bfloat16's largest starts from that; one that is not finite is its first piece.
__device__ __forceinline__ void pieces(float x, bf16 *o) {
    if ((__float_as_uint(x) & 0x7f800000u) == 0x7f800000u) {
        o[0] = (bf16)x, o[1] = o[2] = (bf16)0.f;
        return;
    }
    o[0] = (bf16)fminf(fmaxf(x, -most<bf16>()), most<bf16>());
    const float rest = x - (float)o[0];
    o[1] = (bf16)rest;
    o[2] = (bf16)(rest - (float)o[1]);
}

template <typename E, int NP> __device__ __forceinline__ void split_pack(float x, int v, Pack<E, 8> *o) {
    if constexpr (NP == 3) {
        bf16 p[3];
        pieces(x, p);
#pragma unroll
        for (int n = 0; n < 3; ++n) o[n].v[v] = p[n];
    } else {
        o[0].v[v] = (E)x;
    }
}

// eight elements of a row, zeros behind its end
template <typename T, bool VEC> __device__ __forceinline__ void load8(const T *row, int c, int C, float *f) {
    if constexpr (VEC) {   // (rows in whole eights)
        const Pack<T, 8> p = *reinterpret_cast<const Pack<T, 8> *>(row + c);
#pragma unroll
        for (int v = 0; v < 8; ++v) f[v] = (float)p.v[v];
    } else {
#pragma unroll
        for (int v = 0; v < 8; ++v) f[v] = (float)row[c + v < C ? c + v : 0];
#pragma unroll
        for (int v = 0; v < 8; ++v)
            if (c + v >= C) f[v] = 0.f;
    }
}

// A row-major matrix and its copy with rows of lanes_row eights, in NP pieces, a plane apart
struct LayOut {
    const void *from;
    void *to;
    int64_t rows;
    int C, lanes_row;
    int64_t lanes() const { return rows * lanes_row; }
};

// both operands of a product (the second may have no rows) in one launch
template <typename T, typename E, int NP>
__global__ void __launch_bounds__(TB) lay_out_kernel(LayOut first, LayOut second, int64_t lanes_first, int64_t lanes) {
    for (int64_t n = (int64_t)blockIdx.x * TB + threadIdx.x; n < lanes; n += (int64_t)gridDim.x * TB) {
        const LayOut &m = n < lanes_first ? first : second;
        const int64_t i = n < lanes_first ? n : n - lanes_first, row = i / m.lanes_row;
        const int c = (int)(i - row * m.lanes_row) * 8;
        float f[8];
        if (m.C % 8 == 0) load8<T, true>((const T *)m.from + row * m.C, c, m.C, f);
        else load8<T, false>((const T *)m.from + row * m.C, c, m.C, f);
        Pack<E, 8> o[NP];
#pragma unroll
        for (int v = 0; v < 8; ++v) split_pack<E, NP>(f[v], v, o);
#pragma unroll
        for (int k = 0; k < NP; ++k) *reinterpret_cast<Pack<E, 8> *>((E *)m.to + (k * m.rows * m.lanes_row + i) * 8) = o[k];
    }
}

// dz = dy act'(z) laid out as an operand (where dz is given), and its column sums over a chunk of rows. A workgroup has
// `cols` lanes of 8 channels and TB / cols rows side by side.
template <typename T, typename Z, typename E, int NP, bool VEC>
__global__ void __launch_bounds__(TB) slope_kernel(const T *__restrict__ dy, const Z *__restrict__ pre, E *__restrict__ dz,
                                                   float *__restrict__ part, int64_t rows, int C, int lanes_row, int cols,
                                                   int64_t chunk, int64_t plane, int act) {
    __shared__ float red[TB * 8];
    const int t = threadIdx.x, lanes_r = TB / cols, col = t % cols, rl = t / cols;
    const int j = blockIdx.y * cols + col, c = j * 8;
    const bool active = rl < lanes_r && j < lanes_row;
    const int64_t first = blockIdx.x * chunk, last = first + chunk < rows ? first + chunk : rows;
    float s[8];
#pragma unroll
    for (int v = 0; v < 8; ++v) s[v] = 0.f;
    constexpr int UNROLL = 4;   // rows of a lane in flight
    if (active)
        for (int64_t r0 = first + rl; r0 < last; r0 += (int64_t)lanes_r * UNROLL) {
            float d[UNROLL][8], z[UNROLL][8];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t ru = r0 + (int64_t)u * lanes_r, r = ru < last ? ru : first;
                load8<T, VEC>(dy + r * C, c, C, d[u]);
                if (act != TVDCN_ACT_NONE) load8<Z, VEC>(pre + r * C, c, C, z[u]);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t r = r0 + (int64_t)u * lanes_r;
                if (r >= last) break;
                argument_values<Z, 8>(z[u]);
                act_slopes<is_f32<T>(), 8>(d[u], z[u], act);
#pragma unroll
                for (int v = 0; v < 8; ++v) s[v] += d[u][v];
                if (dz) {
                    Pack<E, 8> o[NP];
#pragma unroll
                    for (int v = 0; v < 8; ++v) split_pack<E, NP>(d[u][v], v, o);
#pragma unroll
                    for (int n = 0; n < NP; ++n)
                        *reinterpret_cast<Pack<E, 8> *>(dz + n * plane + (r * lanes_row + j) * 8) = o[n];
                }
            }
        }
    if (!part) return;
    if (rl < lanes_r)
#pragma unroll
        for (int v = 0; v < 8; ++v) red[(rl * cols + col) * 8 + v] = s[v];
    __syncthreads();
    for (int i = t; i < cols * 8; i += TB) {
        float a = red[i];
        for (int r = 1; r < lanes_r; ++r) a += red[r * cols * 8 + i];
        const int64_t n = (int64_t)blockIdx.y * cols * 8 + i;
        if (n < C) part[(int64_t)blockIdx.x * C + n] = a;
    }
}

constexpr int FIN = 1024;

// dW = the sum of its shares (eight loads in flight per lane); db = the sum of its chunks (16 channels per workgroup, 64
// lanes along the chunks)
template <typename T>
__global__ void __launch_bounds__(FIN) finish_kernel(const float *__restrict__ sums, T *__restrict__ dw, int64_t n,
                                                     int splits, int w_blocks, const float *__restrict__ part,
                                                     T *__restrict__ db, int C, int chunks) {
    __shared__ float red[FIN];
    const int t = threadIdx.x;
    if ((int)blockIdx.x < w_blocks) {
        const int64_t stride = (int64_t)w_blocks * FIN;
        for (int64_t i = (int64_t)blockIdx.x * FIN + t; i < n; i += stride) {
            float a = 0.f;
            for (int k = 0; k < splits; k += 8) {
                float v[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) v[u] = k + u < splits ? sums[(k + u) * n + i] : 0.f;
#pragma unroll
                for (int u = 0; u < 8; ++u) a += v[u];
            }
            dw[i] = (T)a;
        }
        return;
    }
    const int c = ((int)blockIdx.x - w_blocks) * 16 + (t & 15);
    float a = 0.f;
    if (c < C)
        for (int u = t >> 4; u < chunks; u += 4 * (FIN / 16)) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = u + k * (FIN / 16) < chunks ? part[(int64_t)(u + k * (FIN / 16)) * C + c] : 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) a += v[k];
        }
    red[t] = a;
    __syncthreads();
    if (t < 64) {   // four lanes a channel, 16 rows each
        for (int k = 64; k < FIN; k += 64) a += red[t + k];
        a += __shfl_xor(a, 16);
        a += __shfl_xor(a, 32);
        if (t < 16 && c < C) db[c] = (T)a;
    }
}

// ---- host ----

bool f32(const PointwiseArgs &a) { return a.dtype == TVDCN_DTYPE_FLOAT32; }
size_t align256(size_t v) { return (v + 255) / 256 * 256; }

unsigned strided_grid(int64_t lanes) {
    const int64_t b = ceil_div(lanes, TB);
    return (unsigned)(b < 16384 ? b : 16384);
}

template <bool RT, bool CT, int PC> hipError_t launch_pieces(Product &p, hipStream_t s) {
    static std::atomic<unsigned long long> done{0};
    return launch_persistent(pieces_product_kernel<RT, CT, PC>, done, p, 128, 2 * (12 + 2 * PC) * 4096, s);
}
template <bool RT, bool CT> hipError_t launch_float(Product &p, hipStream_t s) {
    p.tiles_r = (int)ceil_div(p.rows, 64);
    p.tiles_c = (int)ceil_div(p.cols, 64);
    float_product_kernel<RT, CT><<<(unsigned)(p.tiles_r * p.tiles_c * p.splits), 256, 0, s>>>(p, p.R.ld % 4 == 0, p.C.ld % 4 == 0);
    return hipGetLastError();
}

// Which tiles an output takes. 16 bits: 256 x 256 or 256 x 128 (of whole eights of columns), one workgroup per CU; 128 x 128 or 64 x
// 64, two per CU. float32: in pieces, 256 x 128, or as it lies, 64 x 64 or (rows of whole fours, whole eights of columns) 256 x 128.
// The least of what they take, in microseconds: launch, first loads and results, and so much per step of 64 along the reduction and
// round of workgroups. Measured in bfloat16, 16 steps: 2048 x 1024 takes 33.6 / 23.7 / 21.1 / 15.6 us in the four; 24 steps, 32768 x
// 256: 47.8 / 35.0 / 43.3 / 79.7; 32 steps, 65536 x 512: 130 / 166 / 253 / -. float32, in pieces / 64 x 64 / 256 x 128: 4 steps, 32768
// x 256: 33.7 / 60.7 / 49; 4 steps, 65536 x 256: - / 110 / 91; 2 steps, 32768 x 128: - / 20.9 / 28.4; 32 steps, 4096 x 2048: 166 /
// 339 / -. (The weight gradient's shares gain nothing of the last: 57.9 us instead of 59.7 at 32768 rows of 256 and 256.)
enum Tiles { WIDE, HALF, BIG, SMALL, PIECES, FLOAT, FLOAT_WIDE };
double tiles_cost(Tiles t, int64_t rows, int64_t cols, int64_t splits, double steps) {
    auto count = [&](int64_t r, int64_t c) { return ceil_div(rows, r) * ceil_div(cols, c) * splits; };
    switch (t) {
        case WIDE: return 10 + 1.75 * steps * (double)ceil_div(count(256, 256), 256);
        case HALF: return 7 + 1.2 * steps * (double)ceil_div(count(256, 128), 256);
        case BIG: return 6 + steps * (count(128, 128) <= 256 ? 0.95 : 1.7 * (double)ceil_div(count(128, 128), 512));
        case SMALL: return 4 + steps * (count(64, 64) <= 256 ? 0.55 : 0.75 * (double)ceil_div(count(64, 64), 512));
        case PIECES: return 10 + 5.2 * steps * (double)ceil_div(count(256, 128), 256);
        case FLOAT_WIDE: return 3 + (12 + 7.5 * steps) * (double)ceil_div(count(256, 128), 256);
        default: return 6 + std::max(2.2 * steps, (1 + 1.28 * steps) * (double)count(64, 64) / 256);
    }
}
Tiles choose_tiles(int64_t rows, int64_t cols, double steps) {   // 16 bits
    Tiles best = SMALL;
    for (Tiles t : {BIG, HALF, WIDE})
        if ((t == BIG || cols % 8 == 0) && tiles_cost(t, rows, cols, 1, steps) < tiles_cost(best, rows, cols, 1, steps)) best = t;
    return best;
}

Tiles choose_float(int64_t rows, int64_t cols, double steps, bool fours) {
    return fours && cols % 8 == 0 && tiles_cost(FLOAT_WIDE, rows, cols, 1, steps) < tiles_cost(FLOAT, rows, cols, 1, steps) ? FLOAT_WIDE : FLOAT;
}

template <typename T, bool RT, bool CT> hipError_t launch_product(Product p, Tiles tiles, hipStream_t s) {
    if constexpr (is_f32<T>()) {
        if (tiles == FLOAT) return launch_float<RT, CT>(p, s);
        if constexpr (!RT) {
            if (tiles == FLOAT_WIDE) return launch_wide<float, RT, CT, 2>(p, s);
        } else {   // (the weight gradient, perhaps of a kept input)
            if (p.pieces_c == 1) return launch_pieces<RT, CT, 1>(p, s);
        }
        return launch_pieces<RT, CT, 3>(p, s);
    } else {
        switch (tiles) {
            case WIDE: return launch_wide<T, RT, CT, 4>(p, s);
            case HALF: return launch_wide<T, RT, CT, 2>(p, s);
            case BIG: return launch_tiles<T, RT, CT, 2, 2, 4, 4, 2, 2>(p, s);
            default: return launch_tiles<T, RT, CT, 2, 2, 2, 2, 3, 2>(p, s);
        }
    }
}

// y or dx: rows in runs whose workgroups HIP takes in one launch
template <typename T, bool CT> hipError_t launch_rows(Product p, bool pieces, int64_t rows, hipStream_t s) {
    const int64_t run = (int64_t)(1 << 22) / ceil_div(p.cols, 64) * 64;
    const char *r = (const char *)p.R.p;
    const int64_t bytes = p.R.ld * (is_f32<T>() && !pieces ? 4 : 2);
    T *out = (T *)p.out, *pre = (T *)p.pre;
    const T *res = (const T *)p.residual;
    for (int64_t first = 0; first < rows; first += run) {
        p.rows = (int)(rows - first < run ? rows - first : run);
        p.R.p = r + first * bytes;
        p.R.width = p.rows;
        p.out = out + first * p.cols;
        p.pre = pre ? pre + first * p.cols : nullptr;
        p.residual = res ? res + first * p.cols : nullptr;
        const double steps = (double)ceil_div(p.share, 64);
        const bool fours = (p.R.ld | p.C.ld | p.R.lim | p.C.lim | p.C.width) % 4 == 0;
        const Tiles tiles = !is_f32<T>() ? choose_tiles(p.rows, p.cols, steps)
                            : pieces     ? PIECES
                                         : choose_float(p.rows, p.cols, steps, fours);
        if (hipError_t e = launch_product<T, false, CT>(p, tiles, s)) return e;
    }
    return hipSuccess;
}

template <typename T, typename E, int NP> hipError_t lay_out(const LayOut &first, const LayOut &second, hipStream_t s) {
    const int64_t lanes = first.lanes() + second.lanes();
    lay_out_kernel<T, E, NP><<<strided_grid(lanes), TB, 0, s>>>(first, second, first.lanes(), lanes);
    return hipGetLastError();
}

// float32 in pieces or as it lies: the pieces' products run at about 190 TFLOP/s against 128 (the weight gradient's, and all
// where the 256 x 128 tiles do not serve: 105; 112 over both of a backward), and cost the operands' copies (10 bytes a value at
// 5 TB/s; in the backward dz in pieces too, 2 bytes a value more) and launches and first loads. The pieces' kernel writes whole
// eights of columns. 16384 x 512 to 512, in pieces / as it lies: forward 70 / 71 us, gradients of x 76 / 79, of W 88 / 105; 65536 x
// 256 to 256: 91 as it lies, 103 / 86, 137 / 106 (each with the copies that the two share).
bool forward_in_pieces(const PointwiseArgs &a) {
    const double saved = 2.0 * a.rows * a.in * a.out * (a.in % 4 == 0 ? 2.55e-9 : 4.26e-9);
    return f32(a) && a.out % 8 == 0 && saved > 5 + a.rows * 2e-6 * a.in;
}
bool backward_in_pieces(const PointwiseArgs &a) {
    const double saved = 4.0 * a.rows * a.in * a.out * (a.out % 4 == 0 ? 3.7e-9 : 4.26e-9);
    return f32(a) && a.in % 8 == 0 && saved > 24 + a.rows * (2e-6 * a.in + 0.4e-6 * a.out);
}

struct Plan {
    bool pieces;                       // (float32)
    int64_t pi, po;                    // pitches of the channels of x and W, of dz
    bool x_laid, w_laid, dz_laid;      // the operand is a copy in the workspace
    size_t x_at, w_at, dz_at, part_at, sums_at, bytes;
    int cols, chunks;                  // bias gradient: lanes of channels, chunks of rows
    int64_t chunk;
    Tiles tiles;                       // weight gradient: its tiles, and shares of the rows
    int splits;
    int64_t share;
    size_t take(size_t n) {
        const size_t at = bytes;
        bytes += align256(n);
        return at;
    }
};

Plan forward_plan(const PointwiseArgs &a) {
    Plan k{};
    k.pieces = forward_in_pieces(a);
    k.x_laid = k.w_laid = k.pieces || (!f32(a) && a.in % 8 != 0);
    k.pi = k.x_laid ? round_up(a.in, 8) : a.in;
    const size_t value = k.pieces ? 6 : 2;
    if (k.w_laid) k.w_at = k.take((size_t)a.out * k.pi * value);
    if (k.x_laid) k.x_at = k.take((size_t)a.rows * k.pi * value);
    return k;
}

Plan backward_plan(const PointwiseArgs &a) {
    Plan k{};
    const bool wide = f32(a), kept = a.codes != nullptr;
    k.pieces = backward_in_pieces(a);
    const bool copies = k.pieces || (!wide && a.in % 8 != 0);
    k.w_laid = copies;
    k.x_laid = copies && !kept;
    k.pi = copies || kept ? round_up(a.in, 8) : a.in;
    k.dz_laid = k.pieces || a.act != TVDCN_ACT_NONE || (!wide && a.out % 8 != 0);
    k.po = k.dz_laid ? round_up(a.out, 8) : a.out;
    const size_t plain = wide ? 4 : 2, value = k.pieces ? 6 : plain;
    if (k.w_laid) k.w_at = k.take((size_t)a.out * k.pi * value);
    if (k.x_laid) k.x_at = k.take((size_t)a.rows * k.pi * value);
    if (kept) k.x_at = k.take((size_t)a.rows * k.pi * (k.pieces ? 2 : plain));
    if (k.dz_laid) k.dz_at = k.take((size_t)a.rows * k.po * value);
    // about 1024 workgroups, at most 256 chunks: the last step adds them up
    const int lanes = (int)ceil_div(a.out, 8);
    k.cols = lanes < 32 ? lanes : 32;
    int64_t chunks = ceil_div(1024, ceil_div(lanes, k.cols));
    const int64_t most = ceil_div(a.rows, (TB / k.cols) * 4);
    chunks = chunks < most ? chunks : most;
    chunks = chunks < 256 ? chunks : 256;
    k.chunk = ceil_div(a.rows, chunks < 1 ? 1 : chunks);
    k.chunks = (int)ceil_div(a.rows, k.chunk < 1 ? 1 : k.chunk);
    k.part_at = k.take((size_t)k.chunks * a.out * 4);
    // shares of the rows: as many as give every CU its workgroups, each share at least four steps (two of the slower float32 ones).
    // The shares' sums are written and read again: 8 bytes per output and share, at about 4 TB/s.
    const int64_t most_splits = std::max<int64_t>(1, a.rows / ((wide ? 2 : 4) * SHARE));
    double least = 0;
    int64_t splits = 0;
    for (const auto &[t, r, c, slots] : {std::tuple<Tiles, int, int, int>{SMALL, 64, 64, 512}, {BIG, 128, 128, 256},
                                         {BIG, 128, 128, 512}, {HALF, 256, 128, 256}, {WIDE, 256, 256, 256},
                                         {PIECES, 256, 128, 256}, {FLOAT, 64, 64, 256}, {FLOAT, 64, 64, 512},
                                         {FLOAT, 64, 64, 1024}}) {
        if (wide ? t != (k.pieces ? PIECES : FLOAT) : t >= PIECES || (t <= HALF && a.in % 8 != 0)) continue;
        const int64_t n = std::min(std::max<int64_t>(1, slots / (ceil_div(a.out, r) * ceil_div(a.in, c))), most_splits);
        const double steps = (double)ceil_div(ceil_div(a.rows, n), SHARE);
        const double cost = tiles_cost(t, a.out, a.in, n, steps) + (n > 1 ? (double)(n * a.out) * a.in * 2e-6 : 0.0);
        if (splits == 0 || cost < least) least = cost, splits = n, k.tiles = t;
    }
    k.share = round_up(ceil_div(a.rows, splits), SHARE);
    k.splits = (int)ceil_div(a.rows, k.share < 1 ? 1 : k.share);
    k.sums_at = k.splits > 1 ? k.take((size_t)k.splits * a.out * a.in * 4) : 0;
    return k;
}

// The operands that are copied: x (unless it is kept in 8 bits, or not asked for) and W
template <typename T> hipError_t lay_out_operands(const PointwiseArgs &a, const Plan &k, bool x, bool w, hipStream_t s) {
    const int lanes = (int)(k.pi / 8);
    LayOut first{a.x, a.work + k.x_at, x && k.x_laid ? a.rows : 0, a.in, lanes};
    LayOut second{a.weight, a.work + k.w_at, w && k.w_laid ? a.out : 0, a.in, lanes};
    if (first.rows + second.rows == 0) return hipSuccess;
    if constexpr (is_f32<T>()) return lay_out<T, bf16, 3>(first, second, s);
    else return lay_out<T, T, 1>(first, second, s);
}

template <typename T> hipError_t forward(const PointwiseArgs &a, hipStream_t s) {
    const Plan k = forward_plan(a);
    if (hipError_t e = lay_out_operands<T>(a, k, true, true, s)) return e;
    Product p{};
    p.R = {k.x_laid ? a.work + k.x_at : a.x, k.pi, a.rows * k.pi, k.pi, a.rows};
    p.C = {k.w_laid ? a.work + k.w_at : a.weight, k.pi, a.out * k.pi, k.pi, a.out};
    p.pieces_c = 3;
    p.cols = a.out;
    p.splits = 1;
    p.share = k.pi;
    p.out = a.y;
    p.bias = a.bias;
    p.residual = a.residual;
    p.pre = a.pre;
    p.act = a.act;
    return launch_rows<T, false>(p, k.pieces, a.rows, s);
}

// dz as an operand (to == null: not needed so) and the bias gradient's chunks (part == null: not needed). Z: what pre holds.
template <typename T, typename Z, typename E, int NP>
hipError_t slopes_of(const PointwiseArgs &a, const Plan &k, void *to, float *part, hipStream_t s) {
    const int lanes = (int)ceil_div(a.out, 8);
    const auto kernel = a.out % 8 == 0 ? slope_kernel<T, Z, E, NP, true> : slope_kernel<T, Z, E, NP, false>;
    kernel<<<dim3(k.chunks, (unsigned)ceil_div(lanes, k.cols)), TB, 0, s>>>(
        (const T *)a.dy, (const Z *)a.pre, (E *)to, part, a.rows, a.out, lanes, k.cols, k.chunk, a.rows * k.po, a.act);
    return hipGetLastError();
}

template <typename T, typename E, int NP> hipError_t slopes(const PointwiseArgs &a, const Plan &k, void *to, float *part, hipStream_t s) {
    if (a.act == TVDCN_ACT_SILU || a.act == TVDCN_ACT_GELU) return slopes_of<T, typename Argument<T>::type, E, NP>(a, k, to, part, s);
    return slopes_of<T, T, E, NP>(a, k, to, part, s);
}

template <typename T> hipError_t backward(const PointwiseArgs &a, hipStream_t s) {
    const Plan k = backward_plan(a);
    const bool any = a.rows > 0, need_dx = any && a.dx, need_dw = any && a.dweight;
    float *part = a.dbias ? (float *)(a.work + k.part_at) : nullptr;
    void *laid = (need_dx || need_dw) && k.dz_laid ? a.work + k.dz_at : nullptr;
    const void *dz = laid ? laid : a.dy;
    if (any && (part || laid)) {
        hipError_t e;
        if constexpr (is_f32<T>()) e = k.pieces ? slopes<T, bf16, 3>(a, k, laid, part, s) : slopes<T, float, 1>(a, k, laid, part, s);
        else e = slopes<T, T, 1>(a, k, laid, part, s);
        if (e) return e;
    }
    if (hipError_t e = lay_out_operands<T>(a, k, need_dw, need_dx, s)) return e;
    // (as they lie, float32 operands end at their own channels; copies are zeros up to their pitch)
    const bool lies = f32(a) && !k.pieces;
    if (need_dx) {
        Product p{};
        p.R = {dz, k.po, a.rows * k.po, lies ? a.out : k.po, a.rows};
        p.C = {k.w_laid ? a.work + k.w_at : a.weight, k.w_laid ? k.pi : a.in, a.out * k.pi, a.out, k.w_laid ? k.pi : a.in};
        p.pieces_c = 3;
        p.cols = a.in;
        p.splits = 1;
        p.share = lies ? a.out : k.po;
        p.out = a.dx;
        if (hipError_t e = launch_rows<T, true>(p, k.pieces, a.rows, s)) return e;
    }
    if (need_dw) {
        const void *x = a.codes || k.x_laid ? a.work + k.x_at : a.x;
        if (a.codes)
            if (hipError_t e = launch_expand(a.dtype, k.pieces, a.rows, a.in, k.pi, a.codes, a.exps, a.work + k.x_at, s)) return e;
        Product p{};
        p.R = {dz, k.po, a.rows * k.po, a.rows, lies ? a.out : k.po};
        p.C = {x, k.pi, a.rows * k.pi, a.rows, lies ? a.in : k.pi};
        p.pieces_c = a.codes ? 1 : 3;
        p.rows = a.out;
        p.cols = a.in;
        p.splits = k.splits;
        p.share = k.share;
        p.sums = k.splits > 1;
        p.out = p.sums ? (void *)(a.work + k.sums_at) : a.dweight;
        if (hipError_t e = launch_product<T, true, true>(p, k.tiles, s)) return e;
    }
    // (no rows: zeros, the sum of nothing)
    const bool sum_w = a.dweight && (k.splits > 1 || !any);
    const int64_t n = (int64_t)a.out * a.in;
    const int w_blocks = sum_w ? (int)std::min<int64_t>(ceil_div(n, FIN), 4096) : 0, b_blocks = a.dbias ? (int)ceil_div(a.out, 16) : 0;
    if (w_blocks + b_blocks == 0) return hipSuccess;
    finish_kernel<T><<<(unsigned)(w_blocks + b_blocks), FIN, 0, s>>>((const float *)(a.work + k.sums_at), (T *)a.dweight, n,
                                                                   any ? k.splits : 0, w_blocks, part, (T *)a.dbias,
                                                                   a.out, any ? k.chunks : 0);
    return hipGetLastError();
}

}  // namespace

size_t pointwise_forward_bytes(const PointwiseArgs &a) { return forward_plan(a).bytes; }
size_t pointwise_backward_bytes(const PointwiseArgs &a) { return backward_plan(a).bytes; }

hipError_t launch_pointwise_forward(const PointwiseArgs &a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return forward<float>(a, s);
        case TVDCN_DTYPE_FLOAT16: return forward<f16>(a, s);
        default: return forward<bf16>(a, s);
    }
}

hipError_t launch_pointwise_backward(const PointwiseArgs &a, hipStream_t s) {
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return backward<float>(a, s);
        case TVDCN_DTYPE_FLOAT16: return backward<f16>(a, s);
        default: return backward<bf16>(a, s);
    }
}

}  // namespace tvdcn_hip
