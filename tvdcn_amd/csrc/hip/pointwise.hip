// The pointwise convolution over channels-last maps: y = act(x W^T + b) + r, and its gradients
//   dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum dz.
//
// One matrix product kernel serves the three contractions, out[r][c] = sum_t R(r, t) C(c, t), on 16x16x32 MFMAs. An
// operand is either t-contiguous ([r][t]: x, W and dz in y and dx) or t-major ([t][r]: W in dx, dz and x in dW); a
// t-major tile goes through LDS as it lies in memory and its fragments are transposed by the LDS read
// (ds_read_b64_tr_b16), so no operand is ever transposed in memory. The operand of the output's contiguous side takes
// the MFMA's row side: a lane then holds neighbouring output channels of one pixel and stores them together, with bias,
// activation and residual applied on the way.
//
// Tiles of 64 along t are staged by direct-to-LDS loads, double-buffered: the next tile's loads are in flight while the
// current one is multiplied. LDS chunks of 16 bytes are swizzled (on the global side of the load, since the LDS side is
// fixed by the lane) so that the lanes of a read fall into different banks. Values beyond an operand's edge are read as
// zeros by the buffer's own bounds check.
//
// float32 maps run as three bfloat16 pieces per value (exact) and the six products of pieces that reach
// float32's precision, smallest first: 2^-24 relative to the operands' products, at a sixth of the 16-bit rate (2.6 times
// the rate of the float32 MFMAs). An infinite operand may turn into a NaN where float32 would keep an infinity.
#include "maps.h"

namespace tvdcn_hip {
namespace {

typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));

constexpr int TB = 256;
constexpr int BK = 64;   // reduction per staged tile

__device__ __forceinline__ fvec4 mfma(const bf16x8 &a, const bf16x8 &b, const fvec4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ fvec4 mfma(const f16x8 &a, const f16x8 &b, const fvec4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
template <typename E> struct Frag;
template <> struct Frag<bf16> { typedef bf16x8 type; };
template <> struct Frag<f16> { typedef f16x8 type; };

// A matrix of 16-bit elements. t-contiguous: `width` rows of `lim` elements; t-major: `lim` rows of `width` elements.
// Rows are `ld` apart, a multiple of 8; so are lim (t-contiguous) and width (t-major). Pieces are `plane` apart.
struct Operand {
    const void *p;
    int64_t ld, plane, lim, width;
};

struct Product {
    Operand R, C;
    int npair;
    int8_t pr[6], pc[6];      // pieces of each product
    int rows, cols;           // of the output
    int64_t share;            // reduction per workgroup (a multiple of BK, or all of it)
    int tiles_r, tiles_c, splits;
    void *out;                // [rows][cols]; float32 sums [splits][rows][cols] where sums
    const void *bias, *residual;
    void *pre;
    int act;
    bool sums;
};

// 64 lanes x 16 bytes from a buffer into 1 KB of LDS at `lds` (uniform)
__device__ __forceinline__ void load_to_lds(const u32x4 &rsrc, uint32_t offset, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                 :
                 : "s"(lds), "v"(offset), "s"(rsrc)
                 : "memory");
}

template <int N> constexpr int log2_of() { return N <= 1 ? 0 : 1 + log2_of<N / 2>(); }

// Stages tiles of an operand: B rows (columns of the output, or rows) x BK. Wave w of 4 issues B / 32 loads of 1 KB.
//  t-contiguous: LDS row of 64 elements, 128 bytes, per output index; chunk j of row n at j ^ swz(n)
//  t-major:      LDS row of B elements per t; chunk j of row t at j ^ 2 swz(t)
template <bool TM, bool PERM, int B, int F> struct Stager {
    static constexpr int LOADS = B / 32;
    uint32_t off[LOADS];
    bool in[LOADS];          // t-contiguous: the row exists; t-major: the columns do
    int at[LOADS];           // first reduction index of the lane's chunk

    // which of 8 chunk positions a row is turned by: the 16 rows that one fragment read covers differ in it or in the
    // row's parity (an LDS pass of 256 bytes covers two rows)
    static __device__ __forceinline__ int swz(int n) {
        if (TM) return (n & 3) | ((n >> 3) & 1) << 2;
        if (PERM) return ((n >> 1) & 1) | ((n >> log2_of<4 * F>()) & 3) << 1;
        return (n >> 1) & 7;
    }
    __device__ __forceinline__ void init(const Operand &o, int64_t first, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int idx = wave * LOADS + i;
            if (TM) {
                constexpr int CH = B / 8;
                const int t = idx * (512 / B) + lane / CH, chunk = (lane % CH) ^ ((2 * swz(t)) & (CH - 1));
                off[i] = (uint32_t)(t * (int)o.ld + chunk * 8) * 2u;
                in[i] = first + chunk * 8 < o.width;
                at[i] = t;
            } else {
                const int row = idx * 8 + lane / 8, chunk = (lane % 8) ^ swz(row);
                off[i] = (uint32_t)(row * (int)o.ld + chunk * 8) * 2u;
                in[i] = first + row < o.width;
                at[i] = chunk * 8;
            }
        }
    }
    __device__ __forceinline__ void load(const Operand &o, int piece, int64_t first, int64_t k0, int64_t kend, uint32_t lds,
                                         int wave) const {
        const int64_t lim = kend < o.lim ? kend : o.lim;
        const int left = (int)(lim - k0 < BK ? lim - k0 : BK);
        const uint64_t base = (uint64_t)o.p + 2 * (uint64_t)(o.plane * piece + (TM ? k0 * o.ld + first : first * o.ld + k0));
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
                const char *p = tile + t * (B * 2) + (((c >> 3) ^ ((2 * swz(t)) & (B / 8 - 1))) << 4) + (c & 7) * 2;
                typedef __attribute__((address_space(3))) s16x4 *lds_t;
                u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_t)p);
            }
            return u.f;
        } else {
            // PERM: the MFMA's row r is output index (r / 4) 4F + 4i + r % 4, so that a lane's F fragments are 4F
            // neighbouring indexes
            const int n = origin + (PERM ? (r >> 2) * (4 * F) + i * 4 + (r & 3) : i * 16 + r);
            return *reinterpret_cast<const typename Frag<E>::type *>(tile + n * 128 + (((kk * 4 + q) ^ swz(n)) << 4));
        }
    }
};

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
#pragma unroll
            for (int v = 0; v < RUN; ++v) o.v[v] = (T)z[v];
            *reinterpret_cast<P *>((T *)p.pre + at) = o;
        }
#pragma unroll
        for (int v = 0; v < RUN; ++v) o.v[v] = (T)(act_value<is_f32<T>()>(z[v], p.act) + r[v]);
        *reinterpret_cast<P *>((T *)p.out + at) = o;
    } else {
#pragma unroll
        for (int v = 0; v < RUN; ++v) {
            if (col + v >= p.cols) break;
            float zv = acc[v];
            if (p.bias) zv += (float)((const T *)p.bias)[col + v];
            if (p.pre) ((T *)p.pre)[at + v] = (T)zv;
            float o = act_value<is_f32<T>()>(zv, p.act);
            if (p.residual) o += (float)((const T *)p.residual)[at + v];
            ((T *)p.out)[at + v] = (T)o;
        }
    }
}

// 4 waves as 2 x 2, each FR x FC fragments of 16 x 16: a tile of 32 FR rows x 32 FC columns
template <typename E, typename T, bool RT, bool CT, int FR, int FC>
__global__ void __launch_bounds__(TB) product_kernel(Product p) {
    constexpr int BR = 32 * FR, BC = 32 * FC, TILE = (BR + BC) * BK * 2;
    __shared__ __align__(1024) char smem[2 * TILE];
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
    const int nk = (int)((kend - kbeg + BK - 1) / BK), iters = nk * p.npair;

    typedef Stager<RT, false, BR, FR> SR;
    typedef Stager<CT, !CT, BC, FC> SC;
    SR sr;
    SC sc;
    sr.init(p.R, row0, wave, lane);
    sc.init(p.C, col0, wave, lane);
    typedef __attribute__((address_space(3))) char *lds_t;
    const uint32_t lds = (uint32_t)(uintptr_t)(lds_t)smem;
    const int wr = wave >> 1, wc = wave & 1;

    fvec4 acc[FC][FR];
#pragma unroll
    for (int i = 0; i < FC; ++i)
#pragma unroll
        for (int j = 0; j < FR; ++j) acc[i][j] = fvec4{0.f, 0.f, 0.f, 0.f};

    int pair = 0, step = 0;   // of the next tile to stage
    auto stage = [&](int buf) {
        const int64_t k0 = kbeg + (int64_t)step * BK;
        sr.load(p.R, p.pr[pair], row0, k0, kend, lds + buf * TILE, wave);
        sc.load(p.C, p.pc[pair], col0, k0, kend, lds + buf * TILE + BR * BK * 2, wave);
        if (++step == nk) step = 0, ++pair;
    };
    if (iters > 0) stage(0);
    for (int it = 0; it < iters; ++it) {
        // this tile's loads have landed, and every wave has read the tile before it
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (it + 1 < iters) stage((it + 1) & 1);
        const char *tr = smem + (it & 1) * TILE, *tc = tr + BR * BK * 2;
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
template <typename T> __device__ __forceinline__ void load8(const T *row, int c, int C, bool vec, float *f) {
    if (vec) {
        const Pack<T, 8> p = *reinterpret_cast<const Pack<T, 8> *>(row + c);
#pragma unroll
        for (int v = 0; v < 8; ++v) f[v] = (float)p.v[v];
    } else {
#pragma unroll
        for (int v = 0; v < 8; ++v) f[v] = c + v < C ? (float)row[c + v] : 0.f;
    }
}

template <typename T, typename E, int NP>
__global__ void __launch_bounds__(TB) lay_out_kernel(const T *__restrict__ x, E *__restrict__ y, int64_t rows, int C,
                                                     int lanes_row, int64_t plane) {
    const bool vec = C % 8 == 0;
    const int64_t lanes = rows * lanes_row;
    for (int64_t i = (int64_t)blockIdx.x * TB + threadIdx.x; i < lanes; i += (int64_t)gridDim.x * TB) {
        const int64_t row = i / lanes_row;
        const int c = (int)(i - row * lanes_row) * 8;
        float f[8];
        load8(x + row * C, c, C, vec, f);
        Pack<E, 8> o[NP];
#pragma unroll
        for (int v = 0; v < 8; ++v) split_pack<E, NP>(f[v], v, o);
#pragma unroll
        for (int n = 0; n < NP; ++n) *reinterpret_cast<Pack<E, 8> *>(y + n * plane + i * 8) = o[n];
    }
}

// dz = dy act'(z) laid out as an operand (where dz is given), and its column sums over a chunk of rows. A workgroup has
// `cols` lanes of 8 channels and TB / cols rows side by side.
template <typename T, typename E, int NP>
__global__ void __launch_bounds__(TB) slope_kernel(const T *__restrict__ dy, const T *__restrict__ pre, E *__restrict__ dz,
                                                   float *__restrict__ part, int64_t rows, int C, int lanes_row, int cols,
                                                   int64_t chunk, int64_t plane, int act) {
    __shared__ float red[TB * 8];
    const int t = threadIdx.x, lanes_r = TB / cols, col = t % cols, rl = t / cols;
    const int j = blockIdx.y * cols + col, c = j * 8;
    const bool active = rl < lanes_r && j < lanes_row, vec = C % 8 == 0;
    const int64_t first = blockIdx.x * chunk, last = first + chunk < rows ? first + chunk : rows;
    float s[8];
#pragma unroll
    for (int v = 0; v < 8; ++v) s[v] = 0.f;
    if (active)
        for (int64_t r = first + rl; r < last; r += lanes_r) {
            float d[8], z[8];
            load8(dy + r * C, c, C, vec, d);
            if (act != TVDCN_ACT_NONE) {
                load8(pre + r * C, c, C, vec, z);
#pragma unroll
                for (int v = 0; v < 8; ++v) d[v] *= act_slope<is_f32<T>()>(z[v], act);
            }
#pragma unroll
            for (int v = 0; v < 8; ++v) s[v] += d[v];
            if (dz) {
                Pack<E, 8> o[NP];
#pragma unroll
                for (int v = 0; v < 8; ++v) split_pack<E, NP>(d[v], v, o);
#pragma unroll
                for (int n = 0; n < NP; ++n)
                    *reinterpret_cast<Pack<E, 8> *>(dz + n * plane + (r * lanes_row + j) * 8) = o[n];
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

// dW = the sum of its shares; db = the sum of its chunks (64 channels per workgroup, four waves along the chunks)
template <typename T>
__global__ void __launch_bounds__(TB) finish_kernel(const float *__restrict__ sums, T *__restrict__ dw, int64_t n,
                                                    int splits, int w_blocks, const float *__restrict__ part,
                                                    T *__restrict__ db, int C, int chunks) {
    __shared__ float red[TB];
    const int t = threadIdx.x;
    if ((int)blockIdx.x < w_blocks) {
        const int64_t stride = (int64_t)w_blocks * TB;
        for (int64_t i = (int64_t)blockIdx.x * TB + t; i < n; i += stride) {
            float a = 0.f;
            for (int k = 0; k < splits; ++k) a += sums[k * n + i];
            dw[i] = (T)a;
        }
        return;
    }
    const int c = ((int)blockIdx.x - w_blocks) * 64 + (t & 63);
    float a = 0.f;
    if (c < C)
        for (int u = t >> 6; u < chunks; u += TB / 64) a += part[(int64_t)u * C + c];
    red[t] = a;
    __syncthreads();
    if (t < 64 && c < C) db[c] = (T)(red[t] + red[t + 64] + red[t + 128] + red[t + 192]);
}

// ---- host ----

bool f32(const PointwiseArgs &a) { return a.dtype == TVDCN_DTYPE_FLOAT32; }
size_t align256(size_t v) { return (v + 255) / 256 * 256; }

unsigned strided_grid(int64_t lanes) {
    const int64_t b = ceil_div(lanes, TB);
    return (unsigned)(b < 16384 ? b : 16384);
}

// The pieces' products: all of one piece, or float32's six in rising order of size (three where the columns' operand has
// one piece)
void set_pairs(Product &p, int nr, int nc) {
    static const int8_t six[6][2] = {{2, 0}, {0, 2}, {1, 1}, {1, 0}, {0, 1}, {0, 0}};
    p.npair = 0;
    for (const auto &s : six)
        if (s[0] < nr && s[1] < nc) p.pr[p.npair] = s[0], p.pc[p.npair] = s[1], ++p.npair;
}

template <typename E, typename T, bool RT, bool CT, int F> hipError_t launch_tiles(Product &p, hipStream_t s) {
    p.tiles_r = (int)ceil_div(p.rows, 32 * F);
    p.tiles_c = (int)ceil_div(p.cols, 32 * F);
    product_kernel<E, T, RT, CT, F, F><<<(unsigned)(p.tiles_r * p.tiles_c * p.splits), TB, 0, s>>>(p);
    return hipGetLastError();
}

// 128 x 128 tiles where they fill the 256 CUs, else 64 x 64
bool big_tiles(int64_t rows, int64_t cols, int64_t splits) { return ceil_div(rows, 128) * ceil_div(cols, 128) * splits >= 256; }

template <typename E, typename T, bool RT, bool CT> hipError_t launch_product(Product p, hipStream_t s) {
    return big_tiles(p.rows, p.cols, p.splits) ? launch_tiles<E, T, RT, CT, 4>(p, s) : launch_tiles<E, T, RT, CT, 2>(p, s);
}

// y or dx: rows in runs whose workgroups HIP takes in one launch
template <typename E, typename T, bool CT> hipError_t launch_rows(Product p, int64_t rows, hipStream_t s) {
    const int64_t run = (int64_t)(1 << 22) / ceil_div(p.cols, 64) * 64;
    const char *r = (const char *)p.R.p;
    const int64_t ld = p.R.ld;
    T *out = (T *)p.out, *pre = (T *)p.pre;
    const T *res = (const T *)p.residual;
    for (int64_t first = 0; first < rows; first += run) {
        p.rows = (int)(rows - first < run ? rows - first : run);
        p.R.p = r + first * ld * 2;
        p.R.width = p.rows;
        p.out = out + first * p.cols;
        p.pre = pre ? pre + first * p.cols : nullptr;
        p.residual = res ? res + first * p.cols : nullptr;
        if (hipError_t e = launch_product<E, T, false, CT>(p, s)) return e;
    }
    return hipSuccess;
}

template <typename T, typename E, int NP>
hipError_t lay_out(const void *x, void *y, int64_t rows, int C, hipStream_t s) {
    const int lanes_row = (int)ceil_div(C, 8);
    lay_out_kernel<T, E, NP><<<strided_grid(rows * lanes_row), TB, 0, s>>>((const T *)x, (E *)y, rows, C, lanes_row,
                                                                        rows * lanes_row * 8);
    return hipGetLastError();
}

struct Plan {
    int64_t pi, po;                    // pitches of the channels
    bool x_laid, w_laid, dz_laid;      // the operand is a copy in the workspace
    int np, npx;                       // pieces per value; of x in the backward
    size_t x_at, w_at, dz_at, part_at, sums_at, forward, backward;
    int cols, chunks;                  // bias gradient: lanes of channels, chunks of rows
    int64_t chunk;
    int splits;                        // weight gradient: shares of the rows
    int64_t share;
};

Plan make_plan(const PointwiseArgs &a) {
    Plan k{};
    const bool wide = f32(a);
    k.pi = round_up(a.in, 8);
    k.po = round_up(a.out, 8);
    k.np = wide ? 3 : 1;
    const bool odd_in = a.in % 8 != 0, odd_out = a.out % 8 != 0;
    k.w_laid = wide || odd_in;
    k.x_laid = wide || odd_in;   // forward
    size_t off = 0;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off += align256(bytes);
        return at;
    };
    k.w_at = k.w_laid ? take((size_t)a.out * k.pi * 2 * k.np) : 0;
    k.x_at = k.x_laid ? take((size_t)a.rows * k.pi * 2 * k.np) : 0;
    k.forward = off;

    off = 0;
    const bool kept = a.codes != nullptr;
    k.npx = wide && !kept ? 3 : 1;
    k.dz_laid = wide || odd_out || a.act != TVDCN_ACT_NONE;
    if (k.w_laid) k.w_at = take((size_t)a.out * k.pi * 2 * k.np);
    if (k.x_laid || kept) k.x_at = take((size_t)a.rows * k.pi * 2 * k.npx);
    k.dz_at = k.dz_laid ? take((size_t)a.rows * k.po * 2 * k.np) : 0;
    // about 1024 workgroups, at most 256 chunks: the last step adds them up
    const int lanes = (int)(k.po / 8);
    k.cols = lanes < 32 ? lanes : 32;
    int64_t chunks = ceil_div(1024, ceil_div(lanes, k.cols));
    const int64_t most = ceil_div(a.rows, (TB / k.cols) * 4);
    chunks = chunks < most ? chunks : most;
    chunks = chunks < 256 ? chunks : 256;
    k.chunk = ceil_div(a.rows, chunks < 1 ? 1 : chunks);
    k.chunks = (int)ceil_div(a.rows, k.chunk < 1 ? 1 : k.chunk);
    k.part_at = take((size_t)k.chunks * a.out * 4);
    // shares of the rows: two 128 x 128 workgroups per CU, each at least four steps
    const int64_t tiles = ceil_div(a.out, 128) * ceil_div(a.in, 128);
    int64_t splits = ceil_div(512, tiles);
    const int64_t most_splits = ceil_div(a.rows, 4 * BK);
    splits = splits < most_splits ? splits : most_splits;
    k.share = round_up(ceil_div(a.rows, splits < 1 ? 1 : splits), BK);
    k.splits = (int)ceil_div(a.rows, k.share < 1 ? 1 : k.share);
    k.sums_at = k.splits > 1 ? take((size_t)k.splits * a.out * a.in * 4) : 0;
    k.backward = off;
    return k;
}

template <typename T, typename E, int NP> hipError_t forward(const PointwiseArgs &a, hipStream_t s) {
    const Plan k = make_plan(a);
    const void *x = a.x, *w = a.weight;
    if (k.w_laid) {
        if (hipError_t e = lay_out<T, E, NP>(w, a.work + k.w_at, a.out, a.in, s)) return e;
        w = a.work + k.w_at;
    }
    if (k.x_laid) {
        if (hipError_t e = lay_out<T, E, NP>(x, a.work + k.x_at, a.rows, a.in, s)) return e;
        x = a.work + k.x_at;
    }
    Product p{};
    p.R = {x, k.pi, a.rows * k.pi, k.pi, a.rows};
    p.C = {w, k.pi, a.out * k.pi, k.pi, a.out};
    set_pairs(p, NP, NP);
    p.cols = a.out;
    p.splits = 1;
    p.share = k.pi;
    p.out = a.y;
    p.bias = a.bias;
    p.residual = a.residual;
    p.pre = a.pre;
    p.act = a.act;
    return launch_rows<E, T, false>(p, a.rows, s);
}

template <typename T, typename E, int NP> hipError_t backward(const PointwiseArgs &a, hipStream_t s) {
    const Plan k = make_plan(a);
    const void *dz = a.dy, *w = a.weight, *x = a.x;
    float *part = a.dbias ? (float *)(a.work + k.part_at) : nullptr;
    const bool need_dz = a.dx || a.dweight;
    if (a.rows > 0 && (a.dbias || (need_dz && k.dz_laid))) {
        const int lanes = (int)(k.po / 8);
        E *to = need_dz && k.dz_laid ? (E *)(a.work + k.dz_at) : nullptr;
        slope_kernel<T, E, NP><<<dim3(k.chunks, (unsigned)ceil_div(lanes, k.cols)), TB, 0, s>>>(
            (const T *)a.dy, (const T *)a.pre, to, part, a.rows, a.out, lanes, k.cols, k.chunk, a.rows * k.po, a.act);
        if (hipError_t e = hipGetLastError()) return e;
        if (to) dz = to;
    }
    if (a.dx && a.rows > 0) {
        if (k.w_laid) {
            if (hipError_t e = lay_out<T, E, NP>(w, a.work + k.w_at, a.out, a.in, s)) return e;
            w = a.work + k.w_at;
        }
        Product p{};
        p.R = {dz, k.po, a.rows * k.po, k.po, a.rows};
        p.C = {w, k.pi, a.out * k.pi, a.out, k.pi};
        set_pairs(p, NP, NP);
        p.cols = a.in;
        p.splits = 1;
        p.share = k.po;
        p.out = a.dx;
        if (hipError_t e = launch_rows<E, T, true>(p, a.rows, s)) return e;
    }
    if (a.dweight && a.rows > 0) {
        if (a.codes) {
            if (hipError_t e = launch_expand(a.dtype, f32(a), a.rows, a.in, k.pi, a.codes, a.exps, a.work + k.x_at, s)) return e;
            x = a.work + k.x_at;
        } else if (k.x_laid) {
            if (hipError_t e = lay_out<T, E, NP>(x, a.work + k.x_at, a.rows, a.in, s)) return e;
            x = a.work + k.x_at;
        }
        Product p{};
        p.R = {dz, k.po, a.rows * k.po, a.rows, k.po};
        p.C = {x, k.pi, a.rows * k.pi, a.rows, k.pi};
        set_pairs(p, NP, k.npx);
        p.rows = a.out;
        p.cols = a.in;
        p.splits = k.splits;
        p.share = k.share;
        p.sums = k.splits > 1;
        p.out = p.sums ? (void *)(a.work + k.sums_at) : a.dweight;
        if (hipError_t e = launch_product<E, T, true, true>(p, s)) return e;
    }
    // (no rows: zeros, the sum of nothing)
    const bool sum_w = a.dweight && (k.splits > 1 || a.rows == 0);
    const int64_t n = (int64_t)a.out * a.in;
    const int w_blocks = sum_w ? (int)strided_grid(n) : 0, b_blocks = a.dbias ? (int)ceil_div(a.out, 64) : 0;
    if (w_blocks + b_blocks == 0) return hipSuccess;
    finish_kernel<T><<<(unsigned)(w_blocks + b_blocks), TB, 0, s>>>((const float *)(a.work + k.sums_at), (T *)a.dweight, n,
                                                                   a.rows ? k.splits : 0, w_blocks, part, (T *)a.dbias,
                                                                   a.out, a.rows ? k.chunks : 0);
    return hipGetLastError();
}

}  // namespace

size_t pointwise_forward_bytes(const PointwiseArgs &a) { return make_plan(a).forward; }
size_t pointwise_backward_bytes(const PointwiseArgs &a) { return make_plan(a).backward; }

hipError_t launch_pointwise_forward(const PointwiseArgs &a, hipStream_t s) {
    if (a.rows == 0) return hipSuccess;
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return forward<float, bf16, 3>(a, s);
        case TVDCN_DTYPE_FLOAT16: return forward<f16, f16, 1>(a, s);
        default: return forward<bf16, bf16, 1>(a, s);
    }
}

hipError_t launch_pointwise_backward(const PointwiseArgs &a, hipStream_t s) {
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return backward<float, bf16, 3>(a, s);
        case TVDCN_DTYPE_FLOAT16: return backward<f16, f16, 1>(a, s);
        default: return backward<bf16, bf16, 1>(a, s);
    }
}

}  // namespace tvdcn_hip
