// Group normalisation with affine map and activation over channels-last maps [batch][pixels][channels]:
//
//   n = (x - mean) rstd,  z = w n + b,  y = act(z);  mean and variance over the pixels and the Cg channels of a
//   (batch, group);  dz = dy act'(z),  dn = w dz,  dx = rstd (dn - avg(dn) - n avg(dn n)),  dw = sum dz n,  db = sum dz
//
// Bound by memory. Groups that a workgroup can hold in registers are read once, in one launch (below). For larger ones the
// statistics read x once, the second pass reads it again (from the 256 MB last-level cache where it fits) and writes y. A
// workgroup takes a run of pixels of one image and all channels (in tiles of 256
// lanes), so every access is a run of whole rows; a lane keeps its 16 bytes of channels over all its pixels, and with
// them the parameters of those channels. Sums are float32, those of the statistics of deviations from running means (large means
// against small spreads do not cancel, nor does a value unlike the rest), joined in a fixed order.

#include "maps.h"

namespace tvdcn_hip {
namespace {

constexpr int TB = 256;
constexpr int UNROLL = 4;   // pixels of a lane in flight

// How a map is cut: tiles of `cols` lanes of channels, chunks of `rows` pixels.
struct Cut {
    int cols;          // lanes along the channels in a tile
    int lanes_r;       // pixels side by side in a workgroup
    int tiles;
    int chunks;        // per image
    int64_t rows;      // pixels per chunk
    int64_t units;     // batch * chunks
};

Cut make_cut(int64_t batch, int64_t pixels, int channels, int vec) {
    Cut k;
    const int cv = (channels + vec - 1) / vec;
    k.cols = cv < TB ? cv : TB;
    k.lanes_r = TB / k.cols;
    k.tiles = (cv + k.cols - 1) / k.cols;
    // about 1024 workgroups (four per CU), each lane at least UNROLL pixels, at most 256 chunks of an image: the second
    // step reads their sums
    int64_t chunks = ceil_div(1024, batch * k.tiles);
    const int64_t most = ceil_div(pixels, (int64_t)k.lanes_r * UNROLL);
    chunks = chunks < most ? chunks : most;
    chunks = chunks < 256 ? chunks : 256;
    chunks = chunks < 1 ? 1 : chunks;
    k.rows = ceil_div(pixels, chunks);
    k.chunks = (int)ceil_div(pixels, k.rows);
    k.units = batch * k.chunks;
    return k;
}

// A lane's VEC channels of a pixel, from the map or its 8-bit form: as they lie (so that several are on their way before the
// first is looked at), and as values
template <typename T, int VEC, bool KEPT> struct Source {
    const T *x;
    const int8_t *codes;
    const uint8_t *exps;
    int C, blocks;
    struct Raw {
        Pack<std::conditional_t<KEPT, int8_t, T>, VEC> p;
        uint8_t e;
    };
    // where channel c of a row lies, and its exponent
    __device__ __forceinline__ int64_t at(int64_t row, int c) const { return row * C + c; }
    __device__ __forceinline__ int64_t block(int64_t row, int c) const { return KEPT ? row * blocks + c / kKeptBlock : 0; }
    __device__ __forceinline__ Raw load(int64_t at, int64_t block) const {
        Raw r;
        if constexpr (KEPT) {
            r.p = *reinterpret_cast<const decltype(r.p) *>(codes + at);
            r.e = exps[block];
        } else {
            r.p = *reinterpret_cast<const decltype(r.p) *>(x + at);
        }
        return r;
    }
    static __device__ __forceinline__ void values(const Raw &r, float *f) {
        if constexpr (KEPT) {
            kept_values<T, VEC>(r.p.v, r.e, f);
        } else {
#pragma unroll
            for (int v = 0; v < VEC; ++v) f[v] = (float)r.p.v[v];
        }
    }
};

template <typename T, int VEC> __device__ __forceinline__ void params(const void *w, int c, float *f, float none) {
    if (w == nullptr) {
#pragma unroll
        for (int v = 0; v < VEC; ++v) f[v] = none;
        return;
    }
    const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC> *>((const T *)w + c);
#pragma unroll
    for (int v = 0; v < VEC; ++v) f[v] = (float)p.v[v];
}

// The groups of VEC channels from c on
template <int VEC> struct Groups {
    int g[VEC];
    __device__ __forceinline__ Groups(int c, int Cg) {
        int group = c / Cg, left = (group + 1) * Cg - c;
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            g[v] = group;
            if (--left == 0) ++group, left = Cg;
        }
    }
    // their values of one image
    template <typename V> __device__ __forceinline__ void get(const V *__restrict__ from, V *to) const {
#pragma unroll
        for (int v = 0; v < VEC; ++v) to[v] = from[g[v]];
    }
};

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}
__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v += __shfl_xor(v, m);
    return v;
}

// Adds a workgroup's per-lane pairs over its pixel lanes; the sums of channel lane i end in red[i].
template <int VEC> __device__ __forceinline__ void sum_pixel_lanes(float2 *red, const float *s, const float *q, int t,
                                                                    const Cut &k, bool active) {
    const int col = t % k.cols, rl = t / k.cols, n = k.cols * VEC;
    if (rl < k.lanes_r) {
#pragma unroll
        for (int v = 0; v < VEC; ++v)
            red[rl * n + col * VEC + v] = active ? make_float2(s[v], q[v]) : make_float2(0.f, 0.f);
    }
    __syncthreads();
    for (int i = t; i < n; i += TB) {
        float2 a = red[i];
        for (int r = 1; r < k.lanes_r; ++r) {
            a.x += red[r * n + i].x;
            a.y += red[r * n + i].y;
        }
        red[i] = a;
    }
    __syncthreads();
}

// part[(unit * tiles + tile) * G + g] = the mean of the tile's values of the group, and their squared deviations from it
//
// A lane carries a channel's mean m and sum of squared deviations M over its n pixels so far, and takes UNROLL more at a time:
// with s and q the sums of d = x - m and of d^2 over the k new ones, m' = m + s / (n + k), M' = M + q - s^2 / (n + k). What is
// subtracted is at most k / (n + k) of q, so nothing cancels, whatever the first values are (m starts as the first, and a value
// unlike the rest costs no more bits than it adds to the spread). Means are then joined over lanes and channels, and M by their
// deviations from the joint one: M = sum M_i + n_i (m_i - m)^2. The whole forward (statistics, finish, apply) of 4 x 256 x 128 x
// 128 in 32 groups, bfloat16: 26.3 us, 100 MB of traffic at 3.8 TB/s; with each wave summing group after group instead, 31.9.
template <typename T, int VEC>
__global__ void __launch_bounds__(TB) norm_stats_kernel(const T *__restrict__ x, float2 *__restrict__ part, int64_t P,
                                                        int C, int G, int Cg, Cut k) {
    __shared__ float2 red[TB * VEC];
    const int t = threadIdx.x, col = t % k.cols, rl = t / k.cols, tile = blockIdx.y, n = k.cols * VEC;
    const int c0 = (tile * k.cols + col) * VEC;
    const bool active = rl < k.lanes_r && c0 < C;
    const int base = tile * n, end = min(base + n, C), g0 = base / Cg, g1 = (end - 1) / Cg;
    int per = 64;
    while (per > 1 && (g1 - g0 + 1) * per > TB) per /= 2;
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float mean[VEC], sq[VEC], count = 0.f;
#pragma unroll
        for (int v = 0; v < VEC; ++v) mean[v] = sq[v] = 0.f;
        if (active) {
            const T *xb = x + b * P * C + c0;
            const Pack<T, VEC> p0 = *reinterpret_cast<const Pack<T, VEC> *>(xb + (first + rl < last ? first + rl : first) * C);
#pragma unroll
            for (int v = 0; v < VEC; ++v) mean[v] = (float)p0.v[v];
            for (int64_t r = first + rl; r < last; r += (int64_t)k.lanes_r * UNROLL) {
                Pack<T, VEC> p[UNROLL];
                float s[VEC], q[VEC];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const int64_t ru = r + (int64_t)u * k.lanes_r;
                    p[u] = *reinterpret_cast<const Pack<T, VEC> *>(xb + (ru < last ? ru : first) * C);
                }
#pragma unroll
                for (int v = 0; v < VEC; ++v) s[v] = q[v] = 0.f;
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    if (r + (int64_t)u * k.lanes_r >= last) break;
                    count += 1.f;
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const float d = (float)p[u].v[v] - mean[v];
                        s[v] += d;
                        q[v] = fmaf(d, d, q[v]);
                    }
                }
                const float inv = __builtin_amdgcn_rcpf(count);   // (a last bit off moves m by as much of its step)
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    const float step = s[v] * inv;
                    mean[v] += step;
                    sq[v] += q[v] > 3.402823466e38f ? q[v] : fmaf(-s[v], step, q[v]);   // (beyond float32: infinite, not a NaN)
                }
            }
        }
        if (rl < k.lanes_r)
#pragma unroll
            for (int v = 0; v < VEC; ++v) red[rl * n + col * VEC + v] = make_float2(mean[v], sq[v]);
        __syncthreads();
        // over a group's channels and pixel lanes (lane r holds pixels r, r + lanes_r, ... of the chunk): `per` lanes to a group, a
        // wave at most, so that a workgroup's groups are summed side by side
        const int64_t rows = last - first, whole = rows / k.lanes_r;
        const int more = (int)(rows - whole * k.lanes_r), lanes = whole ? k.lanes_r : more;
        for (int g = g0 + t / per; g <= g1; g += TB / per) {
            const int lo = max(g * Cg, base) - base, w = min((g + 1) * Cg, end) - base - lo, l = t % per, dr = per / w;
            const int di = per - dr * w;
            auto each = [&](auto f) {
                for (int r = l / w, i = l - r * w; r < lanes;) {
                    f((float)(whole + (r < more)), red[r * n + lo + i]);
                    r += dr, i += di;
                    if (i >= w) i -= w, ++r;
                }
            };
            auto sum = [&](float v) {
                for (int m = 1; m < per; m <<= 1) v += __shfl_xor(v, m);
                return v;
            };
            const float m0 = red[lo].x;
            float m = 0.f, a = 0.f;
            each([&](float count, const float2 &v) { m = fmaf(count, v.x - m0, m); });
            m = m0 + sum(m) / ((float)rows * (float)w);
            each([&](float count, const float2 &v) { a += fmaf(count, (v.x - m) * (v.x - m), v.y); });
            a = sum(a);
            if (l == 0) part[(unit * k.tiles + tile) * G + g] = make_float2(m, a);
        }
        __syncthreads();
    }
}

// mean and rstd of a (batch, group) from its chunks' and tiles': a wave each
__global__ void __launch_bounds__(64) norm_finish_kernel(const float2 *__restrict__ part, float *__restrict__ mean,
                                                         float *__restrict__ rstd, int64_t BG, int64_t P, int G, int Cg,
                                                         int tile_c, float eps, Cut k) {
    for (int64_t i = blockIdx.x; i < BG; i += gridDim.x) {
        const int64_t b = i / G;
        const int g = (int)(i - b * G);
        const int t0 = g * Cg / tile_c, nt = ((g + 1) * Cg - 1) / tile_c - t0 + 1;
        const double m0 = part[(b * k.chunks * k.tiles + t0) * G + g].x;
        double s = 0.0, q = 0.0;
        for (int j = threadIdx.x; j < k.chunks * nt; j += 64) {
            const int chunk = j / nt, tile = t0 + j % nt;
            const float2 v = part[((b * k.chunks + chunk) * k.tiles + tile) * G + g];
            const int64_t first = chunk * k.rows, rows = P - first < k.rows ? P - first : k.rows;
            const double n = (double)rows * (min((g + 1) * Cg, (tile + 1) * tile_c) - max(g * Cg, tile * tile_c)), d = v.x - m0;
            s += n * d;
            q += v.y + n * d * d;
        }
        s = wave_sum(s);
        q = wave_sum(q);
        if (threadIdx.x == 0) {
            const double n = (double)P * Cg, m = s / n;
            const double var = q / n - m * m;
            mean[i] = (float)(m0 + m);
            rstd[i] = (float)(1.0 / sqrt((var > 0.0 || var != var ? var : 0.0) + (double)eps));
        }
    }
}

template <typename T, int VEC>
__global__ void __launch_bounds__(TB) norm_apply_kernel(const T *__restrict__ x, const void *__restrict__ w,
                                                        const void *__restrict__ bias, const float *__restrict__ mean,
                                                        const float *__restrict__ rstd, T *__restrict__ y, int64_t P,
                                                        int C, int G, int Cg, int act, Cut k) {
    const int t = threadIdx.x, col = t % k.cols, rl = t / k.cols;
    const int c0 = (blockIdx.y * k.cols + col) * VEC;
    if (rl >= k.lanes_r || c0 >= C) return;
    float wv[VEC], bv[VEC];
    params<T, VEC>(w, c0, wv, 1.f);
    params<T, VEC>(bias, c0, bv, 0.f);
    const Groups<VEC> of(c0, Cg);
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float mu[VEC], sc[VEC];
        of.get(mean + b * G, mu);
        of.get(rstd + b * G, sc);
#pragma unroll
        for (int v = 0; v < VEC; ++v) sc[v] *= wv[v];
        const int64_t base = b * P * C + c0;
        for (int64_t r = first + rl; r < last; r += (int64_t)k.lanes_r * UNROLL) {
            Pack<T, VEC> p[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t ru = r + (int64_t)u * k.lanes_r;
                p[u] = *reinterpret_cast<const Pack<T, VEC> *>(x + base + (ru < last ? ru : first) * C);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t ru = r + (int64_t)u * k.lanes_r;
                if (ru >= last) break;
                float z[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) z[v] = fmaf((float)p[u].v[v] - mu[v], sc[v], bv[v]);
                act_values<is_f32<T>(), VEC>(z, act);
#pragma unroll
                for (int v = 0; v < VEC; ++v) p[u].v[v] = (T)z[v];
                *reinterpret_cast<Pack<T, VEC> *>(y + base + ru * C) = p[u];
            }
        }
    }
}

// ---- backward ----

// part[unit * C + c] = the chunk's sums of dz and dz n
template <typename T, int VEC, bool KEPT>
__global__ void __launch_bounds__(TB) norm_sums_kernel(Source<T, VEC, KEPT> src, const T *__restrict__ dy,
                                                       const void *__restrict__ w, const void *__restrict__ bias,
                                                       const float *__restrict__ mean, const float *__restrict__ rstd,
                                                       float2 *__restrict__ part, int64_t P, int C, int G, int Cg,
                                                       int act, Cut k) {
    __shared__ float2 red[TB * VEC];
    const int t = threadIdx.x, col = t % k.cols, rl = t / k.cols, tile = blockIdx.y;
    const int c0 = (tile * k.cols + col) * VEC;
    const bool active = rl < k.lanes_r && c0 < C;
    const int step = k.lanes_r * C, step_e = k.lanes_r * src.blocks;   // (under 2^21)
    float wv[VEC], bv[VEC];
    if (active) {
        params<T, VEC>(w, c0, wv, 1.f);
        params<T, VEC>(bias, c0, bv, 0.f);
    }
    const Groups<VEC> of(active ? c0 : 0, Cg);
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float s[VEC], q[VEC], mu[VEC], rs[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) s[v] = q[v] = 0.f;
        if (active) {
            of.get(mean + b * G, mu);
            of.get(rstd + b * G, rs);
            int64_t at = src.at(b * P + first + rl, c0), block = src.block(b * P + first + rl, c0);
            for (int64_t r = first + rl; r < last; r += (int64_t)k.lanes_r * UNROLL, at += UNROLL * step, block += UNROLL * step_e) {
                Pack<T, VEC> d[UNROLL];
                typename Source<T, VEC, KEPT>::Raw raw[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {   // (past the chunk's end: the first of them again)
                    const bool in = r + u * k.lanes_r < last;
                    const int64_t at_u = at + (in ? u * step : 0);
                    d[u] = *reinterpret_cast<const Pack<T, VEC> *>(dy + at_u);
                    raw[u] = src.load(at_u, block + (in ? u * step_e : 0));
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    if (r + u * k.lanes_r >= last) break;
                    float f[VEC], z[VEC], dz[VEC];
                    src.values(raw[u], f);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        f[v] = (f[v] - mu[v]) * rs[v];
                        z[v] = fmaf(f[v], wv[v], bv[v]);
                        dz[v] = (float)d[u].v[v];
                    }
                    act_slopes<is_f32<T>(), VEC>(dz, z, act);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        s[v] += dz[v];
                        q[v] = fmaf(dz[v], f[v], q[v]);
                    }
                }
            }
        }
        sum_pixel_lanes<VEC>(red, s, q, t, k, active);
        const int base = tile * k.cols * VEC;
        for (int i = t; i < k.cols * VEC && base + i < C; i += TB) part[unit * C + base + i] = red[i];
        __syncthreads();
    }
}

constexpr int FIN = 1024;   // lanes of the step that adds up the chunks' sums: 4 loads each in flight cover 256 chunks in one go

// The first BG workgroups: avg(dn) and avg(dn n) of a (batch, group) into avg. The others: 16 channels of dw and db each, 64
// lanes along the chunks of all images.
template <typename T>
__global__ void __launch_bounds__(FIN) norm_bwd_finish_kernel(const float2 *__restrict__ part, const void *__restrict__ w,
                                                              float2 *__restrict__ avg, T *__restrict__ dw,
                                                              T *__restrict__ db, int64_t BG, int64_t P, int C, int G,
                                                              int Cg, int chunks, int64_t units) {
    __shared__ float2 red[FIN];
    const int t = threadIdx.x;
    const int64_t jobs = BG + (dw || db ? (C + 15) / 16 : 0);
    for (int64_t job = blockIdx.x; job < jobs; job += gridDim.x) {
        float s = 0.f, q = 0.f;
        if (job < BG) {
            const int64_t b = job / G;
            const int g = (int)(job - b * G);
            for (int64_t i = t; i < (int64_t)chunks * Cg; i += FIN) {
                const int64_t chunk = i / Cg;
                const int c = g * Cg + (int)(i - chunk * Cg);
                const float2 v = part[(b * chunks + chunk) * C + c];
                const float wc = w ? (float)((const T *)w)[c] : 1.f;
                s = fmaf(v.x, wc, s);
                q = fmaf(v.y, wc, q);
            }
            s = wave_sum(s);
            q = wave_sum(q);
            if ((t & 63) == 0) red[t >> 6] = make_float2(s, q);
            __syncthreads();
            if (t < 64) {
                const float2 v = t < FIN / 64 ? red[t] : make_float2(0.f, 0.f);
                const float n = (float)((double)P * Cg);
                s = wave_sum(v.x) / n;
                q = wave_sum(v.y) / n;
                if (t == 0) avg[job] = make_float2(s, q);
            }
        } else {
            const int c = (int)(job - BG) * 16 + (t & 15);
            if (c < C)
                for (int64_t u = t >> 4; u < units; u += 4 * (FIN / 16)) {
                    float2 v[4];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int64_t uk = u + k * (FIN / 16);
                        v[k] = uk < units ? part[uk * C + c] : make_float2(0.f, 0.f);
                    }
#pragma unroll
                    for (int k = 0; k < 4; ++k) s += v[k].x, q += v[k].y;
                }
            red[t] = make_float2(s, q);
            __syncthreads();
            if (t < 64) {   // four lanes a channel, 16 rows each
                float2 a = red[t];
                for (int k = 64; k < FIN; k += 64) a.x += red[t + k].x, a.y += red[t + k].y;
                a.x += __shfl_xor(a.x, 16), a.y += __shfl_xor(a.y, 16);
                a.x += __shfl_xor(a.x, 32), a.y += __shfl_xor(a.y, 32);
                if (t < 16 && c < C) {
                    if (db) db[c] = (T)a.x;
                    if (dw) dw[c] = (T)a.y;
                }
            }
        }
        __syncthreads();
    }
}

template <typename T, int VEC, bool KEPT>
__global__ void __launch_bounds__(TB) norm_dx_kernel(Source<T, VEC, KEPT> src, const T *__restrict__ dy,
                                                     const void *__restrict__ w, const void *__restrict__ bias,
                                                     const float *__restrict__ mean, const float *__restrict__ rstd,
                                                     const float2 *__restrict__ avg, T *__restrict__ dx, int64_t P,
                                                     int C, int G, int Cg, int act, Cut k) {
    const int t = threadIdx.x, col = t % k.cols, rl = t / k.cols;
    const int c0 = (blockIdx.y * k.cols + col) * VEC;
    if (rl >= k.lanes_r || c0 >= C) return;
    const int step = k.lanes_r * C, step_e = k.lanes_r * src.blocks;
    float wv[VEC], bv[VEC];
    params<T, VEC>(w, c0, wv, 1.f);
    params<T, VEC>(bias, c0, bv, 0.f);
    const Groups<VEC> of(c0, Cg);
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float mu[VEC], rs[VEC];
        float2 av[VEC];
        of.get(mean + b * G, mu);
        of.get(rstd + b * G, rs);
        of.get(avg + b * G, av);
        int64_t at = src.at(b * P + first + rl, c0), block = src.block(b * P + first + rl, c0);
        for (int64_t r = first + rl; r < last; r += (int64_t)k.lanes_r * UNROLL, at += UNROLL * step, block += UNROLL * step_e) {
            Pack<T, VEC> d[UNROLL];
            typename Source<T, VEC, KEPT>::Raw raw[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const bool in = r + u * k.lanes_r < last;
                const int64_t at_u = at + (in ? u * step : 0);
                d[u] = *reinterpret_cast<const Pack<T, VEC> *>(dy + at_u);
                raw[u] = src.load(at_u, block + (in ? u * step_e : 0));
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                if (r + u * k.lanes_r >= last) break;
                float f[VEC], z[VEC], dz[VEC];
                src.values(raw[u], f);
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    f[v] = (f[v] - mu[v]) * rs[v];
                    z[v] = fmaf(f[v], wv[v], bv[v]);
                    dz[v] = (float)d[u].v[v];
                }
                act_slopes<is_f32<T>(), VEC>(dz, z, act);
#pragma unroll
                for (int v = 0; v < VEC; ++v) d[u].v[v] = (T)(rs[v] * (dz[v] * wv[v] - av[v].x - f[v] * av[v].y));
                *reinterpret_cast<Pack<T, VEC> *>(dx + at + u * step) = d[u];
            }
        }
    }
}

// ---- whole groups: a group's values stay in registers between the sums and the results, so a map is read once and one launch
// does it. TG lanes per group (several groups to a workgroup of 256 where TG < 256), NV accesses of VEC channels per lane. ----

constexpr int block_of(int TG) { return TG > 256 ? TG : 256; }

// Workgroups go to the 8 XCDs in turn: each gets a run of neighbouring groups, which share lines of the map in one L2
__device__ __forceinline__ int64_t xcd_run(int64_t id, int64_t total) {
    const int64_t per = total / 8, extra = total % 8, xcd = id % 8;
    return xcd * per + (xcd < extra ? xcd : extra) + id / 8;
}

template <int TG> __device__ __forceinline__ float group_sum(float v, float *red, int t) {
    constexpr int W = TG < 64 ? TG : 64;
#pragma unroll
    for (int m = 1; m < W; m <<= 1) v += __shfl_xor(v, m);
    if constexpr (TG > 64) {
        __syncthreads();   // (the last sum's values have been read)
        if ((t & 63) == 0) red[t >> 6] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TG / 64; ++w) v += red[t / TG * (TG / 64) + w];
    }
    return v;
}

// A lane's place: group, first channel of its accesses, and its pixels first, first + rows, ...
template <int TG, int VEC> struct Place {
    int64_t bg, b;
    int g, c0, first, rows, cv;
    bool on;   // lanes beyond the last whole row of accesses, or beyond the groups, hold nothing
    __device__ __forceinline__ Place(int64_t groups, int64_t blocks, int G, int Cg, int64_t P) {
        const int t = threadIdx.x, l = t % TG;
        bg = xcd_run(blockIdx.x, blocks) * (block_of(TG) / TG) + t / TG;
        on = bg < groups;
        if (!on) bg = groups - 1;
        b = bg / G;
        g = (int)(bg - b * G);
        cv = Cg / VEC;
        rows = TG / cv;
        first = l / cv;
        c0 = g * Cg + (l - first * cv) * VEC;
        on = on && first < rows;
        if (!on) first = (int)P;
    }
};

template <typename T, int VEC, int TG, int NV>
__global__ void __launch_bounds__(block_of(TG)) norm_group_kernel(const T *__restrict__ x, const void *__restrict__ w,
                                                                  const void *__restrict__ bias, T *__restrict__ y,
                                                                  float *__restrict__ mean, float *__restrict__ rstd,
                                                                  int64_t groups, int64_t blocks, int64_t P, int C, int G, int Cg,
                                                                  float eps, int act) {
    __shared__ float red[block_of(TG) / 64];
    const int t = threadIdx.x;
    const Place<TG, VEC> at(groups, blocks, G, Cg, P);
    const int64_t base = at.b * P * C + at.c0;
    Pack<T, VEC> p[NV];
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int r = at.first + i * at.rows;
        if (r < P) p[i] = *reinterpret_cast<const Pack<T, VEC> *>(x + base + (int64_t)r * C);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at.first + i * at.rows < P)
#pragma unroll
            for (int v = 0; v < VEC; ++v) s += (float)p[i].v[v];
    const float n = (float)(P * Cg), mu = group_sum<TG>(s, red, t) / n;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at.first + i * at.rows < P)
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const float d = (float)p[i].v[v] - mu;
                s = fmaf(d, d, s);
            }
    const float rs = 1.f / sqrtf(group_sum<TG>(s, red, t) / n + eps);
    if (!at.on) return;
    if (t % TG == 0) mean[at.bg] = mu, rstd[at.bg] = rs;
    float sc[VEC], bv[VEC];
    params<T, VEC>(w, at.c0, sc, 1.f);
    params<T, VEC>(bias, at.c0, bv, 0.f);
#pragma unroll
    for (int v = 0; v < VEC; ++v) sc[v] *= rs;
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int r = at.first + i * at.rows;
        if (r >= P) break;
        float z[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) z[v] = fmaf((float)p[i].v[v] - mu, sc[v], bv[v]);
        act_values<is_f32<T>(), VEC>(z, act);
#pragma unroll
        for (int v = 0; v < VEC; ++v) p[i].v[v] = (T)z[v];
        *reinterpret_cast<Pack<T, VEC> *>(y + base + (int64_t)r * C) = p[i];
    }
}

// dx, and the group's sums of dz and dz n per channel: part[b * C + c], or dw and db themselves where there is one image. n and
// dz stay in registers too, so these are smaller groups.
template <typename T, int VEC, int TG, int NV, bool KEPT>
__global__ void __launch_bounds__(block_of(TG))
    norm_group_bwd_kernel(Source<T, VEC, KEPT> src, const T *__restrict__ dy, const void *__restrict__ w,
                          const void *__restrict__ bias, const float *__restrict__ mean, const float *__restrict__ rstd,
                          T *__restrict__ dx, float2 *__restrict__ part, T *__restrict__ dw, T *__restrict__ db,
                          int64_t groups, int64_t blocks, int64_t P, int C, int G, int Cg, int act) {
    __shared__ float2 sums[block_of(TG) * VEC];
    float *red = (float *)sums;   // (before the sums)
    const int t = threadIdx.x;
    const Place<TG, VEC> at(groups, blocks, G, Cg, P);
    const int64_t base = at.b * P * C + at.c0;
    const float mu = mean[at.bg], rs = rstd[at.bg];
    float wv[VEC], bv[VEC], s[VEC], q[VEC];
    params<T, VEC>(w, at.c0, wv, 1.f);
    params<T, VEC>(bias, at.c0, bv, 0.f);
#pragma unroll
    for (int v = 0; v < VEC; ++v) s[v] = q[v] = 0.f;
    float f[NV][VEC], d[NV][VEC];   // n, dz
    typename Source<T, VEC, KEPT>::Raw raw[NV];
    Pack<T, VEC> g[NV];
#pragma unroll
    for (int i = 0; i < NV; ++i) {
        const int r = at.first + i * at.rows;
        if (r < P) {
            raw[i] = src.load(src.at(at.b * P + r, at.c0), src.block(at.b * P + r, at.c0));
            g[i] = *reinterpret_cast<const Pack<T, VEC> *>(dy + base + (int64_t)r * C);
        }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i)
        if (at.first + i * at.rows < P) {
            float z[VEC];
            src.values(raw[i], f[i]);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                d[i][v] = (float)g[i].v[v];
                f[i][v] = (f[i][v] - mu) * rs;
                z[v] = fmaf(f[i][v], wv[v], bv[v]);
            }
            act_slopes<is_f32<T>(), VEC>(d[i], z, act);
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                s[v] += d[i][v];
                q[v] = fmaf(d[i][v], f[i][v], q[v]);
            }
        }
    float a1 = 0.f, a2 = 0.f;
#pragma unroll
    for (int v = 0; v < VEC; ++v) a1 = fmaf(s[v], wv[v], a1), a2 = fmaf(q[v], wv[v], a2);
    const float n = (float)(P * Cg);
    a1 = group_sum<TG>(a1, red, t) / n;
    a2 = group_sum<TG>(a2, red, t) / n;
    if (dx)
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int r = at.first + i * at.rows;
            if (r >= P) break;
            Pack<T, VEC> p;
#pragma unroll
            for (int v = 0; v < VEC; ++v) p.v[v] = (T)(rs * (d[i][v] * wv[v] - a1 - f[i][v] * a2));
            *reinterpret_cast<Pack<T, VEC> *>(dx + base + (int64_t)r * C) = p;
        }
    if (!part && !dw && !db) return;
    // per channel: the lanes of its accesses, added up by one wave (or by the group's lanes) per channel
    const int l = t % TG, own = t / TG * TG * VEC;
    __syncthreads();
    if (at.on)
#pragma unroll
        for (int v = 0; v < VEC; ++v) sums[own + l * VEC + v] = make_float2(s[v], q[v]);
    __syncthreads();
    const int used = min(at.rows, (int)(P < TG ? P : TG));   // lanes along the pixels that held any
    auto write = [&](int c, float sc, float qc) {
        const int64_t to = at.b * C + at.g * Cg + c;
        if (part) part[to] = make_float2(sc, qc);
        if (!part && db) db[to] = (T)sc;
        if (!part && dw) dw[to] = (T)qc;
    };
    const bool there = xcd_run(blockIdx.x, blocks) * (block_of(TG) / TG) + t / TG < groups;
    if constexpr (TG > 64) {
        for (int c = l >> 6; c < Cg; c += TG / 64) {
            float sc = 0.f, qc = 0.f;
            for (int r = l & 63; r < used; r += 64) {
                const float2 a = sums[own + r * Cg + c];
                sc += a.x, qc += a.y;
            }
            sc = wave_sum(sc);
            qc = wave_sum(qc);
            if ((l & 63) == 0 && there) write(c, sc, qc);
        }
    } else if (there) {
        for (int c = l; c < Cg; c += TG) {
            float sc = 0.f, qc = 0.f;
            for (int r = 0; r < used; ++r) {
                const float2 a = sums[own + r * Cg + c];
                sc += a.x, qc += a.y;
            }
            write(c, sc, qc);
        }
    }
}

constexpr int64_t MOST_GROUPS = 1 << 22;   // a workgroup each: HIP takes fewer than 2^32 threads along x

// What a group takes: lanes, and accesses per lane (0: a workgroup does not hold it, or not at a gain). Forward, groups of up to 64
// / 512 / 4096 / 16384 / 65536 values of 16 bits whose channels come in eights (half as many float32 ones in fours; an eighth to
// a half of that one by one): (8, 256, 64 x 64) in 32 groups 15.7 us instead of 18.5, (16, 512, 4096) 31.2 instead of 41.2,
// bfloat16 (in a graph). Backward, up to 16384 (2048 one by one): (8, 256, 32 x 32) 13.7 us instead of 17.4; four times that does not fit
// beside the sums and takes 35.3 instead of 33.1 read twice.
struct Whole {
    int TG, NV;
};
template <int VEC> Whole whole_of(const NormArgs &a, bool backward) {
    const int Cg = a.channels / a.groups, cv = Cg / VEC;
    if (Cg % VEC || a.batch * a.groups >= MOST_GROUPS) return {0, 0};
    constexpr int FEW = VEC > 1 ? 2 : 8, MANY = VEC > 1 ? 8 : 32;
    for (const Whole &k : {Whole{4, FEW}, Whole{32, FEW}, Whole{256, FEW}, Whole{256, MANY}, Whole{1024, MANY}}) {
        if (backward && (k.TG == 1024 || k.NV == 32)) break;
        if (cv <= k.TG && a.pixels <= (int64_t)(k.TG / cv) * k.NV) return k;
    }
    return {0, 0};
}

constexpr int64_t MOST_BLOCKS = 1 << 20;   // (HIP takes fewer than 2^32 threads along x; the kernels stride)
dim3 grid_of(const Cut &k) { return dim3((unsigned)(k.units < MOST_BLOCKS ? k.units : MOST_BLOCKS), (unsigned)k.tiles); }
unsigned grid_1d(int64_t n) { return (unsigned)(n < MOST_BLOCKS ? n : MOST_BLOCKS); }

// Channels per access: 16 bytes where the rows allow it. (Where the rows do and the groups do not, whole groups go one by one if
// they fit, else the rows in whole accesses.)
template <typename T> int vec_of(const NormArgs &a, bool backward) {
    constexpr int V = 16 / sizeof(T);
    if (a.channels % V) return 1;
    return a.channels / a.groups % V && whole_of<1>(a, backward).TG ? 1 : V;
}
int vec_of(const NormArgs &a, bool backward) {
    return a.dtype == TVDCN_DTYPE_FLOAT32 ? vec_of<float>(a, backward) : vec_of<f16>(a, backward);
}

template <typename T, int VEC, int TG, int NV> hipError_t forward_groups(const NormArgs &a, hipStream_t s) {
    const int64_t groups = a.batch * a.groups, blocks = ceil_div(groups, block_of(TG) / TG);
    norm_group_kernel<T, VEC, TG, NV><<<(unsigned)blocks, block_of(TG), 0, s>>>(
        (const T *)a.x, a.weight, a.bias, (T *)a.y, a.mean, a.rstd, groups, blocks, a.pixels, a.channels, a.groups,
        a.channels / a.groups, a.eps, a.act);
    return hipGetLastError();
}

template <typename T, int VEC, int TG, int NV, bool KEPT> hipError_t backward_groups(const NormArgs &a, hipStream_t s) {
    const int C = a.channels;
    const int64_t groups = a.batch * a.groups, blocks = ceil_div(groups, block_of(TG) / TG);
    const bool params = a.dweight || a.dbias, one = a.batch == 1;
    float2 *part = params && !one ? (float2 *)a.part : nullptr;
    const Source<T, VEC, KEPT> src{(const T *)a.x, a.codes, a.exps, C, (int)ceil_div(C, kKeptBlock)};
    norm_group_bwd_kernel<T, VEC, TG, NV, KEPT><<<(unsigned)blocks, block_of(TG), 0, s>>>(
        src, (const T *)a.dy, a.weight, a.bias, a.mean, a.rstd, (T *)a.dx, part, one ? (T *)a.dweight : nullptr,
        one ? (T *)a.dbias : nullptr, groups, blocks, a.pixels, C, a.groups, C / a.groups, a.act);
    if (hipError_t e = hipGetLastError()) return e;
    if (part)
        norm_bwd_finish_kernel<T><<<grid_1d(ceil_div(C, 16)), FIN, 0, s>>>(part, a.weight, nullptr, (T *)a.dweight, (T *)a.dbias,
                                                                          0, 0, C, a.groups, C / a.groups, 0, a.batch);
    return hipGetLastError();
}

template <typename T, int VEC> hipError_t forward(const NormArgs &a, hipStream_t s) {
    const int C = a.channels, G = a.groups, Cg = C / G;
    constexpr int FEW = VEC > 1 ? 2 : 8, MANY = VEC > 1 ? 8 : 32;
    if (const Whole k = whole_of<VEC>(a, false); k.TG) {
        if (k.TG == 4) return forward_groups<T, VEC, 4, FEW>(a, s);
        if (k.TG == 32) return forward_groups<T, VEC, 32, FEW>(a, s);
        if (k.TG == 1024) return forward_groups<T, VEC, 1024, MANY>(a, s);
        return k.NV == FEW ? forward_groups<T, VEC, 256, FEW>(a, s) : forward_groups<T, VEC, 256, MANY>(a, s);
    }
    const Cut k = make_cut(a.batch, a.pixels, C, VEC);
    const T *x = (const T *)a.x;
    norm_stats_kernel<T, VEC><<<grid_of(k), TB, 0, s>>>(x, (float2 *)a.part, a.pixels, C, G, Cg, k);
    if (hipError_t e = hipGetLastError()) return e;
    norm_finish_kernel<<<grid_1d(a.batch * G), 64, 0, s>>>((const float2 *)a.part, a.mean, a.rstd, a.batch * G, a.pixels, G, Cg,
                                                           k.cols * VEC, a.eps, k);
    if (hipError_t e = hipGetLastError()) return e;
    norm_apply_kernel<T, VEC><<<grid_of(k), TB, 0, s>>>(x, a.weight, a.bias, a.mean, a.rstd, (T *)a.y, a.pixels, C, G,
                                                        Cg, a.act, k);
    return hipGetLastError();
}

template <typename T, int VEC, bool KEPT> hipError_t backward(const NormArgs &a, hipStream_t s) {
    const int C = a.channels, G = a.groups, Cg = C / G;
    if (a.batch == 0 || a.pixels == 0) {   // sums of nothing
        if (a.dweight || a.dbias)
            norm_bwd_finish_kernel<T><<<grid_1d(ceil_div(C, 16)), FIN, 0, s>>>(nullptr, a.weight, nullptr, (T *)a.dweight,
                                                                             (T *)a.dbias, 0, 0, C, G, Cg, 0, 0);
        return hipGetLastError();
    }
    constexpr int FEW = VEC > 1 ? 2 : 8;
    if (const Whole k = whole_of<VEC>(a, true); k.TG) {
        if (k.TG == 4) return backward_groups<T, VEC, 4, FEW, KEPT>(a, s);
        if (k.TG == 32) return backward_groups<T, VEC, 32, FEW, KEPT>(a, s);
        return k.NV == FEW ? backward_groups<T, VEC, 256, FEW, KEPT>(a, s) : backward_groups<T, VEC, 256, 8, KEPT>(a, s);
    }
    const Cut k = make_cut(a.batch, a.pixels, C, VEC);
    const int64_t BG = a.batch * G;
    float2 *avg = (float2 *)a.part, *part = avg + BG;
    const Source<T, VEC, KEPT> src{(const T *)a.x, a.codes, a.exps, C, (int)ceil_div(C, kKeptBlock)};
    norm_sums_kernel<T, VEC, KEPT><<<grid_of(k), TB, 0, s>>>(src, (const T *)a.dy, a.weight, a.bias, a.mean, a.rstd,
                                                             part, a.pixels, C, G, Cg, a.act, k);
    if (hipError_t e = hipGetLastError()) return e;
    norm_bwd_finish_kernel<T><<<grid_1d(BG + ceil_div(C, 16)), FIN, 0, s>>>(
        part, a.weight, avg, (T *)a.dweight, (T *)a.dbias, BG, a.pixels, C, G, Cg, k.chunks, k.units);
    if (hipError_t e = hipGetLastError()) return e;
    if (a.dx)
        norm_dx_kernel<T, VEC, KEPT><<<grid_of(k), TB, 0, s>>>(src, (const T *)a.dy, a.weight, a.bias, a.mean, a.rstd,
                                                               avg, (T *)a.dx, a.pixels, C, G, Cg, a.act, k);
    return hipGetLastError();
}

template <typename T> hipError_t forward_of(const NormArgs &a, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    return vec_of<T>(a, false) == V ? forward<T, V>(a, s) : forward<T, 1>(a, s);
}
template <typename T> hipError_t backward_of(const NormArgs &a, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    if (vec_of<T>(a, true) == V) return a.codes ? backward<T, V, true>(a, s) : backward<T, V, false>(a, s);
    return a.codes ? backward<T, 1, true>(a, s) : backward<T, 1, false>(a, s);
}

}  // namespace

int64_t norm_part_floats(const NormArgs &a, bool backward) {
    const int vec = vec_of(a, backward);
    const Whole whole = vec == 1 ? whole_of<1>(a, backward) : vec == 4 ? whole_of<4>(a, backward) : whole_of<8>(a, backward);
    if (whole.TG) return backward && a.batch > 1 ? 2 * a.batch * a.channels : 0;
    const Cut k = make_cut(a.batch, a.pixels, a.channels, vec);
    return backward ? 2 * (a.batch * a.groups + k.units * a.channels) : 2 * k.units * k.tiles * a.groups;
}

hipError_t launch_norm_forward(const NormArgs &a, hipStream_t s) {
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return forward_of<float>(a, s);
        case TVDCN_DTYPE_FLOAT16: return forward_of<f16>(a, s);
        default: return forward_of<bf16>(a, s);
    }
}

hipError_t launch_norm_backward(const NormArgs &a, hipStream_t s) {
    switch (a.dtype) {
        case TVDCN_DTYPE_FLOAT32: return backward_of<float>(a, s);
        case TVDCN_DTYPE_FLOAT16: return backward_of<f16>(a, s);
        default: return backward_of<bf16>(a, s);
    }
}

}  // namespace tvdcn_hip
