// Group normalisation with affine map and activation over channels-last maps [batch][pixels][channels]:
//
//   n = (x - mean) rstd,  z = w n + b,  y = act(z);  mean and variance over the pixels and the Cg channels of a
//   (batch, group);  dz = dy act'(z),  dn = w dz,  dx = rstd (dn - avg(dn) - n avg(dn n)),  dw = sum dz n,  db = sum dz
//
// Bound by memory. Forward: the statistics read x once, the second pass reads it again (from the 256 MB last-level
// cache where it fits) and writes y. A workgroup takes a run of pixels of one image and all channels (in tiles of 256
// lanes), so every access is a run of whole rows; a lane keeps its 16 bytes of channels over all its pixels, and with
// them the parameters of those channels. Sums are float32, of deviations from the group's first value (large means
// against small spreads do not cancel), combined in a fixed order.
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

// A lane's VEC channels of a pixel, from the map or its 8-bit form
template <typename T, int VEC, bool KEPT> struct Source {
    const T *x;
    const int8_t *codes;
    const uint8_t *exps;
    int C, blocks;
    __device__ __forceinline__ void get(int64_t row, int c, float *f) const {
        if constexpr (KEPT) {
            const Pack<int8_t, VEC> q = *reinterpret_cast<const Pack<int8_t, VEC> *>(codes + row * C + c);
            const float scale = kept_scale<T>(exps[row * blocks + c / kKeptBlock]);
#pragma unroll
            for (int v = 0; v < VEC; ++v) f[v] = kept_value<T>(q.v[v], scale);
        } else {
            const Pack<T, VEC> p = *reinterpret_cast<const Pack<T, VEC> *>(x + row * C + c);
#pragma unroll
            for (int v = 0; v < VEC; ++v) f[v] = (float)p.v[v];
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

// part[(unit * tiles + tile) * G + g] = the tile's sums of x - shift and its square, shift = the group's first value
template <typename T, int VEC>
__global__ void __launch_bounds__(TB) norm_stats_kernel(const T *__restrict__ x, float2 *__restrict__ part, int64_t P,
                                                        int C, int G, int Cg, Cut k) {
    __shared__ float2 red[TB * VEC];
    const int t = threadIdx.x, col = t % k.cols, rl = t / k.cols, tile = blockIdx.y;
    const int c0 = (tile * k.cols + col) * VEC;
    const bool active = rl < k.lanes_r && c0 < C;
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float s[VEC], q[VEC], shift[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) s[v] = q[v] = shift[v] = 0.f;
        if (active) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) shift[v] = (float)x[b * P * C + (c0 + v) / Cg * Cg];
            const T *xb = x + b * P * C + c0;
            for (int64_t r = first + rl; r < last; r += (int64_t)k.lanes_r * UNROLL) {
                Pack<T, VEC> p[UNROLL];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    const int64_t ru = r + (int64_t)u * k.lanes_r;
                    p[u] = *reinterpret_cast<const Pack<T, VEC> *>(xb + (ru < last ? ru : first) * C);
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    if (r + (int64_t)u * k.lanes_r >= last) break;
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        const float d = (float)p[u].v[v] - shift[v];
                        s[v] += d;
                        q[v] = fmaf(d, d, q[v]);
                    }
                }
            }
        }
        sum_pixel_lanes<VEC>(red, s, q, t, k, active);
        // a wave per group of the tile
        const int base = tile * k.cols * VEC, end = min(base + k.cols * VEC, C);
        for (int g = base / Cg + t / 64; g <= (end - 1) / Cg; g += TB / 64) {
            const int lo = max(g * Cg, base), hi = min((g + 1) * Cg, end);
            float a = 0.f, c = 0.f;
            for (int i = lo + (t & 63); i < hi; i += 64) {
                a += red[i - base].x;
                c += red[i - base].y;
            }
            a = wave_sum(a);
            c = wave_sum(c);
            if ((t & 63) == 0) part[(unit * k.tiles + tile) * G + g] = make_float2(a, c);
        }
        __syncthreads();
    }
}

// mean and rstd of a (batch, group) from its chunks' sums: a wave each
template <typename T>
__global__ void __launch_bounds__(64) norm_finish_kernel(const T *__restrict__ x, const float2 *__restrict__ part,
                                                         float *__restrict__ mean, float *__restrict__ rstd, int64_t BG,
                                                         int64_t P, int C, int G, int Cg, int tile_c, float eps, Cut k) {
    for (int64_t i = blockIdx.x; i < BG; i += gridDim.x) {
        const int64_t b = i / G;
        const int g = (int)(i - b * G);
        const int t0 = g * Cg / tile_c, nt = ((g + 1) * Cg - 1) / tile_c - t0 + 1;
        double s = 0.0, q = 0.0;
        for (int j = threadIdx.x; j < k.chunks * nt; j += 64) {
            const float2 v = part[((b * k.chunks + j / nt) * k.tiles + t0 + j % nt) * G + g];
            s += v.x;
            q += v.y;
        }
        s = wave_sum(s);
        q = wave_sum(q);
        if (threadIdx.x == 0) {
            const double n = (double)P * Cg, m = s / n;
            const double var = q / n - m * m;
            mean[i] = (float)((double)(float)x[b * P * C + (int64_t)g * Cg] + m);
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
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float mu[VEC], sc[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int64_t i = b * G + (c0 + v) / Cg;
            mu[v] = mean[i];
            sc[v] = rstd[i] * wv[v];
        }
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
    float wv[VEC], bv[VEC];
    if (active) {
        params<T, VEC>(w, c0, wv, 1.f);
        params<T, VEC>(bias, c0, bv, 0.f);
    }
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float s[VEC], q[VEC], mu[VEC], rs[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) s[v] = q[v] = 0.f;
        if (active) {
#pragma unroll
            for (int v = 0; v < VEC; ++v) {
                const int64_t i = b * G + (c0 + v) / Cg;
                mu[v] = mean[i];
                rs[v] = rstd[i];
            }
            const T *dyb = dy + b * P * C + c0;
            for (int64_t r = first + rl; r < last; r += (int64_t)k.lanes_r * UNROLL) {
                Pack<T, VEC> d[UNROLL];
                float f[UNROLL][VEC];
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    int64_t ru = r + (int64_t)u * k.lanes_r;
                    ru = ru < last ? ru : first;
                    d[u] = *reinterpret_cast<const Pack<T, VEC> *>(dyb + ru * C);
                    src.get(b * P + ru, c0, f[u]);
                }
#pragma unroll
                for (int u = 0; u < UNROLL; ++u) {
                    if (r + (int64_t)u * k.lanes_r >= last) break;
                    float z[VEC], dz[VEC];
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        f[u][v] = (f[u][v] - mu[v]) * rs[v];
                        z[v] = fmaf(f[u][v], wv[v], bv[v]);
                        dz[v] = (float)d[u].v[v];
                    }
                    act_slopes<is_f32<T>(), VEC>(dz, z, act);
#pragma unroll
                    for (int v = 0; v < VEC; ++v) {
                        s[v] += dz[v];
                        q[v] = fmaf(dz[v], f[u][v], q[v]);
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
    float wv[VEC], bv[VEC];
    params<T, VEC>(w, c0, wv, 1.f);
    params<T, VEC>(bias, c0, bv, 0.f);
    for (int64_t unit = blockIdx.x; unit < k.units; unit += gridDim.x) {
        const int64_t b = unit / k.chunks, chunk = unit - b * k.chunks;
        const int64_t first = chunk * k.rows, last = first + k.rows < P ? first + k.rows : P;
        float mu[VEC], rs[VEC], a1[VEC], a2[VEC];
#pragma unroll
        for (int v = 0; v < VEC; ++v) {
            const int64_t i = b * G + (c0 + v) / Cg;
            mu[v] = mean[i];
            rs[v] = rstd[i];
            a1[v] = avg[i].x;
            a2[v] = avg[i].y;
        }
        const int64_t base = b * P * C + c0;
        for (int64_t r = first + rl; r < last; r += (int64_t)k.lanes_r * UNROLL) {
            Pack<T, VEC> d[UNROLL];
            float f[UNROLL][VEC];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                int64_t ru = r + (int64_t)u * k.lanes_r;
                ru = ru < last ? ru : first;
                d[u] = *reinterpret_cast<const Pack<T, VEC> *>(dy + base + ru * C);
                src.get(b * P + ru, c0, f[u]);
            }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u) {
                const int64_t ru = r + (int64_t)u * k.lanes_r;
                if (ru >= last) break;
                float z[VEC], dz[VEC];
#pragma unroll
                for (int v = 0; v < VEC; ++v) {
                    f[u][v] = (f[u][v] - mu[v]) * rs[v];
                    z[v] = fmaf(f[u][v], wv[v], bv[v]);
                    dz[v] = (float)d[u].v[v];
                }
                act_slopes<is_f32<T>(), VEC>(dz, z, act);
#pragma unroll
                for (int v = 0; v < VEC; ++v) d[u].v[v] = (T)(rs[v] * (dz[v] * wv[v] - a1[v] - f[u][v] * a2[v]));
                *reinterpret_cast<Pack<T, VEC> *>(dx + base + ru * C) = d[u];
            }
        }
    }
}

constexpr int64_t MOST_BLOCKS = 1 << 20;   // (HIP takes fewer than 2^32 threads along x; the kernels stride)
dim3 grid_of(const Cut &k) { return dim3((unsigned)(k.units < MOST_BLOCKS ? k.units : MOST_BLOCKS), (unsigned)k.tiles); }
unsigned grid_1d(int64_t n) { return (unsigned)(n < MOST_BLOCKS ? n : MOST_BLOCKS); }

template <typename T> int vec_of(const NormArgs &a) { return a.channels % (16 / sizeof(T)) == 0 ? 16 / sizeof(T) : 1; }
int vec_of(const NormArgs &a) { return a.dtype == TVDCN_DTYPE_FLOAT32 ? vec_of<float>(a) : vec_of<f16>(a); }

template <typename T, int VEC> hipError_t forward(const NormArgs &a, hipStream_t s) {
    const int C = a.channels, G = a.groups, Cg = C / G;
    const Cut k = make_cut(a.batch, a.pixels, C, VEC);
    const T *x = (const T *)a.x;
    norm_stats_kernel<T, VEC><<<grid_of(k), TB, 0, s>>>(x, (float2 *)a.part, a.pixels, C, G, Cg, k);
    if (hipError_t e = hipGetLastError()) return e;
    norm_finish_kernel<T><<<grid_1d(a.batch * G), 64, 0, s>>>(x, (const float2 *)a.part, a.mean, a.rstd, a.batch * G,
                                                              a.pixels, C, G, Cg, k.cols * VEC, a.eps, k);
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
    return vec_of<T>(a) == V ? forward<T, V>(a, s) : forward<T, 1>(a, s);
}
template <typename T> hipError_t backward_of(const NormArgs &a, hipStream_t s) {
    constexpr int V = 16 / sizeof(T);
    if (vec_of<T>(a) == V) return a.codes ? backward<T, V, true>(a, s) : backward<T, V, false>(a, s);
    return a.codes ? backward<T, 1, true>(a, s) : backward<T, 1, false>(a, s);
}

}  // namespace

int64_t norm_part_floats(const NormArgs &a, bool backward) {
    const Cut k = make_cut(a.batch, a.pixels, a.channels, vec_of(a));
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
