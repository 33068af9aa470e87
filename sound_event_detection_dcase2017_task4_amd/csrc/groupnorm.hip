// Group normalisation with an activation on channels-last activations x [N][S][C], forward and backward.
//
//   mean, rstd over the S rows and the C/G channels of a group;  xhat = (x - mean) rstd;  z = xhat w + b;  y = act(z)
//   gz = gy act'(z);  gw = sum gz xhat;  gb = sum gz;  h = gz w;  gx = rstd (h - mean_g(h) - xhat mean_g(h xhat))
//
// Bound by HBM.  The statistics of a group need every row of a sample before any element of it can be written.
//
// A thread owns V channels (16 bytes) of every RT-th row of a chunk of rows, whatever the group width: sums are held per channel and
// folded to groups afterwards.  A row that is not a multiple of V channels ends in a vector that overlaps its neighbour (the twice
// computed channels are written twice with the same value, and counted once), and loads need no more than element alignment.
#include "common.h"
#include "sed_hip.h"

SED_OBJECT_FLAGS(groupnorm)

namespace {

constexpr int THREADS = 256;
constexpr int UNROLL = 4;

// How a launch cuts the tensor: CT column vectors (of K a row) x RT row lanes per workgroup, `tiles` column tiles, chunks of rows.
struct Cut {
    int V, K, CT, RT, tiles;
    long rows, chunks, blocks;          // rows per chunk, chunks per sample, workgroups of the launch
};
Cut cut_of(long N, long S, int C, int esize) {
    Cut c;
    c.V = C >= 16 / esize ? 16 / esize : 1;
    c.K = (C + c.V - 1) / c.V;
    c.CT = c.K < THREADS ? c.K : THREADS;
    c.RT = THREADS / c.CT;
    c.tiles = (c.K + c.CT - 1) / c.CT;
    // enough workgroups to fill 256 CUs eight times over, at least UNROLL rows per thread, at most 64 so that a sum's chain stays short
    const long want = (2048 + N * c.tiles - 1) / (N * c.tiles);
    long rows = (S + want - 1) / want;
    const long lo = (long)c.RT * UNROLL, hi = (long)c.RT * 64;
    rows = rows < lo ? lo : (rows > hi ? hi : rows);
    c.rows = (rows + lo - 1) / lo * lo;
    c.chunks = (S + c.rows - 1) / c.rows;
    c.blocks = N * c.chunks * c.tiles;
    return c;
}

struct NormP {
    const void* x;
    const void* gy;
    const void* w;
    const void* b;
    void* y;                             // y, or gx
    const float* mean;
    const float* rstd;
    const float* coef;                   // [N][G][2]: mean_g(h), mean_g(h xhat)
    float* parts;                        // [N][chunks][2][C]
    long S, rows, chunks;
    int C, G, CT, RT, tiles, K, wdtype;
};

template <typename T, int V> struct Vec { T v[V]; };
template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_vec(const T* p) {       // element alignment is enough
    Vec<T, V> r;
    __builtin_memcpy(&r, p, sizeof(r));
    return r;
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& r) { __builtin_memcpy(p, &r, sizeof(r)); }

__device__ __forceinline__ float load_param(const void* p, int type, int c, float none) {
    if (!p) return none;
    if (type == SED_F32) return reinterpret_cast<const float*>(p)[c];
    if (type == SED_F16) return (float)reinterpret_cast<const _Float16*>(p)[c];
    return (float)reinterpret_cast<const __bf16*>(p)[c];
}

// where this thread works: sample, chunk, first channel, row lane
struct Place {
    long n, chunk, s0, s1;
    int c0, own, r;                      // first channel; channels below `own` belong to the neighbour; row lane
    bool on;
};
template <int V> __device__ __forceinline__ Place place_of(const NormP& p) {
    Place q;
    long id = blockIdx.x;
    const int tile = (int)(id % p.tiles);
    id /= p.tiles;
    q.chunk = id % p.chunks;
    q.n = id / p.chunks;
    q.s0 = q.chunk * p.rows;
    q.s1 = min(p.S, q.s0 + p.rows);
    const int t = threadIdx.x, col = tile * p.CT + t % p.CT;
    q.r = t / p.CT;
    q.on = q.r < p.RT && col < p.K;
    q.own = col * V;
    q.c0 = min(q.own, p.C - V);
    return q;
}

// sums a[V], b[V] of every thread over the row lanes; the first row lane leaves them in out [2][C]
template <int V, typename F> __device__ __forceinline__ void fold_rows(const NormP& p, const Place& q, const float (&a)[V], const float (&b)[V], F write) {
    __shared__ float red[2][THREADS * V];
    const int t = threadIdx.x;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        red[0][t * V + j] = a[j];
        red[1][t * V + j] = b[j];
    }
    __syncthreads();
    for (int k = t; k < p.CT * V; k += THREADS) {
        float sa = 0.f, sb = 0.f;
        for (int r = 0; r < p.RT; ++r) {
            sa += red[0][r * p.CT * V + k];
            sb += red[1][r * p.CT * V + k];
        }
        const int tile = (int)(blockIdx.x % p.tiles), col = tile * p.CT + k / V;
        if (col < p.K) {
            const int own = col * V, c = min(own, p.C - V) + k % V;
            if (c >= own) write(c, sa, sb);
        }
    }
}

// per chunk and channel: mean and sum of squared deviations.  The sums run over x - (the channel's value in the chunk's first row): a
// member of the set, so that the square of a large common offset never enters a sum.
template <typename T, int V> __global__ __launch_bounds__(THREADS) void norm_stats_kernel(NormP p) {
    const Place q = place_of<V>(p);
    const T* const x = reinterpret_cast<const T*>(p.x) + q.n * p.S * p.C + q.c0;
    float s1[V] = {}, s2[V] = {}, k0[V];
    if (q.on) {
        const auto f = load_vec<T, V>(x + q.s0 * p.C);
#pragma unroll
        for (int j = 0; j < V; ++j) k0[j] = (float)f.v[j];
        for (long s = q.s0 + q.r; s < q.s1; s += (long)p.RT * UNROLL) {
            Vec<T, V> v[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                if (s + (long)u * p.RT < q.s1) v[u] = load_vec<T, V>(x + (s + (long)u * p.RT) * p.C);
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                if (s + (long)u * p.RT < q.s1)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float d = (float)v[u].v[j] - k0[j];
                        s1[j] += d;
                        s2[j] = fmaf(d, d, s2[j]);
                    }
        }
    }
    const float inv = 1.f / (float)(q.s1 - q.s0);
    float* const out = p.parts + (q.n * p.chunks + q.chunk) * 2 * p.C;
    const T* const first = reinterpret_cast<const T*>(p.x) + (q.n * p.S + q.s0) * p.C;
    fold_rows<V>(p, q, s1, s2, [&](int c, float a, float b) {
        const float m = a * inv;
        out[c] = (float)first[c] + m;
        out[p.C + c] = fmaxf(fmaf(-a, m, b), 0.f) + (b - b);              // b - b: 0, or the NaN that fmaxf would drop
    });
}

// mean and 1 / sqrt(variance + eps) of a group from its chunks' means and squared deviations: two passes over numbers in the caches
__global__ __launch_bounds__(128) void norm_finalize_kernel(const float* parts, long S, long rows, long chunks, int C, int G, float eps, float* mean, float* rstd) {
    __shared__ float red[2];
    const long n = blockIdx.x / G;
    const int g = (int)(blockIdx.x % G), cg = C / G;
    const float* const base = parts + n * chunks * 2 * C + g * cg;
    const long total = chunks * cg;
    const float scale = 1.f / ((float)S * (float)cg);
    float a = 0.f;
    for (long e = threadIdx.x; e < total; e += 128) {
        const long i = e / cg;
        const float cnt = (float)min(rows, S - i * rows);
        a = fmaf(cnt * scale, base[i * 2 * C + e % cg], a);
    }
    a = wave_sum(a);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a;
    __syncthreads();
    const float m = red[0] + red[1];
    __syncthreads();
    float v = 0.f;
    for (long e = threadIdx.x; e < total; e += 128) {
        const long i = e / cg;
        const float cnt = (float)min(rows, S - i * rows), d = base[i * 2 * C + e % cg] - m;
        v += fmaf(cnt * d, d, base[i * 2 * C + C + e % cg]) * scale;
    }
    v = wave_sum(v);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    if (threadIdx.x == 0) {
        mean[blockIdx.x] = m;
        rstd[blockIdx.x] = 1.f / sqrtf(red[0] + red[1] + eps);
    }
}

template <typename T, int V, int ACT> __global__ __launch_bounds__(THREADS) void norm_apply_kernel(NormP p) {
    const Place q = place_of<V>(p);
    if (!q.on) return;
    const T* const x = reinterpret_cast<const T*>(p.x) + q.n * p.S * p.C + q.c0;
    T* const y = reinterpret_cast<T*>(p.y) + q.n * p.S * p.C + q.c0;
    const int cg = p.C / p.G;
    float m[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = q.c0 + j;
        const long ng = q.n * p.G + c / cg;
        m[j] = p.mean[ng];
        a[j] = p.rstd[ng] * load_param(p.w, p.wdtype, c, 1.f);
        b[j] = load_param(p.b, p.wdtype, c, 0.f);
    }
    for (long s = q.s0 + q.r; s < q.s1; s += (long)p.RT * UNROLL) {
        Vec<T, V> v[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (s + (long)u * p.RT < q.s1) v[u] = load_vec<T, V>(x + (s + (long)u * p.RT) * p.C);
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (s + (long)u * p.RT < q.s1) {
#pragma unroll
                for (int j = 0; j < V; ++j) v[u].v[j] = (T)sed_act<ACT>(fmaf((float)v[u].v[j] - m[j], a[j], b[j]));
                store_vec<T, V>(y + (s + (long)u * p.RT) * p.C, v[u]);
            }
    }
}

// per chunk and channel: sum gz and sum gz xhat
template <typename T, int V, int ACT> __global__ __launch_bounds__(THREADS) void norm_bwd_sums_kernel(NormP p) {
    const Place q = place_of<V>(p);
    float s1[V] = {}, s2[V] = {};
    if (q.on) {
        const long at = q.n * p.S * p.C + q.c0;
        const T* const x = reinterpret_cast<const T*>(p.x) + at;
        const T* const gy = reinterpret_cast<const T*>(p.gy) + at;
        const int cg = p.C / p.G;
        float m[V], r[V], w[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = q.c0 + j;
            const long ng = q.n * p.G + c / cg;
            m[j] = p.mean[ng];
            r[j] = p.rstd[ng];
            w[j] = load_param(p.w, p.wdtype, c, 1.f);
            b[j] = load_param(p.b, p.wdtype, c, 0.f);
        }
        for (long s = q.s0 + q.r; s < q.s1; s += (long)p.RT * UNROLL) {
            Vec<T, V> v[UNROLL], g[UNROLL];
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                if (s + (long)u * p.RT < q.s1) {
                    v[u] = load_vec<T, V>(x + (s + (long)u * p.RT) * p.C);
                    g[u] = load_vec<T, V>(gy + (s + (long)u * p.RT) * p.C);
                }
#pragma unroll
            for (int u = 0; u < UNROLL; ++u)
                if (s + (long)u * p.RT < q.s1)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float xh = ((float)v[u].v[j] - m[j]) * r[j];
                        const float gz = (float)g[u].v[j] * sed_act_grad<ACT>(fmaf(xh, w[j], b[j]));
                        s1[j] += gz;
                        s2[j] = fmaf(gz, xh, s2[j]);
                    }
        }
    }
    float* const out = p.parts + (q.n * p.chunks + q.chunk) * 2 * p.C;
    fold_rows<V>(p, q, s1, s2, [&](int c, float a, float b) {
        out[c] = a;
        out[p.C + c] = b;
    });
}

// one workgroup per (sample, group): the chunks' sums per channel, chan [N][2][C], and the group's two means, coef [N][G][2]
__global__ __launch_bounds__(128) void norm_bwd_fold_kernel(const float* parts, long S, long chunks, int C, int G, const void* w, int wdtype, float* chan, float* coef) {
    __shared__ float red[2][2];
    const long n = blockIdx.x / G;
    const int g = (int)(blockIdx.x % G), cg = C / G;
    const float* const base = parts + n * chunks * 2 * C + g * cg;
    float ga = 0.f, gb = 0.f;
    for (int k = threadIdx.x; k < cg; k += 128) {
        float a = 0.f, b = 0.f;
        for (long i = 0; i < chunks; ++i) {
            a += base[i * 2 * C + k];
            b += base[i * 2 * C + C + k];
        }
        const int c = g * cg + k;
        chan[n * 2 * C + c] = a;
        chan[n * 2 * C + C + c] = b;
        const float wc = load_param(w, wdtype, c, 1.f);
        ga = fmaf(wc, a, ga);
        gb = fmaf(wc, b, gb);
    }
    ga = wave_sum(ga);
    gb = wave_sum(gb);
    if ((threadIdx.x & 63) == 0) {
        red[0][threadIdx.x >> 6] = ga;
        red[1][threadIdx.x >> 6] = gb;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const float scale = 1.f / ((float)S * (float)cg);
        coef[blockIdx.x * 2l] = (red[0][0] + red[0][1]) * scale;
        coef[blockIdx.x * 2l + 1] = (red[1][0] + red[1][1]) * scale;
    }
}

// gbias, gweight [C]: the sums of chan [N][2][C] over the samples; 16 channels x 16 sample lanes per workgroup
__global__ __launch_bounds__(256) void norm_bwd_params_kernel(const float* chan, long N, int C, float* gw, float* gb) {
    __shared__ float red[2][16][17];
    const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, c = blockIdx.x * 16 + lane;
    float a = 0.f, b = 0.f;
    if (c < C)
        for (long n = row; n < N; n += 16) {
            a += chan[n * 2 * C + c];
            b += chan[n * 2 * C + C + c];
        }
    red[0][row][lane] = a;
    red[1][row][lane] = b;
    __syncthreads();
    if (row == 0 && c < C) {
        for (int k = 1; k < 16; ++k) {
            a += red[0][k][lane];
            b += red[1][k][lane];
        }
        if (gb) gb[c] = a;
        if (gw) gw[c] = b;
    }
}

template <typename T, int V, int ACT> __global__ __launch_bounds__(THREADS) void norm_bwd_apply_kernel(NormP p) {
    const Place q = place_of<V>(p);
    if (!q.on) return;
    const long at = q.n * p.S * p.C + q.c0;
    const T* const x = reinterpret_cast<const T*>(p.x) + at;
    const T* const gy = reinterpret_cast<const T*>(p.gy) + at;
    T* const gx = reinterpret_cast<T*>(p.y) + at;
    const int cg = p.C / p.G;
    float m[V], r[V], w[V], b[V], c1[V], c2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = q.c0 + j;
        const long ng = q.n * p.G + c / cg;
        m[j] = p.mean[ng];
        r[j] = p.rstd[ng];
        w[j] = load_param(p.w, p.wdtype, c, 1.f);
        b[j] = load_param(p.b, p.wdtype, c, 0.f);
        c1[j] = p.coef[2 * ng];
        c2[j] = p.coef[2 * ng + 1];
    }
    for (long s = q.s0 + q.r; s < q.s1; s += (long)p.RT * UNROLL) {
        Vec<T, V> v[UNROLL], g[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (s + (long)u * p.RT < q.s1) {
                v[u] = load_vec<T, V>(x + (s + (long)u * p.RT) * p.C);
                g[u] = load_vec<T, V>(gy + (s + (long)u * p.RT) * p.C);
            }
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
            if (s + (long)u * p.RT < q.s1) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xh = ((float)v[u].v[j] - m[j]) * r[j];
                    const float gz = (float)g[u].v[j] * sed_act_grad<ACT>(fmaf(xh, w[j], b[j]));
                    v[u].v[j] = (T)(r[j] * (fmaf(gz, w[j], -c1[j]) - xh * c2[j]));
                }
                store_vec<T, V>(gx + (s + (long)u * p.RT) * p.C, v[u]);
            }
    }
}

int esize_of(int dtype) { return dtype == SED_F32 ? 4 : 2; }
bool bad_shape(int dtype, int wdtype, long N, long S, int C, int G, int act) {
    return dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2 || N < 1 || S < 1 || C < 1 || G < 1 || C % G || act < 0 || act > 3 ||
           N * G > 0x7fffffffL || cut_of(N, S, C, esize_of(dtype)).blocks > 0x7fffffffL;
}
NormP params_of(const Cut& c, const void* x, const void* w, const void* b, int wdtype, long S, int C, int G, float* ws) {
    NormP p{};
    p.x = x; p.w = w; p.b = b; p.wdtype = wdtype;
    p.S = S; p.rows = c.rows; p.chunks = c.chunks; p.C = C; p.G = G; p.CT = c.CT; p.RT = c.RT; p.tiles = c.tiles; p.K = c.K;
    p.parts = ws;
    return p;
}

#define NORM_ACT(KERNEL, T, V)                                                                              \
    switch (act) {                                                                                          \
        case SED_ACT_NONE: hipLaunchKernelGGL((KERNEL<T, V, 0>), grid, dim3(THREADS), 0, stream, p); break; \
        case SED_ACT_RELU: hipLaunchKernelGGL((KERNEL<T, V, 1>), grid, dim3(THREADS), 0, stream, p); break; \
        case SED_ACT_SILU: hipLaunchKernelGGL((KERNEL<T, V, 2>), grid, dim3(THREADS), 0, stream, p); break; \
        default: hipLaunchKernelGGL((KERNEL<T, V, 3>), grid, dim3(THREADS), 0, stream, p);                  \
    }
#define NORM_TYPE(WHAT, ...)                                                                     \
    if (c.V == 1) {                                                                              \
        if (dtype == SED_F32) { WHAT(__VA_ARGS__, float, 1) }                                    \
        else if (dtype == SED_F16) { WHAT(__VA_ARGS__, _Float16, 1) }                            \
        else { WHAT(__VA_ARGS__, __bf16, 1) }                                                    \
    } else {                                                                                     \
        if (dtype == SED_F32) { WHAT(__VA_ARGS__, float, 4) }                                    \
        else if (dtype == SED_F16) { WHAT(__VA_ARGS__, _Float16, 8) }                            \
        else { WHAT(__VA_ARGS__, __bf16, 8) }                                                    \
    }
#define NORM_PLAIN(KERNEL, T, V) hipLaunchKernelGGL((KERNEL<T, V>), grid, dim3(THREADS), 0, stream, p);

}  // namespace

SED_API long sed_group_norm_ws_floats(long N, long S, int C, int G, int backward) {
    if (bad_shape(SED_F32, SED_F32, N, S, C, G, 0) || bad_shape(SED_F16, SED_F32, N, S, C, G, 0)) return 0;
    const long a = cut_of(N, S, C, 4).chunks, b = cut_of(N, S, C, 2).chunks;
    const long parts = N * (a > b ? a : b) * 2 * C;
    return backward ? parts + N * 2 * C + N * 2 * G : parts;
}

SED_API int sed_group_norm_fwd(const void* x, const void* weight, const void* bias, int dtype, int wdtype, long N, long S, int C, int G,
                               float eps, int act, void* y, float* mean, float* rstd, float* ws, sed_stream_t stream) {
    if (!x || !y || !mean || !rstd || !ws || !(eps >= 0.f) || bad_shape(dtype, wdtype, N, S, C, G, act)) return SED_EINVAL;
    const Cut c = cut_of(N, S, C, esize_of(dtype));
    const dim3 grid((unsigned)c.blocks);
    NormP p = params_of(c, x, weight, bias, wdtype, S, C, G, ws);
    p.y = y; p.mean = mean; p.rstd = rstd;
    NORM_TYPE(NORM_PLAIN, norm_stats_kernel)
    hipLaunchKernelGGL(norm_finalize_kernel, dim3((unsigned)(N * G)), dim3(128), 0, stream, ws, S, c.rows, c.chunks, C, G, eps, mean, rstd);
    NORM_TYPE(NORM_ACT, norm_apply_kernel)
    SED_LAUNCH_CHECK();
    return 0;
}

SED_API int sed_group_norm_bwd(const void* x, const void* gy, const void* weight, const void* bias, int dtype, int wdtype, long N, long S,
                               int C, int G, int act, const float* mean, const float* rstd, void* gx, float* gweight, float* gbias,
                               float* ws, sed_stream_t stream) {
    if (!x || !gy || !mean || !rstd || !ws || bad_shape(dtype, wdtype, N, S, C, G, act)) return SED_EINVAL;
    const Cut c = cut_of(N, S, C, esize_of(dtype));
    const dim3 grid((unsigned)c.blocks);
    NormP p = params_of(c, x, weight, bias, wdtype, S, C, G, ws);
    float* const chan = ws + N * c.chunks * 2 * C;
    float* const coef = chan + N * 2 * C;
    p.gy = gy; p.y = gx; p.mean = mean; p.rstd = rstd; p.coef = coef;
    NORM_TYPE(NORM_ACT, norm_bwd_sums_kernel)
    hipLaunchKernelGGL(norm_bwd_fold_kernel, dim3((unsigned)(N * G)), dim3(128), 0, stream, ws, S, c.chunks, C, G, weight, wdtype, chan, coef);
    if (gweight || gbias)
        hipLaunchKernelGGL(norm_bwd_params_kernel, dim3((unsigned)sed_cdiv(C, 16)), dim3(256), 0, stream, chan, N, C, gweight, gbias);
    if (gx) { NORM_TYPE(NORM_ACT, norm_bwd_apply_kernel) }
    SED_LAUNCH_CHECK();
    return 0;
}
