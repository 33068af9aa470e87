// Group normalisation with an activation on channels-last activations x [N][S][C], forward and backward.
//
//   mean, rstd over the S rows and the C/G channels of a group;  xhat = (x - mean) rstd;  z = xhat w + b;  y = act(z)
//   gz = gy act'(z);  gw = sum gz xhat;  gb = sum gz;  h = gz w;  gx = rstd (h - mean_g(h) - xhat mean_g(h xhat))
//
// Bound by HBM.  The statistics of a group need every row of a sample before any element of it can be written.  Where the rows of some
// groups fit the registers of a workgroup they are read once (the one-pass kernels); beyond that a first pass leaves statistics per
// chunk of rows and channel, a small kernel joins them, and a second pass reads the rows again -- forward, and from 384 MB on, only where
// a sample does not fit the registers of 128 workgroups either.
//
// A thread owns V channels (16 bytes) of every RT-th row of a chunk of rows, whatever the group width: sums are held per channel and
// folded to groups afterwards.  A row that is not a multiple of V channels ends in a vector that overlaps its neighbour (the twice
// computed channels are written twice with the same value, and counted once), and loads need no more than element alignment.
#include "act.h"
#include "common.h"
#include "sed_hip.h"

SED_OBJECT_FLAGS(groupnorm)

namespace {

constexpr int THREADS = 256;
// rows that a thread has in flight: the backward passes read two tensors, and are slower with more registers a thread (65 M bf16 elements,
// sums and gx: 63 and 73 us with two rows, 79 and 97 with four, 74 and 73 with one)
constexpr int UNROLL = 4, BWD_UNROLL = 2;

// How a launch cuts the tensor: CT column vectors (of K a row) x RT row lanes per workgroup, `tiles` column tiles, chunks of rows.
struct Cut {
    int V, K, CT, RT, tiles;
    long rows, chunks, blocks;          // rows per chunk, chunks per sample, workgroups of the launch
};
Cut cut_of(long N, long S, int C, int esize) {
    Cut c;
    c.V = C >= 16 / esize ? 16 / esize : 1;
    c.K = (C + c.V - 1) / c.V;
    // up to 1 KB of a row, so that a chunk has many rows: its sums, which are written and read again, are then little beside them
    c.tiles = (c.K + 63) / 64;
    c.CT = (c.K + c.tiles - 1) / c.tiles;
    c.RT = THREADS / c.CT;
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

__device__ __forceinline__ void store_param(void* p, int type, int c, float v) {
    if (type == SED_F32) reinterpret_cast<float*>(p)[c] = v;
    else if (type == SED_F16) reinterpret_cast<_Float16*>(p)[c] = (_Float16)v;
    else reinterpret_cast<__bf16*>(p)[c] = (__bf16)v;
}

// the groups of V consecutive channels, by one division
template <int V> __device__ __forceinline__ void groups_of(int c0, int cg, int (&g)[V]) {
    int q = c0 / cg, r = c0 - q * cg;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        g[j] = q;
        if (++r == cg) { r = 0; ++q; }
    }
}

// where this thread works: sample, chunk, first channel, row lane
struct Place {
    long n, chunk, s0, s1;
    int c0, own, r;                      // first channel; channels below `own` belong to the neighbour; row lane
    bool on;
};
template <int V> __device__ __forceinline__ Place place_of(const NormP& p, unsigned bid) {
    Place q;
    long id = bid;
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

// Statistics of a column of numbers in one reading: the sums run over d = x - k0, k0 the column's first number.  A column is what one
// thread reads of a channel, 64 rows at most: whatever k0 is -- a padded row, an outlier -- the squares that cancel are at most 64 times
// what k0 itself adds to the group's squares, and the variance keeps 24 - 6 bits of it.
template <int V> __device__ __forceinline__ void column_stats(int count, const float (&k0)[V], float (&s1)[V], float (&s2)[V]) {      // -> mean, squared deviations
    const float inv = count ? 1.f / (float)count : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const float d = s1[j] * inv;
        s2[j] = fmaxf(fmaf(-s1[j], d, s2[j]), 0.f) + (s2[j] - s2[j]);         // the difference: 0, or the NaN that fmaxf would drop
        s1[j] = count ? k0[j] + d : 0.f;
    }
}
// Means and squared deviations of every thread's columns, joined over the row lanes: write(channel, mean, squares).  `count` rows are dealt
// out to RT lanes; scratch holds 2 * T * V floats, part T.
template <int V, typename F> __device__ __forceinline__ void join_columns(int T, int CT, int RT, int count, const float (&mean)[V], const float (&sq)[V], float* scratch, float* part, F write) {
    const int t = threadIdx.x, NC = CT * V, share = max(1, min(T / NC, 16)), lane = NC < T ? t / NC : 0, full = count / RT, more = count % RT;
    float* const ra = scratch;
    float* const rb = scratch + T * V;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        ra[t * V + j] = mean[j];
        rb[t * V + j] = sq[j];
    }
    __syncthreads();
    const float inv = 1.f / (float)count;
    for (int base = 0; base < NC; base += T) {     // once where there is more than one thread for a channel
        const int k = base + (NC < T ? t % NC : t);
        const bool on = lane < share && k < NC;
        // means are averaged as differences from one of them: a common offset is rounded once, not with every term
        const float ref = on ? ra[k] : 0.f;
        float m = 0.f, q = 0.f;
        if (on)
            for (int r = lane; r < RT; r += share) m = fmaf((float)(full + (r < more)) * inv, ra[r * NC + k] - ref, m);
        if (share > 1) {
            part[t] = m;
            __syncthreads();
            m = 0.f;
            if (on)
                for (int i = 0; i < share; ++i) m += part[i * NC + k];
            __syncthreads();
        }
        m += ref;
        if (on)
            for (int r = lane; r < RT; r += share) {
                const float d = ra[r * NC + k] - m;
                q += fmaf((float)(full + (r < more)) * d, d, rb[r * NC + k]);
            }
        if (share > 1) {
            part[t] = q;
            __syncthreads();
            if (on && lane == 0)
                for (int i = 1; i < share; ++i) q += part[i * NC + k];
        }
        if (on && lane == 0) write(k, m, q);
    }
    __syncthreads();
}

// per chunk and channel: mean and sum of squared deviations
template <typename T, int V> __global__ __launch_bounds__(THREADS) void norm_stats_kernel(NormP p) {
    __shared__ float scratch[2 * THREADS * V], part[THREADS];
    const Place q = place_of<V>(p, blockIdx.x);
    const T* const x = reinterpret_cast<const T*>(p.x) + q.n * p.S * p.C + q.c0;
    float s1[V] = {}, s2[V] = {}, k0[V] = {};
    const int rows = (int)(q.s1 - q.s0);
    if (q.on && q.r < rows) {
        const auto f = load_vec<T, V>(x + (q.s0 + q.r) * p.C);
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
    column_stats<V>(q.r < rows ? (rows - 1 - q.r) / p.RT + 1 : 0, k0, s1, s2);
    float* const out = p.parts + (q.n * p.chunks + q.chunk) * 2 * p.C;
    const int tile = (int)(blockIdx.x % p.tiles);
    join_columns<V>(THREADS, p.CT, p.RT, rows, s1, s2, scratch, part, [&](int k, float m, float sq) {
        const int col = tile * p.CT + k / V, own = col * V, c = min(own, p.C - V) + k % V;
        if (col < p.K && c >= own) {
            out[c] = m;
            out[p.C + c] = sq;
        }
    });
}

// The kernels that join a sample's chunks take a bundle of groups each, all of a workgroup's threads on channels x chunks: f(chunk, channel)
// summed over the chunks, per channel, into out[channel - c0] (LDS) for the channels from c0 to c1.  scratch: JOIN floats.
constexpr int JOIN = 1024;
constexpr int MAX_BUNDLE = 1024;         // channels of a bundle, and of a group that is held in LDS
template <typename F, typename W> __device__ __forceinline__ void chunk_sums(long chunks, int c0, int c1, float* scratch, F f, W write) {
    const int t = threadIdx.x, T = blockDim.x, lanes = min(T, c1 - c0), share = T / lanes, lane = t % lanes, first = t / lanes;
    for (int c = c0; c < c1; c += lanes) {
        const int k = c + lane;
        float a = 0.f;
        if (first < share && k < c1)
#pragma unroll 4
            for (long i = first; i < chunks; i += share) a += f(i, k);
        __syncthreads();
        scratch[t] = a;
        // halves of the lanes' shares, added pairwise
        for (int n = share; n > 1;) {
            const int half = (n + 1) / 2;
            __syncthreads();
            if (first + half < n) scratch[t] += scratch[t + half * lanes];
            n = half;
        }
        __syncthreads();
        if (t < lanes && k < c1) write(k, scratch[t]);
    }
    __syncthreads();
}
// How they cut: 64 channels' worth of groups in a workgroup, as far as there are 256 workgroups, and a thread for eight numbers
struct Join {
    int per, threads;
    long blocks;
};
Join join_of(long N, long chunks, int C, int G) {
    const int cg = C / G;
    Join j;
    j.per = cg >= 64 ? 1 : 64 / cg < G ? 64 / cg : G;
    const long most = N * G / 256;
    if (j.per > most) j.per = most > 1 ? (int)most : 1;
    const long want = chunks * j.per * cg / 8;
    j.threads = 64;
    while (j.threads < JOIN && j.threads < want) j.threads *= 2;
    j.blocks = N * ((G + j.per - 1) / j.per);
    return j;
}

// mean and 1 / sqrt(variance + eps) of a group from its chunks' means and squared deviations: two passes over numbers in the caches
__global__ __launch_bounds__(JOIN) void norm_finalize_kernel(const float* parts, long S, long rows, long chunks, int C, int G, int per, float eps, float* mean, float* rstd) {
    __shared__ float scratch[JOIN], chan[MAX_BUNDLE], means[64];
    const int bundles = (G + per - 1) / per, cg = C / G;
    const long n = blockIdx.x / bundles;
    const int g0 = (int)(blockIdx.x % bundles) * per, g1 = min(G, g0 + per), t = threadIdx.x;
    const float* const base = parts + n * chunks * 2 * C;
    const float scale = 1.f / ((float)S * (float)cg);
    auto count = [&](long i) { return (float)min(rows, S - i * rows); };
    // sums over a group's channels; a channel beyond the LDS is added to the one that it shares a place with
    auto group_sum = [&](int g) {
        float a = 0.f;
        for (int k = t & 63; k < min(cg, MAX_BUNDLE); k += 64) a += chan[(g - g0) * cg + k];
        return wave_sum(a);
    };
    auto add = [&](int k, float v) {
        const int at = k - g0 * cg;
        chan[at % MAX_BUNDLE] = at < MAX_BUNDLE ? v : chan[at % MAX_BUNDLE] + v;
    };
    chunk_sums(chunks, g0 * cg, g1 * cg, scratch, [&](long i, int c) { return count(i) * scale * (base[i * 2 * C + c] - base[per == 1 ? g0 * cg : c / cg * cg]); }, add);
    for (int g = g0 + (t >> 6); g < g1; g += (int)blockDim.x / 64) {
        const float m = group_sum(g) + base[g * cg];          // averaged as differences from the first chunk's first channel
        if ((t & 63) == 0) means[g - g0] = m;
    }
    __syncthreads();
    chunk_sums(chunks, g0 * cg, g1 * cg, scratch, [&](long i, int c) {
        const float k = count(i), d = base[i * 2 * C + c] - means[per == 1 ? 0 : c / cg - g0];
        return fmaf(k * d, d, base[i * 2 * C + C + c]) * scale;
    }, add);
    for (int g = g0 + (t >> 6); g < g1; g += (int)blockDim.x / 64) {
        const float v = group_sum(g);
        if ((t & 63) == 0) {
            mean[n * G + g] = means[g - g0];
            rstd[n * G + g] = 1.f / sqrtf(v + eps);
        }
    }
}

template <typename T, int V, int ACT> __global__ __launch_bounds__(THREADS) void norm_apply_kernel(NormP p) {
    const Place q = place_of<V>(p, blockIdx.x);
    if (!q.on) return;
    const T* const x = reinterpret_cast<const T*>(p.x) + q.n * p.S * p.C + q.c0;
    T* const y = reinterpret_cast<T*>(p.y) + q.n * p.S * p.C + q.c0;
    int gr[V];
    groups_of<V>(q.c0, p.C / p.G, gr);
    float m[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = q.c0 + j;
        const long ng = q.n * p.G + gr[j];
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
    const Place q = place_of<V>(p, blockIdx.x);
    float s1[V] = {}, s2[V] = {};
    if (q.on) {
        const long at = q.n * p.S * p.C + q.c0;
        const T* const x = reinterpret_cast<const T*>(p.x) + at;
        const T* const gy = reinterpret_cast<const T*>(p.gy) + at;
        int gr[V];
        groups_of<V>(q.c0, p.C / p.G, gr);
        float m[V], r[V], w[V], b[V];
#pragma unroll
        for (int j = 0; j < V; ++j) {
            const int c = q.c0 + j;
            const long ng = q.n * p.G + gr[j];
            m[j] = p.mean[ng];
            r[j] = p.rstd[ng];
            w[j] = load_param(p.w, p.wdtype, c, 1.f);
            b[j] = load_param(p.b, p.wdtype, c, 0.f);
        }
        for (long s = q.s0 + q.r; s < q.s1; s += (long)p.RT * BWD_UNROLL) {
            Vec<T, V> v[BWD_UNROLL], g[BWD_UNROLL];
#pragma unroll
            for (int u = 0; u < BWD_UNROLL; ++u)
                if (s + (long)u * p.RT < q.s1) {
                    v[u] = load_vec<T, V>(x + (s + (long)u * p.RT) * p.C);
                    g[u] = load_vec<T, V>(gy + (s + (long)u * p.RT) * p.C);
                }
#pragma unroll
            for (int u = 0; u < BWD_UNROLL; ++u)
                if (s + (long)u * p.RT < q.s1)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const float xh = ((float)v[u].v[j] - m[j]) * r[j];
                        const float gz = sed_act_gz<ACT>((float)g[u].v[j], fmaf(xh, w[j], b[j]));
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

// per (sample, bundle of `per` groups): the chunks' sums per channel, chan [N][2][C], and the groups' two means, coef [N][G][2]
__global__ __launch_bounds__(JOIN) void norm_bwd_fold_kernel(const float* parts, long S, long chunks, int C, int G, int per, const void* w, int wdtype, float* chan, float* coef) {
    __shared__ float scratch[JOIN];
    const int bundles = (G + per - 1) / per, cg = C / G;
    const long n = blockIdx.x / bundles;
    const int g0 = (int)(blockIdx.x % bundles) * per, g1 = min(G, g0 + per), t = threadIdx.x;
    const float* const base = parts + n * chunks * 2 * C;
#pragma unroll
    for (int which = 0; which < 2; ++which)
        chunk_sums(chunks, g0 * cg, g1 * cg, scratch, [&](long i, int c) { return base[(i * 2 + which) * C + c]; },
                   [&](int c, float v) { chan[(n * 2 + which) * C + c] = v; });
    // the workgroup's own stores to chan are read back
    for (int g = g0 + (t >> 6); g < g1; g += (int)blockDim.x / 64) {
        float a = 0.f, b = 0.f;
        for (int k = t & 63; k < cg; k += 64) {
            const int c = g * cg + k;
            const float wc = load_param(w, wdtype, c, 1.f);
            a = fmaf(wc, chan[n * 2 * C + c], a);
            b = fmaf(wc, chan[n * 2 * C + C + c], b);
        }
        a = wave_sum(a);
        b = wave_sum(b);
        if ((t & 63) == 0) {
            const float scale = 1.f / ((float)S * (float)cg);
            coef[(n * G + g) * 2] = a * scale;
            coef[(n * G + g) * 2 + 1] = b * scale;
        }
    }
}

// gbias, gweight [C] of wdtype: the sums of chan [N][2][C] over the samples; 16 channels x ROWS sample lanes per workgroup
struct ParamsP {
    const float* chan;
    long N;
    int C, wdtype;
    void* gw;
    void* gb;
    int blocks;                          // 0: neither is wanted
};
template <int ROWS> __device__ __forceinline__ void param_sums(const ParamsP& p, int bid) {
    __shared__ float red[2][ROWS][17];
    const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, c = bid * 16 + lane;
    float a = 0.f, b = 0.f;
    if (c < p.C)
        for (long n = row; n < p.N; n += ROWS) {
            a += p.chan[n * 2 * p.C + c];
            b += p.chan[n * 2 * p.C + p.C + c];
        }
    red[0][row][lane] = a;
    red[1][row][lane] = b;
    __syncthreads();
    for (int s = ROWS / 2; s > 0; s >>= 1) {
        if (row < s) {
            red[0][row][lane] += red[0][row + s][lane];
            red[1][row][lane] += red[1][row + s][lane];
        }
        __syncthreads();
    }
    if (row == 0 && c < p.C) {
        if (p.gb) store_param(p.gb, p.wdtype, c, red[0][0][lane]);
        if (p.gw) store_param(p.gw, p.wdtype, c, red[1][0][lane]);
    }
}
__global__ __launch_bounds__(1024) void norm_bwd_params_kernel(ParamsP p) { param_sums<64>(p, blockIdx.x); }

// gx; the first params.blocks workgroups add up the parameters' gradients
template <typename T, int V, int ACT> __global__ __launch_bounds__(THREADS) void norm_bwd_apply_kernel(NormP p, ParamsP params) {
    if ((int)blockIdx.x < params.blocks) { param_sums<THREADS / 16>(params, blockIdx.x); return; }
    const Place q = place_of<V>(p, blockIdx.x - params.blocks);
    if (!q.on) return;
    const long at = q.n * p.S * p.C + q.c0;
    const T* const x = reinterpret_cast<const T*>(p.x) + at;
    const T* const gy = reinterpret_cast<const T*>(p.gy) + at;
    T* const gx = reinterpret_cast<T*>(p.y) + at;
    int gr[V];
    groups_of<V>(q.c0, p.C / p.G, gr);
    float m[V], r[V], w[V], b[V], c1[V], c2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = q.c0 + j;
        const long ng = q.n * p.G + gr[j];
        m[j] = p.mean[ng];
        r[j] = p.rstd[ng];
        w[j] = load_param(p.w, p.wdtype, c, 1.f);
        b[j] = load_param(p.b, p.wdtype, c, 0.f);
        c1[j] = p.coef[2 * ng];
        c2[j] = p.coef[2 * ng + 1];
    }
    for (long s = q.s0 + q.r; s < q.s1; s += (long)p.RT * BWD_UNROLL) {
        Vec<T, V> v[BWD_UNROLL], g[BWD_UNROLL];
#pragma unroll
        for (int u = 0; u < BWD_UNROLL; ++u)
            if (s + (long)u * p.RT < q.s1) {
                v[u] = load_vec<T, V>(x + (s + (long)u * p.RT) * p.C);
                g[u] = load_vec<T, V>(gy + (s + (long)u * p.RT) * p.C);
            }
#pragma unroll
        for (int u = 0; u < BWD_UNROLL; ++u)
            if (s + (long)u * p.RT < q.s1) {
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    const float xh = ((float)v[u].v[j] - m[j]) * r[j];
                    const float gz = sed_act_gz<ACT>((float)g[u].v[j], fmaf(xh, w[j], b[j]));
                    v[u].v[j] = (T)(r[j] * (fmaf(gz, w[j], -c1[j]) - xh * c2[j]));
                }
                store_vec<T, V>(gx + (s + (long)u * p.RT) * p.C, v[u]);
            }
    }
}

// ---- one pass: the rows of a bundle of whole groups stay in the registers of one workgroup, up to 128 KB (forward) or 2 x 64 KB
// (backward), and are read once.  16-bit rows stay packed: 1000 x 300 x 512 bfloat16 takes 192 us forward and 300 backward, with rows that
// the compiler holds as floats (and half the workgroups on a CU) 489 and 573.
struct OneP {
    const void* x;
    const void* gy;
    const void* w;
    const void* b;
    void* y;                             // y, or gx (nullable)
    float* mean;
    float* rstd;
    float* chan;                         // backward: [N][2][C], sum gz and sum gz xhat
    long S;
    int C, G, per, bundles, wdtype;      // per: groups in a bundle
    int glanes;                          // lanes that add up a group's channels: a power of two up to 64
    float eps;
};
constexpr int ONE_THREADS = 512, ONE_FWD = 16, ONE_BWD = 8;        // threads, and 16-byte vectors of x that one of them holds

// Sums of a[V], b[V] over the row lanes of each of the bundle's channels, left in out[2][channels] (LDS).  scratch: 2 * blockDim * V floats.
template <int V> __device__ __forceinline__ void channel_sums(int CT, int RT, int K, int width, const float (&a)[V], const float (&b)[V], float* scratch, float* out) {
    const int t = threadIdx.x, T = blockDim.x, NC = CT * V;
    float* const ra = scratch;
    float* const rb = scratch + T * V;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j) {
        ra[t * V + j] = a[j];
        rb[t * V + j] = b[j];
    }
    __syncthreads();
    // NC columns of RT numbers: share = how many threads add up one column, in two steps
    const int share = max(1, min(T / NC, 16)), lane = t / NC, k0 = t % NC;
    if (share > 1) {
        float sa = 0.f, sb = 0.f;
        if (lane < share)
            for (int r = lane; r < RT; r += share) {
                sa += ra[r * NC + k0];
                sb += rb[r * NC + k0];
            }
        __syncthreads();
        if (lane < share) {
            ra[lane * NC + k0] = sa;
            rb[lane * NC + k0] = sb;
        }
        __syncthreads();
    }
    const int rows = share > 1 ? share : RT;
    for (int k = t; k < NC; k += T) {
        float sa = 0.f, sb = 0.f;
        for (int r = 0; r < rows; ++r) {
            sa += ra[r * NC + k];
            sb += rb[r * NC + k];
        }
        const int own = k / V * V, c = min(own, width - V) + k % V;
        if (k / V < K && c >= own) {
            out[c] = sa;
            out[MAX_BUNDLE + c] = sb;
        }
    }
    __syncthreads();
}
// sums over a group's channels of two LDS arrays, times f(channel); result to every thread through LDS, per group of the bundle
template <typename F> __device__ __forceinline__ void group_sums(const float* chan, int groups, int cg, F f, float* out) {
    const int t = threadIdx.x, waves = (blockDim.x + 63) >> 6;
    for (int g = t >> 6; g < groups; g += waves) {
        float a = 0.f, b = 0.f;
        for (int k = t & 63; k < cg; k += 64) {
            const float w = f(g * cg + k);
            a = fmaf(w, chan[g * cg + k], a);
            b = fmaf(w, chan[MAX_BUNDLE + g * cg + k], b);
        }
        a = wave_sum(a);
        b = wave_sum(b);
        if ((t & 63) == 0) {
            out[2 * g] = a;
            out[2 * g + 1] = b;
        }
    }
    __syncthreads();
}

// what a lane's 16 bytes hold must stay in 16-bit form between the passes over it: converted once, they would take twice the registers
template <typename T, int V> __device__ __forceinline__ void keep(Vec<T, V>& v) {
    floatx4 q = __builtin_bit_cast(floatx4, v);
    asm volatile("" : "+v"(q));
    v = __builtin_bit_cast(Vec<T, V>, q);
}

__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}
// Mean and sum of squared deviations of each of `groups` groups of cg channels over `count` rows, from its channels' (chan, LDS: the means,
// and MAX_BUNDLE further the squares); `lanes` (a power of two) share a group, and the first of them passes the two to write.
template <typename F> __device__ __forceinline__ void group_stats(const float* chan, int groups, int cg, int count, int lanes, F write) {
    const float share = 1.f / (float)cg;
    const int sub = threadIdx.x % lanes;
    for (int g = threadIdx.x / lanes; g < groups; g += blockDim.x / lanes) {
        float a = 0.f, q = 0.f;
        const float ref = chan[g * cg];
        for (int c = g * cg + sub; c < (g + 1) * cg; c += lanes) a += chan[c] - ref;
        const float m = fmaf(lanes_sum(a, lanes), share, ref);
        for (int c = g * cg + sub; c < (g + 1) * cg; c += lanes) {
            const float d = chan[c] - m;
            q += fmaf((float)count * d, d, chan[MAX_BUNDLE + c]);
        }
        q = lanes_sum(q, lanes);
        if (sub == 0) write(g, m, q);
    }
}

template <typename T, int V, int ACT, int R> __global__ __launch_bounds__(ONE_THREADS, 4) void norm_one_kernel(OneP p) {
    extern __shared__ float scratch[];             // 2 * blockDim * V floats
    __shared__ float chan[2 * MAX_BUNDLE], grp[2 * MAX_BUNDLE], part[ONE_THREADS];
    const long n = blockIdx.x / p.bundles;
    const int g0 = (int)(blockIdx.x % p.bundles) * p.per, groups = min(p.per, p.G - g0), cg = p.C / p.G, width = groups * cg;
    const int K = (width + V - 1) / V, RT = blockDim.x / K, t = threadIdx.x, col = t % K, r0 = t / K;
    const int count = r0 < RT ? (int)p.S : 0;
    const int own = col * V, c0 = min(own, width - V);
    const long at = n * p.S * p.C + g0 * cg + c0;
    const T* const x = reinterpret_cast<const T*>(p.x) + at;
    Vec<T, V> v[R];
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (r0 + u * RT < count) v[u] = load_vec<T, V>(x + (long)(r0 + u * RT) * p.C);
    float s1[V] = {}, s2[V] = {}, k0[V];
#pragma unroll
    for (int j = 0; j < V; ++j) k0[j] = r0 < count ? (float)v[0].v[j] : 0.f;
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (r0 + u * RT < count) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = (float)v[u].v[j] - k0[j];
                s1[j] += d;
                s2[j] = fmaf(d, d, s2[j]);
            }
            keep(v[u]);
        }
    column_stats<V>(r0 < count ? (count - 1 - r0) / RT + 1 : 0, k0, s1, s2);
    join_columns<V>(blockDim.x, K, RT, (int)p.S, s1, s2, scratch, part, [&](int k, float m, float sq) {
        const int own = k / V * V, c = min(own, width - V) + k % V;
        if (c >= own) {
            chan[c] = m;
            chan[MAX_BUNDLE + c] = sq;
        }
    });
    const float scale = 1.f / ((float)p.S * (float)cg);
    group_stats(chan, groups, cg, (int)p.S, p.glanes, [&](int g, float m, float q) {
        const float r = 1.f / sqrtf(q * scale + p.eps);
        grp[2 * g] = m;
        grp[2 * g + 1] = r;
        p.mean[n * p.G + g0 + g] = m;
        p.rstd[n * p.G + g0 + g] = r;
    });
    __syncthreads();
    int gr[V];
    groups_of<V>(c0, cg, gr);
    float m[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        m[j] = grp[2 * gr[j]];
        a[j] = grp[2 * gr[j] + 1] * load_param(p.w, p.wdtype, g0 * cg + c0 + j, 1.f);
        b[j] = load_param(p.b, p.wdtype, g0 * cg + c0 + j, 0.f);
    }
    T* const y = reinterpret_cast<T*>(p.y) + at;
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (r0 + u * RT < count) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[u].v[j] = (T)sed_act<ACT>(fmaf((float)v[u].v[j] - m[j], a[j], b[j]));
            store_vec<T, V>(y + (long)(r0 + u * RT) * p.C, v[u]);
        }
}

template <typename T, int V, int ACT, int R> __global__ __launch_bounds__(ONE_THREADS, 4) void norm_one_bwd_kernel(OneP p) {
    extern __shared__ float scratch[];
    __shared__ float chan[2 * MAX_BUNDLE], grp[2 * MAX_BUNDLE];
    const long n = blockIdx.x / p.bundles;
    const int g0 = (int)(blockIdx.x % p.bundles) * p.per, groups = min(p.per, p.G - g0), cg = p.C / p.G, width = groups * cg;
    const int K = (width + V - 1) / V, RT = blockDim.x / K, t = threadIdx.x, col = t % K, r0 = t / K;
    const bool on = r0 < RT;
    const int own = col * V, c0 = min(own, width - V);
    const long at = n * p.S * p.C + g0 * cg + c0;
    const T* const x = reinterpret_cast<const T*>(p.x) + at;
    const T* const gy = reinterpret_cast<const T*>(p.gy) + at;
    Vec<T, V> v[R], g[R];
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (on && r0 + u * RT < p.S) {
            v[u] = load_vec<T, V>(x + (long)(r0 + u * RT) * p.C);
            g[u] = load_vec<T, V>(gy + (long)(r0 + u * RT) * p.C);
        }
    float s1[V] = {}, s2[V] = {}, m[V], r[V], w[V], b[V];
    int gr[V];
    groups_of<V>(c0, cg, gr);
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int c = g0 * cg + c0 + j;
        const long ng = n * p.G + g0 + gr[j];
        m[j] = p.mean[ng];
        r[j] = p.rstd[ng];
        w[j] = load_param(p.w, p.wdtype, c, 1.f);
        b[j] = load_param(p.b, p.wdtype, c, 0.f);
    }
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (on && r0 + u * RT < p.S) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = ((float)v[u].v[j] - m[j]) * r[j];
                const float gz = sed_act_gz<ACT>((float)g[u].v[j], fmaf(xh, w[j], b[j]));
                s1[j] += gz;
                s2[j] = fmaf(gz, xh, s2[j]);
            }
            keep(v[u]);
            keep(g[u]);
        }
    channel_sums<V>(K, RT, K, width, s1, s2, scratch, chan);
    for (int k = t; k < width; k += blockDim.x) {
        p.chan[n * 2 * p.C + g0 * cg + k] = chan[k];
        p.chan[n * 2 * p.C + p.C + g0 * cg + k] = chan[MAX_BUNDLE + k];
    }
    if (!p.y) return;
    group_sums(chan, groups, cg, [&](int k) { return load_param(p.w, p.wdtype, g0 * cg + k, 1.f); }, grp);
    if (!on) return;
    const float scale = 1.f / ((float)p.S * (float)cg);
    T* const gx = reinterpret_cast<T*>(p.y) + at;
    float c1[V], c2[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        c1[j] = grp[2 * gr[j]] * scale;
        c2[j] = grp[2 * gr[j] + 1] * scale;
    }
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (r0 + u * RT < p.S) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float xh = ((float)v[u].v[j] - m[j]) * r[j];
                const float gz = sed_act_gz<ACT>((float)g[u].v[j], fmaf(xh, w[j], b[j]));
                v[u].v[j] = (T)(r[j] * (fmaf(gz, w[j], -c1[j]) - xh * c2[j]));
            }
            store_vec<T, V>(gx + (long)(r0 + u * RT) * p.C, v[u]);
        }
}

// ---- one pass over samples that a single workgroup cannot hold (forward): the rows of a sample lie in the registers of up to 128
// workgroups, 128 KB each.  Each publishes the statistics of its rows; the one that arrives last joins the sample's and publishes them;
// the others wait for that, and write their rows from registers.  Nothing rests on the workgroups of a sample running together: one that
// has waited WAIT_TICKS gives up (and with it all that wait later), and a second kernel, which normally finds nothing to do, writes
// what was left, from memory.  The results are the same bits either way.
// Taken from 384 MB on: below 256 MB the caches serve the second reading of the two passes.  256 x 64064 x 64 float16 (2.1 GB) takes
// 1062 us, in two passes 1255; 64 x 64064 x 64 float32 459 and 667; 262 MB of either type 149 to 201 and 163 to 179; 131 MB 85 and 80.
// (Backward, with x and gy in registers, the form that was built lost: 65 M bfloat16 elements 190 us, in two passes 146.  A sample then has
// twice the workgroups, and each published a row of channels for the last one to add up; what the waiting ones need is two numbers a
// group and chunk, which was not built.)
constexpr long SHARED_LEAST = 384l << 20;          // bytes of x
constexpr int SHARED_MOST = 128;                   // workgroups of a sample, of the 512 that are resident
constexpr long WAIT_TICKS = 200000;                // of the 100 MHz clock: 2 ms
struct SharedP {
    const void* x;
    const void* w;
    const void* b;
    void* y;
    float* mean;
    float* rstd;
    unsigned long long* stats;           // [N][G][chunks] {mean, sum of squared deviations}
    int* state;                          // zeroed: [N] arrived, [N] ready, given up, [N][chunks] written
    long N, S, wait;
    int rows, chunks, C, G, wdtype;
    int glanes, clanes;                  // lanes that add up a group's channels, and a group's chunks: powers of two up to 64
    float eps;
};
__device__ __forceinline__ float get(const float* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
__device__ __forceinline__ void put(float* p, float v) { __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }
// every store of the workgroup has reached the memory that all XCDs share
__device__ __forceinline__ void published() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}
// true in the workgroup of a sample that arrives last
__device__ __forceinline__ bool arrive(const SharedP& p, long n, int* word) {
    published();
    if (threadIdx.x == 0) *word = __hip_atomic_fetch_add(p.state + n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == p.chunks - 1;
    __syncthreads();
    const bool last = *word;
    __syncthreads();
    return last;
}
__device__ __forceinline__ void announce(const SharedP& p, long n) {
    published();
    if (threadIdx.x == 0) __hip_atomic_store(p.state + p.N + n, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// waits for the sample's sums; false: given up
__device__ __forceinline__ bool await(const SharedP& p, long n, int* word) {
    if (threadIdx.x == 0) {
        const long until = wall_clock64() + p.wait;
        int ok = 0;
        while (!(ok = __hip_atomic_load(p.state + p.N + n, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT))) {
            if (__hip_atomic_load(p.state + 2 * p.N, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT)) break;
            if ((long)wall_clock64() >= until) {
                __hip_atomic_store(p.state + 2 * p.N, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                break;
            }
            __builtin_amdgcn_s_sleep(8);
        }
        *word = ok;
    }
    __syncthreads();
    return *word != 0;
}
__device__ __forceinline__ void written(const SharedP& p) {
    if (threadIdx.x == 0) p.state[2 * p.N + 1 + blockIdx.x] = 1;
}
template <typename T, int V, int ACT, int R> __global__ __launch_bounds__(ONE_THREADS, 4) void norm_shared_kernel(SharedP p) {
    extern __shared__ float scratch[];             // 2 * ONE_THREADS * V floats
    __shared__ float chan[2 * MAX_BUNDLE], grp[2 * MAX_BUNDLE], part[ONE_THREADS];
    __shared__ int word;
    const long n = blockIdx.x / p.chunks;
    const int chunk = (int)(blockIdx.x % p.chunks), cg = p.C / p.G, K = (p.C + V - 1) / V, RT = ONE_THREADS / K;
    const int t = threadIdx.x, col = t % K, r0 = t / K, c0 = min(col * V, p.C - V);
    const long s0 = (long)chunk * p.rows;
    const int count = r0 < RT ? (int)min((long)p.rows, p.S - s0) : 0, all = (int)min((long)p.rows, p.S - s0);
    const long first = (n * p.S + s0) * p.C, at = first + c0;
    const T* const x = reinterpret_cast<const T*>(p.x) + at;
    Vec<T, V> v[R];
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (r0 + u * RT < count) v[u] = load_vec<T, V>(x + (long)(r0 + u * RT) * p.C);
    float s1[V] = {}, s2[V] = {}, k0[V];
#pragma unroll
    for (int j = 0; j < V; ++j) k0[j] = r0 < count ? (float)v[0].v[j] : 0.f;
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (r0 + u * RT < count) {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float d = (float)v[u].v[j] - k0[j];
                s1[j] += d;
                s2[j] = fmaf(d, d, s2[j]);
            }
            keep(v[u]);
        }
    column_stats<V>(r0 < count ? (count - 1 - r0) / RT + 1 : 0, k0, s1, s2);
    join_columns<V>(ONE_THREADS, K, RT, all, s1, s2, scratch, part, [&](int k, float m, float sq) {
        const int own = k / V * V, c = min(own, p.C - V) + k % V;
        if (c >= own) {
            chan[c] = m;
            chan[MAX_BUNDLE + c] = sq;
        }
    });
    group_stats(chan, p.G, cg, all, p.glanes, [&](int g, float m, float q) {
        __hip_atomic_store(p.stats + (n * p.G + g) * p.chunks + chunk, (unsigned long long)__float_as_uint(q) << 32 | __float_as_uint(m), __ATOMIC_RELAXED,
                           __HIP_MEMORY_SCOPE_AGENT);
    });
    if (arrive(p, n, &word)) {
        const float scale = 1.f / (float)p.S, share = 1.f / (float)cg;
        const int L = p.clanes, sub = t % L;
#pragma unroll 2
        for (int g = t / L; g < p.G; g += ONE_THREADS / L) {
            float m[SHARED_MOST / 64], q[SHARED_MOST / 64], cnt[SHARED_MOST / 64], a = 0.f, b = 0.f;
#pragma unroll
            for (int i = 0; i < SHARED_MOST / 64; ++i) {
                const int k = i * L + sub;
                unsigned long long e = 0;
                if (k < p.chunks) e = __hip_atomic_load(p.stats + (n * p.G + g) * p.chunks + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                cnt[i] = k < p.chunks ? (float)min((long)p.rows, p.S - (long)k * p.rows) * scale : 0.f;
                m[i] = __uint_as_float((unsigned)e);
                q[i] = __uint_as_float((unsigned)(e >> 32));
            }
            const float ref = __shfl(m[0], (t & 63) - sub, 64);          // the first chunk's
#pragma unroll
            for (int i = 0; i < SHARED_MOST / 64; ++i) a = fmaf(cnt[i], m[i] - ref, a);
            const float mean = lanes_sum(a, L) + ref;
#pragma unroll
            for (int i = 0; i < SHARED_MOST / 64; ++i) {
                const float d = m[i] - mean;
                b += fmaf(cnt[i] * d, d, q[i] * share * scale);
            }
            b = lanes_sum(b, L);
            if (sub == 0) {
                grp[2 * g] = mean;
                grp[2 * g + 1] = 1.f / sqrtf(b + p.eps);
                put(p.mean + n * p.G + g, mean);
                put(p.rstd + n * p.G + g, grp[2 * g + 1]);
            }
        }
        announce(p, n);
    } else {
        if (!await(p, n, &word)) return;
        for (int g = t; g < p.G; g += ONE_THREADS) {
            grp[2 * g] = get(p.mean + n * p.G + g);
            grp[2 * g + 1] = get(p.rstd + n * p.G + g);
        }
        __syncthreads();
    }
    written(p);
    int gr[V];
    groups_of<V>(c0, cg, gr);
    float m[V], a[V], b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) {
        m[j] = grp[2 * gr[j]];
        a[j] = grp[2 * gr[j] + 1] * load_param(p.w, p.wdtype, c0 + j, 1.f);
        b[j] = load_param(p.b, p.wdtype, c0 + j, 0.f);
    }
    T* const y = reinterpret_cast<T*>(p.y) + at;
#pragma unroll
    for (int u = 0; u < R; ++u)
        if (r0 + u * RT < count) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[u].v[j] = (T)sed_act<ACT>(fmaf((float)v[u].v[j] - m[j], a[j], b[j]));
            store_vec<T, V>(y + (long)(r0 + u * RT) * p.C, v[u]);
        }
}

// the rows of the chunks that were given up
template <typename T, int V, int ACT> __global__ __launch_bounds__(ONE_THREADS) void norm_rest_kernel(SharedP p) {
    __shared__ int list[ONE_THREADS], left;
    const long total = p.N * p.chunks;
    const int t = threadIdx.x, K = (p.C + V - 1) / V, RT = ONE_THREADS / K, c0 = min(t % K * V, p.C - V), r0 = t / K;
    int gr[V];
    groups_of<V>(c0, p.C / p.G, gr);
    for (long base = (long)blockIdx.x * ONE_THREADS; base < total; base += (long)gridDim.x * ONE_THREADS) {
        __syncthreads();
        if (t == 0) left = 0;
        __syncthreads();
        if (base + t < total && !p.state[2 * p.N + 1 + base + t]) list[atomicAdd(&left, 1)] = (int)(base + t);
        __syncthreads();
        for (int i = 0; i < left; ++i) {
            const long n = list[i] / p.chunks, s0 = (long)(list[i] % p.chunks) * p.rows, at = (n * p.S + s0) * p.C + c0;
            const int count = r0 < RT ? (int)min((long)p.rows, p.S - s0) : 0;
            float m[V], a[V], b[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                m[j] = p.mean[n * p.G + gr[j]];
                a[j] = p.rstd[n * p.G + gr[j]] * load_param(p.w, p.wdtype, c0 + j, 1.f);
                b[j] = load_param(p.b, p.wdtype, c0 + j, 0.f);
            }
            for (int s = r0; s < count; s += RT) {
                auto v = load_vec<T, V>(reinterpret_cast<const T*>(p.x) + at + (long)s * p.C);
#pragma unroll
                for (int j = 0; j < V; ++j) v.v[j] = (T)sed_act<ACT>(fmaf((float)v.v[j] - m[j], a[j], b[j]));
                store_vec<T, V>(reinterpret_cast<T*>(p.y) + at + (long)s * p.C, v);
            }
        }
    }
}
__global__ __launch_bounds__(256) void norm_zero_kernel(int* p, long n) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long)gridDim.x * 256) p[i] = 0;
}

int esize_of(int dtype) { return dtype == SED_F32 ? 4 : 2; }
bool bad_shape(int dtype, int wdtype, long N, long S, int C, int G, int act) {
    return dtype < 0 || dtype > 2 || wdtype < 0 || wdtype > 2 || N < 1 || S < 1 || C < 1 || G < 1 || C % G || act < 0 || act > 3 ||
           // a launch takes fewer than 2^32 threads: 1024 a workgroup for the joins and the parameters' sums, 256 for the passes
           N * G >= 1L << 22 || C / 16 + 1 >= 1L << 22 || cut_of(N, S, C, esize_of(dtype)).blocks + C / 16 + 1 >= 1L << 24;
}
// How the one-pass kernels cut: bundles of whole groups with at least 128 bytes of a row (or all of it), a workgroup of so many threads
// that each holds up to R vectors.  threads = 0: the rows do not fit, or a row has fewer channels than a vector.
struct One {
    int per, bundles, threads, R;
};
One one_of(long N, long S, int C, int G, int esize, int most) {
    One o{};
    const int V = 16 / esize, cg = C / G;
    o.per = (128 / esize + cg - 1) / cg;
    if (o.per > G) o.per = G;
    // the last bundle has what is left: it must hold a vector too, else it joins its neighbours
    while (o.per < G && (G % o.per ? G % o.per : o.per) * cg < V) ++o.per;
    const long width = (long)o.per * cg;
    o.bundles = (G + o.per - 1) / o.per;
    const long K = (width + V - 1) / V;
    if (C < V || width > MAX_BUNDLE || K > 256 || S > (long)ONE_THREADS * most || N * o.bundles >= (1L << 32) / ONE_THREADS) return o;
    const long want = K * ((S + 3) / 4);           // four vectors a thread, as far as the threads go
    o.threads = (int)(want < 64 ? 64 : want > ONE_THREADS ? ONE_THREADS : (want + 63) / 64 * 64);
    if (o.threads < K) o.threads = (int)((K + 63) / 64 * 64);
    const long each = (S + o.threads / K - 1) / (o.threads / K);
    if (each > most) o.threads = 0;
    else o.R = each <= 4 ? 4 : most;
    return o;
}
// How the kernels that share a sample cut: chunks of rows that fit a workgroup.  chunks = 0: not for them.
struct Shared {
    int rows, chunks;
};
Shared shared_of(long N, long S, int C, int esize) {
    const int V = 16 / esize;
    const long K = (C + V - 1) / V, RT = ONE_THREADS / K;
    if (C < V || C > MAX_BUNDLE || N * S * C * esize < SHARED_LEAST) return {0, 0};
    const long most = RT * ONE_FWD, chunks = (S + most - 1) / most;
    if (chunks > SHARED_MOST || N * chunks >= (1L << 32) / ONE_THREADS) return {0, 0};
    const long rows = ((S + chunks - 1) / chunks + RT - 1) / RT * RT;        // even shares
    return {(int)rows, (int)((S + rows - 1) / rows)};
}
int lanes_of(int n) {
    int l = 1;
    while (l < n && l < 64) l *= 2;
    return l;
}
long state_ints(long N, int chunks) { return 2 * N + 1 + N * chunks; }
NormP params_of(const Cut& c, const void* x, const void* w, const void* b, int wdtype, long S, int C, int G, float* ws) {
    NormP p{};
    p.x = x; p.w = w; p.b = b; p.wdtype = wdtype;
    p.S = S; p.rows = c.rows; p.chunks = c.chunks; p.C = C; p.G = G; p.CT = c.CT; p.RT = c.RT; p.tiles = c.tiles; p.K = c.K;
    p.parts = ws;
    return p;
}

// the counters and flags of a launch, cleared; workgroups of the kernel behind it
unsigned clear(const SharedP& p, hipStream_t stream) {
    const long ints = state_ints(p.N, p.chunks), nb = (ints + 255) / 256, rest = (p.N * p.chunks + ONE_THREADS - 1) / ONE_THREADS;
    hipLaunchKernelGGL(norm_zero_kernel, dim3((unsigned)(nb > 1024 ? 1024 : nb)), dim3(256), 0, stream, p.state, ints);
    return (unsigned)(rest > 1024 ? 1024 : rest);
}

#define NORM_ACT(KERNEL, T, V)                                                                              \
    switch (act) {                                                                                          \
        case SED_ACT_NONE: hipLaunchKernelGGL((KERNEL<T, V, 0>), grid, dim3(THREADS), 0, stream, p); break; \
        case SED_ACT_RELU: hipLaunchKernelGGL((KERNEL<T, V, 1>), grid, dim3(THREADS), 0, stream, p); break; \
        case SED_ACT_SILU: hipLaunchKernelGGL((KERNEL<T, V, 2>), grid, dim3(THREADS), 0, stream, p); break; \
        default: hipLaunchKernelGGL((KERNEL<T, V, 3>), grid, dim3(THREADS), 0, stream, p);                  \
    }
#define NORM_APPLY(KERNEL, T, V)                                                                                          \
    {                                                                                                                     \
        const dim3 with((unsigned)(params.blocks + c.blocks));                                                            \
        switch (act) {                                                                                                    \
            case SED_ACT_NONE: hipLaunchKernelGGL((KERNEL<T, V, 0>), with, dim3(THREADS), 0, stream, p, params); break; \
            case SED_ACT_RELU: hipLaunchKernelGGL((KERNEL<T, V, 1>), with, dim3(THREADS), 0, stream, p, params); break; \
            case SED_ACT_SILU: hipLaunchKernelGGL((KERNEL<T, V, 2>), with, dim3(THREADS), 0, stream, p, params); break; \
            default: hipLaunchKernelGGL((KERNEL<T, V, 3>), with, dim3(THREADS), 0, stream, p, params);                  \
        }                                                                                                                 \
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
#define ONE_ACT(KERNEL, MOST, T, V)                                                                                                          \
    switch (act) {                                                                                                                           \
        case SED_ACT_NONE: ONE_R(KERNEL, MOST, T, V, 0) break;                                                                               \
        case SED_ACT_RELU: ONE_R(KERNEL, MOST, T, V, 1) break;                                                                               \
        case SED_ACT_SILU: ONE_R(KERNEL, MOST, T, V, 2) break;                                                                               \
        default: ONE_R(KERNEL, MOST, T, V, 3)                                                                                                \
    }
#define ONE_R(KERNEL, MOST, T, V, ACT)                                                                                                       \
    if (one.R == 4) hipLaunchKernelGGL((KERNEL<T, V, ACT, 4>), grid, dim3(one.threads), 2 * one.threads * V * 4, stream, p);                 \
    else hipLaunchKernelGGL((KERNEL<T, V, ACT, MOST>), grid, dim3(one.threads), 2 * one.threads * V * 4, stream, p);
#define ONE_TYPE(KERNEL, MOST)                                        \
    if (dtype == SED_F32) { ONE_ACT(KERNEL, MOST, float, 4) }         \
    else if (dtype == SED_F16) { ONE_ACT(KERNEL, MOST, _Float16, 8) } \
    else { ONE_ACT(KERNEL, MOST, __bf16, 8) }
#define SHARED(T, V, ACT)                                                                                                                             \
    hipLaunchKernelGGL((norm_shared_kernel<T, V, ACT, ONE_FWD>), dim3((unsigned)(N * sh.chunks)), dim3(ONE_THREADS), 2 * ONE_THREADS * V * 4, stream, p); \
    hipLaunchKernelGGL((norm_rest_kernel<T, V, ACT>), dim3(rest), dim3(ONE_THREADS), 0, stream, p);
#define SHARED_ACT(T, V)                        \
    switch (act) {                              \
        case SED_ACT_NONE: SHARED(T, V, 0) break; \
        case SED_ACT_RELU: SHARED(T, V, 1) break; \
        case SED_ACT_SILU: SHARED(T, V, 2) break; \
        default: SHARED(T, V, 3)                \
    }
#define NORM_PLAIN(KERNEL, T, V) hipLaunchKernelGGL((KERNEL<T, V>), grid, dim3(THREADS), 0, stream, p);

}  // namespace

SED_API long sed_group_norm_ws_floats(int dtype, long N, long S, int C, int G, int backward) {
    if (bad_shape(dtype, SED_F32, N, S, C, G, 0)) return 0;
    if (one_of(N, S, C, G, esize_of(dtype), backward ? ONE_BWD : ONE_FWD).threads) return backward ? N * 2 * C : 0;
    const Shared sh = shared_of(N, S, C, esize_of(dtype));
    if (!backward && sh.chunks) return 1 + N * G * sh.chunks * 2 + state_ints(N, sh.chunks);
    const long parts = N * cut_of(N, S, C, esize_of(dtype)).chunks * 2 * C;
    return backward ? parts + N * 2 * C + N * 2 * G : parts;
}

SED_API int sed_group_norm_fwd(const void* x, const void* weight, const void* bias, int dtype, int wdtype, long N, long S, int C, int G,
                               float eps, int act, void* y, float* mean, float* rstd, float* ws, sed_stream_t stream) {
    if (!x || !y || !mean || !rstd || !(eps >= 0.f) || bad_shape(dtype, wdtype, N, S, C, G, act)) return SED_EINVAL;
    const One one = one_of(N, S, C, G, esize_of(dtype), ONE_FWD);
    if (!one.threads && !ws) return SED_EINVAL;
    if (one.threads) {
        const dim3 grid((unsigned)(N * one.bundles));
        OneP p{x, nullptr, weight, bias, y, mean, rstd, nullptr, S, C, G, one.per, one.bundles, wdtype, lanes_of(C / G), eps};
        ONE_TYPE(norm_one_kernel, ONE_FWD)
        SED_LAUNCH_CHECK();
        return 0;
    }
    const Shared sh = shared_of(N, S, C, esize_of(dtype));
    if (sh.chunks) {
        float* const stats = ws + (reinterpret_cast<uintptr_t>(ws) & 7) / 4;          // 8-byte numbers
        const SharedP p{x, weight, bias, y, mean, rstd, reinterpret_cast<unsigned long long*>(stats), reinterpret_cast<int*>(stats + N * G * sh.chunks * 2),
                        N, S, sed_spin_limit__() < WAIT_TICKS ? sed_spin_limit__() : WAIT_TICKS, sh.rows, sh.chunks, C, G, wdtype, lanes_of(C / G), lanes_of(sh.chunks), eps};
        const unsigned rest = clear(p, stream);
        if (dtype == SED_F32) { SHARED_ACT(float, 4) }
        else if (dtype == SED_F16) { SHARED_ACT(_Float16, 8) }
        else { SHARED_ACT(__bf16, 8) }
        SED_LAUNCH_CHECK();
        return 0;
    }
    const Cut c = cut_of(N, S, C, esize_of(dtype));
    const dim3 grid((unsigned)c.blocks);
    NormP p = params_of(c, x, weight, bias, wdtype, S, C, G, ws);
    p.y = y; p.mean = mean; p.rstd = rstd;
    NORM_TYPE(NORM_PLAIN, norm_stats_kernel)
    const Join j = join_of(N, c.chunks, C, G);
    hipLaunchKernelGGL(norm_finalize_kernel, dim3((unsigned)j.blocks), dim3(j.threads), 0, stream, ws, S, c.rows, c.chunks, C, G, j.per, eps, mean, rstd);
    NORM_TYPE(NORM_ACT, norm_apply_kernel)
    SED_LAUNCH_CHECK();
    return 0;
}

SED_API int sed_group_norm_bwd(const void* x, const void* gy, const void* weight, const void* bias, int dtype, int wdtype, long N, long S,
                               int C, int G, int act, const float* mean, const float* rstd, void* gx, void* gweight, void* gbias,
                               float* ws, sed_stream_t stream) {
    if (!x || !gy || !mean || !rstd || !ws || bad_shape(dtype, wdtype, N, S, C, G, act)) return SED_EINVAL;
    const One one = one_of(N, S, C, G, esize_of(dtype), ONE_BWD);
    if (one.threads) {
        const dim3 grid((unsigned)(N * one.bundles));
        OneP p{x, gy, weight, bias, gx, const_cast<float*>(mean), const_cast<float*>(rstd), ws, S, C, G, one.per, one.bundles, wdtype, 0, 0.f};
        ONE_TYPE(norm_one_bwd_kernel, ONE_BWD)
        const ParamsP params{ws, N, C, wdtype, gweight, gbias, gweight || gbias ? sed_cdiv(C, 16) : 0};
        if (params.blocks) hipLaunchKernelGGL(norm_bwd_params_kernel, dim3((unsigned)params.blocks), dim3(1024), 0, stream, params);
        SED_LAUNCH_CHECK();
        return 0;
    }
    const Cut c = cut_of(N, S, C, esize_of(dtype));
    const dim3 grid((unsigned)c.blocks);
    NormP p = params_of(c, x, weight, bias, wdtype, S, C, G, ws);
    float* const chan = ws + N * c.chunks * 2 * C;
    float* const coef = chan + N * 2 * C;
    p.gy = gy; p.y = gx; p.mean = mean; p.rstd = rstd; p.coef = coef;
    NORM_TYPE(NORM_ACT, norm_bwd_sums_kernel)
    const Join j = join_of(N, c.chunks, C, G);
    hipLaunchKernelGGL(norm_bwd_fold_kernel, dim3((unsigned)j.blocks), dim3(j.threads), 0, stream, ws, S, c.chunks, C, G, j.per, weight, wdtype, chan, coef);
    const ParamsP params{chan, N, C, wdtype, gweight, gbias, gweight || gbias ? sed_cdiv(C, 16) : 0};
    if (gx) { NORM_TYPE(NORM_APPLY, norm_bwd_apply_kernel) }
    else if (params.blocks) hipLaunchKernelGGL(norm_bwd_params_kernel, dim3((unsigned)params.blocks), dim3(1024), 0, stream, params);
    SED_LAUNCH_CHECK();
    return 0;
}
