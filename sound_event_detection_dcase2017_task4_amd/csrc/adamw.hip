// AdamW over many tensors in one launch, moments held in 32 or in 8 bits.
//
//   m = b1 m + (1 - b1) g      v = b2 v + (1 - b2) g^2      p = (1 - lr wd) p - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// The work is a list of chunks of 4096 elements, each inside one tensor: a 28-tensor model and a single 240-million-element matrix
// fill the chip alike, and no tensor costs a launch.  Bound by HBM: 28 bytes an element with 32-bit moments (parameter, gradient, two
// moments in; parameter, two moments out; 30 for a 16-bit parameter with its 32-bit copy), 16 (18) bytes with 8-bit ones.
//
// A 16-bit parameter is the rounding of its 32-bit copy.  Where it is not, somebody else wrote the parameter since the last step, and
// the step goes on from the parameter: nothing has to be remembered about who wrote it, at two bytes an element.
//
// 8-bit moments: a block of 256 elements -- one wave, four elements a lane -- shares one scale, the block's largest magnitude, held
// in 32 bits.  The codes are powers of a linear grid, because the moments of one block spread over decades and a relative error
// is what the update sees:
//   m = sign(q) (|q| / 127)^2 scale, q = rint(127 sqrt(|m| / scale))       half a step = 0.8 % at the scale, 8 % at a hundredth of it
//   v = (q / 255)^4 scale,           q = rint(255 (v / scale)^(1/4))       half a step of sqrt(v) = 0.4 % at the scale
// A positive v does not decode to 0 (its code is at least 1, which stands for 2.4e-10 of the scale): m / (0 + eps) would be a step of any
// size.  Below a scale of 3e-36 -- gradients of 1e-18 -- the product underflows to 0 all the same, and eps has to hold.  The update itself
// uses the new moments in 32 bits; only what the next step reads is rounded.  A NaN in a block makes its scale NaN, and the block reads back
// as NaN.  An infinite m (or a gradient beyond 1.8e19, whose square is) makes it infinite: the codes are then 0 for m, which reads back as
// NaN; and 1 for a positive v, which reads back as infinity (0 as NaN): where only v overflowed, the block's updates are 0 from there on, as
// a 32-bit element's are.
#include "common.h"
#include "sed_hip.h"

SED_OBJECT_FLAGS(adamw)

namespace {

constexpr int BLK = 256;            // elements of one 8-bit block; every tensor's state begins at a multiple of it
constexpr int CHUNK = 4096;         // elements of one workgroup
constexpr int MAX_GROUPS = 16;
constexpr int ROW = 6;              // longs per tensor: parameter, gradient, first element of its moments, of its copy, elements, group | type << 32

struct Hyper {
    float decay, step_size, b1, omb1, b2, omb2, inv_c2, eps;
};
struct AdamwP {
    const long* rows;
    const int2* chunks;             // (tensor, chunk inside it)
    void* m;
    void* v;
    float* ms;
    float* vs;
    float* master;
    const int* skip_flag;
    int* skipped;
    float grad_scale;
    Hyper h[MAX_GROUPS];
};

template <typename T> struct Vec4;
template <> struct Vec4<float> { typedef float type __attribute__((ext_vector_type(4))); };
template <> struct Vec4<_Float16> { typedef _Float16 type __attribute__((ext_vector_type(4))); };
template <> struct Vec4<__bf16> { typedef __bf16 type __attribute__((ext_vector_type(4))); };

// four elements at e of a tensor of n; wide when the base address allows it
template <typename T> __device__ __forceinline__ void load4(const T* p, long e, long n, bool wide, float (&f)[4]) {
    if (wide && e + 4 <= n) {
        const auto q = *reinterpret_cast<const typename Vec4<T>::type*>(p + e);
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = (float)q[j];
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) f[j] = e + j < n ? (float)p[e + j] : 0.f;
    }
}
template <typename T> __device__ __forceinline__ void store4(T* p, long e, long n, bool wide, const float (&f)[4]) {
    if (wide && e + 4 <= n) {
        typename Vec4<T>::type q;
#pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = (T)f[j];
        *reinterpret_cast<typename Vec4<T>::type*>(p + e) = q;
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (e + j < n) p[e + j] = (T)f[j];
    }
}

// largest of non-negative floats over the wave, compared as bits: a NaN is the largest of all and is not lost.  Lanes trade within quads,
// rows of 16 and across rows by DPP moves, which need no LDS (958 -> 828 us at 240 M elements, now 820); lane 63 ends with the largest.
template <int CTRL> __device__ __forceinline__ int max_dpp(int m) { return max(m, __builtin_amdgcn_update_dpp(m, m, CTRL, 0xf, 0xf, false)); }
__device__ __forceinline__ float wave_max_bits(float a, float b, float c, float d) {
    int m = max(max(__float_as_int(a), __float_as_int(b)), max(__float_as_int(c), __float_as_int(d)));       // no sign bit: int order is float order
    m = max_dpp<0xB1>(m);                          // quad_perm 1 0 3 2
    m = max_dpp<0x4E>(m);                          // quad_perm 2 3 0 1
    m = max_dpp<0x141>(m);                         // row_half_mirror
    m = max_dpp<0x140>(m);                         // row_mirror
    m = max_dpp<0x142>(m);                         // row_bcast 15
    m = max_dpp<0x143>(m);                         // row_bcast 31
    return __int_as_float(__builtin_amdgcn_readlane(m, 63));
}

// The codes and the sums below are formed with one rounding per operation (no fused multiply-add): a code is then the same wherever
// it is formed, and a value next to the border of two codes does not depend on how the compiler groups the terms.
__device__ __forceinline__ float decode_m(int q, float scale) {
#pragma clang fp contract(off)
    const float u = (float)q * (float)(1.0 / 127.0);
    return u * fabsf(u) * scale;
}
__device__ __forceinline__ float decode_v(int q, float scale) {
#pragma clang fp contract(off)
    float u = (float)q * (float)(1.0 / 255.0);
    u = u * u;
    return u * u * scale;
}
// The code is defined by correctly rounded divisions and roots, some hundred instructions for an element's two codes.  The hardware's
// reciprocal and root (1 ulp each) give the same code unless the value lies within their error of the border of two codes: 4.5e-7 of
// it covers both sides' roundings (2 ulp + 1 + 1/2 against 1 and a half).  Then, and for scales whose reciprocal is not a normal
// number, the lane takes the long way: about one wave in fifty does.
__device__ __forceinline__ int encode_m(float m, float scale) {
    const int q = (int)rintf(sqrtf(fabsf(m) / scale) * 127.f);
    return m < 0.f ? -q : q;
}
__device__ __forceinline__ int encode_v(float v, float scale) {
    const int q = (int)rintf(sqrtf(sqrtf(v / scale)) * 255.f);
    return v > 0.f ? max(q, 1) : q;
}
__device__ __forceinline__ bool usual(float scale) { return scale > 1e-30f && scale < 1e30f; }
__device__ __forceinline__ void encode4(const float (&m)[4], const float (&v)[4], float sm, float sv, char4& cm, uchar4& cv) {
    bool near = !usual(sm) || !usual(sv);
    const float rm = __builtin_amdgcn_rcpf(sm), rv = __builtin_amdgcn_rcpf(sv);
    int qm[4], qv[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float um = __builtin_amdgcn_sqrtf(fabsf(m[j]) * rm) * 127.f, nm = rintf(um);
        const float uv = __builtin_amdgcn_sqrtf(__builtin_amdgcn_sqrtf(v[j] * rv)) * 255.f, nv = rintf(uv);
        near |= fabsf(um - nm) > fmaf(um, -4.5e-7f, 0.5f) || fabsf(uv - nv) > fmaf(uv, -4.5e-7f, 0.5f);
        qm[j] = m[j] < 0.f ? -(int)nm : (int)nm;
        qv[j] = v[j] > 0.f ? max((int)nv, 1) : (int)nv;
    }
    if (near)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            qm[j] = encode_m(m[j], sm);
            qv[j] = encode_v(v[j], sv);
        }
    cm = make_char4(qm[0], qm[1], qm[2], qm[3]);
    cv = make_uchar4(qv[0], qv[1], qv[2], qv[3]);
}
// 1 ulp, down to the smallest numbers
__device__ __forceinline__ float root(float v) {
    const bool tiny = v < 0x1p-100f;
    return __builtin_amdgcn_sqrtf(tiny ? v * 0x1p60f : v) * (tiny ? 0x1p-30f : 1.f);
}

template <typename T, bool EIGHT> __device__ __forceinline__ void adamw_chunk(const AdamwP& a, const long* row, long c0) {
    T* const p = reinterpret_cast<T*>(row[0]);
    const T* const g = reinterpret_cast<const T*>(row[1]);
    const long n = row[4], off = row[2], padded = (n + BLK - 1) / BLK * BLK;
    float* const copy = sizeof(T) == 4 ? nullptr : a.master + row[3];
    const Hyper h = a.h[(int)(row[5] & 0xffffffff)];
    const bool wide = ((row[0] | row[1]) & (4 * sizeof(T) - 1)) == 0;
    float pv[4][4], gv[4][4], mv[4][4], vv[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long e = c0 + i * 1024 + threadIdx.x * 4;
        if (e >= padded) continue;
        load4(g, e, n, wide, gv[i]);
        if (sizeof(T) == 4) load4(p, e, n, wide, pv[i]);
        else {
            float q[4];
            load4(copy, e, padded, true, pv[i]);
            load4(p, e, n, wide, q);
#pragma unroll
            for (int j = 0; j < 4; ++j) pv[i][j] = (float)(T)pv[i][j] == q[j] ? pv[i][j] : q[j];
        }
        if (EIGHT) {
            const char4 qm = reinterpret_cast<const char4*>(a.m)[(off + e) >> 2];
            const uchar4 qv = reinterpret_cast<const uchar4*>(a.v)[(off + e) >> 2];
            const float sm = a.ms[(off + e) / BLK], sv = a.vs[(off + e) / BLK];
            mv[i][0] = decode_m(qm.x, sm); mv[i][1] = decode_m(qm.y, sm); mv[i][2] = decode_m(qm.z, sm); mv[i][3] = decode_m(qm.w, sm);
            vv[i][0] = decode_v(qv.x, sv); vv[i][1] = decode_v(qv.y, sv); vv[i][2] = decode_v(qv.z, sv); vv[i][3] = decode_v(qv.w, sv);
        } else {
            load4(reinterpret_cast<const float*>(a.m) + off, e, padded, true, mv[i]);
            load4(reinterpret_cast<const float*>(a.v) + off, e, padded, true, vv[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const long e = c0 + i * 1024 + threadIdx.x * 4;
        if (e >= padded) continue;                 // whole waves: a wave's 256 elements are one block
        {
#pragma clang fp contract(off)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float gj = gv[i][j] * a.grad_scale;
                mv[i][j] = mv[i][j] * h.b1 + gj * h.omb1;
                vv[i][j] = vv[i][j] * h.b2 + gj * gj * h.omb2;
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) pv[i][j] = pv[i][j] * h.decay - h.step_size * mv[i][j] * __builtin_amdgcn_rcpf(fmaf(root(vv[i][j]), h.inv_c2, h.eps));
        if (e < n) {
            store4(p, e, n, wide, pv[i]);
            if (sizeof(T) != 4) store4(copy, e, n, true, pv[i]);
        }
        if (EIGHT) {
            const float sm = wave_max_bits(fabsf(mv[i][0]), fabsf(mv[i][1]), fabsf(mv[i][2]), fabsf(mv[i][3]));
            const float sv = wave_max_bits(fabsf(vv[i][0]), fabsf(vv[i][1]), fabsf(vv[i][2]), fabsf(vv[i][3]));
            const float dm = sm > 0.f ? sm : 1.f, dv = sv > 0.f ? sv : 1.f;
            char4 cm;
            uchar4 cv;
            encode4(mv[i], vv[i], dm, dv, cm, cv);
            reinterpret_cast<char4*>(a.m)[(off + e) >> 2] = cm;
            reinterpret_cast<uchar4*>(a.v)[(off + e) >> 2] = cv;
            if ((threadIdx.x & 63) == 0) {
                a.ms[(off + e) / BLK] = sm;
                a.vs[(off + e) / BLK] = sv;
            }
        } else {
            store4(reinterpret_cast<float*>(a.m) + off, e, n, true, mv[i]);
            store4(reinterpret_cast<float*>(a.v) + off, e, n, true, vv[i]);
        }
    }
}

// five workgroups on a CU: with four 4.7 M elements took 23.5 us for 21.4, with six (and what does not fit the registers in memory) 28.5
template <bool EIGHT> __global__ __launch_bounds__(256, 5) void adamw_kernel(AdamwP a) {
    if (a.skip_flag && __hip_atomic_load(a.skip_flag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0) {
        if (blockIdx.x == 0 && threadIdx.x == 0) atomicAdd(a.skipped, 1);
        return;
    }
    const int2 c = a.chunks[blockIdx.x];
    const long* const row = a.rows + (long)c.x * ROW;
    if (row[1] == 0) return;                       // no gradient in this step: the tensor and its moments stay
    const int type = (int)(row[5] >> 32);
    const long c0 = (long)c.y * CHUNK;
    if (type == SED_F32) adamw_chunk<float, EIGHT>(a, row, c0);
    else if (type == SED_F16) adamw_chunk<_Float16, EIGHT>(a, row, c0);
    else adamw_chunk<__bf16, EIGHT>(a, row, c0);
}

// sed_guard_collect: one thread in front of a step
__global__ void guard_collect_kernel(const float* rank_flag, int* skip_flag, const int* skipped, int* err_host, int* status_host) {
    int bad = __hip_atomic_load(skip_flag, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) != 0;
    if (rank_flag && !(rank_flag[0] == 0.f)) {
        bad = 1;
        __hip_atomic_store(skip_flag, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        if (err_host) __hip_atomic_store(err_host, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
    }
    if (status_host) __hip_atomic_store(status_host, __hip_atomic_load(skipped, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) + bad, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_SYSTEM);
}

__global__ __launch_bounds__(256) void adamw_moments_kernel(const char4* m, const float* ms, const uchar4* v, const float* vs, long n4,
                                                            float4* om, float4* ov) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < n4; i += (long)gridDim.x * 256) {
        const char4 q = m[i];
        const uchar4 r = v[i];
        const float sm = ms[i / (BLK / 4)], sv = vs[i / (BLK / 4)];
        om[i] = make_float4(decode_m(q.x, sm), decode_m(q.y, sm), decode_m(q.z, sm), decode_m(q.w, sm));
        ov[i] = make_float4(decode_v(r.x, sv), decode_v(r.y, sv), decode_v(r.z, sv), decode_v(r.w, sv));
    }
}

}  // namespace

SED_API int sed_adamw_chunk(void) { return CHUNK; }

SED_API int sed_adamw(const long* rows, const int* chunks, long nchunks, void* m, void* v, float* m_scale, float* v_scale,
                      float* master, int state_bits, const double* hyper, int ngroups, int step, float grad_scale, const int* skip_flag,
                      int* skipped, sed_stream_t stream) {
    if (!rows || !chunks || !m || !v || !hyper || nchunks < 1 || nchunks >= 1L << 24 || ngroups < 1 || ngroups > MAX_GROUPS || step < 1)
        return SED_EINVAL;
    if (state_bits != 32 && (state_bits != 8 || !m_scale || !v_scale)) return SED_EINVAL;
    if (skip_flag && !skipped) return SED_EINVAL;
    AdamwP a{};
    a.rows = rows; a.chunks = reinterpret_cast<const int2*>(chunks);
    a.m = m; a.v = v; a.ms = m_scale; a.vs = v_scale; a.master = master;
    a.skip_flag = skip_flag; a.skipped = skipped; a.grad_scale = grad_scale;
    for (int k = 0; k < ngroups; ++k) {
        const double *q = hyper + 5 * k, lr = q[0], b1 = q[1], b2 = q[2], eps = q[3], wd = q[4];
        if (!(b1 >= 0 && b1 < 1 && b2 >= 0 && b2 < 1 && eps >= 0)) return SED_EINVAL;
        // formed in double and rounded once: 1.f - 0.999f is 5e-5 off
        a.h[k] = {(float)(1.0 - lr * wd), (float)(lr / (1.0 - pow(b1, step))), (float)b1, (float)(1.0 - b1), (float)b2, (float)(1.0 - b2),
                  (float)(1.0 / sqrt(1.0 - pow(b2, step))), (float)eps};
    }
    if (state_bits == 8) hipLaunchKernelGGL(adamw_kernel<true>, dim3((unsigned)nchunks), dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(adamw_kernel<false>, dim3((unsigned)nchunks), dim3(256), 0, stream, a);
    SED_LAUNCH_CHECK();
    return 0;
}

SED_API int sed_guard_collect(const float* rank_flag, int* skip_flag, const int* skipped, int* err_host, int* status_host, sed_stream_t stream) {
    if (!skip_flag || (status_host && !skipped)) return SED_EINVAL;
    hipLaunchKernelGGL(guard_collect_kernel, dim3(1), dim3(1), 0, stream, rank_flag, skip_flag, skipped, err_host, status_host);
    SED_LAUNCH_CHECK();
    return 0;
}

SED_API int sed_adamw_moments(const void* m, const float* m_scale, const void* v, const float* v_scale, long n, float* out_m,
                              float* out_v, sed_stream_t stream) {
    if (!m || !m_scale || !v || !v_scale || !out_m || !out_v || n < 1 || n % BLK) return SED_EINVAL;
    const long nb = (n / 4 + 255) / 256;
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)(nb > 16384 ? 16384 : nb)), dim3(256), 0, stream,
                       reinterpret_cast<const char4*>(m), m_scale, reinterpret_cast<const uchar4*>(v), v_scale, n / 4,
                       reinterpret_cast<float4*>(out_m), reinterpret_cast<float4*>(out_v));
    SED_LAUNCH_CHECK();
    return 0;
}
