// Matrix products with bias, activation and residual in their epilogue, forward and backward, for 32- and 16-bit tensors.
//
//   z = x W^T + b;  y = act(z) + r          x [M][K], W [N][K], y, r [M][N]
//   gz = gy act'(z);  gx = gz W;  gW = gz^T x;  gb = sum_m gz;  gr = gy
//
// All three products are out[m][n] = sum_k Q(m, k) P(n, k).  An operand lies in memory with k contiguous (x and W of the forward
// product, gz of gx) or with its rows contiguous (W of gx, both operands of gW).  Either is staged into LDS as it lies, 16 bytes a lane
// straight from memory, and read from there as the matrix instructions want it: 16 bytes of one row, or by transposing reads.
// The matrix instruction takes P as its first operand: a lane then holds four consecutive n of one row m, which it can store together.
// Products of 32-bit tensors run on the fp32 matrix instructions; sums are held in 32 bits for all types.
#include "act.h"
#include "common.h"
#include "sed_hip.h"

SED_OBJECT_FLAGS(linear)

namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 half4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));
typedef short short4t __attribute__((__vector_size__(4 * sizeof(short))));
typedef short short8t __attribute__((ext_vector_type(8)));
typedef unsigned uint4v __attribute__((ext_vector_type(4)));

constexpr unsigned OUTSIDE = 0x80000000u;          // a byte offset behind every descriptor: such a lane receives zeros

struct Epilogue {
    const void* bias;                              // nullable, [N]
    const void* res;                               // nullable, [M][N]
    void* y;                                       // [M][N]
    void* z;                                       // nullable: what the backward pass needs of z, [M][ldz]
    long ldz;
    int btype, act, wide, bwide;                   // wide: y and res can be accessed 16 bytes at a time; bwide: the bias too
};

__device__ __forceinline__ float load_typed(const void* p, int type, long i) {
    if (type == SED_F32) return reinterpret_cast<const float*>(p)[i];
    if (type == SED_F16) return (float)reinterpret_cast<const _Float16*>(p)[i];
    return (float)reinterpret_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void store_typed(void* p, int type, long i, float v) {
    if (type == SED_F32) reinterpret_cast<float*>(p)[i] = v;
    else if (type == SED_F16) reinterpret_cast<_Float16*>(p)[i] = (_Float16)v;
    else reinterpret_cast<__bf16*>(p)[i] = (__bf16)v;
}

// What is kept of z for the backward pass, which reads nothing but act'(z) from it: z in 32 bits, whatever the tensors' type.  (A z of
// 16 bits puts |act''(z) z| 2^-12 into a float16 gradient, as much as its own rounding, and as much into a bias gradient of 32 bits.)
// ReLU keeps 1 or 0, in 16 bits beside 16-bit tensors; a NaN counts as on, so that its gradient passes as in torch.
template <typename T> struct Mask { typedef _Float16 type; };
template <> struct Mask<float> { typedef float type; };
template <typename T, int ACT> struct Kept { typedef float type; };
template <typename T> struct Kept<T, SED_ACT_RELU> { typedef typename Mask<T>::type type; };
__device__ __forceinline__ float act_of(float z, int act) {
    switch (act) {
        case SED_ACT_RELU: return sed_act<1>(z);
        case SED_ACT_SILU: return sed_act<2>(z);
        case SED_ACT_GELU: return sed_act<3>(z);
    }
    return z;
}

template <typename T> struct Type { static constexpr int code = SED_F32; };
template <> struct Type<_Float16> { static constexpr int code = SED_F16; };
template <> struct Type<__bf16> { static constexpr int code = SED_BF16; };
template <typename T, int V> struct Wide { typedef T type __attribute__((ext_vector_type(V))); };
constexpr int RUNTIME = -1;                        // an activation that is not known to the compiler

// V consecutive columns of row m, n a multiple of V: the residual, and everything behind it (v = z - bias)
template <typename T, int V> __device__ __forceinline__ void load_residual(const Epilogue& e, long m, int n, int N, float (&r)[V]) {
    const T* const at = reinterpret_cast<const T*>(e.res) + m * N + n;
    if (!e.res) {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = 0.f;
    } else if (e.wide) {
        const auto q = *reinterpret_cast<const typename Wide<T, V>::type*>(at);
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = (float)q[j];
    } else {
#pragma unroll
        for (int j = 0; j < V; ++j) r[j] = n + j < N ? (float)at[j] : 0.f;
    }
}
template <typename T, int V> __device__ __forceinline__ void load_bias(const Epilogue& e, int n, int N, float (&b)[V]) {
    if (!e.bias) {
#pragma unroll
        for (int r = 0; r < V; ++r) b[r] = 0.f;
    } else if (e.bwide) {                          // of type T
        const auto q = *reinterpret_cast<const typename Wide<T, V>::type*>(reinterpret_cast<const T*>(e.bias) + n);
#pragma unroll
        for (int r = 0; r < V; ++r) b[r] = (float)q[r];
    } else {
#pragma unroll
        for (int r = 0; r < V; ++r) b[r] = n + r < N ? load_typed(e.bias, e.btype, n + r) : 0.f;
    }
}
template <typename T, int V, int ACT> __device__ __forceinline__ void finish(const Epilogue& e, long m, int n, int N, float (&v)[V], const float (&bias)[V], const float (&res)[V]) {
#pragma unroll
    for (int r = 0; r < V; ++r) v[r] += bias[r];
    if (e.z) {                                     // ldz is a multiple of V
        if ((ACT == RUNTIME ? e.act : ACT) == SED_ACT_RELU) {
            typedef typename Mask<T>::type Z;
            typename Wide<Z, V>::type k;
#pragma unroll
            for (int r = 0; r < V; ++r) k[r] = (Z)(v[r] <= 0.f ? 0.f : 1.f);
            *reinterpret_cast<typename Wide<Z, V>::type*>(reinterpret_cast<Z*>(e.z) + m * e.ldz + n) = k;
        } else {
            float* const z = reinterpret_cast<float*>(e.z) + m * e.ldz + n;
#pragma unroll
            for (int r = 0; r < V; r += 4) *reinterpret_cast<floatx4*>(z + r) = floatx4{v[r], v[r + 1], v[r + 2], v[r + 3]};
        }
    }
#pragma unroll
    for (int r = 0; r < V; ++r) v[r] = (ACT == RUNTIME ? act_of(v[r], e.act) : sed_act<ACT>(v[r])) + res[r];
    T* const y = reinterpret_cast<T*>(e.y) + m * N + n;
    if (e.wide) {
        typename Wide<T, V>::type o;
#pragma unroll
        for (int r = 0; r < V; ++r) o[r] = (T)v[r];
        *reinterpret_cast<typename Wide<T, V>::type*>(y) = o;
    } else {
#pragma unroll
        for (int r = 0; r < V; ++r)
            if (n + r < N) y[r] = (T)v[r];
    }
}

// One number as the sum of two of a 16-bit type: what is lost is 2^-18 of it in bfloat16, 2^-24 of it or 2^-36 in float16, which holds half of it
// and the small part times 2^11.  An infinity or NaN is in the large part alone.
template <typename T> struct Split { static constexpr float UNIT = 1.f, LOW = 1.f; };
template <> struct Split<__bf16> { static constexpr float UNIT = 1.f, LOW = 1.f; };
template <> struct Split<_Float16> { static constexpr float UNIT = 0.5f, LOW = 0x1p-11f; };
template <typename T> __device__ __forceinline__ void split(float f, T& large, T& small) {
    f *= Split<T>::UNIT;
    large = (T)f;
    const float rest = f - (float)large;
    small = rest - rest == 0.f ? (T)(rest * (1.f / Split<T>::LOW)) : (T)0.f;
}
// SiLU and GELU beside 16-bit tensors: their gz has more bits than the tensors
bool in_parts(int esize, int act) { return esize == 2 && (act == SED_ACT_SILU || act == SED_ACT_GELU); }

// ---- 16 bytes of k of every row: one instruction in 16 bits, four in 32 (they take the k of a lane in any order, as long as P and Q agree)
template <typename T> struct Frag;
template <> struct Frag<_Float16> { typedef half8 type; };
template <> struct Frag<__bf16> { typedef bf8 type; };
template <> struct Frag<float> { typedef floatx4 type; };
// 16 rows, 64 bytes of k
__device__ __forceinline__ floatx4 mma(half8 p, half8 q, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(p, q, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mma(bf8 p, bf8 q, floatx4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(p, q, c, 0, 0, 0); }
__device__ __forceinline__ floatx4 mma(floatx4 p, floatx4 q, floatx4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(p[j], q[j], c, 0, 0, 0);
    return c;
}
// 32 rows, 32 bytes of k
__device__ __forceinline__ floatx16 mma(half8 p, half8 q, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(p, q, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 mma(bf8 p, bf8 q, floatx16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(p, q, c, 0, 0, 0); }
__device__ __forceinline__ floatx16 mma(floatx4 p, floatx4 q, floatx16 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(p[j], q[j], c, 0, 0, 0);
    return c;
}

// ---------------------------------------------------------------------------------------------------------------- tiles
// A step takes 128 bytes of k: 64 elements in 16 bits, 32 in 32.  One operand's tile of R rows is R * 128 bytes.
//   k contiguous: [R][128 bytes];  rows contiguous: [k][R elements];  16-byte piece c of a line lies at place c ^ swizzle(line), so that
//   the lanes that are served together lie in different banks.
// The backward products of 16-bit tensors behind a SiLU or GELU take gz as the sum of two numbers of the tensors' type, the rounding of gz and
// what it leaves: gx and gW then carry their own rounding only (gz rounded once put as much again into them, and in float16 lost what is
// below 6e-8).  k runs over the small parts first and over the large ones behind them, 0 .. K and half .. half + K, half the next
// multiple of the step.  float16 holds gz / 2, which cannot overflow, and the small part times 2^11, which does not underflow: the sums are
// multiplied by 2^-11 between the parts and by 2 at the end (the float16 kernels of edge 256 spill there, outside the
// loop).  It doubles the two products: forward and backward of 32000 x 2048 x 2048 bf16 take 1302 us, for 848 with gz and z in 16
// bits, of 4000 x 512 x 2048 125 for 116; the error against 64 bits is 1.7e-3 for 2.4e-3, that of the output's rounding.
struct Operand {
    const void* base;
    long ld;                                       // elements from one line to the next
    int rows;                                      // rows (m or n)
    long part;                                     // elements from the small parts to the large ones; 0: the same for both
};
constexpr long ONE_PART = 1L << 62;                // a `half` that k does not reach
struct GemmP {
    Operand p, q;
    int M, N;
    long K;
    long half, end;                                // first k of the second part, end of the last one
    long kslice;                                   // k of one slice, a multiple of the step
    int tm, tn;                                    // tiles
    float* part;                                   // [slices][M][ldp] where the product is cut along k
    long ldp;
    Epilogue e;
};

// Row i = 8a + 4h + b of a fragment of 32 rows comes out in register 4a + b of the lanes of half h.  In 16 bits the rows of P are taken in
// the order 16 (a / 2) + 8h + 4 (a % 2) + b, so that a lane's results are runs of eight consecutive n: 16 bytes to store.
template <typename T, int R, bool ROWS, int THREADS, bool RUNS> struct Stage {
    static constexpr int E = 16 / sizeof(T), STEP = 128 / sizeof(T), PIECES = R * 8, PER = PIECES / THREADS;
    static constexpr int LINE = ROWS ? R / E : 8;            // pieces in a line
    static_assert(PIECES % THREADS == 0 && THREADS % LINE == 0 && (ROWS || THREADS / LINE % 16 == 0), "a lane's pieces repeat the swizzle");
    __device__ __forceinline__ static int swizzle(int line) {
        if (!ROWS) return RUNS ? (line & 3) | (line >> 1 & 4) : line & 7;
        return (sizeof(T) == 2 ? 4 * (line & 3) : 8 * (line >> 2 & 1)) & (LINE - 1);
    }
    __device__ __forceinline__ static int line_of(int i) { return i * (THREADS / LINE) + threadIdx.x / LINE; }
    __device__ __forceinline__ static int piece_of(int i) { return (threadIdx.x % LINE) ^ swizzle(line_of(i)); }
    // byte offset of this lane's i-th piece from the tile's first element, OUTSIDE where its row does not exist
    __device__ __forceinline__ static void offsets(const Operand& o, int row0, unsigned (&off)[PER]) {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const bool ok = row0 + (ROWS ? piece_of(i) * E : line_of(i)) < o.rows;
            off[i] = ok ? (unsigned)(line_of(i) * o.ld * (long)sizeof(T)) + piece_of(i) * 16 : OUTSIDE;
        }
    }
    // where the step that begins at k lies, and how much of it: what is behind K lies outside and comes as zeros -- all of a step
    // behind `stop`, the lines behind K, or, where the last step of a part ends inside the lines, the pieces that are taken out of `off`
    // until the next part begins
    template <bool PARTS> __device__ __forceinline__ static uint4v descriptor(const Operand& o, int row0, long k, long stop, long K, long half, unsigned (&off)[PER]) {
        const bool second = PARTS && k >= half;
        const long in = second ? k - half : k;
        const T* const base = reinterpret_cast<const T*>(o.base) + (second ? o.part : 0);
        const unsigned long at = reinterpret_cast<unsigned long>(base + (ROWS ? in * o.ld + row0 : row0 * o.ld + in));
        const int left = k < stop ? (int)min(K - in, (long)STEP) : 0;
        if (PARTS && !ROWS && k == half) offsets(o, row0, off);
        if (!ROWS && left > 0 && left < STEP)
#pragma unroll
            for (int i = 0; i < PER; ++i) off[i] = piece_of(0) * E < left ? off[i] : OUTSIDE;
        const unsigned size = ROWS ? (unsigned)(left * o.ld * (long)sizeof(T)) : (left > 0 ? 0x7fffffffu : 0u);
        return {(unsigned)at, (unsigned)(at >> 32) & 0xffffu, size, 0x00020000u};
    }
    // The i-th request of a step into the slot of LDS at `lds`.  Written as assembly: it has no register to write, and the compiler, which
    // cannot tell the slots apart, would wait for it at the next transposing read.  The kernel waits in arrived().  (M0 is the
    // compiler's, but for nothing that this file uses.)
    __device__ __forceinline__ static void request(uint4v descriptor, unsigned off, unsigned lds, int i) {
        asm volatile("s_add_u32 m0, %2, %3\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(descriptor), "s"(lds), "n"(i * THREADS * 16) : "memory", "scc");
    }
    // 32 rows from `row` on, the kk-th quarter of the step's k
    __device__ __forceinline__ static typename Frag<T>::type frag(const unsigned char* lds, int row, int kk) {
        typedef typename Frag<T>::type Fr;
        const int lane = threadIdx.x & 63, i = lane & 31, half = lane >> 5;
        if constexpr (!ROWS) {
            const int r = row + (RUNS ? (i & 16) | (i & 4) << 1 | (i & 8) >> 1 | (i & 3) : i);
            return *reinterpret_cast<const Fr*>(lds + r * 128 + (((kk * 2 + half) ^ swizzle(r)) << 4));
        } else if constexpr (sizeof(T) == 2) {
            // a transposing read takes 8-byte pieces of four lines from 16 lanes and gives each lane one column of them
            const int k = kk * 16 + 8 * half + (i >> 2 & 3), j = i & 3, c = row + (i & 16) + (RUNS ? 8 * (j & 1) + 4 * (j >> 1) : 4 * j);
            const unsigned char* const at = lds + k * (R * 2) + (((c >> 3) ^ swizzle(k)) << 4) + (c & 7) * 2;
            typedef __attribute__((address_space(3))) short4t* L;
            const short4t a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L)(at)), b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((L)(at + 4 * (R * 2)));
            return __builtin_bit_cast(Fr, short8t{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]});
        } else {
            Fr f;
            const int c = row + i;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int k = kk * 8 + 4 * half + j;
                f[j] = *reinterpret_cast<const float*>(lds + k * (R * 4) + (((c >> 2) ^ swizzle(k)) << 4) + (c & 3) * 4);
            }
            return f;
        }
    }
};

__device__ __forceinline__ int xcd_spread(int bid, int nblk) {       // neighbours in the result are on one XCD and share its L2
    const int q = nblk >> 3, r = nblk & 7, xcd = bid & 7;
    return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (bid >> 3);
}

// all but the last LATER requests of every wave have been served, and its LDS reads are done
template <int LATER> __device__ __forceinline__ void arrived() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LATER) : "memory");
    __syncthreads();
}

// A step is taken in four quarters with two sets of fragments: while the instructions of one quarter run, the next quarter's fragments
// are read.  In the last quarter every wave holds the rest of the step in registers.
// LDS is a ring of five slots of one operand's step each: P(t), Q(t), P(t+1), Q(t+1) and the one that P(t+2) goes to during the first
// three quarters of step t; Q(t+2) goes to P(t)'s slot in the last one, behind a barrier.  The requests of a step are so spread over
// all of it (a wave that issues sixteen at once waits for the address unit: 57 % of the matrix rate against 72 %), and have at least
// three quarters to arrive.  Steps behind the end are requested and read like any other, as zeros: the loop has no other branch.
// `bid` of `blocks` workgroups; lds: 5 slots.
template <typename T, bool PROWS, bool QROWS, int BM, int BN, int WM, int WN, bool CUT, int ACT, bool PARTS>
__device__ __forceinline__ void gemm_tile(const GemmP& a, int bid, int blocks, unsigned char* lds) {
    constexpr int THREADS = 64 * WM * WN, MI = BM / WM / 32, NI = BN / WN / 32, V = 16 / sizeof(T);
    typedef Stage<T, BN, PROWS, THREADS, V == 8> SP;
    typedef Stage<T, BM, QROWS, THREADS, false> SQ;
    typedef typename Frag<T>::type Fr;
    static_assert(BM == BN, "one size of slot");
    constexpr int SLOT = BM * 128, FRAGS = NI + MI, MFMAS = MI * NI;
    const int tiles = a.tm * a.tn, id = xcd_spread(bid, blocks);
    const int slice = id / tiles, tile = id % tiles;
    // tiles in groups of eight rows of tiles: the 32 that an XCD works on share 8 + 4 operand tiles, not 32 + 1
    const int group = tile / (8 * a.tn), gm = min(8, a.tm - 8 * group), in = tile - group * 8 * a.tn;
    const int m0 = (8 * group + in % gm) * BM, n0 = in / gm * BN;
    static_assert(!PARTS || (PROWS && sizeof(T) == 2), "the backward products of 16-bit tensors");
    const long end = PARTS ? a.end : a.K, k0 = CUT ? slice * a.kslice : 0, k1 = CUT ? min(end, k0 + a.kslice) : end;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int wm = (wave % WM) * (BM / WM), wn = (wave / WM) * (BN / WN);
    unsigned poff[SP::PER], qoff[SQ::PER];
    SP::offsets(a.p, n0, poff);
    SQ::offsets(a.q, m0, qoff);
    // For the epilogue a wave passes 32 rows of its results at a time through LDS: a lane then has V consecutive n of row
    // 32 i + PASS it + lane / LINE, and its neighbours have the rest of the line.  (Stored from where the instructions leave them, 32 bytes
    // a line, a bf16 product of 32000 x 2048 x 2048 with silu, residual and kept z took 402 us, now 335.)
    constexpr int W = BN / WN, LINE = W / V, PASS = 64 / LINE, PASSES = 32 / PASS, PITCH = 4 * W + 16;
    static_assert(4 * 32 * PITCH <= 5 * SLOT, "the waves' rows fit the ring");
    const int n = n0 + wn + lane % LINE * V;
    auto row = [&](int i, int it) { return m0 + wm + 32 * i + PASS * it + lane / LINE; };
    // All of a lane's residual is requested at once, and from the first where registers are left for it (edges 64 and 128): read run by run
    // at the end, its latency was a third of the time of a product with K = 512.
    typedef typename Wide<T, V>::type Run;
    constexpr bool FORWARD = !PROWS && !CUT, EARLY = BM <= 128;          // only the forward product has an epilogue
    Run res[FORWARD ? MI : 1][FORWARD ? PASSES : 1];
    auto fetch = [&]() {
        if (FORWARD && a.e.res && a.e.wide && n < a.N)
#pragma unroll
            for (int i = 0; i < MI; ++i)
#pragma unroll
                for (int it = 0; it < PASSES; ++it)
                    if (row(i, it) < a.M) res[i][it] = *reinterpret_cast<const Run*>(reinterpret_cast<const T*>(a.e.res) + (long)row(i, it) * a.N + n);
    };
    if (EARLY) fetch();
    floatx16 acc[MI][NI] = {};
    Fr p[2][NI], q[2][MI];
    const unsigned lds0 = (unsigned)(size_t)(__attribute__((address_space(3))) unsigned char*)lds + wave * 1024;
    auto ask_p = [&](uint4v d, int slot, int o) { SP::request(d, poff[o], lds0 + slot * SLOT, o); };
    auto ask_q = [&](uint4v d, int slot, int o) { SQ::request(d, qoff[o], lds0 + slot * SLOT, o); };
    auto read = [&](int ps, int qs, int kk, int set, int o) {         // one of the fragments of a quarter
        if (o < NI) p[set][o] = SP::frag(lds + ps * SLOT, wn + 32 * o, kk);
        else q[set][o - NI] = SQ::frag(lds + qs * SLOT, wm + 32 * (o - NI), kk);
    };
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        const uint4v dp = SP::template descriptor<PARTS>(a.p, n0, k0 + t * SP::STEP, k1, a.K, a.half, poff);
        const uint4v dq = SQ::template descriptor<PARTS>(a.q, m0, k0 + t * SP::STEP, k1, a.K, a.half, qoff);
#pragma unroll
        for (int o = 0; o < SP::PER; ++o) ask_p(dp, 2 * t, o);
#pragma unroll
        for (int o = 0; o < SQ::PER; ++o) ask_q(dq, 2 * t + 1, o);
    }
    arrived<SP::PER + SQ::PER>();
#pragma unroll
    for (int o = 0; o < FRAGS; ++o) read(0, 1, 0, 0, o);
    int ps = 0;                                    // P(t)'s slot; the next ones follow around the ring
    auto ring = [&](int i) { return ps + i < 5 ? ps + i : ps + i - 5; };
    auto step = [&](long k) {
        const uint4v dp = SP::template descriptor<PARTS>(a.p, n0, k + 2 * SP::STEP, k1, a.K, a.half, poff);
        const uint4v dq = SQ::template descriptor<PARTS>(a.q, m0, k + 2 * SP::STEP, k1, a.K, a.half, qoff);
        const int qs = ring(1), pn = ring(2), qn = ring(3), spare = ring(4);
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
            if (kk == 3) arrived<SP::PER>();       // the step's fragments are in registers everywhere, the next step is in LDS
            const int first = SP::PER * kk / 3, asked = kk == 3 ? SQ::PER : SP::PER * (kk + 1) / 3 - first, others = FRAGS + asked;
            int o = 0;
#pragma unroll
            for (int f = 0; f < MFMAS; ++f) {
                acc[f / NI][f % NI] = mma(p[kk & 1][f % NI], q[kk & 1][f / NI], acc[f / NI][f % NI]);
#pragma unroll
                for (; o < (f < MFMAS / 2 ? FRAGS * 2 * (f + 1) / MFMAS : FRAGS + (others - FRAGS) * (f + 1 - MFMAS / 2) / (MFMAS - MFMAS / 2)); ++o) {
                    if (o < FRAGS) read(kk == 3 ? pn : ps, kk == 3 ? qn : qs, (kk + 1) & 3, (kk + 1) & 1, o);
                    else if (kk == 3) ask_q(dq, ps, o - FRAGS);
                    else ask_p(dp, spare, first + o - FRAGS);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        ps = pn;
    };
    if constexpr (PARTS) {
        long k = k0;
        do {
            const long stop = min(k1, k < a.half ? a.half : k1);
            for (; k < stop; k += SP::STEP) step(k);
            if constexpr (Split<T>::LOW != 1.f)
                if (k <= a.half)
#pragma unroll
                    for (int f = 0; f < MFMAS; ++f) acc[f / NI][f % NI] *= Split<T>::LOW;
        } while (k < k1);
    } else {
        for (long k = k0; k < k1; k += SP::STEP) step(k);
    }
    arrived<0>();                                  // no request is in flight when the workgroup ends
    if (!EARLY) fetch();
    float bias[V] = {};
    if (FORWARD && n < a.N) load_bias<T, V>(a.e, n, a.N, bias);
    // 16-byte piece c of a line lies at place c ^ (c / 8 % 2): two neighbours' pieces, as a lane reads them in 16 bits, lie in other banks
    unsigned char* const mine = lds + wave * 32 * PITCH;
    auto place = [](int c) { return (c ^ (c >> 3 & 1)) * 16; };
#pragma unroll
    for (int i = 0; i < MI; ++i) {
#pragma unroll
        for (int j = 0; j < NI; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {          // four registers are four consecutive n
                const int half = lane >> 5, c = 8 * j + (V == 8 ? 4 * (r >> 1) + 2 * half + (r & 1) : 2 * r + half);
                *reinterpret_cast<floatx4*>(mine + (lane & 31) * PITCH + place(c)) =
                    floatx4{acc[i][j][4 * r], acc[i][j][4 * r + 1], acc[i][j][4 * r + 2], acc[i][j][4 * r + 3]};
            }
#pragma unroll
        for (int it = 0; it < PASSES; ++it) {
            float v[V];
#pragma unroll
            for (int h = 0; h < V / 4; ++h) {
                const floatx4 q = *reinterpret_cast<const floatx4*>(mine + (PASS * it + lane / LINE) * PITCH + place(lane % LINE * (V / 4) + h));
#pragma unroll
                for (int j = 0; j < 4; ++j) v[4 * h + j] = PARTS ? q[j] * (1.f / Split<T>::UNIT) : q[j];
            }
            const int m = row(i, it);
            if (m >= a.M || n >= a.N) continue;
            if (CUT) {
                float* const to = a.part + ((long)slice * a.M + m) * a.ldp + n;              // ldp is a multiple of 8
#pragma unroll
                for (int h = 0; h < V; h += 4) *reinterpret_cast<floatx4*>(to + h) = floatx4{v[h], v[h + 1], v[h + 2], v[h + 3]};
            } else {
                float r[V] = {};
                if (FORWARD && a.e.res) {
                    if (!a.e.wide) load_residual<T, V>(a.e, m, n, a.N, r);
                    else
#pragma unroll
                        for (int j = 0; j < V; ++j) r[j] = (float)res[FORWARD ? i : 0][FORWARD ? it : 0][j];
                }
                finish<T, V, ACT>(a.e, m, n, a.N, v, bias, r);
            }
        }
    }
}

template <typename T, bool PROWS, bool QROWS, int BM, int BN, int WM, int WN, bool CUT, int ACT, bool PARTS>
__global__ __launch_bounds__(64 * WM * WN, BM * BN > 128 * 128 ? 1 : 2) void gemm_kernel(GemmP a) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[5 * BM * 128];
    gemm_tile<T, PROWS, QROWS, BM, BN, WM, WN, CUT, ACT, PARTS>(a, blockIdx.x, gridDim.x, lds);
}
// gb [N] of `type` = the column sums of sums [chunks][ld]: 16 columns x ROWS lanes, a power of two
struct ColumnsP {
    const float* sums;
    long chunks;
    int ld, N;
    void* gb;
    int type, blocks;
};
template <int ROWS> __device__ __forceinline__ void column_sums(const ColumnsP& p, int bid, float* red) {       // red: ROWS * 17
    const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, c = bid * 16 + lane;
    float v = 0.f;
    if (c < p.N) {
#pragma unroll 4
        for (long i = row; i < p.chunks; i += ROWS) v += p.sums[i * p.ld + c];
    }
    red[row * 17 + lane] = v;
    __syncthreads();
    for (int s = ROWS / 2; s > 0; s >>= 1) {
        if (row < s) red[row * 17 + lane] += red[(row + s) * 17 + lane];
        __syncthreads();
    }
    if (row == 0 && c < p.N) store_typed(p.gb, p.type, c, red[lane]);
}

// both products of a backward pass, and the bias gradient's last sums, in one launch, where both are cut into tiles of 64: the first
// c.blocks workgroups take the sums, the next `first` gz^T x, whose tiles are the longer ones where there are more rows than columns,
// the others gz W.  Forward and backward of 4000 x 512 x 512 bf16 take 27.3 us so and 35.7 in two launches (with gelu, gz in two
// parts, 42.6 and 49.9), of 4000 x 512 x 2048 58.7 and 76.9 (with gelu gW is cut into tiles of 128, and the launches are two: 113), of
// 500 x 96 x 136 fp32 16.7 and 23.1.
template <typename T, bool CUTW, bool CUTX, bool PARTS> __global__ __launch_bounds__(256, 2) void gemm_pair_kernel(GemmP w, GemmP x, int first, ColumnsP c) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[5 * 64 * 128];
    const int bid = (int)blockIdx.x - c.blocks;
    if (bid < 0) column_sums<16>(c, blockIdx.x, reinterpret_cast<float*>(lds));
    else if (bid < first) gemm_tile<T, true, true, 64, 64, 2, 2, CUTW, 0, PARTS>(w, bid, first, lds);
    else gemm_tile<T, true, false, 64, 64, 2, 2, CUTX, 0, PARTS>(x, bid - first, gridDim.x - c.blocks - first, lds);
}

// the slices of a cut product, added in order, and the epilogue
template <typename T> __global__ __launch_bounds__(256) void join_kernel(const float* part, int slices, int M, int N, long ldp, Epilogue e) {
    const long quads = ldp / 4, total = quads * M;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)gridDim.x * 256) {
        const long m = i / quads;
        const int n = (int)(i % quads) * 4;
        if (n >= N) continue;
        floatx4 s = *reinterpret_cast<const floatx4*>(part + m * ldp + n);
        for (int k = 1; k < slices; ++k) s += *reinterpret_cast<const floatx4*>(part + ((long)k * M + m) * ldp + n);
        float v[4] = {s[0], s[1], s[2], s[3]}, b[4], r[4];
        load_bias<T, 4>(e, n, N, b);
        load_residual<T, 4>(e, m, n, N, r);
        finish<T, 4, RUNTIME>(e, m, n, N, v, b, r);
    }
}

// ---------------------------------------------------------------------------------------------------------------- few rows
// Up to 16 * MT rows of x: the product is a pass over W.  A workgroup owns 16 rows of W, its waves split k in runs of U times 64 bytes, all of
// them requested at once; the waves' sums are added through LDS.  No alignment is asked of x and W.  Rows that do not exist are
// read as the first one: they only reach results that are not stored.
template <typename T> __device__ __forceinline__ typename Frag<T>::type piece(const T* row, long k, long K) {
    constexpr int E = 16 / sizeof(T);
    typename Frag<T>::type f;
#pragma unroll
    for (int j = 0; j < E; ++j) f[j] = k + j < K ? row[k + j] : (T)0.f;
    return f;
}
template <typename T, int MT, int U> __global__ __launch_bounds__(1024) void rows_kernel(const T* x, const T* w, int M, int N, long K, Epilogue e) {
    constexpr int E = 16 / sizeof(T), RUN = 4 * E * U;
    __shared__ __attribute__((aligned(16))) floatx4 sums[16][MT][64];
    const int waves = blockDim.x >> 6, wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
    const int n0 = blockIdx.x * 16;
    const T* const wr = w + (long)(n0 + l < N ? n0 + l : 0) * K;
    const T* xr[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xr[i] = x + (long)(i * 16 + l < M ? i * 16 + l : 0) * K;
    floatx4 acc[MT] = {};
    typename Frag<T>::type p[U], q[U][MT];
    for (long k = (long)wave * RUN; k < K; k += (long)waves * RUN) {
        if (k + RUN <= K) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                __builtin_memcpy(&p[u], wr + k + (u * 4 + g) * E, 16);
#pragma unroll
                for (int i = 0; i < MT; ++i) __builtin_memcpy(&q[u][i], xr[i] + k + (u * 4 + g) * E, 16);
            }
        } else {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                p[u] = piece<T>(wr, k + (u * 4 + g) * E, K);
#pragma unroll
                for (int i = 0; i < MT; ++i) q[u][i] = piece<T>(xr[i], k + (u * 4 + g) * E, K);
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < MT; ++i) acc[i] = mma(p[u], q[u][i], acc[i]);
    }
#pragma unroll
    for (int i = 0; i < MT; ++i) sums[wave][i][lane] = acc[i];
    __syncthreads();
    for (int i = wave; i < MT; i += waves) {
        floatx4 v = sums[0][i][lane];
        for (int s = 1; s < waves; ++s) v += sums[s][i][lane];
        const int m = i * 16 + l, n = n0 + 4 * g;
        if (m < M && n < N) {
            float f[4] = {v[0], v[1], v[2], v[3]}, b[4], r[4];
            load_bias<T, 4>(e, n, N, b);
            load_residual<T, 4>(e, m, n, N, r);
            finish<T, 4, RUNTIME>(e, m, n, N, f, b, r);
        }
    }
}
template <typename T, int U> void launch_rows(const T* x, const T* w, int M, int N, long K, const Epilogue& e, hipStream_t stream) {
    const long runs = (K * (long)sizeof(T) + 64 * U - 1) / (64 * U);
    const dim3 grid((unsigned)sed_cdiv(N, 16)), block((unsigned)(64 * (runs < 16 ? runs : 16)));
    if (M <= 16) hipLaunchKernelGGL((rows_kernel<T, 1, U>), grid, block, 0, stream, x, w, M, N, K, e);
    else if (M <= 32) hipLaunchKernelGGL((rows_kernel<T, 2, U>), grid, block, 0, stream, x, w, M, N, K, e);
    else hipLaunchKernelGGL((rows_kernel<T, 4, 2>), grid, block, 0, stream, x, w, M, N, K, e);          // few_rows(): lines of up to 1 KB, U = 2
}

// ---------------------------------------------------------------------------------------------------------------- passes around them
// copies of up to two [R][C] with lines of ld elements, zeros behind the C-th: operands whose lines do not begin at multiples of 16 bytes
struct PadP {
    const void* src[2];
    void* dst[2];
    long R[2];
    int C, ld, blocks;                             // blocks: workgroups that share them, 0 where there is nothing to copy
};
template <typename T> __device__ __forceinline__ void pad_lines(const PadP& p) {
    constexpr int E = 16 / sizeof(T);
    const int per = p.ld / E;
    const long first = p.R[0] * per, total = first + p.R[1] * per;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long)p.blocks * 256) {
        const int which = i >= first;
        const long r = (i - which * first) / per;
        const int c = (int)(i % per) * E;
        const T* const src = reinterpret_cast<const T*>(p.src[which]) + r * p.C + c;
        T v[E];
        if (c + E <= p.C) __builtin_memcpy(v, src, 16);
        else
#pragma unroll
            for (int j = 0; j < E; ++j) v[j] = c + j < p.C ? src[j] : (T)0.f;
        __builtin_memcpy(reinterpret_cast<T*>(p.dst[which]) + r * p.ld + c, v, 16);
    }
}
template <typename T> __global__ __launch_bounds__(256) void pad_kernel(PadP p) { pad_lines<T>(p); }

// gz [M][ld] = gy act'(z) (null: only the sums), its small parts [M][ld] in front of it where it is in parts, and per chunk of rows the column
// sums of gz in 32 bits, before it is rounded.
// A thread owns E columns (16 bytes) of every RT-th row of a chunk.  The first pad.blocks workgroups copy the operands that need it.
struct GradP {
    const void* gy;
    const void* z;
    void* gz;
    float* sums;                                   // nullable, [chunks][ld]
    void* gb;                                      // where there is one chunk, its sums are the result, of btype
    int btype;
    long M, rows;
    int N, ld, CT, RT, tiles, act;
    PadP pad;
};
template <typename T, int ACT, bool WHOLE> __global__ __launch_bounds__(256) void act_grad_kernel(GradP p) {       // WHOLE: N is a multiple of E
    constexpr int E = 16 / sizeof(T), U = 4;
    typedef typename Kept<T, ACT>::type Z;
    __shared__ float red[256 * E];
    if ((int)blockIdx.x < p.pad.blocks) { pad_lines<T>(p.pad); return; }
    const unsigned bid = blockIdx.x - p.pad.blocks;
    const int tile = (int)(bid % p.tiles), t = threadIdx.x, col = tile * p.CT + t % p.CT, r = t / p.CT, c = col * E;
    const long chunk = bid / p.tiles, s0 = chunk * p.rows, s1 = min(p.M, s0 + p.rows);
    const T* const gy = reinterpret_cast<const T*>(p.gy) + c;
    const Z* const kept = reinterpret_cast<const Z*>(p.z) + c;
    constexpr bool PARTS = sizeof(T) == 2 && (ACT == SED_ACT_SILU || ACT == SED_ACT_GELU);
    float sum[E] = {};
    if (r < p.RT && c < p.ld)
        for (long s = s0 + r; s < s1; s += U * p.RT) {
            T g[U][E];
            Z z[U][E];
            // rows behind the chunk are read as its last one and left out of the sums
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long at = min(s + u * p.RT, s1 - 1);
                if (WHOLE) __builtin_memcpy(g[u], gy + at * p.N, 16);
                else
#pragma unroll
                    for (int j = 0; j < E; ++j) g[u][j] = c + j < p.N ? gy[at * p.N + j] : (T)0.f;
                if (ACT) __builtin_memcpy(z[u], kept + at * p.ld, sizeof(z[u]));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const long at = s + u * p.RT;
                if (at >= s1) continue;
                T small[E];
#pragma unroll
                for (int j = 0; j < E; ++j) {
                    float f = (float)g[u][j];
                    if (ACT == SED_ACT_RELU) f = (float)z[u][j] != 0.f ? f : 0.f;             // kept as 1 or 0
                    else if (ACT) f *= sed_act_grad<ACT>((float)z[u][j]);
                    if (!WHOLE && c + j >= p.N) f = 0.f;   // z is not written there
                    sum[j] += f;
                    if constexpr (PARTS) split<T>(f, g[u][j], small[j]);
                    else g[u][j] = (T)f;
                }
                if (!p.gz) continue;
                if constexpr (PARTS) __builtin_memcpy(reinterpret_cast<T*>(p.gz) + at * p.ld + c, small, 16);
                __builtin_memcpy(reinterpret_cast<T*>(p.gz) + ((PARTS ? p.M : 0) + at) * p.ld + c, g[u], 16);
            }
        }
    if (!p.sums && !p.gb) return;
#pragma unroll
    for (int j = 0; j < E; ++j) red[t * E + j] = sum[j];
    __syncthreads();
    for (int k = t; k < p.CT * E; k += 256) {
        float v = 0.f;
        for (int i = 0; i < p.RT; ++i) v += red[i * p.CT * E + k];
        const int n = tile * p.CT * E + k;
        if (p.gb && n < p.N) store_typed(p.gb, p.btype, n, v);
        else if (p.sums && n < p.ld) p.sums[chunk * p.ld + n] = v;
    }
}
template <typename T, bool WHOLE> void launch_act_grad(const GradP& p, unsigned blocks, hipStream_t stream) {
    switch (p.act) {
        case SED_ACT_NONE: hipLaunchKernelGGL((act_grad_kernel<T, 0, WHOLE>), dim3(blocks), dim3(256), 0, stream, p); break;
        case SED_ACT_RELU: hipLaunchKernelGGL((act_grad_kernel<T, 1, WHOLE>), dim3(blocks), dim3(256), 0, stream, p); break;
        case SED_ACT_SILU: hipLaunchKernelGGL((act_grad_kernel<T, 2, WHOLE>), dim3(blocks), dim3(256), 0, stream, p); break;
        default: hipLaunchKernelGGL((act_grad_kernel<T, 3, WHOLE>), dim3(blocks), dim3(256), 0, stream, p);
    }
}
__global__ __launch_bounds__(1024) void column_sums_kernel(ColumnsP p) {
    __shared__ float red[64 * 17];
    column_sums<64>(p, blockIdx.x, red);
}

// ---------------------------------------------------------------------------------------------------------------- host
int esize_of(int dtype) { return dtype == SED_F32 ? 4 : 2; }
long padded(long n, int esize) { return (n + 16 / esize - 1) / (16 / esize) * (16 / esize); }
long up256(long bytes) { return (bytes + 255) / 256 * 256; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
bool needs_pad(const void* p, long ld, int esize) { return !aligned16(p) || ld % (16 / esize); }

long whole_steps(long k, int esize) { const long step = 128 / esize; return (k + step - 1) / step * step; }
// k of a product whose Q is in two parts, or in one
template <typename T> void set_k(GemmP& a, long K, bool parts) {
    a.K = K;
    a.half = parts ? whole_steps(K, sizeof(T)) : ONE_PART;
    a.end = parts ? 2 * a.half : K;
}

// How a product is cut: tile edge, and slices along k that a second pass adds.  The cut with the least time by what was measured on an
// MI355X: a step of 128 bytes of k takes a tile of 64, 128 or 256 the microseconds below when 1, 2, .. of them share a CU (LDS holds 4, 2
// or 1), a tile costs as much again at its ends, and a cut one passes its 32-bit sums through memory.  E.g. bf16
// (rows, N, K) = (4000, 512, 512) takes 7.6 us with edge 64 and 9.4 with 128, (4000, 2048, 512) 15.0 with 128, 18.9 with 64, 25.2 with 256,
// (4096, 4096, 4096) 117 with 256 and 133 with 128.
struct Plan {
    int edge, tm, tn, slices;
    long kslice, part_bytes, ldp;
};
Plan plan_of(long M, long N, long K, int esize) {
    static const int edges[3] = {64, 128, 256}, room[3] = {4, 2, 1};
    static const float ends[3] = {4.f, 6.f, 16.f};
    static const float step16[3][4] = {{.30f, .45f, .65f, .80f}, {.60f, .95f}, {1.65f}}, step32[2][4] = {{.65f, 1.23f, 1.7f, 2.1f}, {2.0f, 3.9f}};
    const long step = 128 / esize, steps = (K + step - 1) / step;
    Plan best{};
    float least = 0.f;
    for (int e = 0; e < (esize == 2 ? 3 : 2); ++e) {
        const float* const us = esize == 2 ? step16[e] : step32[e];
        const long tm = (M + edges[e] - 1) / edges[e], tn = (N + edges[e] - 1) / edges[e];
        if (tm * tn >= 1L << 24) continue;         // 2^32 threads are more than a launch takes; edge 128 fits every shape that is let in
        for (long s = 1; s <= 64 && (s == 1 || (steps / s >= 4 && tm * tn * s <= 2048)); s *= 2) {
            const long per = (steps + s - 1) / s, slices = (steps + per - 1) / per, on = (tm * tn * slices + 255) / 256;
            float t = (float)(on / room[e]) * (per * us[room[e] - 1] + ends[e]);
            if (on % room[e]) t += per * us[on % room[e] - 1] + ends[e];
            if (slices > 1) t += 6.f + (float)slices * M * N * 8.f / 5e6f;
            if (best.edge && t >= least) continue;
            least = t;
            best.edge = edges[e]; best.tm = (int)tm; best.tn = (int)tn; best.slices = (int)slices; best.kslice = per * step;
        }
    }
    best.ldp = (N + 7) / 8 * 8;
    best.part_bytes = best.slices > 1 ? up256(best.slices * M * best.ldp * 4) : 0;
    return best;
}
// A few rows are a pass over W with 16 of its rows per workgroup, which reads all of x: one row of bf16 (1, 4096, 4096) takes 7.4 us, 16
// rows 10.1, 64 rows 24.7 against 15.2 in tiles; (64, 2048, 512) 5.1 against 5.5, (64, 512, 2048) 13.4 against 8.1.
bool few_rows(long M, long K, int esize) { return M <= 64 && K * esize <= (M <= 16 ? 16384 : M <= 32 ? 4096 : 1024); }

template <typename T, bool PROWS, bool QROWS, int EDGE, bool PARTS> void launch_edge(const GemmP& a, const Plan& q, hipStream_t stream) {
    const dim3 grid((unsigned)((long)q.tm * q.tn * q.slices));
    if (q.slices > 1) { hipLaunchKernelGGL((gemm_kernel<T, PROWS, QROWS, EDGE, EDGE, 2, 2, true, 0, PARTS>), grid, dim3(256), 0, stream, a); return; }
    if constexpr (!PROWS) {                        // only the forward product has an epilogue
        switch (a.e.act) {
            case SED_ACT_RELU: hipLaunchKernelGGL((gemm_kernel<T, PROWS, QROWS, EDGE, EDGE, 2, 2, false, 1, PARTS>), grid, dim3(256), 0, stream, a); return;
            case SED_ACT_SILU: hipLaunchKernelGGL((gemm_kernel<T, PROWS, QROWS, EDGE, EDGE, 2, 2, false, 2, PARTS>), grid, dim3(256), 0, stream, a); return;
            case SED_ACT_GELU: hipLaunchKernelGGL((gemm_kernel<T, PROWS, QROWS, EDGE, EDGE, 2, 2, false, 3, PARTS>), grid, dim3(256), 0, stream, a); return;
        }
    }
    hipLaunchKernelGGL((gemm_kernel<T, PROWS, QROWS, EDGE, EDGE, 2, 2, false, 0, PARTS>), grid, dim3(256), 0, stream, a);
}
template <typename T, bool PROWS, bool QROWS, bool PARTS> void launch_edges(const GemmP& a, const Plan& q, hipStream_t stream) {
    if (q.edge == 64) launch_edge<T, PROWS, QROWS, 64, PARTS>(a, q, stream);
    else if (q.edge == 128 || sizeof(T) == 4) launch_edge<T, PROWS, QROWS, 128, PARTS>(a, q, stream);
    else if constexpr (sizeof(T) == 2) launch_edge<T, PROWS, QROWS, 256, PARTS>(a, q, stream);
}
void place(GemmP& a, const Plan& q, float* part) { a.tm = q.tm; a.tn = q.tn; a.kslice = q.kslice; a.part = part; a.ldp = q.ldp; }
template <typename T> void launch_join(const GemmP& a, const Plan& q, hipStream_t stream) {
    if (q.slices < 2) return;
    const long quads = q.ldp / 4 * a.M, nb = (quads + 255) / 256;
    hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(nb > 8192 ? 8192 : nb)), dim3(256), 0, stream, a.part, q.slices, a.M, a.N, q.ldp, a.e);
}
template <typename T, bool PROWS, bool QROWS> void launch_gemm(GemmP a, const Plan& q, float* part, hipStream_t stream) {
    place(a, q, part);
    if (a.half == ONE_PART) launch_edges<T, PROWS, QROWS, false>(a, q, stream);
    else if constexpr (PROWS && sizeof(T) == 2) launch_edges<T, PROWS, QROWS, true>(a, q, stream);
    launch_join<T>(a, q, stream);
}
bool pairs(const Plan& w, const Plan& x) { return w.edge == 64 && x.edge == 64 && (long)w.tm * w.tn * w.slices + (long)x.tm * x.tn * x.slices < (1L << 24) - (1L << 17); }
template <typename T, bool PARTS> void launch_pair(const GemmP& w, bool cutw, const GemmP& x, bool cutx, int first, const ColumnsP& c, dim3 grid, hipStream_t stream) {
    if (cutw && cutx) hipLaunchKernelGGL((gemm_pair_kernel<T, true, true, PARTS>), grid, dim3(256), 0, stream, w, x, first, c);
    else if (cutw) hipLaunchKernelGGL((gemm_pair_kernel<T, true, false, PARTS>), grid, dim3(256), 0, stream, w, x, first, c);
    else if (cutx) hipLaunchKernelGGL((gemm_pair_kernel<T, false, true, PARTS>), grid, dim3(256), 0, stream, w, x, first, c);
    else hipLaunchKernelGGL((gemm_pair_kernel<T, false, false, PARTS>), grid, dim3(256), 0, stream, w, x, first, c);
}
template <typename T> void launch_pair(GemmP w, const Plan& qw, GemmP x, const Plan& qx, const ColumnsP& c, float* part, hipStream_t stream) {
    place(w, qw, part);
    place(x, qx, part + qw.part_bytes / 4);
    const int first = qw.tm * qw.tn * qw.slices;
    const dim3 grid((unsigned)(c.blocks + first + qx.tm * qx.tn * qx.slices));
    if (w.half == ONE_PART) launch_pair<T, false>(w, qw.slices > 1, x, qx.slices > 1, first, c, grid, stream);
    else if constexpr (sizeof(T) == 2) launch_pair<T, true>(w, qw.slices > 1, x, qx.slices > 1, first, c, grid, stream);
    launch_join<T>(w, qw, stream);
    launch_join<T>(x, qx, stream);
}
// x [M][C] and w [N][C] with lines of a multiple of 16 bytes, those of them that need it: from here on they are what lies in ws
template <typename T> PadP pad_of(const void*& x, long M, bool px, const void*& w, long N, bool pw, long C, char*& ws) {
    PadP p{};
    if (!px && !pw) return p;
    p.C = (int)C; p.ld = (int)padded(C, sizeof(T));
    auto take = [&](int i, const void*& src, long R) {
        p.src[i] = src; p.R[i] = R; p.dst[i] = ws;
        src = ws;
        ws += up256(R * p.ld * (long)sizeof(T));
    };
    int used = 0;
    if (px) take(used++, x, M);
    if (pw) take(used++, w, N);
    const long nb = ((p.R[0] + p.R[1]) * (p.ld * (long)sizeof(T) / 16) + 255) / 256;
    p.blocks = (int)(nb > 16384 ? 16384 : nb);
    return p;
}
template <typename T> void launch_pad(const PadP& p, hipStream_t stream) {
    if (p.blocks) hipLaunchKernelGGL((pad_kernel<T>), dim3((unsigned)p.blocks), dim3(256), 0, stream, p);
}

// rows and columns that 32-bit offsets inside a tile and the tiles of one launch can hold: 2^38 elements of x, W or y at most
bool bad_shape(int dtype, long M, long N, long K, int act) {
    return dtype < 0 || dtype > 2 || M < 1 || N < 1 || K < 1 || M > 0x7fffffffL - 256 || N > 1L << 21 || K > 1L << 21 || act < 0 || act > 3 ||
           (M + 127) / 128 * ((N + 127) / 128) >= 1L << 24 || (M + 127) / 128 * ((K + 127) / 128) >= 1L << 24 ||
           (N + 127) / 128 * ((K + 127) / 128) >= 1L << 24;
}

struct GradCut {
    int CT, RT, tiles;
    long rows, chunks;
};
GradCut grad_cut(long M, long ld, int esize) {
    GradCut c;
    const long cols = ld * esize / 16;
    c.CT = (int)(cols < 256 ? cols : 256);
    c.RT = 256 / c.CT;
    c.tiles = (int)((cols + c.CT - 1) / c.CT);
    const long want = (2048 + c.tiles - 1) / c.tiles;
    long rows = (M + want - 1) / want;
    const long lo = (long)c.RT * 4, hi = (long)c.RT * 64;
    rows = rows < lo ? lo : (rows > hi ? hi : rows);
    if (M <= 4 * lo) rows = M;                              // a few rows in one chunk: a launch less
    c.rows = rows;
    c.chunks = (M + rows - 1) / rows;
    return c;
}

template <typename T>
int linear_fwd(const void* x, const void* w, const void* bias, const void* res, int btype, long M, long N, long K, int act, void* y, void* z,
               char* ws, hipStream_t stream) {
    Epilogue e{bias, res, y, z, padded(N, sizeof(T)), btype, act, 0, 0};
    e.wide = N % (16 / sizeof(T)) == 0 && aligned16(y) && aligned16(res);
    e.bwide = bias && N % (16 / sizeof(T)) == 0 && aligned16(bias) && btype == Type<T>::code;
    if (few_rows(M, K, sizeof(T))) {
        const T *xt = reinterpret_cast<const T*>(x), *wt = reinterpret_cast<const T*>(w);
        // as many waves as there are runs, and longer runs once there are more than sixteen
        if (K * (long)sizeof(T) > 16 * 128) launch_rows<T, 4>(xt, wt, (int)M, (int)N, K, e, stream);
        else launch_rows<T, 2>(xt, wt, (int)M, (int)N, K, e, stream);
        SED_LAUNCH_CHECK();
        return 0;
    }
    const long ld = padded(K, sizeof(T));
    launch_pad<T>(pad_of<T>(x, M, needs_pad(x, K, sizeof(T)), w, N, needs_pad(w, K, sizeof(T)), K, ws), stream);
    GemmP a{};
    a.M = (int)M; a.N = (int)N; a.e = e;
    set_k<T>(a, ld, false);
    a.q = {x, ld, (int)M, 0};
    a.p = {w, ld, (int)N, 0};
    launch_gemm<T, false, false>(a, plan_of(M, N, ld, sizeof(T)), reinterpret_cast<float*>(ws), stream);
    SED_LAUNCH_CHECK();
    return 0;
}

long fwd_ws(const void* x, const void* w, int esize, long M, long N, long K) {
    if (few_rows(M, K, esize)) return 0;
    const long ld = padded(K, esize);
    return (needs_pad(x, K, esize) ? up256(M * ld * esize) : 0) + (needs_pad(w, K, esize) ? up256(N * ld * esize) : 0) + plan_of(M, N, ld, esize).part_bytes;
}

Plan plan_gx(long M, long N, long K, int esize, bool parts) { return plan_of(M, K, parts ? 2 * whole_steps(N, esize) : padded(N, esize), esize); }
Plan plan_gw(long M, long N, long K, int esize, bool parts) { return plan_of(N, K, parts ? 2 * whole_steps(M, esize) : M, esize); }

struct BwdNeeds {
    bool gz, px, pw;
};
BwdNeeds bwd_needs(const void* x, const void* w, const void* gy, int esize, long N, long K, int act, bool gx, bool gw) {
    return {(gx || gw) && (act != SED_ACT_NONE || needs_pad(gy, N, esize)), gw && needs_pad(x, K, esize), gx && needs_pad(w, K, esize)};
}
long bwd_ws(const void* x, const void* w, const void* gy, int esize, long M, long N, long K, int act, bool gx, bool gw, bool gb) {
    const BwdNeeds d = bwd_needs(x, w, gy, esize, N, K, act, gx, gw);
    const long ldn = padded(N, esize), ldk = padded(K, esize);
    const bool parts = in_parts(esize, act);
    long b = (d.gz ? up256((parts ? 2 : 1) * M * ldn * esize) : 0) + (d.px ? up256(M * ldk * esize) : 0) + (d.pw ? up256(N * ldk * esize) : 0);
    if (gb) b += up256(grad_cut(M, ldn, esize).chunks * ldn * 4);
    const Plan px = gx ? plan_gx(M, N, K, esize, parts) : Plan{}, pw = gw ? plan_gw(M, N, K, esize, parts) : Plan{};
    if (gx && gw && pairs(pw, px)) return b + pw.part_bytes + px.part_bytes;
    return b + (px.part_bytes > pw.part_bytes ? px.part_bytes : pw.part_bytes);
}

template <typename T>
int linear_bwd(const void* x, const void* w, const void* gy, const void* z, int btype, long M, long N, long K, int act, void* gx, void* gw, void* gb,
               char* ws, hipStream_t stream) {
    const int es = sizeof(T);
    const BwdNeeds d = bwd_needs(x, w, gy, es, N, K, act, gx != nullptr, gw != nullptr);
    const long ldn = padded(N, es), ldk = padded(K, es);
    const GradCut c = grad_cut(M, ldn, es);
    const bool parts = in_parts(es, act);
    T* gz = nullptr;
    if (d.gz) {
        gz = reinterpret_cast<T*>(ws);
        ws += up256((parts ? 2 : 1) * M * ldn * es);
    }
    float* sums = nullptr;
    if (gb) {
        sums = reinterpret_cast<float*>(ws);
        ws += up256(c.chunks * ldn * 4);
    }
    const PadP pad = pad_of<T>(x, M, d.px, w, N, d.pw, K, ws);
    if (!gz && !gb) launch_pad<T>(pad, stream);
    else {
        const bool one = gb && c.chunks == 1;
        GradP p{gy, z, gz, one ? nullptr : sums, one ? gb : nullptr, btype, M, c.rows, (int)N, (int)ldn, c.CT, c.RT, c.tiles, act, pad};
        if (N % (16 / es) == 0) launch_act_grad<T, true>(p, (unsigned)(pad.blocks + c.chunks * c.tiles), stream);
        else launch_act_grad<T, false>(p, (unsigned)(pad.blocks + c.chunks * c.tiles), stream);
    }
    const void* const dz = gz ? gz : gy;
    const bool wide = K % (16 / es) == 0;
    GemmP x_{}, w_{};
    Plan px{}, pw{};
    if (gx) {
        x_.M = (int)M; x_.N = (int)K;
        x_.e.y = gx; x_.e.wide = wide && aligned16(gx);
        x_.q = {dz, ldn, (int)M, M * ldn};
        x_.p = {w, ldk, (int)ldk, 0};
        // gz has zeros behind its N-th column, W has no line there: k ends at N for W's lines and at ldn for gz's pieces
        set_k<T>(x_, N, parts);
        px = plan_gx(M, N, K, es, parts);
    }
    if (gw) {
        w_.M = (int)N; w_.N = (int)K;
        set_k<T>(w_, M, parts);
        w_.e.y = gw; w_.e.wide = wide && aligned16(gw);
        w_.q = {dz, ldn, (int)ldn, M * ldn};
        w_.p = {x, ldk, (int)ldk, 0};
        pw = plan_gw(M, N, K, es, parts);
    }
    float* const part = reinterpret_cast<float*>(ws);
    ColumnsP columns{sums, c.chunks, (int)ldn, (int)N, gb, btype, gb && c.chunks > 1 ? sed_cdiv(N, 16) : 0};
    if (gx && gw && pairs(pw, px)) launch_pair<T>(w_, pw, x_, px, columns, part, stream);
    else {
        if (columns.blocks) hipLaunchKernelGGL(column_sums_kernel, dim3((unsigned)columns.blocks), dim3(1024), 0, stream, columns);
        if (gx) launch_gemm<T, true, false>(x_, px, part, stream);
        if (gw) launch_gemm<T, true, true>(w_, pw, part, stream);
    }
    SED_LAUNCH_CHECK();
    return 0;
}

}  // namespace

SED_API long sed_linear_kept_elements(long M, long N) { return M < 1 || N < 1 ? 0 : M * padded(N, 2); }

SED_API int sed_linear_plan(int dtype, long M, long N, long K, int act, int which) {
    if (bad_shape(dtype, M, N, K, act) || which < 0 || which > 2) return 0;
    const int es = esize_of(dtype);
    if (which == 0 && few_rows(M, K, es)) return 1 + 1024;
    const Plan p = which == 0 ? plan_of(M, N, padded(K, es), es) : which == 1 ? plan_gx(M, N, K, es, in_parts(es, act)) : plan_gw(M, N, K, es, in_parts(es, act));
    return p.edge + 1024 * p.slices;
}

SED_API long sed_linear_fwd_ws_bytes(const void* x, const void* w, int dtype, long M, long N, long K) {
    return bad_shape(dtype, M, N, K, 0) ? 0 : fwd_ws(x, w, esize_of(dtype), M, N, K);
}

SED_API int sed_linear_fwd(const void* x, const void* w, const void* bias, const void* residual, int dtype, int bdtype, long M, long N,
                           long K, int act, void* y, void* z, void* ws, long ws_bytes, sed_stream_t stream) {
    if (!x || !w || !y || !aligned16(z) || bdtype < 0 || bdtype > 2 || bad_shape(dtype, M, N, K, act)) return SED_EINVAL;
    const long need = fwd_ws(x, w, esize_of(dtype), M, N, K);
    if (need && (!ws || ws_bytes < need || !aligned16(ws))) return SED_EINVAL;
    char* const s = reinterpret_cast<char*>(ws);
    if (dtype == SED_F32) return linear_fwd<float>(x, w, bias, residual, bdtype, M, N, K, act, y, z, s, stream);
    if (dtype == SED_F16) return linear_fwd<_Float16>(x, w, bias, residual, bdtype, M, N, K, act, y, z, s, stream);
    return linear_fwd<__bf16>(x, w, bias, residual, bdtype, M, N, K, act, y, z, s, stream);
}

SED_API long sed_linear_bwd_ws_bytes(const void* x, const void* w, const void* gy, int dtype, long M, long N, long K, int act, int gx,
                                     int gw, int gb) {
    return bad_shape(dtype, M, N, K, act) ? 0 : bwd_ws(x, w, gy, esize_of(dtype), M, N, K, act, gx, gw, gb);
}

SED_API int sed_linear_bwd(const void* x, const void* w, const void* gy, const void* z, int dtype, int bdtype, long M, long N, long K,
                           int act, void* gx, void* gw, void* gb, void* ws, long ws_bytes, sed_stream_t stream) {
    if (!gy || (gw && !x) || (gx && !w) || (act != SED_ACT_NONE && !z) || bdtype < 0 || bdtype > 2 || bad_shape(dtype, M, N, K, act)) return SED_EINVAL;
    const long need = bwd_ws(x, w, gy, esize_of(dtype), M, N, K, act, gx, gw, gb);
    if (need && (!ws || ws_bytes < need || !aligned16(ws))) return SED_EINVAL;
    char* const s = reinterpret_cast<char*>(ws);
    if (dtype == SED_F32) return linear_bwd<float>(x, w, gy, z, bdtype, M, N, K, act, gx, gw, gb, s, stream);
    if (dtype == SED_F16) return linear_bwd<_Float16>(x, w, gy, z, bdtype, M, N, K, act, gx, gw, gb, s, stream);
    return linear_bwd<__bf16>(x, w, gy, z, bdtype, M, N, K, act, gx, gw, gb, s, stream);
}
