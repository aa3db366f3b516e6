// Log probabilities of given tokens, entropy and likeliest tokens of rows of logits, cross entropy, and their gradients.
//
// For a row z of V logits with largest value m, in units of bits (L = log2 e, M = L m):
//   s = sum 2^(L z_j - M),   u = sum 2^(L z_j - M) (L z_j - M),   log2 p_j = (L z_j - M) - log2 s,
//   H / ln 2 = log2 s - u / s,   d log p_t / d z_j = delta_jt - p_j,   d H / d z_j = -p_j (log p_j + H).
// L z - M is one fused multiply-add; M rounds, but the same M stands in the sum and in the numerator, so logits far from
// zero lose no digits.  All sums are held in fp32.  A logit of minus infinity has probability zero and adds nothing anywhere.
// A row whose largest value is not finite (all minus infinity, a NaN, plus infinity) has no distribution: its results are
// NaN.  Rows whose token is `ignore` are padding: their results and gradients are zero and their logits are not read.
//
// One block reads a row once with 16-byte loads and keeps a running maximum with the sums relative to it; a row is split
// over a cluster of up to 8 blocks when there are too few rows for all SMs, and the parts are joined through distributed
// shared memory.  What bounds it is the number of instructions per logit, so the inner loop works on pairs: maxima and
// the lower limit on packed bf16 or fp16, multiply-adds and sums on packed fp32.
//
// Measured (device time): 4099 rows of 50,261 bf16 logits with 20 alternatives 84 us (413 MB; 67 us without the
// alternatives, 63 us is the floor), 700 x 10,000 fp32 with 5 of them 9.6 us (7.3 without), 2048 x 32,000 bf16 26 us and its
// gradient 45 us (5.8 TB/s).  Mean loss with gradient of 8192 x 131,072 bf16 775 us (4.3 GB, 5.5 TB/s: logits once from
// memory, once from L2, gradient once to memory), 700 x 10,000 fp32 20 us.  Before the pairs, with 256 threads per block
// and plain loads, these were 184, 15, 38 + 61 and 1017 us.
//
// The likeliest tokens come out of the same pass.  Every thread knows the largest of its logits, so the K-th largest of the
// maxima of 64 pairs of threads, found by sorting them in one warp, is a lower bound for the K-th largest logit.  Every thread
// also keeps the maximum of each four vectors that it read, and only those that reach the bound are looked at again (from
// L2).  What reaches the bound is sorted, 32 keys to a warp.  In the first case: with maxima of the warps' 128 vectors two
// fifths of a row were read again, 94 us; with the bound searched bit by bit, and with the logits of the chosen and of the
// likeliest tokens read at the end, 88 us.
#include <cooperative_groups.h>
#include "api.h"
#include "dtypes.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = 32;
constexpr int kMaxSplits = 8;              // blocks of a cluster that share a row
constexpr int kThreads = 128;              // 8 blocks per SM; with 64 threads the first case above takes 105 us, not 99
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;                 // 16-byte vectors of a thread in a batch
constexpr int kStages = 2;                 // batches of a warp: one in use, one on its way
constexpr int kBatch = 32 * kUnroll;       // vectors that a warp reads at a time
constexpr int kCellBytes = 8192;           // maxima of the threads' batches; neighbouring batches share one beyond that
constexpr int kCandidates = 512;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct RowArgs {
    const void* z;
    long long ld, rows;
    int vocab;
    const void* tokens;
    int wide;
    long long ignore;
    float* logprob;
    float* entropy;            // may be null
    float2* stats;             // {m, log2 s} for the backward pass, may be null
    int top;
    float* top_logprob;        // [rows, top]
    long long* top_tokens;
    int* status;
    int splits;                // blocks (of one cluster) per row
    // cross entropy: gradient of the mean loss, and the loss itself, by the block that is the last to finish
    void* dz;                  // null: none
    long long dz_ld;
    float expected;            // gradient that the loss is expected to get
    const int* count;          // rows that are not padding (1 for a sum), filled by the launch before
    unsigned int* done;        // counter of finished rows, zeroed by the launch before
    float* loss;               // null: none
};

// The fast path.  Values are raised to `low` before they enter a sum, so that no infinity does, and a running maximum
// begins at `start`, so far above `low` that what was raised adds exactly zero.  A row whose maximum does not rise above
// `start`, or whose magnitude is so large that the rounding of M = L m would not stay small (|m| 2^-24 L < 10), takes the
// careful path.  start = -2^27: its product with L is exact.
template <typename T> struct Fast { static constexpr float low = -1073741824.f, start = -134217728.f, end = 1e8f; };
template <> struct Fast<__half> { static constexpr float low = -65504.f, start = -65376.f, end = 1e8f; };

template <typename T>
__device__ __forceinline__ bool careful(float m) { return !(m > Fast<T>::start && m < Fast<T>::end); }

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

__device__ __forceinline__ float warp_max_nan(float x) {
    float r;
    asm volatile("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(x));
    return r;
}

__device__ __forceinline__ float exp2_fast(float x) {                // two units in the last place; 0 for very negative x
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Two fp32 values that one instruction works on.
struct Pair { unsigned long long v; };
__device__ __forceinline__ Pair pair(float a, float b) {
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v)); }
__device__ __forceinline__ Pair fma2(Pair a, Pair b, Pair c) {
    Pair r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
    return r;
}
__device__ __forceinline__ Pair add2(Pair a, Pair b) {
    Pair r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair mul2(Pair a, Pair b) {
    Pair r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
    return r;
}
__device__ __forceinline__ Pair exp2_fast(Pair p) {
    float a, b;
    split(p, a, b);
    return pair(exp2_fast(a), exp2_fast(b));
}

// Whole numbers in the order of the values; NaN above everything, the two zeros equal, never 0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of_key(uint32_t k) {          // NaN above plus infinity, minus infinity below its order
    if (k <= 0x007fffffu) return -INFINITY;
    return k >= 0xff800001u ? mgw_nan() : __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}

// Work on the values of a 16-byte vector in pairs.  largest(): of several vectors, NaN if there is one; values<LIFT>(): as
// fp32, raised to `low` with LIFT; pack(): back to the type.
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    template <int K>
    static __device__ __forceinline__ float largest(const uint4 (&r)[K]) {
        float m = __uint_as_float(r[0].x);
#pragma unroll
        for (int k = 0; k < K; ++k)
            m = max_nan(max_nan(max_nan(m, __uint_as_float(r[k].x)), max_nan(__uint_as_float(r[k].y), __uint_as_float(r[k].z))),
                        __uint_as_float(r[k].w));
        return m;
    }
    template <bool LIFT>
    static __device__ __forceinline__ void values(const uint4& r, Pair (&f)[2]) {
        float a[4] = {__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w)};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (LIFT) a[e] = max_nan(a[e], Fast<float>::low);
        f[0] = pair(a[0], a[1]);
        f[1] = pair(a[2], a[3]);
    }
    static __device__ __forceinline__ uint4 pack(const Pair (&f)[2]) {
        uint4 r;
        float a, b;
        split(f[0], a, b);
        r.x = __float_as_uint(a); r.y = __float_as_uint(b);
        split(f[1], a, b);
        r.z = __float_as_uint(a); r.w = __float_as_uint(b);
        return r;
    }
};
template <typename T2> __device__ __forceinline__ float2 pair_to_float(T2 h);
template <> __device__ __forceinline__ float2 pair_to_float<__half2>(__half2 h) { return __half22float2(h); }
template <> __device__ __forceinline__ float2 pair_to_float<__nv_bfloat162>(__nv_bfloat162 h) { return __bfloat1622float2(h); }
template <typename T2> __device__ __forceinline__ T2 pair_from_float(float a, float b);
template <> __device__ __forceinline__ __half2 pair_from_float<__half2>(float a, float b) { return __floats2half2_rn(a, b); }
template <> __device__ __forceinline__ __nv_bfloat162 pair_from_float<__nv_bfloat162>(float a, float b) { return __floats2bfloat162_rn(a, b); }

template <typename T, typename T2>
struct VecHalf {
    static constexpr int N = 8;
    static __device__ __forceinline__ T2 word(const uint4& r, int k) {
        const uint32_t w = k == 0 ? r.x : k == 1 ? r.y : k == 2 ? r.z : r.w;
        return *reinterpret_cast<const T2*>(&w);
    }
    template <int K>
    static __device__ __forceinline__ float largest(const uint4 (&r)[K]) {
        T2 m = word(r[0], 0);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
            for (int w = 0; w < 4; ++w) m = __hmax2_nan(m, word(r[k], w));
        const float2 f = pair_to_float(m);
        return max_nan(f.x, f.y);
    }
    template <bool LIFT>
    static __device__ __forceinline__ void values(const uint4& r, Pair (&f)[4]) {
        T2 low;
        low.x = low.y = mgw_from_float<T>(Fast<T>::low);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float2 x = pair_to_float(LIFT ? __hmax2_nan(word(r, w), low) : word(r, w));
            f[w] = pair(x.x, x.y);
        }
    }
    static __device__ __forceinline__ uint4 pack(const Pair (&f)[4]) {
        uint32_t w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            float a, b;
            split(f[k], a, b);
            const T2 h = pair_from_float<T2>(a, b);
            w[k] = *reinterpret_cast<const uint32_t*>(&h);
        }
        return make_uint4(w[0], w[1], w[2], w[3]);
    }
};
template <> struct Vec<__half> : VecHalf<__half, __half2> {};
template <> struct Vec<__nv_bfloat16> : VecHalf<__nv_bfloat16, __nv_bfloat162> {};

// A thread's sums, relative to its running maximum m (in bits: M = L m).
struct Sums {
    float m, M;
    Pair s, u;
};

template <bool ENT>
__device__ __forceinline__ void raise_to(Sums& a, float m) {
    // both products rounded, as M is everywhere: a fused subtraction would leave the rounding of the other one behind
    const float M = __fmul_rn(m, kLog2e), d = a.M - M, f = exp2_fast(d);
    if (ENT) a.u = mul2(pair(f, f), fma2(a.s, pair(d, d), a.u));
    a.s = mul2(pair(f, f), a.s);
    a.m = m;
    a.M = M;
}

template <typename T, bool ENT>
__device__ __forceinline__ void add_vector(Sums& a, const uint4& r) {
    constexpr int P = Vec<T>::N / 2;
    Pair f[P];
    Vec<T>::template values<ENT>(r, f);                              // without u a logit of minus infinity does no harm
#pragma unroll
    for (int k = 0; k < P; ++k) {
        const Pair d = fma2(f[k], pair(kLog2e, kLog2e), pair(-a.M, -a.M)), x = exp2_fast(d);
        a.s = add2(a.s, x);
        if (ENT) a.u = fma2(x, d, a.u);
    }
}

struct Stats { float m, s, u; };

// The block's sums: first the maximum of all, then one rescaling, then plain sums.
template <bool ENT>
__device__ __forceinline__ Stats block_join(Sums x, Stats* parts) {
    const float w = warp_max_nan(x.m);
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5].m = w;
    __syncthreads();
    float m = parts[0].m;
#pragma unroll
    for (int k = 1; k < kWarps; ++k) m = max_nan(m, parts[k].m);
    raise_to<ENT>(x, m);
    float s, u = 0.f, t;
    split(x.s, s, t);
    s += t;
    if (ENT) {
        split(x.u, u, t);
        u += t;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        if (ENT) u += __shfl_xor_sync(0xffffffffu, u, o);
    }
    if ((threadIdx.x & 31) == 0) { parts[threadIdx.x >> 5].s = s; parts[threadIdx.x >> 5].u = u; }
    __syncthreads();
    Stats r = {m, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < kWarps; ++k) {
        r.s += parts[k].s;
        if (ENT) r.u += parts[k].u;
    }
    return r;
}

// Two blocks' sums.
template <bool ENT>
__device__ __forceinline__ Stats join(Stats a, Stats b) {
    const float m = max_nan(a.m, b.m), M = __fmul_rn(m, kLog2e);
    const float da = __fmul_rn(a.m, kLog2e) - M, db = __fmul_rn(b.m, kLog2e) - M, fa = exp2_fast(da), fb = exp2_fast(db);
    Stats r = {m, a.s * fa + b.s * fb, 0.f};
    if (ENT) r.u = fa * (a.u + a.s * da) + fb * (b.u + b.s * db);
    return r;
}

// ------------------------------------------------------------------------------------------------ layout of a row
// Elements before the first 16-byte boundary (head), whole vectors, elements behind them (tail).  A block of a cluster
// has the vectors [v0, v1); the first block also has the head, the last one the tail.
template <typename T>
struct Row {
    const T* z;
    int head, n_vec, tail0, vocab, v0, v1;
    bool has_head, has_tail;
    __device__ __forceinline__ Row(const T* z_, int vocab_, int part, int splits) : z(z_), vocab(vocab_) {
        const int h = (int)(((16 - ((unsigned long long)z_ & 15)) & 15) / sizeof(T));
        head = min(h, vocab_);
        n_vec = (vocab_ - head) / Vec<T>::N;
        tail0 = head + n_vec * Vec<T>::N;
        const int per = splits == 1 ? n_vec : (((n_vec + splits - 1) / splits + 31) & ~31);
        v0 = (int)min((long long)n_vec, (long long)part * per);
        v1 = (int)min((long long)n_vec, (long long)v0 + per);
        has_head = part == 0;
        has_tail = part == splits - 1;
    }
    // Calls use(i0, r) for each whole batch of this warp, vectors i0 + 32 k + lane.  The loads run kStages - 1 batches ahead,
    // through a ring in shared memory of which every thread reads only what it has loaded itself.
    template <typename F>
    __device__ __forceinline__ void for_batches(uint4* ring, F use) const {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, first = v0 + warp * kBatch;
        const int n = v1 - first < kBatch ? 0 : (v1 - first - kBatch) / (kWarps * kBatch) + 1;
        const uint4* from = reinterpret_cast<const uint4*>(z + head) + first + lane;
        const uint4* end = from + (long long)n * (kWarps * kBatch);
        const uint4* mine = ring + warp * (kStages * kBatch) + lane;
        const uint32_t base = (uint32_t)__cvta_generic_to_shared(mine);
        uint32_t put = 0, get = 0;                                   // slots, in bytes from the thread's first
        auto fetch = [&]() {
            if (from < end) {
#pragma unroll
                for (int k = 0; k < kUnroll; ++k)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(base + put + k * 512), "l"(from + k * 32) : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            from += kWarps * kBatch;
            put = put == (kStages - 1) * kBatch * 16 ? 0 : put + kBatch * 16;
        };
#pragma unroll
        for (int b = 0; b < kStages - 1; ++b) fetch();
        for (int i0 = first, i1 = first + n * (kWarps * kBatch); i0 < i1; i0 += kWarps * kBatch) {
            fetch();
            asm volatile("cp.async.wait_group %0;" :: "n"(kStages - 1) : "memory");
            uint4 r[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) r[k] = *reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(mine) + get + k * 512);
            get = get == (kStages - 1) * kBatch * 16 ? 0 : get + kBatch * 16;
            use(i0, r);
        }
    }
    // first vector behind this warp's whole batches, for the few that are left (v1 where there are none)
    __device__ __forceinline__ int rest() const {
        const int first = v0 + (threadIdx.x >> 5) * kBatch;
        return v1 - first < kBatch ? first : first + ((v1 - first - kBatch) / (kWarps * kBatch) + 1) * (kWarps * kBatch);
    }
    __device__ __forceinline__ uint4 vec(int i) const { return reinterpret_cast<const uint4*>(z + head)[i]; }
    // the element at the edge that a thread of the block looks after (0 .. 15), or -1
    __device__ __forceinline__ int edge(int thread) const {
        if (thread < 8) return has_head && thread < head ? thread : -1;
        return thread < 16 && has_tail && tail0 + thread - 8 < vocab ? tail0 + thread - 8 : -1;
    }
};

constexpr size_t kRingBytes = (size_t)kWarps * kStages * kBatch * 16;

// Maxima of a thread's batches: 32 of them for 16-bit types, 16 for fp32.
template <typename T> constexpr int kCells = kCellBytes / (kThreads * (int)sizeof(T));

struct TopSpace {                          // in the memory of the ring, which the scan no longer needs
    uint32_t most[kThreads];               // order of the threads' maxima, 0: the thread has no vector
    uint32_t floor;                        // a lower bound of the order of the K-th largest value
    unsigned long long list[kWarps][32];
    unsigned long long candidate[kCandidates];
    int n_candidates;
};
static_assert(sizeof(TopSpace) <= kRingBytes, "it takes the ring's place");

// Sums of this block's part of the row; with TOP also the maxima of the thread's batches and of all its vectors (most: minus
// infinity where it has none).
template <typename T, bool ENT, bool TOP>
__device__ __forceinline__ Sums scan_row(const Row<T>& row, uint4* ring, int shift, T* cells, float& most) {
    const int lane = threadIdx.x & 31;
    Sums a;
    a.m = Fast<T>::start;
    a.M = __fmul_rn(a.m, kLog2e);
    a.s = a.u = pair(0.f, 0.f);
    most = -INFINITY;
    int batch = 0;
    float in_cell = -INFINITY;
    auto note = [&](float m) {
        most = max_nan(most, m);
        in_cell = (batch & ((1 << shift) - 1)) == 0 ? m : max_nan(in_cell, m);
        cells[(batch >> shift) * kThreads + threadIdx.x] = mgw_from_float<T>(in_cell);
        ++batch;
    };
    row.for_batches(ring, [&](int, const uint4 (&r)[kUnroll]) {
        const float m = Vec<T>::largest(r), up = max_nan(a.m, m);
        if (up != a.m) raise_to<ENT>(a, up);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) add_vector<T, ENT>(a, r[k]);
        if (TOP) note(m);
    });
    const int i0 = row.rest();
    if (i0 < row.v1) {                                               // less than a batch
        float m = -INFINITY;
        for (int i = i0 + lane; i < row.v1; i += 32) {
            const uint4 r[1] = {row.vec(i)};
            m = max_nan(m, Vec<T>::largest(r));
            const float up = max_nan(a.m, m);
            if (up != a.m) raise_to<ENT>(a, up);
            add_vector<T, ENT>(a, r[0]);
        }
        if (TOP) note(m);
    }
    const int j = row.edge(threadIdx.x);
    if (j >= 0) {
        const float v = mgw_to_float(row.z[j]);
        const float up = max_nan(a.m, v);
        if (up != a.m) raise_to<ENT>(a, up);
        const float d = fmaf(max_nan(v, Fast<T>::low), kLog2e, -a.M), x = exp2_fast(d);
        a.s = add2(a.s, pair(x, 0.f));
        if (ENT) a.u = fma2(pair(x, 0.f), pair(d, 0.f), a.u);
    }
    return a;
}

// A row whose maximum is at the edge of the type's range: differences first, minus infinity left out.  m may end up
// infinite or NaN; s and u are relative to m, u in bits.
template <typename T>
__device__ __noinline__ Stats careful_row(const T* z, int vocab, Stats* parts) {
    float m = -INFINITY;
    for (int j = threadIdx.x; j < vocab; j += kThreads) m = max_nan(m, mgw_to_float(z[j]));
    m = warp_max_nan(m);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5].m = m;
    __syncthreads();
    for (int w = 0; w < kWarps; ++w) m = max_nan(m, parts[w].m);
    float s = 0.f, u = 0.f;
    for (int j = threadIdx.x; j < vocab; j += kThreads) {
        const float v = mgw_to_float(z[j]);
        const float d = fmaxf((v - m) * kLog2e, -1e4f), x = v == -INFINITY ? 0.f : exp2_fast(d);
        s += x;
        u = fmaf(x, d, u);
    }
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        u += __shfl_xor_sync(0xffffffffu, u, o);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) { parts[threadIdx.x >> 5].s = s; parts[threadIdx.x >> 5].u = u; }
    __syncthreads();
    Stats x = {m, 0.f, 0.f};
    for (int w = 0; w < kWarps; ++w) { x.s += parts[w].s; x.u += parts[w].u; }
    return x;
}

// log2 p of a logit
template <typename T>
__device__ __forceinline__ float log2_prob(float v, float m, float log2_s) {
    return (careful<T>(m) ? (v - m) * kLog2e : fmaf(v, kLog2e, -(m * kLog2e))) - log2_s;
}

// ln p of a logit (one that is itself near the end of the type's range keeps its value: L v would not be finite)
template <typename T>
__device__ __forceinline__ float ln_prob(float v, float m, float log2_s) {
    if (careful<T>(m) || fabsf(v) > 1e30f) return (v - m) - kLn2 * log2_s;
    return kLn2 * (fmaf(v, kLog2e, -(m * kLog2e)) - log2_s);
}

// -------------------------------------------------------------------------------------------------- likeliest tokens
// A key is the value's order and below it the complement of the index, so equal values are ordered by the lower index
// and no two keys are equal; 0 is none.
typedef unsigned long long Key;

__device__ __forceinline__ Key key_of(float v, int index) { return ((Key)order_key(v) << 32) | (0xffffffffu - (uint32_t)index); }

template <typename K>
__device__ __forceinline__ K sort_lanes(K x) {                       // bitonic, descending
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const K y = __shfl_xor_sync(0xffffffffu, x, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);
            x = larger == (y > x) ? y : x;
        }
    return x;
}

template <typename K>
__device__ __forceinline__ K merge_lists(K a, K b) {                 // both descending: the 32 largest of the 64
    const int lane = threadIdx.x & 31;
    const K y = __shfl_sync(0xffffffffu, b, 31 - lane);
    K x = a > y ? a : y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const K z = __shfl_xor_sync(0xffffffffu, x, o);
        x = ((lane & o) == 0) == (z > x) ? z : x;
    }
    return x;
}

// The warps' lists become one, in the first warp.
__device__ __forceinline__ Key join_lists(Key mine, TopSpace* t) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    t->list[warp][lane] = mine;
    __syncthreads();
    if (warp == 0)
        for (int w = 1; w < kWarps; ++w)
            if (t->list[w][0] != 0) mine = merge_lists(mine, t->list[w][lane]);
    return mine;
}

// Many equal or rising values: every warp keeps a sorted list of the 32 largest and goes through its part of the row, 32
// values at a time.
template <typename T>
__device__ __noinline__ Key top_by_lists(const Row<T>& row, float floor, TopSpace* t) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Key mine = 0;
    auto offer = [&](Key x) {
        const Key least = __shfl_sync(0xffffffffu, mine, 31);
        if (__any_sync(0xffffffffu, x > least)) mine = merge_lists(mine, sort_lanes(x));
    };
    for (int i0 = row.v0 + warp * 32; i0 < row.v1; i0 += kWarps * 32) {
        const bool in = i0 + lane < row.v1;
        float f[Vec<T>::N];
        if (in) mgw_unpack<T, Vec<T>::N>(row.vec(i0 + lane), f);
#pragma unroll
        for (int e = 0; e < Vec<T>::N; ++e)
            offer(in && !(f[e] < floor) ? key_of(f[e], row.head + (i0 + lane) * Vec<T>::N + e) : (Key)0);
    }
    if (warp == 0) {
        const int j = row.edge(lane);
        offer(j >= 0 ? key_of(mgw_to_float(row.z[j]), j) : (Key)0);
    }
    return join_lists(mine, t);
}

// Element q of the values in r, by selection: an indexed array would live in memory.
template <typename T>
__device__ __forceinline__ T element(const uint4 (&r)[kUnroll], int q) {
    static_assert(kUnroll == 4, "sixteen words");
    const int w = q * (int)sizeof(T) >> 2;
    const uint4 a = w & 4 ? r[1] : r[0], b = w & 4 ? r[3] : r[2], c = w & 8 ? b : a;
    const uint32_t lo = w & 1 ? c.y : c.x, hi = w & 1 ? c.w : c.z;
    uint32_t word = w & 2 ? hi : lo;
    if (sizeof(T) == 2 && (q & 1)) word >>= 16;
    return *reinterpret_cast<const T*>(&word);
}

// The 32 largest keys of this block's part of the row (at least the `top` largest are right), in the lanes of the first
// warp, the largest first.
template <typename T>
__device__ __forceinline__ Key find_top(const Row<T>& row, int top, int shift, float most, const T* cells, TopSpace* t) {
    constexpr int N = Vec<T>::N;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // the bound: the value that `top` of 64 pairs of threads reach, by sorting the pairs' maxima
    t->most[threadIdx.x] = row.v0 + warp * kBatch + lane < row.v1 ? order_key(most) : 0u;
    if (threadIdx.x == 0) t->n_candidates = 0;
    __syncthreads();
    if (warp == 0) {
        static_assert(kWarps == 4 && kMaxTop == 32, "two sorted lists of 32 become one");
        const uint32_t a = sort_lanes(max(t->most[lane], t->most[64 + lane])), b = sort_lanes(max(t->most[32 + lane], t->most[96 + lane]));
        const uint32_t bound = __shfl_sync(0xffffffffu, merge_lists(a, b), top - 1);
        if (lane == 0) t->floor = bound;
    }
    __syncthreads();
    const uint32_t low = t->floor;
    const float floor = value_of_key(low);
    if (!(most < floor)) {                                           // not many more than `top` threads
        int batch = 0;
        for (int i0 = row.v0 + warp * kBatch + lane; i0 < row.v1; i0 += kWarps * kBatch, ++batch) {
            if (mgw_to_float(cells[(batch >> shift) * kThreads + threadIdx.x]) < floor) continue;
            uint4 r[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k)
                if (i0 + k * 32 < row.v1) r[k] = row.vec(i0 + k * 32);
            uint32_t hits = 0;                                       // which of the kUnroll * N values reach the bound
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                float f[N];
                mgw_unpack<T, N>(r[k], f);
                if (i0 + k * 32 >= row.v1) continue;
#pragma unroll
                for (int e = 0; e < N; ++e) hits |= f[e] < floor ? 0u : 1u << (k * N + e);
            }
            for (; hits != 0; hits &= hits - 1) {
                const int q = __ffs(hits) - 1, at = atomicAdd(&t->n_candidates, 1);      // the order does not matter: keys are sorted
                if (at < kCandidates) t->candidate[at] = key_of(mgw_to_float(element<T>(r, q)), row.head + (i0 + q / N * 32) * N + q % N);
            }
        }
    }
    const int j = row.edge(threadIdx.x);
    if (j >= 0) {
        const float v = mgw_to_float(row.z[j]);
        if (!(v < floor)) {
            const int at = atomicAdd(&t->n_candidates, 1);
            if (at < kCandidates) t->candidate[at] = key_of(v, j);
        }
    }
    __syncthreads();
    const int found = t->n_candidates;
    if (found > kCandidates) return top_by_lists(row, floor, t);
    Key mine = 0;
    for (int at = warp * 32; at < found; at += kThreads) {
        const Key x = sort_lanes(at + lane < found ? t->candidate[at + lane] : (Key)0);
        mine = at == warp * 32 ? x : merge_lists(mine, x);
    }
    return found <= 32 ? mine : join_lists(mine, t);
}

// ------------------------------------------------------------------------------------------- gradient of one row
// The block's part of a row of a gradient.  pairs(Pair logits) and one(logit, column) give the values; the column `t` is
// always done by one().  Whole vectors where logits and gradient start at the same place of a 16-byte block.
template <typename T, bool READ, bool LIFT, typename FP, typename F1>
__device__ __forceinline__ void write_row(const Row<T>& row, uint4* ring, T* dz, long long t, FP pairs, F1 one) {
    constexpr int N = Vec<T>::N;
    if (((unsigned long long)dz & 15) == ((unsigned long long)row.z & 15)) {
        uint4* to = reinterpret_cast<uint4*>(dz + row.head);
        const int ti = t >= row.head && t < row.tail0 ? ((int)t - row.head) / N : -1;      // the vector with column t
        auto finish = [&](const uint4& q, int i) {
            Pair f[N / 2];
            if (READ) Vec<T>::template values<LIFT>(q, f);
#pragma unroll
            for (int k = 0; k < N / 2; ++k) f[k] = pairs(f[k]);
            __stcs(&to[i], Vec<T>::pack(f));                         // not read again here
            if (i == ti) dz[t] = mgw_from_float<T>(one(READ ? mgw_to_float(row.z[t]) : 0.f, (int)t));
        };
        const int lane = threadIdx.x & 31;
        if (READ) {
            row.for_batches(ring, [&](int i0, const uint4 (&r)[kUnroll]) {
#pragma unroll
                for (int k = 0; k < kUnroll; ++k) finish(r[k], i0 + k * 32 + lane);
            });
            for (int i = row.rest() + lane, end = min(row.v1, row.rest() + kBatch); i < end; i += 32) finish(row.vec(i), i);
        } else {
            for (int i = row.v0 + threadIdx.x; i < row.v1; i += kThreads) finish(make_uint4(0, 0, 0, 0), i);
        }
    } else {
        for (int j = row.head + row.v0 * N + threadIdx.x; j < row.head + row.v1 * N; j += kThreads)
            dz[j] = mgw_from_float<T>(one(READ ? mgw_to_float(row.z[j]) : 0.f, j));
    }
    const int j = row.edge(threadIdx.x);
    if (j >= 0) dz[j] = mgw_from_float<T>(one(READ ? mgw_to_float(row.z[j]) : 0.f, j));
}

template <typename T>
__device__ __noinline__ void write_constant(const Row<T>& row, T* dz, float c) {
    write_row<T, false, false>(row, nullptr, dz, -1, [=](Pair) { return pair(c, c); }, [=](float, int) { return c; });
}

// A row whose maximum is at the edge of the range: -p (base + slope log2 p) + g1 delta, one by one.
template <typename T>
__device__ __noinline__ void write_careful(const Row<T>& row, T* dz, float m, float log2_s, float base, float slope, float g1, long long t) {
    const int j0 = row.has_head ? 0 : row.head + row.v0 * Vec<T>::N, j1 = row.has_tail ? row.vocab : row.head + row.v1 * Vec<T>::N;
    for (int j = j0 + threadIdx.x; j < j1; j += kThreads) {
        const float d = fmaxf((mgw_to_float(row.z[j]) - m) * kLog2e - log2_s, -1e4f);      // p = 0 well before
        const float x = -exp2_fast(d) * fmaf(slope, d, base);
        dz[j] = mgw_from_float<T>(j == t ? x + g1 : x);
    }
}

// g (p - delta), the gradient of one row's loss: 2^(L z - M) times g / s
template <typename T>
__device__ __forceinline__ void write_loss_gradient(const Row<T>& row, uint4* ring, T* dz, float m, float log2_s, float g, long long t) {
    if (careful<T>(m)) {
        write_careful(row, dz, m, log2_s, -g, 0.f, -g, t);
        return;
    }
    const float M = __fmul_rn(m, kLog2e), gs = g * exp2f(-log2_s);
    write_row<T, true, false>(
        row, ring, dz, t, [=](Pair v) { return mul2(exp2_fast(fma2(v, pair(kLog2e, kLog2e), pair(-M, -M))), pair(gs, gs)); },
        [=](float v, int j) {
            const float x = exp2_fast(fmaf(v, kLog2e, -M)) * gs;
            return j == t ? x - g : x;
        });
}

// ------------------------------------------------------------------------------------------------------------ forward
template <typename T, bool ENT, bool TOP, bool LOSS>
__global__ void __launch_bounds__(kThreads, 8) logprob_fwd_kernel(RowArgs a) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    uint4* ring = reinterpret_cast<uint4*>(dynamic);
    T* cells = reinterpret_cast<T*>(dynamic + kRingBytes);           // only with TOP
    __shared__ Stats parts[kWarps];
    __shared__ Stats of_block;
    __shared__ Key block_list[kMaxTop];
    const int part = a.splits == 1 ? 0 : blockIdx.x % a.splits;
    const long long r = a.splits == 1 ? blockIdx.x : blockIdx.x / a.splits;
    const long long t = mgw_token(a.tokens, a.wide, r);
    const Row<T> row(static_cast<const T*>(a.z) + r * a.ld, a.vocab, part, a.splits);
    const bool valid = t >= 0 && t < a.vocab;
    T chosen = mgw_from_float<T>(0.f);                               // read now, so that nothing waits for it at the end
    if (part == 0 && threadIdx.x == 0 && valid && t != a.ignore) chosen = row.z[t];
    if (t == a.ignore) {                                             // all blocks of the cluster leave
        if (part == 0) {
            if (threadIdx.x == 0) {
                a.logprob[r] = 0.f;
                if (ENT && a.entropy) a.entropy[r] = 0.f;
                if (a.stats) a.stats[r] = make_float2(0.f, 0.f);
            }
            if (TOP)
                for (int k = threadIdx.x; k < a.top; k += kThreads) {
                    a.top_logprob[r * a.top + k] = 0.f;
                    a.top_tokens[r * a.top + k] = -1;
                }
        }
        if (LOSS && a.dz != nullptr) write_constant(row, static_cast<T*>(a.dz) + r * a.dz_ld, 0.f);
    } else {
        int shift = 0;
        if (TOP)
            while (((row.v1 - row.v0) / (kWarps * kBatch) >> shift) >= kCells<T>) ++shift;
        float most;
        Stats x = block_join<ENT>(scan_row<T, ENT, TOP>(row, ring, shift, cells, most), parts);
        if (a.splits > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (threadIdx.x == 0) of_block = x;
            cluster.sync();
            Stats each[kMaxSplits];                                  // all on their way before the first is needed
#pragma unroll
            for (int k = 0; k < kMaxSplits; ++k)
                if (k < a.splits) each[k] = *cluster.map_shared_rank(&of_block, k);
            x = each[0];
#pragma unroll
            for (int k = 1; k < kMaxSplits; ++k)
                if (k < a.splits) x = join<ENT>(x, each[k]);
        }
        if (careful<T>(x.m)) x = careful_row(row.z, a.vocab, parts);
        const bool fine = fabsf(x.m) < INFINITY;
        const float log2_s = log2f(x.s);
        if (part == 0 && threadIdx.x == 0) {
            if (!valid) mgw_report_token(a.status, MGW_OP_LOGPROB, r, t);
            a.logprob[r] = valid && fine ? ln_prob<T>(mgw_to_float(chosen), x.m, log2_s) : mgw_nan();
            if (ENT && a.entropy) a.entropy[r] = fine ? kLn2 * (log2_s - x.u / x.s) : mgw_nan();
            if (a.stats) a.stats[r] = make_float2(fine ? x.m : mgw_nan(), log2_s);
        }
        if (TOP) {
            const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
            Key mine = find_top(row, a.top, shift, most, cells, reinterpret_cast<TopSpace*>(ring));
            if (a.splits > 1) {
                cg::cluster_group cluster = cg::this_cluster();
                if (warp == 0) block_list[lane] = mine;
                cluster.sync();
                if (part == 0 && warp == 0) {                        // likewise
                    Key other[kMaxSplits - 1];
#pragma unroll
                    for (int k = 1; k < kMaxSplits; ++k) other[k - 1] = k < a.splits ? *cluster.map_shared_rank(&block_list[lane], k) : (Key)0;
#pragma unroll
                    for (int k = 1; k < kMaxSplits; ++k)
                        if (k < a.splits) mine = merge_lists(mine, other[k - 1]);
                }
            }
            if (part == 0 && warp == 0 && lane < a.top && mine != 0) {      // key 0 is no entry: never an index
                const int j = (int)(0xffffffffu - (uint32_t)mine);
                a.top_tokens[r * a.top + lane] = j;
                a.top_logprob[r * a.top + lane] = fine ? ln_prob<T>(value_of_key((uint32_t)(mine >> 32)), x.m, log2_s) : mgw_nan();
            }
        }
        if (LOSS) mgw_wait_for_previous();                               // the count of rows
        if (LOSS && a.dz != nullptr) {                               // the row was just read: it comes from L2
            T* dz = static_cast<T*>(a.dz) + r * a.dz_ld;
            if (fine && valid) write_loss_gradient(row, ring, dz, x.m, log2_s, a.expected / (float)*a.count, t);
            else write_constant(row, dz, mgw_nan());
        }
        if (a.splits > 1) cg::this_cluster().sync();                 // until here the others may read this block's memory
    }
    if (LOSS) mgw_wait_for_previous();                                   // the counter, also for rows that are padding
    if (LOSS && a.loss != nullptr && part == 0) {
        // the block that finishes last adds up the rows: thread i rows i, i + 256, ..., the same order every time
        __shared__ bool last;
        __shared__ double sums[kWarps];
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        if (threadIdx.x == 0) {
            __threadfence();
            last = atomicAdd(a.done, 1u) == (unsigned)(a.rows - 1);
        }
        __syncthreads();
        if (!last) return;
        __threadfence();
        double s = 0.0;
        for (long long i = threadIdx.x; i < a.rows; i += kThreads) s += (double)__ldcg(&a.logprob[i]);
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (lane == 0) sums[warp] = s;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kWarps; ++w) s += sums[w];
            *a.loss = (float)(-s / (double)*a.count);                // no row left: 0 / 0, as the mean of nothing
        }
    }
}

// Rows that are not padding (or 1, for a sum), and the counter of finished rows back to zero.
__global__ void __launch_bounds__(1024) count_rows_kernel(const void* __restrict__ tokens, int wide, long long ignore, long long rows,
                                                          int mean, int* __restrict__ count, unsigned int* __restrict__ done,
                                                          float* __restrict__ loss) {
    __shared__ int kept[32];
    mgw_let_next_start();
    int k = 0;
    if (mean)
        for (long long i = threadIdx.x; i < rows; i += 1024) k += mgw_token(tokens, wide, i) != ignore;
    k = __reduce_add_sync(0xffffffffu, k);
    if ((threadIdx.x & 31) == 0) kept[threadIdx.x >> 5] = k;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) k += kept[w];
        *count = mean ? k : 1;
        *done = 0;
        if (rows == 0) *loss = mean ? mgw_nan() : 0.f;
    }
}

// ----------------------------------------------------------------------------------------------------------- backward
struct GradArgs {
    const void* z;
    long long ld, rows;
    int vocab;
    const void* tokens;
    int wide;
    long long ignore;
    const float2* stats;       // {m, log2 s}
    const float* entropy;      // null: no gradient of the entropy
    const float* g_logprob;    // [rows], or null
    const float* g_entropy;    // [rows], or null
    const float* g_loss;       // one value: gradient of the mean loss, or null
    const int* count;          // rows that are not padding, for g_loss
    int written;               // dz already holds the gradient for g_loss == expected
    float expected;
    void* dz;
    long long dz_ld;
    int splits;                // blocks per row
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 8) logprob_bwd_kernel(GradArgs a) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    uint4* ring = reinterpret_cast<uint4*>(dynamic);
    const float g_loss = a.g_loss != nullptr ? *a.g_loss : 0.f;
    if (a.written && g_loss == a.expected) return;
    // from the last row on: what the forward launch read last is still in L2 (2048 x 32,000 bf16: 45 us, from the first 49)
    for (long long task = a.rows * a.splits - 1 - blockIdx.x; task >= 0; task -= gridDim.x) {
        const long long r = a.splits == 1 ? task : task / a.splits;
        const int part = (int)(task - r * a.splits);
        const long long t = mgw_token(a.tokens, a.wide, r);
        const Row<T> row(static_cast<const T*>(a.z) + r * a.ld, a.vocab, part, a.splits);
        T* dz = static_cast<T*>(a.dz) + r * a.dz_ld;
        if (t == a.ignore) {
            write_constant(row, dz, 0.f);
            continue;
        }
        const float m = a.stats[r].x, log2_s = a.stats[r].y;
        if (t < 0 || t >= a.vocab || m != m) {
            write_constant(row, dz, mgw_nan());
            continue;
        }
        if (a.g_loss != nullptr) {
            write_loss_gradient(row, ring, dz, m, log2_s, g_loss / (float)*a.count, t);
            continue;
        }
        // g1 (delta - p) - g2 p (ln p + H); with d = L z - M:  p = 2^d / s,  ln p = ln 2 (d - log2 s)
        const float h = a.entropy ? a.entropy[r] : 0.f, g1 = a.g_logprob ? a.g_logprob[r] : 0.f, g2 = a.g_entropy ? a.g_entropy[r] : 0.f;
        const float slope = g2 * kLn2, M = __fmul_rn(m, kLog2e);
        if (careful<T>(m)) {
            write_careful(row, dz, m, log2_s, g1 + g2 * h, slope, g1, t);
            continue;
        }
        const float base = g1 + g2 * h - slope * log2_s, rs = -exp2f(-log2_s);
        write_row<T, true, true>(
            row, ring, dz, t,
            [=](Pair v) {
                const Pair d = fma2(v, pair(kLog2e, kLog2e), pair(-M, -M));
                return mul2(mul2(exp2_fast(d), pair(rs, rs)), fma2(pair(slope, slope), d, pair(base, base)));
            },
            [=](float v, int j) {
                const float d = fmaf(max_nan(v, Fast<T>::low), kLog2e, -M);
                const float x = exp2_fast(d) * rs * fmaf(slope, d, base);
                return j == t ? x + g1 : x;
            });
    }
}

bool bad_rows(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens) {
    const int es = dtype == MGW_F32 ? 4 : 2;
    return rows < 0 || rows > 0x7fffffffLL || vocab < 1 || vocab > (1 << 30) || (rows > 1 && ld < vocab) || dtype < MGW_F32 || dtype > MGW_BF16 ||
           (rows > 0 && (z == nullptr || tokens == nullptr || ((uintptr_t)z & (es - 1))));
}

template <typename T, bool ENT, bool TOP, bool LOSS>
int launch_fwd(const RowArgs& a, cudaStream_t stream) {
    const size_t smem = kRingBytes + (TOP ? kCellBytes : 0);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * a.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    int n = 0;
    if (a.splits > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = a.splits; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
        ++n;
    }
    if (LOSS) {                                                      // reads the rows while the launch before counts them
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        ++n;
    }
    cfg.attrs = attr;
    cfg.numAttrs = n;
    MGW_CUDA_CHECK(cudaLaunchKernelEx(&cfg, logprob_fwd_kernel<T, ENT, TOP, LOSS>, a));
    return MGW_OK;
}

template <typename T>
int launch_fwd(const RowArgs& a, cudaStream_t stream) {
    if (a.loss != nullptr) return launch_fwd<T, false, false, true>(a, stream);
    return a.top > 0 ? launch_fwd<T, true, true, false>(a, stream) : launch_fwd<T, true, false, false>(a, stream);
}

constexpr long long kResident = 148 * 8;                               // blocks that run at once
constexpr long long kInL2 = 40LL << 20;                               // bytes of rows that are still in L2 when they are read again:
                                                                      // 8192 x 131,072 bf16 782 us, 902 with a block per row

// Blocks per row: one as soon as the rows alone give 2.7 blocks to every SM, else up to 8 (a portable cluster) that have
// at least 128 vectors each.  550 rows of 50,000 bf16 with 5 likeliest tokens: 19 us with one, 21 with two; 100 such rows
// 10.5 with four, 12.5 with eight; 400 rows without them 13 with one or two, and their gradient 15.5 and 14.  Where rows
// are read twice (`twice`, the loss and its gradient), as many that the rows in flight stay in L2.
int splits_of(long long rows, int vocab, int dtype, bool twice) {
    const int per = dtype == MGW_F32 ? 4 : 8;
    int splits = 1;
    while (splits < kMaxSplits && vocab / per / (splits * 2) >= 128 &&
           (rows * splits < kResident / 3 || (twice && (rows < kResident / splits ? rows : kResident / splits) * vocab * (16 / per) > kInL2)))
        splits *= 2;
    return splits;
}

int launch_fwd(RowArgs& a, int dtype, cudaStream_t stream) {
    a.splits = splits_of(a.rows, a.vocab, dtype, a.dz != nullptr);
    return dtype == MGW_F32 ? launch_fwd<float>(a, stream) : dtype == MGW_F16 ? launch_fwd<__half>(a, stream) : launch_fwd<__nv_bfloat16>(a, stream);
}

}  // namespace

extern "C" int mgw_logprob_fwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide,
                               long long ignore, float* logprob, float* entropy, float* stats, int top, float* top_logprob,
                               long long* top_tokens, int* status, void* stream) {
    if (bad_rows(z, ld, rows, vocab, dtype, tokens) || top < 0 || top > kMaxTop || top > vocab) return MGW_ERR_ARG;
    if (rows == 0) return MGW_OK;
    if (logprob == nullptr || status == nullptr || ((uintptr_t)stats & 7) || (top > 0 && (top_logprob == nullptr || top_tokens == nullptr)))
        return MGW_ERR_ARG;
    RowArgs a = {};
    a.z = z; a.ld = ld; a.rows = rows; a.vocab = vocab; a.tokens = tokens; a.wide = wide; a.ignore = ignore;
    a.logprob = logprob; a.entropy = entropy; a.stats = reinterpret_cast<float2*>(stats);
    a.top = top; a.top_logprob = top_logprob; a.top_tokens = top_tokens; a.status = status;
    return launch_fwd(a, dtype, (cudaStream_t)stream);
}

extern "C" int mgw_logprob_bwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide,
                               long long ignore, const float* stats, const float* entropy, const float* g_logprob,
                               const float* g_entropy, const float* g_loss, const int* count, int written, float expected, void* dz,
                               long long dz_ld, void* stream) {
    if (bad_rows(z, ld, rows, vocab, dtype, tokens)) return MGW_ERR_ARG;
    if (rows == 0) return MGW_OK;
    if (stats == nullptr || dz == nullptr || (rows > 1 && dz_ld < vocab) || (g_entropy != nullptr && entropy == nullptr) ||
        (g_loss != nullptr && count == nullptr) || (written && g_loss == nullptr))
        return MGW_ERR_ARG;
    GradArgs a = {z, ld, rows, vocab, tokens, wide, ignore, reinterpret_cast<const float2*>(stats), g_entropy ? entropy : nullptr,
                  g_logprob, g_entropy, g_loss, count, written, expected, dz, dz_ld, splits_of(rows, vocab, dtype, false)};
    cudaStream_t s = (cudaStream_t)stream;
    const long long tasks = rows * a.splits;
    const unsigned grid = (unsigned)(tasks < 148 * 8 ? tasks : 148 * 8);
    if (dtype == MGW_F32) logprob_bwd_kernel<float><<<grid, kThreads, kRingBytes, s>>>(a);
    else if (dtype == MGW_F16) logprob_bwd_kernel<__half><<<grid, kThreads, kRingBytes, s>>>(a);
    else logprob_bwd_kernel<__nv_bfloat16><<<grid, kThreads, kRingBytes, s>>>(a);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}

// work: 8 bytes {number of rows in the mean, counter}, kept for mgw_logprob_bwd
extern "C" int mgw_cross_entropy_fwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide,
                                     long long ignore, int mean, float expected, float* logprob, float* stats, float* loss, void* dz,
                                     long long dz_ld, int* work, int* status, void* stream) {
    if (bad_rows(z, ld, rows, vocab, dtype, tokens) || loss == nullptr || work == nullptr) return MGW_ERR_ARG;
    if (rows > 0 && (logprob == nullptr || status == nullptr || ((uintptr_t)stats & 7) || (dz != nullptr && rows > 1 && dz_ld < vocab)))
        return MGW_ERR_ARG;
    cudaStream_t s = (cudaStream_t)stream;
    count_rows_kernel<<<1, 1024, 0, s>>>(tokens, wide, ignore, rows, mean, work, reinterpret_cast<unsigned int*>(work + 1), loss);
    MGW_CUDA_CHECK(cudaGetLastError());
    if (rows == 0) return MGW_OK;
    RowArgs a = {};
    a.z = z; a.ld = ld; a.rows = rows; a.vocab = vocab; a.tokens = tokens; a.wide = wide; a.ignore = ignore;
    a.logprob = logprob; a.stats = reinterpret_cast<float2*>(stats); a.status = status;
    a.dz = dz; a.dz_ld = dz_ld; a.expected = expected; a.count = work; a.done = reinterpret_cast<unsigned int*>(work + 1); a.loss = loss;
    return launch_fwd(a, dtype, s);
}
