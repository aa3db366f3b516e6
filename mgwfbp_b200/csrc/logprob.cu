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
// shared memory.  The likeliest tokens come out of the same pass: the largest value of every 32 neighbouring vectors
// (a "group") is kept in shared memory, and only the groups with the K largest of those maxima are looked at again.
#include <cooperative_groups.h>
#include "api.h"
#include "dtypes.cuh"

namespace {

namespace cg = cooperative_groups;

constexpr int kMaxTop = 32;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;
constexpr int kUnroll = 4;                 // 16-byte vectors that a thread keeps in flight
constexpr int kGroups = 4096;              // group maxima that a block keeps; neighbouring groups share one beyond that
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

__device__ __forceinline__ float exp2_fast(float x) {                // two units in the last place; 0 for very negative x
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Whole numbers in the order of the values; NaN above everything, the two zeros equal, never 0.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// The values of a 16-byte vector, raised to `low`, and their largest before that (NaN if there is one).
template <typename T> struct Vec;
template <> struct Vec<float> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float take(const uint4& r, float (&f)[4]) {
        f[0] = __uint_as_float(r.x); f[1] = __uint_as_float(r.y); f[2] = __uint_as_float(r.z); f[3] = __uint_as_float(r.w);
        const float m = max_nan(max_nan(f[0], f[1]), max_nan(f[2], f[3]));
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = max_nan(f[e], Fast<float>::low);
        return m;
    }
};
template <typename T, typename T2>
struct VecHalf {
    static constexpr int N = 8;
    static __device__ __forceinline__ float take(const uint4& r, float (&f)[8]) {
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
        T2 h[4], m, low;
        low.x = low.y = mgw_from_float<T>(Fast<T>::low);
#pragma unroll
        for (int k = 0; k < 4; ++k) h[k] = *reinterpret_cast<const T2*>(&w[k]);
        m = __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3]));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            h[k] = __hmax2_nan(h[k], low);
            f[2 * k] = mgw_to_float(h[k].x);
            f[2 * k + 1] = mgw_to_float(h[k].y);
        }
        return max_nan(mgw_to_float(m.x), mgw_to_float(m.y));
    }
};
template <> struct Vec<__half> : VecHalf<__half, __half2> {};
template <> struct Vec<__nv_bfloat16> : VecHalf<__nv_bfloat16, __nv_bfloat162> {};

struct Stats { float m, s, u; };

// Sums relative to the larger maximum.
template <bool ENT>
__device__ __forceinline__ void raise_to(Stats& a, float m) {
    // both products rounded, as M is everywhere: a fused subtraction would leave the rounding of the other one behind
    const float d = __fmul_rn(a.m, kLog2e) - __fmul_rn(m, kLog2e), f = exp2_fast(d);
    if (ENT) a.u = f * (a.u + a.s * d);
    a.s *= f;
    a.m = m;
}

template <bool ENT>
__device__ __forceinline__ Stats join(Stats a, Stats b) {
    const float m = max_nan(a.m, b.m);
    raise_to<ENT>(a, m);
    raise_to<ENT>(b, m);
    a.s += b.s;
    if (ENT) a.u += b.u;
    return a;
}

template <bool ENT, int N>
__device__ __forceinline__ void add_values(Stats& a, float M, const float (&f)[N]) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float d = fmaf(f[e], kLog2e, -M), x = exp2_fast(d);
        a.s += x;
        if (ENT) a.u = fmaf(x, d, a.u);
    }
}

template <bool ENT>
__device__ __forceinline__ Stats block_join(Stats x, Stats* parts) {
    for (int o = 16; o > 0; o >>= 1) {
        Stats y;
        y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
        y.s = __shfl_xor_sync(0xffffffffu, x.s, o);
        y.u = ENT ? __shfl_xor_sync(0xffffffffu, x.u, o) : 0.f;
        x = join<ENT>(x, y);
    }
    __syncthreads();
    if ((threadIdx.x & 31) == 0) parts[threadIdx.x >> 5] = x;
    __syncthreads();
    x = parts[0];
    for (int w = 1; w < kWarps; ++w) x = join<ENT>(x, parts[w]);
    return x;
}

// ------------------------------------------------------------------------------------------------ layout of a row
// Elements before the first 16-byte boundary (head), whole vectors, elements behind them (tail).  Groups: 0 the head,
// then 32 vectors each, the last one the tail; a block of a cluster has groups [g0, g1).
template <typename T>
struct Row {
    const T* z;
    int head, n_vec, tail0, vocab, groups;
    __device__ __forceinline__ Row(const T* z_, int vocab_) : z(z_), vocab(vocab_) {
        const int h = (int)(((16 - ((unsigned long long)z_ & 15)) & 15) / sizeof(T));
        head = min(h, vocab_);
        n_vec = (vocab_ - head) / Vec<T>::N;
        tail0 = head + n_vec * Vec<T>::N;
        groups = ((n_vec + 31) >> 5) + 2;
    }
    __device__ __forceinline__ uint4 vec(int i) const { return reinterpret_cast<const uint4*>(z + head)[i]; }
};

// Sums and group maxima of this block's groups.
template <typename T, bool ENT, bool TOP>
__device__ __forceinline__ Stats scan_row(const Row<T>& row, int g0, int g1, int shift, uint32_t* group_key) {
    constexpr int N = Vec<T>::N;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    Stats a = {Fast<T>::start, 0.f, 0.f};
    float M = a.m * kLog2e;
    const int b0 = max(g0, 1), b1 = min(g1, row.groups - 1);         // the groups of vectors among them
    for (int g = b0 + warp; g < b1; g += kWarps * kUnroll) {
        uint4 r[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const int i = (g + k * kWarps - 1) * 32 + lane;
            if (g + k * kWarps < b1 && i < row.n_vec) r[k] = row.vec(i);
        }
        float f[kUnroll][N], top[kUnroll], most = Fast<T>::start;
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) {
            const bool in = g + k * kWarps < b1 && (g + k * kWarps - 1) * 32 + lane < row.n_vec;
            if (in) {
                top[k] = Vec<T>::take(r[k], f[k]);
                most = max_nan(most, top[k]);
            } else {
                top[k] = -INFINITY;
#pragma unroll
                for (int e = 0; e < N; ++e) f[k][e] = Fast<T>::low;
            }
            if (TOP && g + k * kWarps < b1) {
                const uint32_t key = __reduce_max_sync(0xffffffffu, in ? order_key(top[k]) : 0u);
                if (lane == 0) {
                    if (shift == 0) group_key[g + k * kWarps - g0] = key;
                    else atomicMax(&group_key[(g + k * kWarps - g0) >> shift], key);
                }
            }
        }
        const float m = max_nan(a.m, most);
        if (m != a.m) {
            raise_to<ENT>(a, m);
            M = m * kLog2e;
        }
#pragma unroll
        for (int k = 0; k < kUnroll; ++k)
            if (g + k * kWarps < b1 && (g + k * kWarps - 1) * 32 + lane < row.n_vec) add_values<ENT, N>(a, M, f[k]);
    }
    // the few elements of head and tail: one per lane of the first warp
    if (warp == 0) {
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const int g = side == 0 ? 0 : row.groups - 1;
            if (g < g0 || g >= g1) continue;
            const int j = side == 0 ? lane : row.tail0 + lane;
            const bool in = j < (side == 0 ? row.head : row.vocab);
            const float v = in ? mgw_to_float(row.z[j]) : -INFINITY;
            if (TOP) {
                const uint32_t key = __reduce_max_sync(0xffffffffu, in ? order_key(v) : 0u);
                if (lane == 0) {
                    if (shift == 0) group_key[g - g0] = key;
                    else atomicMax(&group_key[(g - g0) >> shift], key);
                }
            }
            if (in) {
                const float m = max_nan(a.m, v);
                if (m != a.m) raise_to<ENT>(a, m);
                const float f[1] = {max_nan(v, Fast<T>::low)};
                add_values<ENT, 1>(a, a.m * kLog2e, f);
            }
        }
    }
    return a;
}

// A row whose maximum is at the edge of the type's range: differences first, minus infinity left out.  m may end up
// infinite or NaN; s and u are relative to m, u in bits.
template <typename T>
__device__ Stats careful_row(const T* z, int vocab, Stats* parts) {
    float m = -INFINITY;
    for (int j = threadIdx.x; j < vocab; j += kThreads) m = max_nan(m, mgw_to_float(z[j]));
    for (int o = 16; o > 0; o >>= 1) m = max_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
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
// A warp's list: the 32 largest keys seen so far, one per lane, largest first.  A key is the value's order and below
// it the complement of the index, so equal values are ordered by the lower index and no two keys are equal; 0 is none.
typedef unsigned long long Key;

__device__ __forceinline__ Key key_of(float v, int index) { return ((Key)order_key(v) << 32) | (0xffffffffu - (uint32_t)index); }

__device__ __forceinline__ Key sort_lanes(Key x) {                   // bitonic, descending
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const Key y = __shfl_xor_sync(0xffffffffu, x, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0);
            x = larger == (y > x) ? y : x;
        }
    return x;
}

__device__ __forceinline__ Key merge_lists(Key a, Key b) {           // both descending: the 32 largest of the 64
    const int lane = threadIdx.x & 31;
    const Key y = __shfl_sync(0xffffffffu, b, 31 - lane);
    Key x = a > y ? a : y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const Key z = __shfl_xor_sync(0xffffffffu, x, o);
        x = ((lane & o) == 0) == (z > x) ? z : x;
    }
    return x;
}

struct TopSpace {
    uint32_t group_key[kGroups];
    Key list[kWarps][32];
    Key chosen[32];                        // the groups to look at again, by their maxima
    Key candidate[kCandidates];
    int n_candidates;
};

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

// The elements of a group (of 2^shift neighbouring groups), one call of `use` per vector element and all lanes at once.
template <typename T, typename F>
__device__ __forceinline__ void for_group(const Row<T>& row, int local, int g0, int g1, int shift, F use) {
    const int lane = threadIdx.x & 31;
    const int from = g0 + (local << shift), to = min(g1, from + (1 << shift));
    for (int g = from; g < to; ++g) {
        if (g == 0 || g == row.groups - 1) {
            const int j = g == 0 ? lane : row.tail0 + lane;
            const bool in = j < (g == 0 ? row.head : row.vocab);
            use(in ? key_of(mgw_to_float(row.z[j]), j) : (Key)0);
            continue;
        }
        const int i = (g - 1) * 32 + lane;
        const bool in = i < row.n_vec;
        float f[Vec<T>::N];
        if (in) mgw_unpack<T, Vec<T>::N>(row.vec(i), f);
#pragma unroll
        for (int e = 0; e < Vec<T>::N; ++e) use(in ? key_of(f[e], row.head + i * Vec<T>::N + e) : (Key)0);
    }
}

// The largest keys of this block's groups, in the first warp (other warps return nothing of use).
template <typename T>
__device__ Key top_of_block(const Row<T>& row, int g0, int g1, int shift, int top, TopSpace* t) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int n = (g1 - g0 + (1 << shift) - 1) >> shift;
    Key mine = 0;
    for (int at = warp * 32; at < n; at += kThreads) {
        const Key k = at + lane < n && t->group_key[at + lane] != 0
                          ? ((Key)t->group_key[at + lane] << 32) | (0xffffffffu - (uint32_t)(at + lane)) : (Key)0;
        mine = merge_lists(mine, sort_lanes(k));
    }
    mine = join_lists(mine, t);
    if (warp == 0) t->chosen[lane] = lane < top ? mine : (Key)0;
    if (threadIdx.x == 0) t->n_candidates = 0;
    __syncthreads();
    // every wanted element is in one of these groups and not below the smallest of their maxima
    const uint32_t floor_key = (uint32_t)(t->chosen[top - 1] >> 32);
    for (int k = warp; k < top; k += kWarps) {
        const Key c = t->chosen[k];
        if (c == 0) break;
        for_group(row, (int)(0xffffffffu - (uint32_t)c), g0, g1, shift, [&](Key x) {
            const bool good = x != 0 && (uint32_t)(x >> 32) >= floor_key;
            const unsigned who = __ballot_sync(0xffffffffu, good);
            if (who == 0) return;
            int at = 0;
            if (lane == 0) at = atomicAdd(&t->n_candidates, __popc(who));
            at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1u));
            if (good && at < kCandidates) t->candidate[at] = x;
        });
    }
    __syncthreads();
    mine = 0;
    const int found = t->n_candidates;
    if (found <= kCandidates) {                                      // their order does not matter: keys are unique
        if (found <= 64) {
            if (warp == 0)
                for (int at = 0; at < found; at += 32) mine = merge_lists(mine, sort_lanes(at + lane < found ? t->candidate[at + lane] : (Key)0));
            return mine;
        }
        for (int at = warp * 32; at < found; at += kThreads)
            mine = merge_lists(mine, sort_lanes(at + lane < found ? t->candidate[at + lane] : (Key)0));
    } else {                                                         // many equal or rising values: go through the groups
        for (int k = warp; k < top; k += kWarps) {
            const Key c = t->chosen[k];
            if (c == 0) break;
            for_group(row, (int)(0xffffffffu - (uint32_t)c), g0, g1, shift, [&](Key x) {
                const Key least = __shfl_sync(0xffffffffu, mine, 31);
                if (__any_sync(0xffffffffu, x > least)) mine = merge_lists(mine, sort_lanes(x));
            });
        }
    }
    return join_lists(mine, t);
}

// ------------------------------------------------------------------------------------------------------------ forward
// One row (the columns of groups [g0, g1)) of a gradient: value(logit, column).  Whole vectors where logits and gradient
// start at the same place of a 16-byte block, single elements otherwise.  READ: the logits are needed.
template <typename T, bool READ, typename F>
__device__ __forceinline__ void write_row(const Row<T>& row, T* dz, int g0, int g1, F value) {
    constexpr int N = Vec<T>::N;
    const int v0 = (max(g0, 1) - 1) * 32, v1 = min(row.n_vec, (min(g1, row.groups - 1) - 1) * 32);
    if (((unsigned long long)dz & 15) == ((unsigned long long)row.z & 15)) {
        uint4* to = reinterpret_cast<uint4*>(dz + row.head);
        for (int i0 = v0 + threadIdx.x; i0 < v1; i0 += kThreads * kUnroll) {
            uint4 q[kUnroll];
#pragma unroll
            for (int k = 0; k < kUnroll; ++k)
                if (READ && i0 + k * kThreads < v1) q[k] = row.vec(i0 + k * kThreads);
#pragma unroll
            for (int k = 0; k < kUnroll; ++k) {
                const int i = i0 + k * kThreads;
                if (i >= v1) continue;
                float f[N];
                if (READ) mgw_unpack<T, N>(q[k], f);
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] = value(READ ? f[e] : 0.f, row.head + i * N + e);
                to[i] = mgw_pack<T, N>(f);
            }
        }
    } else {
        for (int j = row.head + v0 * N + threadIdx.x; j < row.head + v1 * N; j += kThreads)
            dz[j] = mgw_from_float<T>(value(READ ? mgw_to_float(row.z[j]) : 0.f, j));
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        const int g = side == 0 ? 0 : row.groups - 1, j = (side == 0 ? 0 : row.tail0) + threadIdx.x;
        if (g >= g0 && g < g1 && j < (side == 0 ? row.head : row.vocab))
            dz[j] = mgw_from_float<T>(value(READ ? mgw_to_float(row.z[j]) : 0.f, j));
    }
}

// g (p - delta), the gradient of one row's loss
template <typename T>
__device__ __forceinline__ void write_loss_gradient(const Row<T>& row, T* dz, int g0, int g1, float m, float log2_s, float g, long long t) {
    if (careful<T>(m)) {
        write_row<T, true>(row, dz, g0, g1, [=](float v, int j) {
            const float p = exp2_fast(log2_prob<T>(v, m, log2_s));
            return g * (j == t ? p - 1.f : p);
        });
        return;
    }
    const float M = m * kLog2e;
    write_row<T, true>(row, dz, g0, g1, [=](float v, int j) {
        const float p = exp2_fast(fmaf(v, kLog2e, -M) - log2_s);
        return g * (j == t ? p - 1.f : p);
    });
}

template <typename T>
__device__ __forceinline__ void write_constant(const Row<T>& row, T* dz, int g0, int g1, float c) {
    write_row<T, false>(row, dz, g0, g1, [=](float, int) { return c; });
}

template <typename T, bool ENT, bool TOP, bool LOSS>
__global__ void __launch_bounds__(kThreads) logprob_fwd_kernel(RowArgs a) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    TopSpace* top = reinterpret_cast<TopSpace*>(dynamic);            // only with TOP
    __shared__ Stats parts[kWarps];
    __shared__ Stats of_block;
    __shared__ Key block_list[32];
    const int part = blockIdx.x % a.splits;
    const long long r = blockIdx.x / a.splits;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long t = mgw_token(a.tokens, a.wide, r);
    const Row<T> row(static_cast<const T*>(a.z) + r * a.ld, a.vocab);
    const int per = (row.groups + a.splits - 1) / a.splits;
    const int g0 = min(row.groups, part * per), g1 = min(row.groups, g0 + per);
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
        if (LOSS && a.dz != nullptr) write_constant(row, static_cast<T*>(a.dz) + r * a.dz_ld, g0, g1, 0.f);
    } else {
        int shift = 0;
        if (TOP) {
            while (((g1 - g0) >> shift) >= kGroups) ++shift;
            if (shift > 0) {
                for (int k = threadIdx.x; k < kGroups; k += kThreads) top->group_key[k] = 0;
                __syncthreads();
            }
        }
        Stats x = block_join<ENT>(scan_row<T, ENT, TOP>(row, g0, g1, shift, top->group_key), parts);
        if (a.splits > 1) {
            cg::cluster_group cluster = cg::this_cluster();
            if (threadIdx.x == 0) of_block = x;
            cluster.sync();
            x = *cluster.map_shared_rank(&of_block, 0);
            for (int k = 1; k < a.splits; ++k) x = join<ENT>(x, *cluster.map_shared_rank(&of_block, k));
        }
        if (careful<T>(x.m)) x = careful_row(row.z, a.vocab, parts);
        const bool fine = fabsf(x.m) < INFINITY;
        const float log2_s = log2f(x.s);
        const bool valid = t >= 0 && t < a.vocab;
        if (part == 0 && threadIdx.x == 0) {
            if (!valid) mgw_report_token(a.status, MGW_OP_LOGPROB, r, t);
            a.logprob[r] = valid && fine ? ln_prob<T>(mgw_to_float(row.z[t]), x.m, log2_s) : mgw_nan();
            if (ENT && a.entropy) a.entropy[r] = fine ? kLn2 * (log2_s - x.u / x.s) : mgw_nan();
            if (a.stats) a.stats[r] = make_float2(fine ? x.m : mgw_nan(), log2_s);
        }
        if (TOP) {
            Key mine = top_of_block(row, g0, g1, shift, a.top, top);
            if (a.splits > 1) {
                cg::cluster_group cluster = cg::this_cluster();
                if (warp == 0) block_list[lane] = mine;
                cluster.sync();
                if (part == 0 && warp == 0)
                    for (int k = 1; k < a.splits; ++k) mine = merge_lists(mine, *cluster.map_shared_rank(&block_list[lane], k));
            }
            if (part == 0 && warp == 0 && lane < a.top) {
                const int j = (int)(0xffffffffu - (uint32_t)mine);
                a.top_tokens[r * a.top + lane] = j;
                a.top_logprob[r * a.top + lane] = fine ? ln_prob<T>(mgw_to_float(row.z[j]), x.m, log2_s) : mgw_nan();
            }
        }
        if (LOSS && a.dz != nullptr) {                               // the row was just read: it comes from L2
            T* dz = static_cast<T*>(a.dz) + r * a.dz_ld;
            if (fine && valid) write_loss_gradient(row, dz, g0, g1, x.m, log2_s, a.expected / (float)*a.count, t);
            else write_constant(row, dz, g0, g1, mgw_nan());
        }
        if (a.splits > 1) cg::this_cluster().sync();                 // until here the others may read this block's memory
    }
    if (LOSS && a.loss != nullptr && part == 0) {
        // the block that finishes last adds up the rows: thread i rows i, i + 256, ..., the same order every time
        __shared__ bool last;
        __shared__ double sums[kWarps];
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
__global__ void __launch_bounds__(kThreads) logprob_bwd_kernel(GradArgs a) {
    const float g_loss = a.g_loss != nullptr ? *a.g_loss : 0.f;
    if (a.written && g_loss == a.expected) return;
    for (long long task = blockIdx.x; task < a.rows * a.splits; task += gridDim.x) {
        const long long r = task / a.splits;
        const int part = (int)(task - r * a.splits);
        const long long t = mgw_token(a.tokens, a.wide, r);
        const Row<T> row(static_cast<const T*>(a.z) + r * a.ld, a.vocab);
        T* dz = static_cast<T*>(a.dz) + r * a.dz_ld;
        const int per = (row.groups + a.splits - 1) / a.splits;
        const int g0 = min(row.groups, part * per), g1 = min(row.groups, g0 + per);
        if (t == a.ignore) {
            write_constant(row, dz, g0, g1, 0.f);
            continue;
        }
        const float m = a.stats[r].x, log2_s = a.stats[r].y;
        if (t < 0 || t >= a.vocab || m != m) {
            write_constant(row, dz, g0, g1, mgw_nan());
            continue;
        }
        if (a.g_loss != nullptr) {
            write_loss_gradient(row, dz, g0, g1, m, log2_s, g_loss / (float)*a.count, t);
            continue;
        }
        // g1 (delta - p) - g2 p (ln p + H)
        const float h = a.entropy ? a.entropy[r] : 0.f, g1v = a.g_logprob ? a.g_logprob[r] : 0.f, g2 = a.g_entropy ? a.g_entropy[r] : 0.f;
        const float base = g1v + g2 * h, slope = g2 * kLn2, M = m * kLog2e;
        const bool edge = careful<T>(m);
        write_row<T, true>(row, dz, g0, g1, [=](float v, int j) {
            const float d = fmaxf((edge ? (v - m) * kLog2e : fmaf(v, kLog2e, -M)) - log2_s, -1e4f);      // p = 0 well before
            const float x = -exp2_fast(d) * fmaf(slope, d, base);
            return j == t ? x + g1v : x;
        });
    }
}

bool bad_rows(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens) {
    const int es = dtype == MGW_F32 ? 4 : 2;
    return rows < 0 || rows > 0x7fffffffLL || vocab < 1 || (rows > 1 && ld < vocab) || dtype < MGW_F32 || dtype > MGW_BF16 ||
           (rows > 0 && (z == nullptr || tokens == nullptr || ((uintptr_t)z & (es - 1))));
}

template <typename T, bool ENT, bool TOP, bool LOSS>
int launch_fwd(const RowArgs& a, cudaStream_t stream) {
    const size_t smem = TOP ? sizeof(TopSpace) : 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.rows * a.splits));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = a.splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = a.splits > 1 ? 1 : 0;
    MGW_CUDA_CHECK(cudaLaunchKernelEx(&cfg, logprob_fwd_kernel<T, ENT, TOP, LOSS>, a));
    return MGW_OK;
}

template <typename T>
int launch_fwd(const RowArgs& a, cudaStream_t stream) {
    if (a.loss != nullptr) return launch_fwd<T, false, false, true>(a, stream);
    return a.top > 0 ? launch_fwd<T, true, true, false>(a, stream) : launch_fwd<T, true, false, false>(a, stream);
}

// Blocks per row: one as long as the rows alone give two blocks to every SM, else up to 8 (a portable cluster) that have
// at least 128 vectors each.
int splits_of(long long rows, int vocab, int dtype) {
    const int per = dtype == MGW_F32 ? 4 : 8;
    int splits = 1;
    while (splits < 8 && rows * splits < 148 * 2 && vocab / per / (splits * 2) >= 128) splits *= 2;
    return splits;
}

int launch_fwd(RowArgs& a, int dtype, cudaStream_t stream) {
    a.splits = splits_of(a.rows, a.vocab, dtype);
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
                  g_logprob, g_entropy, g_loss, count, written, expected, dz, dz_ld, splits_of(rows, vocab, dtype)};
    cudaStream_t s = (cudaStream_t)stream;
    const long long tasks = rows * a.splits;
    const unsigned grid = (unsigned)(tasks < 148 * 8 ? tasks : 148 * 8);
    if (dtype == MGW_F32) logprob_bwd_kernel<float><<<grid, kThreads, 0, s>>>(a);
    else if (dtype == MGW_F16) logprob_bwd_kernel<__half><<<grid, kThreads, 0, s>>>(a);
    else logprob_bwd_kernel<__nv_bfloat16><<<grid, kThreads, 0, s>>>(a);
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
