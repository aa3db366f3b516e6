// Global norm of many gradient tensors and their scaling to a largest norm, for any mix of fp32, fp16 and bf16.
//
//   n = |a g|,  g <- a c g  with  c = min(1, max_norm / (n + 1e-6))        a: factor of the caller, e.g. 1 / loss scale
//
// Two launches and no table in device memory: the tensors' addresses and lengths travel as kernel arguments (which a
// captured graph keeps), so nothing is uploaded and nothing has to be kept between calls.  The first launch leaves one sum
// per block, in the second every block adds those up for itself (in a fixed order, so that all get the same factor) and
// scales its part.  A thread adds the squares of the 16 or 32 values that it has in flight in fp32 and that sum to an
// fp64 total, so that hundreds of millions of values keep their digits; where the values' magnitude would let squares leave
// the range of fp32 (gradients of 1e-25 or 1e25 have a norm too), they are squared in fp64 instead.
//
// Both launches are bound by memory.  66 M fp32 values (264 MB): norm 41 us = 6.4 TB/s, scaling 86 us = 6.1 TB/s read and
// written; 25.6 M values (102 MB, mostly still in L2 for the second launch): 20 + 32 us.  Squaring everything in fp64 took
// 138 us for the norm (one block per SM: 72 registers, and a conversion for each value).  The scaling launch takes 128 us in
// all with two blocks of 512 threads per SM, 140 with one, and 170 with three (its 63 registers a thread no longer fit);
// stores that are marked as not read again are worth 1 %, the backward order of the second launch 2 %.
#include <algorithm>
#include <cstdio>
#include <new>
#include <vector>
#include "api.h"
#include "dtypes.cuh"

namespace {

constexpr int kThreads = 512;
constexpr int kUnroll = 4;                                  // 16-byte vectors that a thread keeps in flight
constexpr int kChunkBytes = kThreads * kUnroll * 16;        // the unit of work of a block
constexpr int kBlocks = 148 * 3;                            // three resident blocks per SM read ...
constexpr int kScaleBlocks = 148 * 2;                       // ... and two read and write

enum { kNorm2 = 0, kNorm1 = 1, kNormMax = 2 };

// Tensors of one launch.  A chunk is kChunkBytes of one tensor, counted from its first 16-byte boundary; chunk 0 has
// the elements before that boundary too.
template <int CAP>
struct ClipTable {
    int n, chunks;
    int first[CAP];                                         // number of the tensor's first chunk
    void* ptr[CAP];
    long long numel[CAP];
    unsigned char dtype[CAP];
};

struct Piece {                                              // one chunk: elements [e0, e1) of a tensor, whole vectors [v0, v1)
    char* base;
    long long e0, e1, v0, v1;                               // v0, v1: element indices, 16-byte aligned addresses
    int dtype;
};

template <int CAP>
__device__ __forceinline__ Piece piece_of(const ClipTable<CAP>& t, int chunk) {
    int lo = 0, hi = t.n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (t.first[mid] <= chunk) lo = mid; else hi = mid - 1;
    }
    Piece p;
    p.base = static_cast<char*>(t.ptr[lo]);
    p.dtype = t.dtype[lo];
    const int shift = p.dtype == MGW_F32 ? 2 : 1;
    const long long n = t.numel[lo];
    const long long head = ((16 - ((unsigned long long)p.base & 15)) & 15) >> shift;
    const long long c = chunk - t.first[lo], per = kChunkBytes >> shift;
    p.e0 = c == 0 ? 0 : head + c * per;
    p.e1 = min(n, head + (c + 1) * per);
    p.v0 = min(p.e1, head + c * per);
    p.v1 = p.v0 + (((p.e1 - p.v0) << shift) >> 4 << 4 >> shift);
    return p;
}

template <int NORM>
__device__ __forceinline__ void add_value(double& acc, float x) {
    if (NORM == kNorm2) acc = fma((double)x, (double)x, acc);
    else if (NORM == kNorm1) acc += (double)fabsf(x);
    else acc = !(fabsf(x) <= acc) && acc == acc ? (double)fabsf(x) : acc;      // the largest; a NaN stays
}

template <int NORM>
__device__ __forceinline__ double join_values(double a, double b) {
    if (NORM != kNormMax) return a + b;
    return !(b <= a) && a == a ? b : a;
}

// The values of one thread's vectors.  Two-norm: with the largest magnitude in (2^-40, 2^50) no sum of 32 squares
// overflows, and what underflows is below 2^-46 of the largest square.
template <int NORM, int N>
__device__ __forceinline__ void add_batch(double& acc, const float (&f)[N], float most, float sum) {
    if (NORM == kNorm2) {
        if (most > 0x1p-40f && most < 0x1p50f) {
            acc += (double)sum;
            return;
        }
        if (most == 0.f) return;
    } else if (NORM == kNorm1 && most < 0x1p100f) {
        acc += (double)sum;
        return;
    }
#pragma unroll
    for (int e = 0; e < N; ++e) add_value<NORM>(acc, f[e]);
}

__device__ __forceinline__ float max_nan(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

template <typename T, int NORM>
__device__ __forceinline__ void sum_piece(const Piece& p, double& acc) {
    constexpr int V = 16 / sizeof(T);
    const T* x = reinterpret_cast<const T*>(p.base);
    const uint4* src = reinterpret_cast<const uint4*>(x + p.v0);
    const int vecs = (int)((p.v1 - p.v0) / V);
    uint4 r[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        r[k] = make_uint4(0, 0, 0, 0);
        if (threadIdx.x + k * kThreads < vecs) r[k] = src[threadIdx.x + k * kThreads];
    }
    float f[kUnroll * V], most = 0.f, sum = 0.f;
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        float g[V];
        mgw_unpack<T, V>(r[k], g);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            f[k * V + e] = g[e];
            most = max_nan(most, fabsf(g[e]));
            if (NORM == kNorm2) sum = fmaf(g[e], g[e], sum);
            else if (NORM == kNorm1) sum += fabsf(g[e]);
        }
    }
    if (NORM == kNormMax) acc = join_values<NORM>(acc, (double)most);
    else add_batch<NORM>(acc, f, most, sum);
    const long long head = p.v0 - p.e0, edge = head + (p.e1 - p.v1);           // fewer than 8 elements on either side
    if (threadIdx.x < edge) add_value<NORM>(acc, mgw_to_float(x[threadIdx.x < head ? p.e0 + threadIdx.x : p.v1 + threadIdx.x - head]));
}

template <int NORM>
__device__ __forceinline__ double block_join(double v, double* red) {
    for (int o = 16; o > 0; o >>= 1) v = join_values<NORM>(v, __shfl_xor_sync(0xffffffffu, v, o));
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = red[0];
    for (int w = 1; w < kThreads / 32; ++w) v = join_values<NORM>(v, red[w]);
    return v;
}

template <int CAP, int NORM>
__global__ void __launch_bounds__(kThreads, 3) norm_kernel(const __grid_constant__ ClipTable<CAP> t, double* __restrict__ partials) {
    __shared__ double red[kThreads / 32];
    double acc = 0.0;
    for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
        const Piece p = piece_of(t, c);
        if (p.dtype == MGW_F32) sum_piece<float, NORM>(p, acc);
        else if (p.dtype == MGW_F16) sum_piece<__half, NORM>(p, acc);
        else sum_piece<__nv_bfloat16, NORM>(p, acc);
    }
    const double v = block_join<NORM>(acc, red);
    if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

template <int NORM>
__device__ __forceinline__ double norm_of(const double* __restrict__ partials, int n, double scale, double* red) {
    double v = 0.0;
    for (int i = threadIdx.x; i < n; i += kThreads) v = join_values<NORM>(v, partials[i]);
    v = block_join<NORM>(v, red);
    return fabs(scale) * (NORM == kNorm2 ? sqrt(v) : v);
}

template <typename T>
__device__ __forceinline__ void scale_piece(const Piece& p, float factor, float rest) {
    constexpr int V = 16 / sizeof(T);
    T* x = reinterpret_cast<T*>(p.base);
    uint4* at = reinterpret_cast<uint4*>(x + p.v0);
    const int vecs = (int)((p.v1 - p.v0) / V);
    uint4 r[kUnroll];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k)
        if (threadIdx.x + k * kThreads < vecs) r[k] = at[threadIdx.x + k * kThreads];
#pragma unroll
    for (int k = 0; k < kUnroll; ++k) {
        if (threadIdx.x + k * kThreads >= vecs) continue;
        float f[V];
        mgw_unpack<T, V>(r[k], f);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = f[e] * factor * rest;
        __stcs(&at[threadIdx.x + k * kThreads], mgw_pack<T, V>(f));
    }
    const long long head = p.v0 - p.e0, edge = head + (p.e1 - p.v1);
    if (threadIdx.x < edge) {
        T* q = x + (threadIdx.x < head ? p.e0 + threadIdx.x : p.v1 + threadIdx.x - head);
        *q = mgw_from_float<T>(mgw_to_float(*q) * factor * rest);
    }
}

template <int CAP, int NORM>
__global__ void __launch_bounds__(kThreads, 2) scale_kernel(const __grid_constant__ ClipTable<CAP> t, const double* __restrict__ partials,
                                                         int n_partials, double scale, double max_norm, float* __restrict__ norm_out) {
    __shared__ double red[kThreads / 32];
    const double norm = norm_of<NORM>(partials, n_partials, scale, red);
    if (blockIdx.x == 0 && threadIdx.x == 0 && norm_out != nullptr) *norm_out = (float)norm;
    double c = max_norm / (norm + 1e-6);
    if (c > 1.0) c = 1.0;                                   // a NaN norm gives NaN gradients, an infinite one zeros
    // Gradients near the largest fp32 value need a factor below the smallest normal one: it is applied in two parts, the
    // second a power of two (exact), so that it keeps its digits.
    const bool small = scale * c < 0x1p-100;
    const float factor = (float)(small ? scale * c * 0x1p64 : scale * c), rest = small ? 0x1p-64f : 1.f;
    if (c == 1.0 && scale == 1.0) return;                   // a norm within the limit: nothing to change
    // from the end: what the first launch read last is still in L2
    for (int i = t.chunks - 1 - (int)blockIdx.x; i >= 0; i -= (int)gridDim.x) {
        const Piece p = piece_of(t, i);
        if (p.dtype == MGW_F32) scale_piece<float>(p, factor, rest);
        else if (p.dtype == MGW_F16) scale_piece<__half>(p, factor, rest);
        else scale_piece<__nv_bfloat16>(p, factor, rest);
    }
}

template <int NORM>
__global__ void __launch_bounds__(kThreads) finish_kernel(const double* __restrict__ partials, int n_partials, double scale,
                                                          float* __restrict__ norm_out) {
    __shared__ double red[kThreads / 32];
    const double norm = norm_of<NORM>(partials, n_partials, scale, red);
    if (threadIdx.x == 0) *norm_out = (float)norm;
}

struct Tensor {
    void* ptr;
    long long numel;
    int dtype;
};

int chunks_of(const Tensor& t) {
    const int es = t.dtype == MGW_F32 ? 4 : 2;
    const long long head = ((16 - ((unsigned long long)(uintptr_t)t.ptr & 15)) & 15) / es, per = kChunkBytes / es;
    return t.numel <= head ? 1 : (int)((t.numel - head + per - 1) / per);
}

struct Call {
    const Tensor* t;
    int n;
    double* partials;
    double scale, max_norm;
    float* norm_out;
    bool clip;
    cudaStream_t stream;
};

template <int CAP>
void fill(ClipTable<CAP>& table, const Tensor* t, int n) {
    table.n = n;
    table.chunks = 0;
    for (int i = 0; i < n; ++i) {
        table.first[i] = table.chunks;
        table.ptr[i] = t[i].ptr;
        table.numel[i] = t[i].numel;
        table.dtype[i] = (unsigned char)t[i].dtype;
        table.chunks += chunks_of(t[i]);
    }
}

template <int CAP, int NORM>
int launch(const Call& c) {
    ClipTable<CAP> table;
    int n_partials = 0;
    for (int at = 0; at < c.n; at += CAP) {
        fill(table, c.t + at, std::min(CAP, c.n - at));
        const int grid = std::min(kBlocks, table.chunks);
        norm_kernel<CAP, NORM><<<grid, kThreads, 0, c.stream>>>(table, c.partials + n_partials);
        MGW_CUDA_CHECK(cudaGetLastError());
        n_partials += grid;
    }
    if (!c.clip) {
        finish_kernel<NORM><<<1, kThreads, 0, c.stream>>>(c.partials, n_partials, c.scale, c.norm_out);
        MGW_CUDA_CHECK(cudaGetLastError());
        return MGW_OK;
    }
    for (int at = 0; at < c.n; at += CAP) {
        if (c.n > CAP) fill(table, c.t + at, std::min(CAP, c.n - at));
        scale_kernel<CAP, NORM><<<std::min(kScaleBlocks, table.chunks), kThreads, 0, c.stream>>>(table, c.partials, n_partials, c.scale, c.max_norm,
                                                                                         at == 0 ? c.norm_out : nullptr);
        MGW_CUDA_CHECK(cudaGetLastError());
    }
    return MGW_OK;
}

template <int CAP>
int launch_norm(const Call& c, int norm) {
    return norm == kNorm2 ? launch<CAP, kNorm2>(c) : norm == kNorm1 ? launch<CAP, kNorm1>(c) : launch<CAP, kNormMax>(c);
}

constexpr int kSmall = 64, kMedium = 256, kLarge = 1024;    // tensors per launch: kernel arguments of 1.4, 5.4 and 21 KB

int fail(const char* text) {
    mgw_set_last_error(cudaErrorInvalidValue, text, __FILE__, __LINE__);
    return MGW_ERR_ARG;
}

}  // namespace

extern "C" size_t mgw_grad_clip_bytes(int n) {
    return n < 1 ? 8 : (size_t)((n + kSmall - 1) / kSmall) * kBlocks * sizeof(double);
}

// Tensors listed twice (same address, length and type) count once; tensors that share memory in any other way are refused.
extern "C" int mgw_grad_clip(const unsigned long long* ptrs, const long long* numels, const unsigned char* dtypes, int n, int norm,
                             double scale, double max_norm, int clip, void* work, size_t work_bytes, float* norm_out, void* stream) {
    if (n < 0 || norm < kNorm2 || norm > kNormMax || norm_out == nullptr || (n > 0 && (ptrs == nullptr || numels == nullptr || dtypes == nullptr)))
        return fail("arguments");
    if (work == nullptr || ((uintptr_t)work & 7) || work_bytes < mgw_grad_clip_bytes(n)) return fail("work area");
    try {
        std::vector<Tensor> t;
        t.reserve(n);
        for (int i = 0; i < n; ++i) {
            if (numels[i] == 0) continue;
            if (numels[i] < 0 || numels[i] > (1LL << 40) || dtypes[i] > MGW_BF16 || ptrs[i] == 0 ||
                (ptrs[i] & (dtypes[i] == MGW_F32 ? 3 : 1)))
                return fail("a tensor's address, length or type");
            t.push_back(Tensor{reinterpret_cast<void*>((uintptr_t)ptrs[i]), numels[i], dtypes[i]});
        }
        std::vector<int> order(t.size());
        for (size_t i = 0; i < order.size(); ++i) order[i] = (int)i;
        // gradients mostly come in the order of their addresses (one merged buffer, one backward pass)
        const auto before = [&](int a, int b) { return t[a].ptr < t[b].ptr || (t[a].ptr == t[b].ptr && a < b); };
        if (!std::is_sorted(order.begin(), order.end(), before)) std::sort(order.begin(), order.end(), before);
        std::vector<char> drop(t.size(), 0);
        uintptr_t end = 0;
        for (size_t k = 0; k < order.size(); ++k) {
            const Tensor& x = t[order[k]];
            const uintptr_t at = (uintptr_t)x.ptr;
            if (k > 0 && at < end) {
                const Tensor& y = t[order[k - 1]];
                if (y.ptr != x.ptr || y.numel != x.numel || y.dtype != x.dtype) return fail("two gradients share memory in part");
                drop[order[k]] = 1;
            }
            end = at + (uintptr_t)x.numel * (x.dtype == MGW_F32 ? 4 : 2);
        }
        size_t m = 0;
        long long chunks = 0;
        for (size_t i = 0; i < t.size(); ++i)
            if (!drop[i]) {
                chunks += chunks_of(t[i]);
                t[m++] = t[i];
            }
        if (chunks > 0x7fffffffLL) return fail("more than 2^31 chunks of 32 KB");
        const Call c = {t.data(), (int)m, static_cast<double*>(work), scale, max_norm, norm_out, clip != 0 && m > 0, (cudaStream_t)stream};
        return m <= (size_t)kSmall ? launch_norm<kSmall>(c, norm) : m <= (size_t)kMedium ? launch_norm<kMedium>(c, norm) : launch_norm<kLarge>(c, norm);
    } catch (const std::bad_alloc&) {
        return fail("out of host memory");
    }
}
