// Log probabilities of given tokens, entropy and likeliest tokens of rows of logits, cross entropy, and their gradients.
//
// For a row z of V logits with largest value m:   s = sum exp(z_j - m),   u = sum exp(z_j - m) (z_j - m),
//   lse = m + ln s,   log p_j = z_j - lse,   H = -sum p_j log p_j = ln s - u / s,
//   d log p_t / d z_j = delta_jt - p_j,   d H / d z_j = -p_j (log p_j + H).
// All sums are held in fp32.  A logit of minus infinity has probability zero and adds nothing anywhere.  A row whose
// largest value is not finite (all minus infinity, a NaN, plus infinity) has no distribution: its results are NaN.
// Rows whose token is `ignore` are padding: their results and gradients are zero and their logits are not read.
#include "api.h"
#include "dtypes.cuh"

namespace {

constexpr int kMaxTop = 32;
constexpr int kThreads = 256;
constexpr int kWarps = kThreads / 32;

struct RowArgs {
    const void* z;
    long long ld, rows;
    int vocab;
    const void* tokens;
    int wide;
    long long ignore;
    float* logprob;
    float* entropy;            // may be null
    float2* stats;             // {m, ln s} for the backward pass, may be null
    int top;
    float* top_logprob;        // [rows, top]
    long long* top_tokens;
    int* status;
};

// Whole numbers in the order of the values; NaN above everything, the two zeros equal.
__device__ __forceinline__ uint32_t order_key(float x) {
    if (x != x) return 0xffffffffu;
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Stats { float m, s, u; };

// Two parts of a row put together: sums taken relative to the larger of the two maxima.
__device__ __forceinline__ Stats join(const Stats& a, const Stats& b) {
    Stats r;
    r.m = a.m > b.m || a.m != a.m ? a.m : b.m;
    if (r.m == -INFINITY) { r.s = 0.f; r.u = 0.f; return r; }
    const float da = fmaxf(a.m - r.m, -1e4f), db = fmaxf(b.m - r.m, -1e4f);       // an empty part has s = 0
    const float fa = expf(da), fb = expf(db);
    r.s = a.s * fa + b.s * fb;
    r.u = fa * (a.u + a.s * da) + fb * (b.u + b.s * db);
    return r;
}

__device__ __forceinline__ Stats join_lanes(Stats x) {
    for (int o = 16; o > 0; o >>= 1) {
        Stats y;
        y.m = __shfl_xor_sync(0xffffffffu, x.m, o);
        y.s = __shfl_xor_sync(0xffffffffu, x.s, o);
        y.u = __shfl_xor_sync(0xffffffffu, x.u, o);
        x = join(x, y);
    }
    return x;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_fwd_kernel(RowArgs a) {
    __shared__ Stats parts[kWarps];
    __shared__ unsigned long long best[kWarps];
    const long long row = blockIdx.x;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const long long t = mgw_token(a.tokens, a.wide, row);
    if (t == a.ignore) {
        if (threadIdx.x == 0) {
            a.logprob[row] = 0.f;
            if (a.entropy) a.entropy[row] = 0.f;
            if (a.stats) a.stats[row] = make_float2(0.f, 0.f);
        }
        for (int k = threadIdx.x; k < a.top; k += kThreads) {
            a.top_logprob[row * a.top + k] = 0.f;
            a.top_tokens[row * a.top + k] = -1;
        }
        return;
    }
    const T* z = static_cast<const T*>(a.z) + row * a.ld;
    Stats x = {-INFINITY, 0.f, 0.f};
    for (int j = threadIdx.x; j < a.vocab; j += kThreads) {
        const float v = mgw_to_float(z[j]);
        if (x.m == x.m && !(v <= x.m)) {                             // larger, or the first NaN
            const float d = fmaxf(x.m - v, -1e4f), f = expf(d);
            x.u = f * (x.u + x.s * d);
            x.s *= f;
            x.m = v;
        }
        const float d = fmaxf(v - x.m, -1e4f), e = v == -INFINITY ? 0.f : expf(d);
        x.s += e;
        x.u += e * d;
    }
    x = join_lanes(x);
    if (lane == 0) parts[warp] = x;
    __syncthreads();
    x = parts[0];
    for (int w = 1; w < kWarps; ++w) x = join(x, parts[w]);
    const bool fine = fabsf(x.m) < INFINITY;
    const float ln_s = logf(x.s);
    if (threadIdx.x == 0) {
        const bool valid = t >= 0 && t < a.vocab;
        if (!valid) mgw_report_token(a.status, MGW_OP_LOGPROB, row, t);
        a.logprob[row] = valid && fine ? (mgw_to_float(z[t]) - x.m) - ln_s : mgw_nan();
        if (a.entropy) a.entropy[row] = fine ? ln_s - x.u / x.s : mgw_nan();
        if (a.stats) a.stats[row] = make_float2(fine ? x.m : mgw_nan(), ln_s);
    }
    // the `top` largest values: the next one below the last, the lower index first
    unsigned long long below = ~0ull;
    for (int k = 0; k < a.top; ++k) {
        unsigned long long mine = 0;
        for (int j = threadIdx.x; j < a.vocab; j += kThreads) {
            const unsigned long long key = ((unsigned long long)order_key(mgw_to_float(z[j])) << 32) | (0xffffffffu - (uint32_t)j);
            if (key > mine && (k == 0 || key < below)) mine = key;
        }
        for (int o = 16; o > 0; o >>= 1) {
            const unsigned long long other = __shfl_xor_sync(0xffffffffu, mine, o);
            if (other > mine) mine = other;
        }
        __syncthreads();
        if (lane == 0) best[warp] = mine;
        __syncthreads();
        for (int w = 0; w < kWarps; ++w)
            if (best[w] > mine) mine = best[w];
        below = mine;
        if (threadIdx.x == 0) {
            const uint32_t j = 0xffffffffu - (uint32_t)mine;
            a.top_tokens[row * a.top + k] = j;
            a.top_logprob[row * a.top + k] = fine ? (mgw_to_float(z[j]) - x.m) - ln_s : mgw_nan();
        }
    }
}

struct GradArgs {
    const void* z;
    long long ld, rows;
    int vocab;
    const void* tokens;
    int wide;
    long long ignore;
    const float2* stats;       // {m, ln s}: kept apart, so that logits far from zero lose no digits
    const float* entropy;      // null: no gradient of the entropy
    const float* g_logprob;    // [rows], or null
    const float* g_entropy;    // [rows], or null
    const float* g_loss;       // one value: gradient of the mean loss, or null
    const float* count;        // rows that are not padding, for g_loss
    void* dz;
    long long dz_ld;
};

template <typename T>
__global__ void __launch_bounds__(kThreads) logprob_bwd_kernel(GradArgs a) {
    const long long row = blockIdx.x;
    const long long t = mgw_token(a.tokens, a.wide, row);
    T* dz = static_cast<T*>(a.dz) + row * a.dz_ld;
    if (t == a.ignore) {
        for (int j = threadIdx.x; j < a.vocab; j += kThreads) dz[j] = mgw_from_float<T>(0.f);
        return;
    }
    const T* z = static_cast<const T*>(a.z) + row * a.ld;
    const bool valid = t >= 0 && t < a.vocab;
    const float2 st = a.stats[row];
    const float m = valid ? st.x : mgw_nan(), ln_s = st.y;
    const float h = a.entropy ? a.entropy[row] : 0.f;
    float g1 = a.g_logprob ? a.g_logprob[row] : 0.f;
    if (a.g_loss) g1 = -(*a.g_loss / *a.count);
    const float g2 = a.g_entropy ? a.g_entropy[row] : 0.f;
    for (int j = threadIdx.x; j < a.vocab; j += kThreads) {
        const float d = m == m ? fmaxf((mgw_to_float(z[j]) - m) - ln_s, -1e4f) : mgw_nan();
        const float p = expf(d);
        float g = -p * (g1 + g2 * (d + h));
        if (j == t) g += g1;
        dz[j] = mgw_from_float<T>(g);
    }
}

// loss = -(sum of logprob) / count over the rows that are not padding, in one block: thread i sums rows i, i + 1024, ...
__global__ void __launch_bounds__(1024) mean_loss_kernel(const float* __restrict__ logprob, const void* __restrict__ tokens, int wide,
                                                         long long ignore, long long rows, int mean, float* __restrict__ loss,
                                                         float* __restrict__ count) {
    __shared__ double sums[32];
    __shared__ long long kept[32];
    double s = 0.0;
    long long k = 0;
    for (long long i = threadIdx.x; i < rows; i += 1024) {
        s += (double)logprob[i];                                     // zero where the row is padding
        k += mgw_token(tokens, wide, i) != ignore;
    }
    for (int o = 16; o > 0; o >>= 1) {
        s += __shfl_xor_sync(0xffffffffu, s, o);
        k += __shfl_xor_sync(0xffffffffu, k, o);
    }
    if ((threadIdx.x & 31) == 0) { sums[threadIdx.x >> 5] = s; kept[threadIdx.x >> 5] = k; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < 32; ++w) { s += sums[w]; k += kept[w]; }
        *count = mean ? (float)k : 1.f;
        *loss = (float)(-s / (mean ? (double)k : 1.0));              // no row left: 0 / 0, as the mean of nothing
    }
}

bool bad_rows(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens) {
    return rows < 0 || rows > 0x7fffffffLL || vocab < 1 || (rows > 1 && ld < vocab) || dtype < MGW_F32 || dtype > MGW_BF16 ||
           (rows > 0 && (z == nullptr || tokens == nullptr));
}

}  // namespace

extern "C" int mgw_logprob_fwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide,
                               long long ignore, float* logprob, float* entropy, float* stats, int top, float* top_logprob,
                               long long* top_tokens, int* status, void* stream) {
    if (bad_rows(z, ld, rows, vocab, dtype, tokens) || top < 0 || top > kMaxTop || top > vocab) return MGW_ERR_ARG;
    if (rows == 0) return MGW_OK;
    if (logprob == nullptr || status == nullptr || (top > 0 && (top_logprob == nullptr || top_tokens == nullptr))) return MGW_ERR_ARG;
    RowArgs a = {z, ld, rows, vocab, tokens, wide, ignore, logprob, entropy, reinterpret_cast<float2*>(stats), top, top_logprob, top_tokens, status};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == MGW_F32) logprob_fwd_kernel<float><<<(unsigned)rows, kThreads, 0, s>>>(a);
    else if (dtype == MGW_F16) logprob_fwd_kernel<__half><<<(unsigned)rows, kThreads, 0, s>>>(a);
    else logprob_fwd_kernel<__nv_bfloat16><<<(unsigned)rows, kThreads, 0, s>>>(a);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}

extern "C" int mgw_logprob_bwd(const void* z, long long ld, long long rows, int vocab, int dtype, const void* tokens, int wide,
                               long long ignore, const float* stats, const float* entropy, const float* g_logprob,
                               const float* g_entropy, const float* g_loss, const float* count, void* dz, long long dz_ld, void* stream) {
    if (bad_rows(z, ld, rows, vocab, dtype, tokens)) return MGW_ERR_ARG;
    if (rows == 0) return MGW_OK;
    if (stats == nullptr || dz == nullptr || (rows > 1 && dz_ld < vocab) || (g_entropy != nullptr && entropy == nullptr) ||
        (g_loss != nullptr && count == nullptr))
        return MGW_ERR_ARG;
    GradArgs a = {z, ld, rows, vocab, tokens, wide, ignore, reinterpret_cast<const float2*>(stats), g_entropy ? entropy : nullptr, g_logprob, g_entropy, g_loss, count, dz, dz_ld};
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == MGW_F32) logprob_bwd_kernel<float><<<(unsigned)rows, kThreads, 0, s>>>(a);
    else if (dtype == MGW_F16) logprob_bwd_kernel<__half><<<(unsigned)rows, kThreads, 0, s>>>(a);
    else logprob_bwd_kernel<__nv_bfloat16><<<(unsigned)rows, kThreads, 0, s>>>(a);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}

extern "C" int mgw_mean_loss(const float* logprob, const void* tokens, int wide, long long ignore, long long rows, int mean, float* loss,
                             float* count, void* stream) {
    if (rows < 0 || loss == nullptr || count == nullptr || (rows > 0 && (logprob == nullptr || tokens == nullptr))) return MGW_ERR_ARG;
    mean_loss_kernel<<<1, 1024, 0, (cudaStream_t)stream>>>(logprob, tokens, wide, ignore, rows, mean, loss, count);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}
