// Embedding lookup with scaling, and the dense gradient of the table by sorted tokens.
//
//   out[i, :] = scale * W[t_i, :]                      dW[v, :] = scale * sum over i with t_i = v of dy[i, :]
//
// The gradient's sums are taken in fp32 in the order of the positions i, so the result does not depend on how blocks
// are scheduled, and rounded once: the tokens are sorted (stable), the sorted list is cut into chunks of equal length --
// however often a single word occurs -- and a warp adds up the rows of one chunk for 512 bytes of columns.  A run of equal
// tokens inside a chunk is stored at once.  A run that crosses the borders of chunks is put together in the order of the
// chunks, in shared memory within a block and through fp32 partial sums and a second launch between blocks.  Rows that no
// token names are filled with zeros by other blocks of the same launch, beside the sort where they can; or the
// sort runs beside a long lookup, whose launch then leaves the sorted list for the gradient.
//
// Everything here is bound by memory once the lists are long: 262,144 rows of 2048 bf16 values of a table of 131,072 take
// 221 us to look up (1.3 GB, 6.0 TB/s) and 305 us to add up (1.6 GB, 5.3 TB/s; of it 40 us are the sort, which has nothing
// to hide behind).  700 rows of 1500 fp32 values of a table of 10,000: 2.7 + 14 us, the latter 64 MB of which 60 MB are zeros.
#include <cooperative_groups.h>
#include <atomic>
#include <mutex>
#include "api.h"
#include "dtypes.cuh"

namespace {

namespace cg = cooperative_groups;

// The kernels of the gradient follow each other closely: each is launched while the one before still runs.
template <typename... P, typename... A>
int launch_dependent(void (*kernel)(P...), long long grid, int threads, size_t smem, cudaStream_t stream, A... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    MGW_CUDA_CHECK(cudaLaunchKernelEx(&cfg, kernel, args...));
    return MGW_OK;
}

// A tile of the radix sort: 2048 entries by 512 threads (by 256 threads with 8 each a pass of 262,144 entries took 15 us
// instead of 9).
constexpr int kSortThreads = 512;
constexpr int kSortItems = 4;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigitBits = 10;

// --------------------------------------------------------------------------------------------------- blocks of a row
// How a warp moves 512 bytes of a row, 16 for each lane:
//   kExact  all rows of both matrices begin on 16-byte boundaries and consist of whole blocks of 16 bytes, one per lane;
//   kWords  rows begin and end on 4-byte boundaries: a lane has four words, 32 words apart, which moves whole lines as well
//           and needs no shifting.  200,000 rows of 1023 fp32 values: gradient 210 us, lookup 165 us (rows of 1024, kExact:
//           199 and 155 us; the rows of 1023 by kShift: 259 and 214 us);
//   kShift  anything else (16-bit types, odd widths): blocks are cut out of two aligned vectors when they are read, and put
//           together from two lanes' values when they are stored.  20,011 rows of 1023 fp16 values: lookup 17 us, 23 us with
//           single 16-bit accesses (rows of 1024: 11 us).
enum { kExact = 0, kWords = 1, kShift = 2 };

template <typename T> constexpr int per_block() { return 16 / (int)sizeof(T); }

// Elements between the last 16-byte boundary and the row.
template <typename T>
__device__ __forceinline__ int lead_of(const T* row) { return (int)(((unsigned long long)row & 15) / sizeof(T)); }

struct Cut { uint4 x, y; int at; };        // 16 bytes from byte `at` of the 32 in x, y

// Whether the vectors around every block of a row lie in the matrix [lo, hi), also those that its edges are cut out of.
template <typename T>
__device__ __forceinline__ bool inside(const T* row, int dim, const char* lo, const char* hi) {
    return reinterpret_cast<const char*>(row) - 31 >= lo && reinterpret_cast<const char*>(row + dim) + 32 <= hi;
}

// Elements from one word of a lane to its next, and the first column of a lane in the row's 512-byte part `part`.
template <typename T> constexpr int word_step() { return 128 / (int)sizeof(T); }
template <typename T, int MODE>
__device__ __forceinline__ int column_of(int part, int lane) {
    return part * 32 * per_block<T>() + lane * (MODE == kWords ? 4 / (int)sizeof(T) : per_block<T>());
}

// A lane's values from column c0 on.  kShift: c0 may be up to N - 1 below the row's first column, or in its last block.
template <typename T, int MODE>
__device__ __forceinline__ Cut load_block(const T* row, int c0, int dim) {
    Cut r;
    r.at = 0;
    const char* s = reinterpret_cast<const char*>(row + c0);
    if (MODE == kWords) {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(s);
        r.x.x = c0 < dim ? w[0] : 0u;
        r.x.y = c0 + word_step<T>() < dim ? w[32] : 0u;
        r.x.z = c0 + 2 * word_step<T>() < dim ? w[64] : 0u;
        r.x.w = c0 + 3 * word_step<T>() < dim ? w[96] : 0u;
        return r;
    }
    if (MODE == kShift) r.at = (int)((unsigned long long)s & 15);
    r.x = *reinterpret_cast<const uint4*>(s - r.at);
    if (MODE == kShift) r.y = *reinterpret_cast<const uint4*>(s - r.at + 16);
    return r;
}

// The same for a row at the ends of the matrix: element by element, zero outside [0, dim).
template <typename T>
__device__ __noinline__ uint4 gather_block(const T* row, int c0, int dim) {
    MgwVec<T, per_block<T>()> v;
    v.raw = make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int e = 0; e < per_block<T>(); ++e)
        if (c0 + e >= 0 && c0 + e < dim) v.v[e] = row[c0 + e];
    return v.raw;
}

// The block that a Cut holds.  (Selects instead of a branch for each offset: these kernels are large enough that a copy
// of their inner loop for each offset costs more in instruction fetches than it saves.)
template <int MODE>
__device__ __forceinline__ uint4 take(const Cut& c) {
    if (MODE != kShift) return c.x;
    const uint32_t bits = (c.at & 3) * 8;
    const bool two = c.at & 8, one = c.at & 4;
    const uint32_t a0 = two ? c.x.z : c.x.x, a1 = two ? c.x.w : c.x.y, a2 = two ? c.y.x : c.x.z, a3 = two ? c.y.y : c.x.w,
                   a4 = two ? c.y.z : c.y.x, a5 = two ? c.y.w : c.y.y;
    const uint32_t b0 = one ? a1 : a0, b1 = one ? a2 : a1, b2 = one ? a3 : a2, b3 = one ? a4 : a3, b4 = one ? a5 : a4;
    return make_uint4(__funnelshift_r(b0, b1, bits), __funnelshift_r(b1, b2, bits), __funnelshift_r(b2, b3, bits),
                      __funnelshift_r(b3, b4, bits));
}

// The elements [begin, stop) of a block (of a 16-bit type) at a 16-byte boundary: one store for a whole block, else up to three towards the
// middle and three behind it, each as wide as its place allows.
template <typename T>
__device__ __forceinline__ void store_part(T* at, const uint4& v, int begin, int stop) {
    if (begin <= 0 && stop >= 8) {
        __stcs(reinterpret_cast<uint4*>(at), v);
        return;
    }
    auto word = [&](int e) { return e & 4 ? (e & 2 ? v.w : v.z) : (e & 2 ? v.y : v.x); };
    char* p = reinterpret_cast<char*>(at);
    int e = max(begin, 0);
    stop = min(stop, 8);
    if (e & 1 && e < stop) { *reinterpret_cast<uint16_t*>(p + 2 * e) = (uint16_t)(word(e) >> 16); ++e; }
    if (e & 2 && e + 2 <= stop) { *reinterpret_cast<uint32_t*>(p + 2 * e) = word(e); e += 2; }
    if (e == 4 && stop == 8) { *reinterpret_cast<uint2*>(p + 8) = make_uint2(v.z, v.w); return; }
    if (e == 0 && stop >= 4) { *reinterpret_cast<uint2*>(p) = make_uint2(v.x, v.y); e = 4; }
    if (e + 2 <= stop) { *reinterpret_cast<uint32_t*>(p + 2 * e) = word(e); e += 2; }
    if (e < stop) *reinterpret_cast<uint16_t*>(p + 2 * e) = (uint16_t)word(e);
}

template <typename T>
__device__ __forceinline__ void store_words(T* row, int c0, int dim, const uint4& v) {
    uint32_t* w = reinterpret_cast<uint32_t*>(row + c0);
    if (c0 < dim) __stcs(w, v.x);
    if (c0 + word_step<T>() < dim) __stcs(w + 32, v.y);
    if (c0 + 2 * word_step<T>() < dim) __stcs(w + 64, v.z);
    if (c0 + 3 * word_step<T>() < dim) __stcs(w + 96, v.w);
}

// A lane's values from column c0 on; kShift: the part in [0, dim) of a block that begins on a boundary.
template <typename T, int MODE>
__device__ __forceinline__ void store_block(T* row, int c0, int dim, const uint4& v) {
    if constexpr (MODE == kExact) __stcs(reinterpret_cast<uint4*>(row + c0), v);
    else if constexpr (MODE == kWords) store_words(row, c0, dim, v);
    else store_part(row + c0, v, -c0, dim - c0);
}

// A warp's part of a row, the lane's values from column c0 on (all lanes take part; those with c0 >= dim have nothing).
// kShift: with the row `lead` elements behind a boundary, a lane stores the block that begins `lead` before its own: the last elements of
// the lane before it and its own first ones.
template <typename T, int MODE>
__device__ __forceinline__ void store_blocks(T* row, int c0, int dim, const uint4& v) {
    if constexpr (MODE != kShift) {
        if (c0 < dim) store_block<T, MODE>(row, c0, dim, v);
    } else {
        constexpr int N = per_block<T>();
        const int lane = threadIdx.x & 31, lead = lead_of(row), at = c0 - lead;
        Cut c;
        c.x.x = __shfl_up_sync(0xffffffffu, v.x, 1);
        c.x.y = __shfl_up_sync(0xffffffffu, v.y, 1);
        c.x.z = __shfl_up_sync(0xffffffffu, v.z, 1);
        c.x.w = __shfl_up_sync(0xffffffffu, v.w, 1);
        c.y = v;
        c.at = 16 - lead * (int)sizeof(T);                            // 16: the own block
        if (at < dim) store_part(row + at, lead == 0 ? v : take<kShift>(c), lane == 0 ? lead : 0, dim - at);
        if (lane == 31 && lead > 0 && at + N < dim) {                 // nobody comes behind it
            c.x = v;
            store_part(row + at + N, take<kShift>(c), 0, min(lead, dim - at - N));
        }
    }
}

// ------------------------------------------------------------------------------------------------------------ lookup
// Blocks that a lane keeps in flight; one more for rows between boundaries, which may have a block more than their length.
constexpr int lookup_unroll(int mode) { return mode == kShift ? 5 : 4; }

template <typename T, int MODE>
__global__ void __launch_bounds__(256, 3)
embedding_fwd_kernel(const void* __restrict__ tokens, int wide, long long n, const T* __restrict__ weight, long long ld,
                     long long vocab, int dim, float scale, T* __restrict__ out, int segments, int beside_sort, int* status) {
    constexpr int N = per_block<T>(), U = lookup_unroll(MODE);
    const int lane = threadIdx.x & 31;
    const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
    const char* lo = reinterpret_cast<const char*>(weight);
    const char* hi = reinterpret_cast<const char*>(weight + (vocab - 1) * ld + dim);
    for (long long task = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); task < n * segments; task += warps) {
        const long long i = segments == 1 ? task : task / segments;
        const int seg = (int)(task - i * segments);
        const long long t = mgw_token(tokens, wide, i);
        T* dst = out + i * dim;
        const bool valid = t >= 0 && t < vocab;
        if (!valid && lane == 0 && seg == 0) mgw_report_token(status, MGW_OP_EMBEDDING, i, t);
        const T* src = weight + (valid ? t : 0) * ld;
        auto put = [&](uint4 v, int c) {                             // blocks begin on boundaries of the output
            if (!valid || scale != 1.f) {                            // a factor of one copies the bits
                float f[N];
                mgw_unpack<T, N>(v, f);
#pragma unroll
                for (int e = 0; e < N; ++e) f[e] = valid ? f[e] * scale : mgw_nan();
                v = mgw_pack<T, N>(f);
            }
            store_block<T, MODE>(dst, c, dim, v);
        };
        const int c = column_of<T, MODE>(seg * U, lane) - (MODE == kShift ? lead_of(dst) : 0);
        if (MODE != kShift || inside(src, dim, lo, hi)) {
            Cut r[U];
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (c + 32 * N * k < dim) r[k] = load_block<T, MODE>(src, c + 32 * N * k, dim);
#pragma unroll
            for (int k = 0; k < U; ++k)
                if (c + 32 * N * k < dim) put(take<MODE>(r[k]), c + 32 * N * k);
        } else {
#pragma unroll 1
            for (int k = 0; k < U; ++k)
                if (c + 32 * N * k < dim) put(gather_block(src, c + 32 * N * k, dim), c + 32 * N * k);
        }
    }
    // the sort was launched first and may still run: what follows this launch in the stream follows the sort too
    if (beside_sort && blockIdx.x == gridDim.x - 1) mgw_wait_for_previous();
}

// -------------------------------------------------------------------------------------------------------------- sort
// Least-significant-digit radix sort of (token, position): per pass a histogram of every tile, a scan over the tiles
// for each digit, and a stable scatter.  Tokens outside the vocabulary and the padding token get the key `vocab`: they
// end up behind all others and take part in no sum.
struct SortPass {
    const void* tokens;        // first pass: the tokens themselves
    int wide;
    const uint2* in;           // later passes: {key, position} (null in the first)
    uint2* out;
    uint32_t* counts;          // [bins][tiles], in the scatter: counts of the tiles before
    uint32_t* totals;          // [bins]
    long long n;
    int tiles, shift, bits;
    long long vocab, padding;
    int* status;               // may be null: nothing is reported
};

__device__ __forceinline__ uint2 sort_entry(const SortPass& p, long long i, bool report) {
    if (p.in != nullptr) return p.in[i];
    const long long t = mgw_token(p.tokens, p.wide, i);
    if (t < 0 || t >= p.vocab) {
        if (report && p.status != nullptr) mgw_report_token(p.status, MGW_OP_EMBEDDING_GRAD, i, t);
        return make_uint2((uint32_t)p.vocab, (uint32_t)i);
    }
    return make_uint2(t == p.padding ? (uint32_t)p.vocab : (uint32_t)t, (uint32_t)i);
}

__global__ void __launch_bounds__(kSortThreads) sort_hist_kernel(SortPass p) {
    extern __shared__ uint32_t hist[];
    const int bins = 1 << p.bits;
    mgw_let_next_start();
    mgw_wait_for_previous();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) hist[b] = 0;
    __syncthreads();
    const long long i0 = (long long)blockIdx.x * kSortTile;
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        const long long i = i0 + j * kSortThreads + threadIdx.x;
        if (i < p.n) atomicAdd(&hist[(sort_entry(p, i, true).x >> p.shift) & (bins - 1)], 1u);      // whole numbers: any order
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) p.counts[(long long)b * p.tiles + blockIdx.x] = hist[b];
}

// One warp per digit: exclusive scan over the tiles, total of the digit.
__global__ void __launch_bounds__(256) sort_scan_kernel(uint32_t* __restrict__ counts, uint32_t* __restrict__ totals, int bins, int tiles) {
    const int bin = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    mgw_let_next_start();
    mgw_wait_for_previous();
    if (bin >= bins) return;
    uint32_t* row = counts + (long long)bin * tiles;
    uint32_t before = 0;
    for (int t0 = 0; t0 < tiles; t0 += 32) {
        const uint32_t c = t0 + lane < tiles ? row[t0 + lane] : 0u;
        uint32_t s = c;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        if (t0 + lane < tiles) row[t0 + lane] = before + s - c;
        before += __shfl_sync(0xffffffffu, s, 31);
    }
    if (lane == 0) totals[bin] = before;
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortPass p) {
    extern __shared__ uint32_t smem[];
    const int bins = 1 << p.bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    constexpr int kWarps = kSortThreads / 32;
    uint32_t* base = smem;                                            // [bins] where this tile's entries of a digit start
    uint16_t* cnt = reinterpret_cast<uint16_t*>(smem + bins);         // [warps][bins] entries of the warps
    __shared__ uint32_t warp_sum[kWarps];
    for (int b = threadIdx.x; b < bins * kWarps; b += kSortThreads) cnt[b] = 0;
    mgw_let_next_start();
    mgw_wait_for_previous();
    // exclusive scan of the digits' totals: a thread owns bins / 512 neighbouring digits
    const int per = (bins + kSortThreads - 1) / kSortThreads;
    uint32_t mine = 0;
    for (int k = 0; k < per; ++k) {
        const int b = threadIdx.x * per + k;
        if (b < bins) mine += p.totals[b];
    }
    uint32_t s = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += v;
    }
    if (lane == 31) warp_sum[warp] = s;
    __syncthreads();
    uint32_t before = s - mine;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    for (int k = 0; k < per; ++k) {
        const int b = threadIdx.x * per + k;
        if (b < bins) {
            base[b] = before + p.counts[(long long)b * p.tiles + blockIdx.x];
            before += p.totals[b];
        }
    }
    // rank of every entry among its warp's entries of the same digit; a warp owns a contiguous part of the tile
    const long long i0 = (long long)blockIdx.x * kSortTile + warp * (kSortTile / kWarps);
    uint2 e[kSortItems];
    uint32_t rank[kSortItems];
    uint16_t* mycnt = cnt + warp * bins;
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        const long long i = i0 + j * 32 + lane;
        if (i < p.n) e[j] = sort_entry(p, i, false);
    }
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        const bool in = i0 + j * 32 + lane < p.n;
        const uint32_t d = in ? (e[j].x >> p.shift) & (bins - 1) : 0xffffffffu;
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        if (in) rank[j] = mycnt[d] + __popc(peers & ((1u << lane) - 1u));
        __syncwarp();
        if (in && lane == 31 - __clz(peers)) mycnt[d] = (uint16_t)(rank[j] + 1);       // the last of them knows how many there are
        __syncwarp();
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kSortThreads) {          // entries of the warps before
        uint32_t sum = 0;
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = cnt[w * bins + b];
            cnt[w * bins + b] = (uint16_t)sum;
            sum += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        if (i0 + j * 32 + lane >= p.n) break;
        const uint32_t d = (e[j].x >> p.shift) & (bins - 1);
        p.out[base[d] + mycnt[d] + rank[j]] = e[j];
    }
}

// Lists of up to 65,536 tokens: the whole sort in one launch of one cluster, which keeps the list in its shared memory.  A
// block has a contiguous part of it; per pass the blocks read each other's histograms and write every entry to its new place,
// which may be another block's memory.  10 us up to 8192 tokens, 18 us for 32,768, 30 us for 65,536, where the six launches
// of the tiled sort are as fast.
constexpr int kCluster = 8;
constexpr int kClusterThreads = 1024;
constexpr int kClusterItems = 8;
constexpr int kClusterPart = kClusterThreads * kClusterItems;         // entries of a block
constexpr int kClusterList = kCluster * kClusterPart;
constexpr int kClusterBits = 9;

struct ClusterSmem {
    uint2 list[2][kClusterPart];                                      // {key, position}, before and after a pass
    uint16_t cnt[kClusterThreads / 32][1 << kClusterBits];            // entries of a warp with a digit, then of the warps before
    uint32_t hist[1 << kClusterBits], base[1 << kClusterBits];
    uint32_t warp_sum[(1 << kClusterBits) / 32];
};

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kClusterThreads) sort_cluster_kernel(SortPass p, int passes) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    ClusterSmem& m = *reinterpret_cast<ClusterSmem*>(dynamic);
    cg::cluster_group cluster = cg::this_cluster();
    mgw_let_next_start();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int bins = 1 << p.bits, n = (int)p.n, rank_in_cluster = (int)cluster.block_rank();
    const int items = (n + kCluster * kClusterThreads - 1) / (kCluster * kClusterThreads);
    const int part = items * kClusterThreads;                         // entries of a block (of the last ones: fewer)
    const int first = rank_in_cluster * part;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * p.bits, from = (pass + 1) & 1, to = pass & 1;
        for (int b = tid; b < bins * (kClusterThreads / 32); b += kClusterThreads) m.cnt[b >> p.bits][b & (bins - 1)] = 0;
        __syncthreads();
        uint2 e[kClusterItems];
        uint32_t rank[kClusterItems];
#pragma unroll
        for (int j = 0; j < kClusterItems; ++j) {
            const int local = (warp * items + j) * 32 + lane, i = first + local;
            if (j < items && i < n) e[j] = pass == 0 ? sort_entry(p, i, true) : m.list[from][local];
        }
#pragma unroll
        for (int j = 0; j < kClusterItems; ++j) {
            if (j >= items) break;
            const bool in = first + (warp * items + j) * 32 + lane < n;
            const uint32_t d = in ? (e[j].x >> shift) & (bins - 1) : 0xffffffffu;
            const unsigned peers = __match_any_sync(0xffffffffu, d);
            if (in) rank[j] = m.cnt[warp][d] + __popc(peers & ((1u << lane) - 1u));
            __syncwarp();
            if (in && lane == 31 - __clz(peers)) m.cnt[warp][d] = (uint16_t)(rank[j] + 1);
            __syncwarp();
        }
        __syncthreads();
        if (tid < bins) {                                             // a digit's entries in the warps before, and in the block
            uint32_t sum = 0, c[kClusterThreads / 32];
#pragma unroll
            for (int w = 0; w < kClusterThreads / 32; ++w) c[w] = m.cnt[w][tid];
#pragma unroll
            for (int w = 0; w < kClusterThreads / 32; ++w) {
                m.cnt[w][tid] = (uint16_t)sum;
                sum += c[w];
            }
            m.hist[tid] = sum;
        }
        cluster.sync();
        uint32_t before = 0, total = 0, s = 0;
        if (tid < bins) {
            uint32_t h[kCluster];
#pragma unroll
            for (int c = 0; c < kCluster; ++c) h[c] = cluster.map_shared_rank(m.hist, c)[tid];
#pragma unroll
            for (int c = 0; c < kCluster; ++c) {
                if (c < rank_in_cluster) before += h[c];
                total += h[c];
            }
            s = total;
        }
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        if (lane == 31 && warp < (1 << kClusterBits) / 32) m.warp_sum[warp] = s;
        __syncthreads();
        if (tid < bins) {
            for (int w = 0; w < warp; ++w) before += m.warp_sum[w];
            m.base[tid] = before + s - total;
        }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < kClusterItems; ++j) {
            if (j >= items || first + (warp * items + j) * 32 + lane >= n) break;
            const uint32_t d = (e[j].x >> shift) & (bins - 1);
            const uint32_t at = m.base[d] + m.cnt[warp][d] + rank[j];
            if (pass == passes - 1) {
                p.out[at] = e[j];
            } else {
                const uint32_t c = at / (uint32_t)part;
                cluster.map_shared_rank(m.list[to], c)[at - c * part] = e[j];
            }
        }
        cluster.sync();                                               // the list is in its new order; histograms are free
    }
}

// The same within one block of 1024 threads, for at most 1024 tokens, one per thread; the sorted list is left in shared memory.
constexpr int kSmallWarps = 32;
constexpr int kSmallList = kSmallWarps * 32;                          // up to here one launch does it all: 12.3 instead of 12.6 us
                                                                      // for 700 tokens (10000 x 512), 14.7 instead of 13.7 for 1024

struct SmallSort {
    uint16_t cnt[kSmallWarps][1 << kClusterBits];
    uint32_t base[1 << kClusterBits], warp_sum[(1 << kClusterBits) / 32];
};

__device__ __forceinline__ const uint2* sort_in_block(const SortPass& p, int passes, uint2 (*list)[kSmallList], SmallSort& m) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, bins = 1 << p.bits, n = (int)p.n;
    const bool in = tid < n;
    for (int pass = 0; pass < passes; ++pass) {
        const int shift = pass * p.bits;
        for (int b = tid; b < bins * kSmallWarps; b += kSmallWarps * 32) m.cnt[b >> p.bits][b & (bins - 1)] = 0;
        uint2 e = make_uint2(0, 0);
        if (in) e = pass == 0 ? sort_entry(p, tid, true) : list[(pass + 1) & 1][tid];
        const uint32_t d = in ? (e.x >> shift) & (bins - 1) : 0xffffffffu;
        __syncthreads();
        const unsigned peers = __match_any_sync(0xffffffffu, d);
        const uint32_t rank = __popc(peers & ((1u << lane) - 1u));
        if (in && lane == 31 - __clz(peers)) m.cnt[warp][d] = (uint16_t)(rank + 1);
        __syncthreads();
        uint32_t total = 0, s = 0;
        if (tid < bins) {                                             // a digit's entries in the warps before, and in all
            uint32_t c[kSmallWarps];
#pragma unroll
            for (int w = 0; w < kSmallWarps; ++w) c[w] = m.cnt[w][tid];
#pragma unroll
            for (int w = 0; w < kSmallWarps; ++w) {
                m.cnt[w][tid] = (uint16_t)total;
                total += c[w];
            }
        }
        s = total;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t v = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += v;
        }
        if (lane == 31 && warp < (1 << kClusterBits) / 32) m.warp_sum[warp] = s;
        __syncthreads();
        if (tid < bins) {
            uint32_t before = 0;
            for (int w = 0; w < warp; ++w) before += m.warp_sum[w];
            m.base[tid] = before + s - total;
        }
        __syncthreads();
        if (in) list[pass & 1][m.base[d] + m.cnt[warp][d] + rank] = e;
        __syncthreads();
    }
    return list[(passes - 1) & 1];
}

// -------------------------------------------------------------------------------------------------------------- sums
struct GradArgs {
    const uint2* list;         // {token, position}, sorted
    long long n;
    const void* dy;
    long long dy_ld;
    void* dw;                  // [vocab, dim]
    long long vocab;
    int dim;
    float scale;
    int chunk;                 // entries of the sorted list that one warp adds up; the 8 warps of a block have neighbouring ones
    int groups, slabs;         // group: the chunks of a block; slab: 32 blocks of a row, one per lane
    float* partial;            // [groups][2][slabs * 32 * N]: the run that comes in, the run that goes on
    int zero_blocks;           // blocks of the launch that fill rows without tokens
    int zero_rows;             // rows of each of them
    int by_tokens;             // they look at the tokens themselves (short lists), not at the sorted list
    const void* tokens;
    int wide;
    long long padding;
};

constexpr int kZeroRows = 1024;            // most rows of a block that fills

constexpr int kSumWarps = 8;
constexpr int kMaxChunk = 64;              // 262,144 tokens: 307 us; 314 with 256, 316 with 512 (fewer, less even parts)

// fp32 partial sums of a slab: the values of a lane one behind the other
template <typename T>
__device__ __forceinline__ float4* partial_of(const GradArgs& a, long long group, int which, int slab, int lane) {
    return reinterpret_cast<float4*>(a.partial) + (((group * 2 + which) * a.slabs + slab) * 32 + lane) * (per_block<T>() / 4);
}

// A block's rows that no token names.
template <typename T, int MODE>
__device__ __forceinline__ void fill_rows(const GradArgs& a, long long block) {
    __shared__ uint32_t named[kZeroRows / 32];
    const long long r0 = block * a.zero_rows, r1 = min(a.vocab, r0 + a.zero_rows);
    for (int k = threadIdx.x; k < kZeroRows / 32; k += blockDim.x) named[k] = 0;
    __syncthreads();
    if (a.by_tokens) {                                                // needs no order, so the sort may still be running
        constexpr int U = 8;
        for (long long i0 = threadIdx.x; i0 < a.n; i0 += blockDim.x * U) {
            long long t[U];
#pragma unroll
            for (int u = 0; u < U; ++u) t[u] = i0 + u * blockDim.x < a.n ? mgw_token(a.tokens, a.wide, i0 + u * blockDim.x) : -1;
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (t[u] >= r0 && t[u] < r1 && t[u] != a.padding) atomicOr(&named[(t[u] - r0) >> 5], 1u << ((t[u] - r0) & 31));
        }
    } else {
        mgw_wait_for_previous();
        for (long long r = r0 + threadIdx.x; r < r1; r += blockDim.x) {
            long long lo = 0, hi = a.n;                               // first entry that is not below the row
            while (lo < hi) {
                const long long mid = (lo + hi) >> 1;
                if (a.list[mid].x < (uint32_t)r) lo = mid + 1; else hi = mid;
            }
            if (lo < a.n && a.list[lo].x == (uint32_t)r) atomicOr(&named[(r - r0) >> 5], 1u << ((r - r0) & 31));
        }
    }
    __syncthreads();
    const int lane = threadIdx.x & 31;
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (long long r = r0 + (threadIdx.x >> 5); r < r1; r += blockDim.x >> 5) {
        if (named[(r - r0) >> 5] >> ((r - r0) & 31) & 1) continue;
        T* row = static_cast<T*>(a.dw) + r * a.dim;
        for (int c = column_of<T, MODE>(0, lane) - (MODE == kShift ? lead_of(row) : 0); c < a.dim; c += 32 * per_block<T>())
            store_block<T, MODE>(row, c, a.dim, zero);
    }
}

// What the warps of a block share: a chunk's run that comes in and its run that goes on, and the keys around the borders.
template <typename T, int WARPS>
struct SumSpace {
    float parts[WARPS][2][per_block<T>()][32];
    uint32_t key_last[WARPS], key_next[WARPS];
};

// The chunks of a group, one per warp, for the columns of a slab.
template <typename T, int MODE, int WARPS>
__device__ __forceinline__ void sum_group(const GradArgs& a, const uint2* list, long long group, int slab, SumSpace<T, WARPS>& m) {
    constexpr int N = per_block<T>(), U = 4;                          // rows in flight
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c0 = column_of<T, MODE>(slab, lane);
    const int c = MODE == kWords ? c0 : min(c0, (a.dim - 1) / N * N); // lanes behind the row's end read its last block
    const T* dy = static_cast<const T*>(a.dy);
    const char* lo = static_cast<const char*>(a.dy);
    const char* hi = reinterpret_cast<const char*>(dy + (a.n - 1) * a.dy_ld + a.dim);
    T* dw = static_cast<T*>(a.dw);
    const uint32_t none = (uint32_t)a.vocab;                          // key of what is skipped, and of nothing
    const long long i0 = min(a.n, (group * WARPS + warp) * a.chunk), i1 = min(a.n, i0 + a.chunk);
    const uint32_t first = i0 < i1 ? list[i0].x : none, last = i0 < i1 ? list[i1 - 1].x : none;
    const uint32_t before = i0 > 0 && i0 < i1 ? list[i0 - 1].x : none, next = i1 < a.n ? list[i1].x : none;
    if (lane == 0) {
        m.key_last[warp] = last;
        m.key_next[warp] = next;
    }
    uint32_t run = first;
    bool comes_in = first != none && before == first;
    float acc[N];
#pragma unroll
    for (int e = 0; e < N; ++e) acc[e] = 0.f;
    auto store = [&](uint32_t key) {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] *= a.scale;
        store_blocks<T, MODE>(dw + (long long)key * a.dim, c0, a.dim, mgw_pack<T, N>(acc));
    };
    auto flush = [&](bool goes_on) {
        if (comes_in || goes_on) {
#pragma unroll
            for (int e = 0; e < N; ++e) m.parts[warp][comes_in ? 0 : 1][e][lane] = acc[e];
        } else {
            store(run);
        }
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = 0.f;
        comes_in = false;
    };
    auto add = [&](uint32_t key, const uint4& v) {
        if (key != run) {
            flush(false);
            run = key;
        }
        float f[N];
        mgw_unpack<T, N>(v, f);
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] += f[e];
    };
    const bool whole = comes_in && last == first;                     // nothing but the run that comes in
    for (long long b0 = i0; b0 < i1 && first != none; b0 += 32) {     // 32 entries at a time, one per lane
        const uint2 mine = b0 + lane < i1 ? list[b0 + lane] : make_uint2(none, 0u);
        const int here = __popc(__ballot_sync(0xffffffffu, mine.x != none));
        // rows at the ends of dy, whose blocks cannot be cut out of vectors
        const bool edge = MODE == kShift && lane < here && !inside(dy + (long long)mine.y * a.dy_ld, a.dim, lo, hi);
        const unsigned edges = MODE != kShift ? 0u : __ballot_sync(0xffffffffu, edge);
        for (int j = 0; j < here; ) {
            if (j + U <= here && (edges >> j & ((1u << U) - 1u)) == 0) {
                Cut r[U];
#pragma unroll
                for (int u = 0; u < U; ++u)
                    r[u] = load_block<T, MODE>(dy + (long long)__shfl_sync(0xffffffffu, mine.y, j + u) * a.dy_ld, c, a.dim);
#pragma unroll
                for (int u = 0; u < U; ++u) add(__shfl_sync(0xffffffffu, mine.x, j + u), take<MODE>(r[u]));
                j += U;
            } else {
                const T* row = dy + (long long)__shfl_sync(0xffffffffu, mine.y, j) * a.dy_ld;
                const uint32_t key = __shfl_sync(0xffffffffu, mine.x, j);
                add(key, MODE == kShift ? gather_block(row, c, a.dim) : load_block<T, MODE>(row, c, a.dim).x);
                ++j;
            }
        }
        if (here < 32) break;
    }
    const bool goes_on = run != none && last == run && next == run;
    if (run != none) flush(goes_on);
    __syncthreads();
    // Runs that cross borders within the block: the warp in which a run starts adds up the parts in their order (and the
    // first warp those of the run that comes into the block).  What crosses the block's border goes to memory.
    auto follow = [&](uint32_t key, int from) {                       // adds the parts behind chunk `from`; true: the run ends here
        for (int w = from; ; ++w) {
            if (!(m.key_last[w] == key && m.key_next[w] == key)) return true;
            if (w + 1 == WARPS) return false;
#pragma unroll
            for (int e = 0; e < N; ++e) acc[e] += m.parts[w + 1][0][e][lane];
        }
    };
    auto keep = [&](int which) {
        float4* to = partial_of<T>(a, group, which, slab, lane);
#pragma unroll
        for (int q = 0; q < N / 4; ++q) to[q] = make_float4(acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]);
    };
    if (warp == 0 && first != none && before == first) {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = m.parts[0][0][e][lane];
        follow(first, 0);
        keep(0);
    }
    if (goes_on && !whole) {
#pragma unroll
        for (int e = 0; e < N; ++e) acc[e] = m.parts[warp][1][e][lane];
        if (follow(last, warp)) store(last);
        else keep(1);
    }
}

template <typename T, int MODE>
__global__ void __launch_bounds__(32 * kSumWarps, MODE == kShift ? 3 : 4) grad_chunks_kernel(GradArgs a) {
    __shared__ SumSpace<T, kSumWarps> m;
    mgw_let_next_start();
    if ((int)blockIdx.x < a.zero_blocks) {
        fill_rows<T, MODE>(a, blockIdx.x);
        return;
    }
    mgw_wait_for_previous();
    const long long task = blockIdx.x - a.zero_blocks, group = task / a.slabs;
    sum_group<T, MODE, kSumWarps>(a, a.list, group, (int)(task - group * a.slabs), m);
}

// Everything in one launch, for at most 1024 tokens: every slab's block sorts the list for itself and is the only group.
struct SmallSpace {
    uint2 list[2][kSmallList];
    unsigned char rest[];                  // SmallSort, then SumSpace
};

template <typename T, int MODE>
__global__ void __launch_bounds__(32 * kSmallWarps) grad_small_kernel(GradArgs a, SortPass p, int passes) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    SmallSpace& m = *reinterpret_cast<SmallSpace*>(dynamic);
    if ((int)blockIdx.x >= a.slabs) {
        fill_rows<T, MODE>(a, blockIdx.x - a.slabs);
        return;
    }
    if (blockIdx.x > 0) p.status = nullptr;                           // one report is enough
    const uint2* list = sort_in_block(p, passes, m.list, *reinterpret_cast<SmallSort*>(m.rest));
    sum_group<T, MODE, kSmallWarps>(a, list, 0, blockIdx.x, *reinterpret_cast<SumSpace<T, kSmallWarps>*>(m.rest));
}

// Runs that cross borders of groups: the warp of the group in which a run starts adds up its partial sums, for one slab.
template <typename T, int MODE>
__global__ void __launch_bounds__(256) grad_join_kernel(GradArgs a) {
    constexpr int N = per_block<T>(), Q = N / 4, U = 8;               // partial sums in flight, added in their order
    mgw_wait_for_previous();
    const int lane = threadIdx.x & 31;
    const long long task = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (task >= (long long)(a.groups - 1) * a.slabs) return;
    const long long group = task / a.slabs, size = (long long)kSumWarps * a.chunk;
    const int slab = (int)(task - group * a.slabs);
    const uint32_t none = (uint32_t)a.vocab;
    const long long i0 = group * size, i1 = i0 + size;                // not the last group: it is full
    // where the run that crosses the group's end started: in this group if the group has another key or it does not come in
    const uint32_t run = a.list[i1 - 1].x, next = a.list[i1].x, first = a.list[i0].x, before = i0 > 0 ? a.list[i0 - 1].x : none;
    if (run == none || next != run || (first == run && before == run)) return;
    long long end = group + 1;                                        // the run's first group that is not its own
    for (bool more = true; more; ) {
        const long long g = end + lane;
        const unsigned same = __ballot_sync(0xffffffffu, g < a.groups && a.list[g * size].x == run);
        const int k = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
        end += k;
        more = k == 32;
    }
    float4 x[Q];
    const float4* from = partial_of<T>(a, group, 1, slab, lane);
#pragma unroll
    for (int q = 0; q < Q; ++q) x[q] = from[q];
    const long long step = 2LL * a.slabs * 32 * Q;
    from = partial_of<T>(a, group + 1, 0, slab, lane);
    for (long long g = group + 1; g < end; g += U, from += U * step) {
        float4 y[U][Q];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < Q; ++q) y[u][q] = g + u < end ? from[u * step + q] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < Q; ++q) { x[q].x += y[u][q].x; x[q].y += y[u][q].y; x[q].z += y[u][q].z; x[q].w += y[u][q].w; }
    }
    float acc[N];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        acc[4 * q] = x[q].x * a.scale; acc[4 * q + 1] = x[q].y * a.scale;
        acc[4 * q + 2] = x[q].z * a.scale; acc[4 * q + 3] = x[q].w * a.scale;
    }
    store_blocks<T, MODE>(static_cast<T*>(a.dw) + (long long)run * a.dim, column_of<T, MODE>(slab, lane), a.dim, mgw_pack<T, N>(acc));
}

int element_size(int dtype) { return dtype == MGW_F32 ? 4 : 2; }

// How the rows of a matrix can be moved.
int mode_of(const void* base, long long ld, int dim, int dtype) {
    const int es = element_size(dtype);
    const unsigned long long x = (unsigned long long)(uintptr_t)base | (unsigned long long)(ld * es) | (unsigned long long)((long long)dim * es);
    return (x & 15) == 0 ? kExact : (x & 3) == 0 ? kWords : kShift;
}

// f<type, mode>(...) for the type and for the mode that suits both matrices
#define MGW_BY_TYPE(f, mode, ...)                                                                                  \
    (dtype == MGW_F32   ? ((mode) == kExact ? f<float, kExact>(__VA_ARGS__) : f<float, kWords>(__VA_ARGS__))       \
     : dtype == MGW_F16 ? ((mode) == kExact   ? f<__half, kExact>(__VA_ARGS__)                                     \
                           : (mode) == kWords ? f<__half, kWords>(__VA_ARGS__) : f<__half, kShift>(__VA_ARGS__))   \
                        : ((mode) == kExact   ? f<__nv_bfloat16, kExact>(__VA_ARGS__)                              \
                           : (mode) == kWords ? f<__nv_bfloat16, kWords>(__VA_ARGS__) : f<__nv_bfloat16, kShift>(__VA_ARGS__)))

// The sort: digits per pass and scratch memory.
struct SortPlan {
    int passes, bits, tiles;
    size_t list_bytes, counts_bytes, totals_bytes;
};

SortPlan sort_plan(long long n, long long vocab) {
    SortPlan p;
    int bits = 1;
    while ((vocab >> bits) != 0) ++bits;                              // keys 0 .. vocab
    p.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    if (p.passes < 2) p.passes = 2;                                   // two passes of few digits: small histograms
    p.bits = (bits + p.passes - 1) / p.passes;
    if (n <= kClusterList) {                                          // one cluster: digits of at most 9 bits
        p.passes = (bits + kClusterBits - 1) / kClusterBits;
        p.bits = (bits + p.passes - 1) / p.passes;
    }
    p.tiles = (int)((n + kSortTile - 1) / kSortTile);
    p.list_bytes = ((size_t)n * 8 + 255) & ~(size_t)255;
    p.counts_bytes = (((size_t)1 << p.bits) * p.tiles * 4 + 255) & ~(size_t)255;
    p.totals_bytes = (((size_t)1 << p.bits) * 4 + 255) & ~(size_t)255;
    return p;
}

struct SumPlan {
    int slabs, chunk, groups;
    size_t partial_bytes;
};

SumPlan sum_plan(long long n, int dim, int dtype) {
    SumPlan s;
    const int per = 16 / element_size(dtype);
    s.slabs = (dim + 32 * per - 1) / (32 * per);
    // A warp's part of the list: short enough that there are blocks for every SM, long enough that they run as one wave
    // where that is possible (four of them per SM) and that few runs cross its borders.  16,384 tokens of 10000 x 512: 26 us
    // as one wave, 30 us as one and three quarters.
    const long long even = (n * s.slabs + kSumWarps * 148 * 4 - 1) / (kSumWarps * 148 * 4);
    s.chunk = (int)(even < 8 ? 8 : even > kMaxChunk ? kMaxChunk : (even + 3) / 4 * 4);
    s.groups = (int)((n + (long long)kSumWarps * s.chunk - 1) / ((long long)kSumWarps * s.chunk));
    s.partial_bytes = (size_t)s.groups * 2 * s.slabs * 32 * per * sizeof(float);
    return s;
}

// Lets a kernel use more than 48 KB of shared memory: once for every device.
template <typename... P>
int allow_smem(void (*kernel)(P...), size_t bytes, std::atomic<unsigned long long>& done) {
    int dev = 0;
    MGW_CUDA_CHECK(cudaGetDevice(&dev));
    const unsigned long long bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return MGW_OK;
    MGW_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes));
    done.fetch_or(bit, std::memory_order_relaxed);
    return MGW_OK;
}

template <typename T, int MODE>
int launch_small(const GradArgs& a, const SortPass& p, int passes, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    const size_t rest = sizeof(SmallSort) > sizeof(SumSpace<T, kSmallWarps>) ? sizeof(SmallSort) : sizeof(SumSpace<T, kSmallWarps>);
    const size_t smem = sizeof(SmallSpace) + rest;
    const int rc = allow_smem(grad_small_kernel<T, MODE>, smem, done);
    if (rc != MGW_OK) return rc;
    grad_small_kernel<T, MODE><<<a.slabs + a.zero_blocks, 32 * kSmallWarps, smem, stream>>>(a, p, passes);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}

template <typename T, int MODE>
int launch_sums(const GradArgs& a, bool behind_sort, cudaStream_t stream) {
    const long long grid = (long long)a.groups * a.slabs + a.zero_blocks;
    if (behind_sort) {
        const int rc = launch_dependent(grad_chunks_kernel<T, MODE>, grid, 32 * kSumWarps, 0, stream, a);
        if (rc != MGW_OK) return rc;
    } else {                                                         // some other kernel is before it: start when that is done
        grad_chunks_kernel<T, MODE><<<(unsigned)grid, 32 * kSumWarps, 0, stream>>>(a);
        MGW_CUDA_CHECK(cudaGetLastError());
    }
    if (a.groups == 1) return MGW_OK;
    return launch_dependent(grad_join_kernel<T, MODE>, ((long long)(a.groups - 1) * a.slabs + 7) / 8, 256, 0, stream, a);
}

template <typename T, int MODE>
int launch_fwd(const void* tokens, int wide, long long n, const void* weight, long long ld, long long vocab, int dim, float scale,
               void* out, bool beside_sort, int* status, cudaStream_t stream) {
    const int per = 32 * lookup_unroll(MODE) * per_block<T>(), segments = (dim + (MODE == kShift ? per_block<T>() - 1 : 0) + per - 1) / per;
    const long long blocks = (n * segments + 7) / 8;
    const unsigned grid = (unsigned)(blocks < 148LL * 64 ? blocks : 148LL * 64);
    if (beside_sort)
        return launch_dependent(embedding_fwd_kernel<T, MODE>, grid, 256, 0, stream, tokens, wide, n, static_cast<const T*>(weight), ld, vocab,
                                dim, scale, static_cast<T*>(out), segments, 1, status);
    embedding_fwd_kernel<T, MODE><<<grid, 256, 0, stream>>>(tokens, wide, n, static_cast<const T*>(weight), ld, vocab, dim, scale,
                                                             static_cast<T*>(out), segments, 0, status);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}

bool bad_sizes(long long n, long long vocab, int dim, int dtype) {
    return n < 0 || n > 0x7fffffffLL || vocab < 1 || vocab > 0x7ffffffeLL || dim < 1 || dim > (1 << 30) || dtype < MGW_F32 || dtype > MGW_BF16;
}

int launch_cluster_sort(const SortPass& a, int passes, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    const int rc = allow_smem(sort_cluster_kernel, sizeof(ClusterSmem), done);
    if (rc != MGW_OK) return rc;
    sort_cluster_kernel<<<kCluster, kClusterThreads, sizeof(ClusterSmem), stream>>>(a, passes);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}

SortPass sort_of(const void* tokens, int wide, long long n, long long vocab, long long padding, const SortPlan& p, int* status) {
    SortPass a = {};
    a.tokens = tokens; a.wide = wide;
    a.n = n; a.tiles = p.tiles; a.bits = p.bits;
    a.vocab = vocab; a.padding = padding; a.status = status;
    return a;
}

}  // namespace

// One block of pinned, device-visible words per process: where the kernels record a token outside the vocabulary.
extern "C" int mgw_token_status(int** out) {
    if (out == nullptr) return MGW_ERR_ARG;
    static std::mutex lock;
    static int* words = nullptr;
    std::lock_guard<std::mutex> hold(lock);
    if (words == nullptr) {
        // may be the first call inside a stream capture, where an allocation is only allowed in relaxed mode
        cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
        MGW_CUDA_CHECK(cudaThreadExchangeStreamCaptureMode(&mode));
        void* p = nullptr;
        const cudaError_t e = cudaHostAlloc(&p, 8 * sizeof(int), cudaHostAllocPortable | cudaHostAllocMapped);
        cudaThreadExchangeStreamCaptureMode(&mode);
        MGW_CUDA_CHECK(e);
        for (int i = 0; i < 8; ++i) static_cast<int*>(p)[i] = 0;
        words = static_cast<int*>(p);
    }
    *out = words;
    return MGW_OK;
}

// The sort of a list that one cluster takes needs 8 SMs and 10 to 30 us, mostly waiting.  Beside a lookup that is as long it
// costs nothing; otherwise the zeros of the gradient are a better thing to do meanwhile.  Lookup and gradient, with the sort
// beside the lookup and beside the zeros: 20,011 x 1023 fp16 of 32,003 60 and 69 us, 65,536 x 2048 bf16 of 32,000 137 and 155,
// 16,384 x 512 fp32 of 10,000 32 and 37; but 4096 x 768 bf16 of 50,000 31 and 25, 1500 x 1500 fp32 of 10,000 27 and 23 (sort
// 10 us, lookup 3 us).  Lists of up to 1024 are sorted where they are added up, those above 65,536 by six launches there.
constexpr long long kLongLookup = 32LL << 20;                          // bytes that the lookup writes

extern "C" size_t mgw_embedding_order_bytes(long long n, long long vocab, int dim, int dtype) {
    if (bad_sizes(n, vocab, dim, dtype) || n <= kSmallList || n > kClusterList || n * dim * element_size(dtype) < kLongLookup) return 0;
    return sort_plan(n, vocab).list_bytes;
}

extern "C" int mgw_embedding_fwd(const void* tokens, int wide, long long n, const void* weight, long long ld, long long vocab,
                                 int dim, int dtype, float scale, void* out, void* order, long long padding, int* status,
                                 void* stream) {
    if (bad_sizes(n, vocab, dim, dtype) || ld < dim) return MGW_ERR_ARG;
    if (n == 0) return MGW_OK;
    if (tokens == nullptr || weight == nullptr || out == nullptr || status == nullptr) return MGW_ERR_ARG;
    if (((uintptr_t)weight | (uintptr_t)out) & (element_size(dtype) - 1)) return MGW_ERR_ARG;
    const int wm = mode_of(weight, ld, dim, dtype), om = mode_of(out, dim, dim, dtype), mode = wm > om ? wm : om;
    if (order != nullptr) {
        if (mgw_embedding_order_bytes(n, vocab, dim, dtype) == 0 || ((uintptr_t)order & 15)) return MGW_ERR_ARG;
        const SortPlan p = sort_plan(n, vocab);
        SortPass a = sort_of(tokens, wide, n, vocab, padding, p, nullptr);              // the lookup reports
        a.out = static_cast<uint2*>(order);
        const int rc = launch_cluster_sort(a, p.passes, (cudaStream_t)stream);
        if (rc != MGW_OK) return rc;
    }
    return MGW_BY_TYPE(launch_fwd, mode, tokens, wide, n, weight, ld, vocab, dim, scale, out, order != nullptr, status,
                       (cudaStream_t)stream);
}

extern "C" size_t mgw_embedding_grad_bytes(long long n, long long vocab, int dim, int dtype) {
    if (bad_sizes(n, vocab, dim, dtype) || n == 0) return 0;
    if (n <= kSmallList) return 0;
    const SortPlan p = sort_plan(n, vocab);
    return 2 * p.list_bytes + p.counts_bytes + p.totals_bytes + sum_plan(n, dim, dtype).partial_bytes;
}

extern "C" int mgw_embedding_grad(const void* dy, long long dy_ld, const void* tokens, int wide, long long n, long long vocab, int dim,
                                  int dtype, float scale, long long padding, const void* order, void* dw, void* work, size_t work_bytes,
                                  int* status, void* stream) {
    if (bad_sizes(n, vocab, dim, dtype) || dw == nullptr) return MGW_ERR_ARG;
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        MGW_CUDA_CHECK(cudaMemsetAsync(dw, 0, (size_t)vocab * dim * element_size(dtype), s));
        return MGW_OK;
    }
    if (dy == nullptr || tokens == nullptr || status == nullptr || (n > 1 && dy_ld < dim)) return MGW_ERR_ARG;
    if (((uintptr_t)dy | (uintptr_t)dw) & (element_size(dtype) - 1)) return MGW_ERR_ARG;
    const SortPlan p = sort_plan(n, vocab);
    const SumPlan q = sum_plan(n, dim, dtype);
    SortPass a = sort_of(tokens, wide, n, vocab, padding, p, status);
    if (order != nullptr && (mgw_embedding_order_bytes(n, vocab, dim, dtype) == 0 || ((uintptr_t)order & 15))) return MGW_ERR_ARG;
    // Rows without tokens are filled by blocks of the same launch as the sums.  Those of a list of up to 65,536 tokens read
    // all tokens and start while the sort runs (20,011 tokens of a table of 32,003: 54 us, 63 us when the sorted list is
    // searched instead); of a longer list every block would read too much.  Four blocks per SM where they read little
    // (262,144 tokens, searched: 315 us, with one per SM 323), one where each reads a long list, two where the list is sorted
    // already (32,768 x 1024 bf16 of 131,072: 92 us, 101 with one, 90 with four; 20,011 x 1023 fp16 of 32,003: 60, 60, 64).
    GradArgs g = {};
    g.n = n; g.dy = dy; g.dy_ld = dy_ld; g.dw = dw; g.vocab = vocab; g.dim = dim; g.scale = scale;
    g.chunk = q.chunk; g.groups = q.groups; g.slabs = q.slabs;
    g.by_tokens = n <= kClusterList && order == nullptr;
    g.tokens = tokens; g.wide = wide; g.padding = padding;
    const int ym = mode_of(dy, dy_ld, dim, dtype), wm = mode_of(dw, dim, dim, dtype), mode = ym > wm ? ym : wm;
    const bool small = n <= kSmallList;
    const int fillers = small ? (q.slabs < 74 ? 148 - q.slabs : 74) : order != nullptr ? 148 * 2 : !g.by_tokens || n <= 4096 ? 148 * 4 : 148;
    g.zero_rows = (int)((vocab + fillers - 1) / fillers);
    if (g.zero_rows > kZeroRows) g.zero_rows = kZeroRows;
    g.zero_blocks = (int)((vocab + g.zero_rows - 1) / g.zero_rows);
    if (small) {
        g.chunk = (int)((n + kSmallWarps - 1) / kSmallWarps);
        return MGW_BY_TYPE(launch_small, mode, g, a, p.passes, s);
    }
    if (work == nullptr || work_bytes < mgw_embedding_grad_bytes(n, vocab, dim, dtype) || ((uintptr_t)work & 15)) return MGW_ERR_ARG;
    char* at = static_cast<char*>(work);
    uint2* list[2];
    for (int i = 0; i < 2; ++i) {
        list[i] = reinterpret_cast<uint2*>(at);
        at += p.list_bytes;
    }
    a.out = list[0];
    a.counts = reinterpret_cast<uint32_t*>(at); at += p.counts_bytes;
    a.totals = reinterpret_cast<uint32_t*>(at); at += p.totals_bytes;
    if (order != nullptr) {                                          // mgw_embedding_fwd has sorted the tokens
    } else if (n <= kClusterList) {
        const int rc = launch_cluster_sort(a, p.passes, s);
        if (rc != MGW_OK) return rc;
    } else {
        const int bins = 1 << p.bits;
        const size_t hist_smem = (size_t)bins * 4, scatter_smem = (size_t)bins * 4 + (size_t)bins * 2 * (kSortThreads / 32);
        for (int k = 0; k < p.passes; ++k) {
            a.in = k == 0 ? nullptr : list[(k + 1) & 1];
            a.out = list[k & 1];
            a.shift = k * p.bits;
            int rc = launch_dependent(sort_hist_kernel, p.tiles, kSortThreads, hist_smem, s, a);
            if (rc == MGW_OK) rc = launch_dependent(sort_scan_kernel, (bins + 7) / 8, 256, 0, s, a.counts, a.totals, bins, p.tiles);
            if (rc == MGW_OK) rc = launch_dependent(sort_scatter_kernel, p.tiles, kSortThreads, scatter_smem, s, a);
            if (rc != MGW_OK) return rc;
        }
    }
    g.list = order != nullptr ? static_cast<const uint2*>(order) : list[n > kClusterList ? (p.passes - 1) & 1 : 0];
    g.partial = reinterpret_cast<float*>(at);
    return MGW_BY_TYPE(launch_sums, mode, g, order == nullptr, s);
}
