// Embedding lookup with scaling, and the dense gradient of the table by sorted tokens.
//
//   out[i, :] = scale * W[t_i, :]                      dW[v, :] = scale * sum over i with t_i = v of dy[i, :]
//
// The gradient's sums are taken in fp32 in the order of the positions i, so the result does not depend on how blocks
// are scheduled: the tokens are sorted (stable), the sorted list is cut into chunks of equal length -- however often
// a single word occurs -- and a warp adds up the rows of one chunk for 32 vectors of columns.  A run of equal tokens
// that lies inside a chunk is stored at once; a run that crosses a border leaves fp32 partial sums, which a second kernel
// adds up in the order of the chunks.  Rows that no token names are filled with zeros by the same launch.
#include <cooperative_groups.h>
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

constexpr int kSortThreads = 512;
constexpr int kSortItems = 4;
constexpr int kSortTile = kSortThreads * kSortItems;
constexpr int kMaxDigitBits = 10;

// ------------------------------------------------------------------------------------------------------------ lookup
constexpr int lookup_unroll(int bytes) { return bytes >= 16 ? 4 : bytes == 4 ? 8 : 16; }

template <typename T, int VEC>
__global__ void __launch_bounds__(256)
embedding_fwd_kernel(const void* __restrict__ tokens, int wide, long long n, const T* __restrict__ weight, long long ld,
                     long long vocab, int dim, float scale, T* __restrict__ out, int segments, int* status) {
    typedef typename MgwRaw<VEC * sizeof(T)>::type Raw;
    constexpr int U = lookup_unroll(VEC * (int)sizeof(T));           // vectors that a lane keeps in flight
    const int lane = threadIdx.x & 31;
    const long long warps = (long long)gridDim.x * (blockDim.x >> 5);
    const int n_vec = dim / VEC;
    for (long long task = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); task < n * segments; task += warps) {
        const long long i = task / segments;
        const int seg = (int)(task - i * segments);
        const long long t = mgw_token(tokens, wide, i);
        Raw* dst = reinterpret_cast<Raw*>(out + i * dim);
        const bool valid = t >= 0 && t < vocab;
        if (!valid && lane == 0 && seg == 0) mgw_report_token(status, MGW_OP_EMBEDDING, i, t);
        const Raw* src = reinterpret_cast<const Raw*>(weight + (valid ? t : 0) * ld);
        const int c0 = seg * 32 * U + lane;
        Raw r[U];
#pragma unroll
        for (int k = 0; k < U; ++k)
            if (valid && c0 + 32 * k < n_vec) r[k] = src[c0 + 32 * k];
#pragma unroll
        for (int k = 0; k < U; ++k) {
            if (c0 + 32 * k >= n_vec) continue;
            if (!valid || scale != 1.f) {                            // a factor of one copies the bits
                float f[VEC];
                if (valid) mgw_unpack<T, VEC>(r[k], f);
#pragma unroll
                for (int e = 0; e < VEC; ++e) f[e] = valid ? f[e] * scale : mgw_nan();
                r[k] = mgw_pack<T, VEC>(f);
            }
            dst[c0 + 32 * k] = r[k];
        }
    }
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
    int* status;
};

__device__ __forceinline__ uint2 sort_entry(const SortPass& p, long long i, bool report) {
    if (p.in != nullptr) return p.in[i];
    const long long t = mgw_token(p.tokens, p.wide, i);
    if (t < 0 || t >= p.vocab) {
        if (report) mgw_report_token(p.status, MGW_OP_EMBEDDING_GRAD, i, t);
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

// Short lists: the whole sort in one launch of one cluster, which keeps the list in its shared memory.  A block has a
// contiguous part of it; per pass the blocks read each other's histograms and write every entry to its new place, which may
// be another block's memory.
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

// Zeros for a stretch of memory (bytes a multiple of the element size), by blocks [0, blocks).
__device__ __forceinline__ void fill_zero(char* at, long long bytes, int block, int blocks) {
    const long long head = min(bytes, (long long)((16 - ((unsigned long long)at & 15)) & 15)), n = (bytes - head) >> 4;
    uint4* v = reinterpret_cast<uint4*>(at + head);
    const uint4 zero = make_uint4(0, 0, 0, 0);
    for (long long i = (long long)block * blockDim.x + threadIdx.x; i < n; i += (long long)blocks * blockDim.x) v[i] = zero;
    if (block == 0) {
        if (threadIdx.x < head) at[threadIdx.x] = 0;
        if (threadIdx.x < bytes - head - (n << 4)) at[head + (n << 4) + threadIdx.x] = 0;
    }
}

// The first cluster sorts; the others, if there are any, fill `zeros` meanwhile.
__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kClusterThreads) sort_cluster_kernel(SortPass p, int passes, char* zeros,
                                                                                                        long long zero_bytes) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    ClusterSmem& m = *reinterpret_cast<ClusterSmem*>(dynamic);
    cg::cluster_group cluster = cg::this_cluster();
    mgw_let_next_start();
    if (blockIdx.x >= kCluster) {
        fill_zero(zeros, zero_bytes, blockIdx.x - kCluster, gridDim.x - kCluster);
        return;
    }
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
#pragma unroll
            for (int c = 0; c < kCluster; ++c) {
                const uint32_t h = cluster.map_shared_rank(m.hist, c)[tid];
                if (c < rank_in_cluster) before += h;
                total += h;
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
    int chunk;                 // entries of the sorted list that one warp adds up
    int chunks, slabs;         // slab: the columns that a warp covers
    float* partial;            // [chunks][2][slabs * 32 * NV * VEC]: the run that comes in, the run that goes on
    int zero_blocks;           // blocks of the launch that fill rows without tokens (0: they are zero already)
};

constexpr int kZeroRows = 8;   // rows that one warp checks and fills

// Columns of a lane: NV vectors of VEC elements, 32 vectors apart.
template <typename T, int VEC, int NV>
struct Columns {
    typedef typename MgwRaw<VEC * sizeof(T)>::type Raw;
    int c[NV];
    int n_vec;
    __device__ __forceinline__ Columns(int slab, int lane, int dim) : n_vec(dim / VEC) {
#pragma unroll
        for (int k = 0; k < NV; ++k) c[k] = (slab * NV + k) * 32 + lane;
    }
    __device__ __forceinline__ void load(const T* row, Raw (&r)[NV]) const {
#pragma unroll
        for (int k = 0; k < NV; ++k)
            if (c[k] < n_vec) r[k] = reinterpret_cast<const Raw*>(row)[c[k]];
    }
    __device__ __forceinline__ void add(const Raw (&r)[NV], float (&acc)[NV][VEC]) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (c[k] >= n_vec) continue;
            float f[VEC];
            mgw_unpack<T, VEC>(r[k], f);
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[k][e] += f[e];
        }
    }
    __device__ __forceinline__ void store_row(T* row, float (&acc)[NV][VEC], float scale) const {
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            if (c[k] >= n_vec) continue;
            float f[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[e] = acc[k][e] * scale;
            reinterpret_cast<Raw*>(row)[c[k]] = mgw_pack<T, VEC>(f);
        }
    }
};

// fp32 partial sums of a slab: the elements of a lane (a multiple of four) one behind the other
template <int VEC, int NV>
__device__ __forceinline__ float4* partial_of(const GradArgs& a, long long chunk, int which, int slab, int lane) {
    static_assert(NV * VEC % 4 == 0, "whole float4s");
    return reinterpret_cast<float4*>(a.partial) + (((chunk * 2 + which) * a.slabs + slab) * 32 + lane) * (NV * VEC / 4);
}

template <typename T, int VEC>
__device__ __forceinline__ void zero_rows(const GradArgs& a, long long block) {
    typedef typename MgwRaw<VEC * sizeof(T)>::type Raw;
    const int lane = threadIdx.x & 31;
    const long long r0 = (block * (blockDim.x >> 5) + (threadIdx.x >> 5)) * kZeroRows;
    bool empty = false;
    if (lane < kZeroRows && r0 + lane < a.vocab) {
        long long lo = 0, hi = a.n;                                   // first entry that is not below the row
        while (lo < hi) {
            const long long mid = (lo + hi) >> 1;
            if (a.list[mid].x < (uint32_t)(r0 + lane)) lo = mid + 1; else hi = mid;
        }
        empty = lo >= a.n || a.list[lo].x != (uint32_t)(r0 + lane);
    }
    unsigned todo = __ballot_sync(0xffffffffu, empty);
    const int n_vec = a.dim / VEC;
    Raw zero;
    memset(&zero, 0, sizeof(zero));
    while (todo) {
        const int r = __ffs(todo) - 1;
        todo &= todo - 1;
        Raw* row = reinterpret_cast<Raw*>(static_cast<T*>(a.dw) + (r0 + r) * a.dim);
        for (int c = lane; c < n_vec; c += 32) row[c] = zero;
    }
}

template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(256) grad_chunks_kernel(GradArgs a) {
    mgw_let_next_start();
    mgw_wait_for_previous();
    if ((int)blockIdx.x < a.zero_blocks) {
        zero_rows<T, VEC>(a, blockIdx.x);
        return;
    }
    typedef typename MgwRaw<VEC * sizeof(T)>::type Raw;
    constexpr int U = 4;                                              // rows in flight
    const int lane = threadIdx.x & 31;
    const long long task = (long long)(blockIdx.x - a.zero_blocks) * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (task >= (long long)a.chunks * a.slabs) return;
    const long long chunk = task / a.slabs;
    const int slab = (int)(task - chunk * a.slabs);
    const Columns<T, VEC, NV> col(slab, lane, a.dim);
    const T* dy = static_cast<const T*>(a.dy);
    T* dw = static_cast<T*>(a.dw);
    const long long i0 = chunk * a.chunk;
    const long long i1 = i0 + a.chunk < a.n ? i0 + a.chunk : a.n;
    const uint32_t none = (uint32_t)a.vocab;
    uint32_t run = a.list[i0].x;
    if (run == none) return;                                          // nothing but skipped tokens from here on
    bool comes_in = i0 > 0 && a.list[i0 - 1].x == run;
    const uint32_t next_key = i1 < a.n ? a.list[i1].x : none;
    float acc[NV][VEC];
#pragma unroll
    for (int k = 0; k < NV; ++k)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[k][e] = 0.f;
    auto flush = [&](bool goes_on) {
        if (comes_in || goes_on) {
            float4* to = partial_of<VEC, NV>(a, chunk, comes_in ? 0 : 1, slab, lane);
            const float* x = &acc[0][0];
#pragma unroll
            for (int q = 0; q < NV * VEC / 4; ++q) to[q] = make_float4(x[4 * q], x[4 * q + 1], x[4 * q + 2], x[4 * q + 3]);
        } else {
            col.store_row(dw + (long long)run * a.dim, acc, a.scale);
        }
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[k][e] = 0.f;
        comes_in = false;
    };
    for (long long b0 = i0; b0 < i1; b0 += 32) {                      // 32 entries at a time, one per lane
        const uint2 mine = b0 + lane < i1 ? a.list[b0 + lane] : make_uint2(none, 0u);
        const int m = __popc(__ballot_sync(0xffffffffu, mine.x != none));
        for (int j = 0; j < m; j += U) {
            Raw r[U][NV];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t p = __shfl_sync(0xffffffffu, mine.y, (j + u) & 31);
                if (j + u < m) col.load(dy + (long long)p * a.dy_ld, r[u]);
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const uint32_t k = __shfl_sync(0xffffffffu, mine.x, (j + u) & 31);
                if (j + u < m) {
                    if (k != run) {
                        flush(false);
                        run = k;
                    }
                    col.add(r[u], acc);
                }
            }
        }
        if (m < 32) break;
    }
    flush(next_key == run);
}

// Runs that cross borders of chunks: the warp of the chunk in which a run starts adds up the partial sums.
template <typename T, int VEC, int NV>
__global__ void __launch_bounds__(256) grad_join_kernel(GradArgs a) {
    mgw_wait_for_previous();
    const int lane = threadIdx.x & 31;
    const long long task = (long long)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5);
    if (task >= (long long)(a.chunks - 1) * a.slabs) return;
    const long long chunk = task / a.slabs;
    const int slab = (int)(task - chunk * a.slabs);
    const long long i0 = chunk * a.chunk, i1 = i0 + a.chunk;          // not the last chunk: it is full
    const uint32_t run = a.list[i1 - 1].x;
    if (run == (uint32_t)a.vocab || a.list[i1].x != run) return;
    if (i0 > 0 && a.list[i0 - 1].x == run) return;                      // it started further left
    long long end = chunk + 1;                                        // the run's first chunk that is not its own
    for (bool more = true; more; ) {
        const long long c = end + lane;
        const unsigned same = __ballot_sync(0xffffffffu, c < a.chunks && a.list[c * a.chunk].x == run);
        const int k = same == 0xffffffffu ? 32 : __ffs(~same) - 1;
        end += k;
        more = k == 32;
    }
    constexpr int Q = NV * VEC / 4, U = 8;                            // partial sums in flight, added in their order
    float4 x[Q];
    const float4* from = partial_of<VEC, NV>(a, chunk, 1, slab, lane);
#pragma unroll
    for (int q = 0; q < Q; ++q) x[q] = from[q];
    const long long step = 2LL * a.slabs * 32 * Q;
    from = partial_of<VEC, NV>(a, chunk + 1, 0, slab, lane);
    for (long long c = chunk + 1; c < end; c += U, from += U * step) {
        float4 y[U][Q];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < Q; ++q) y[u][q] = c + u < end ? from[u * step + q] : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int q = 0; q < Q; ++q) { x[q].x += y[u][q].x; x[q].y += y[u][q].y; x[q].z += y[u][q].z; x[q].w += y[u][q].w; }
    }
    float acc[NV][VEC];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        float* to = &acc[0][0] + 4 * q;
        to[0] = x[q].x; to[1] = x[q].y; to[2] = x[q].z; to[3] = x[q].w;
    }
    const Columns<T, VEC, NV> col(slab, lane, a.dim);
    col.store_row(static_cast<T*>(a.dw) + (long long)run * a.dim, acc, a.scale);
}

int element_size(int dtype) { return dtype == MGW_F32 ? 4 : 2; }

// Widest access in bytes that every row of a matrix allows: 16, 4 or one element.
int access_bytes(const void* base, long long ld, int dim, int dtype) {
    const int es = element_size(dtype);
    const unsigned long long a = (unsigned long long)(uintptr_t)base | (unsigned long long)(ld * es) | (unsigned long long)((long long)dim * es);
    return (a & 15) == 0 ? 16 : (a & 3) == 0 ? 4 : es;
}

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
    int vec, nv, slabs, chunk, chunks;
    size_t partial_bytes;
};

SumPlan sum_plan(long long n, int dim, int dtype, int bytes) {
    SumPlan s;
    const int es = element_size(dtype);
    s.vec = bytes / es;
    s.nv = s.vec >= 4 ? 1 : es == 2 && s.vec == 1 ? 8 : 4;            // narrow accesses: several per lane and row
    const int n_vec = dim / s.vec;
    s.slabs = (n_vec + 32 * s.nv - 1) / (32 * s.nv);
    // a warp's part of the list: long enough that partial sums are few, short enough that there are warps for every SM
    s.chunk = 8;
    while (s.chunk < 512 && (n / s.chunk) * s.slabs > 148LL * 64) s.chunk *= 2;
    s.chunks = (int)((n + s.chunk - 1) / s.chunk);
    s.partial_bytes = (size_t)s.chunks * 2 * s.slabs * 32 * s.nv * s.vec * sizeof(float);
    return s;
}

template <typename T, int VEC, int NV>
int launch_sums(const GradArgs& a, cudaStream_t stream) {
    const long long tasks = (long long)a.chunks * a.slabs;
    const long long blocks = (tasks + 7) / 8 + a.zero_blocks;
    const int rc = launch_dependent(grad_chunks_kernel<T, VEC, NV>, blocks, 256, 0, stream, a);
    if (rc != MGW_OK || a.chunks == 1) return rc;
    return launch_dependent(grad_join_kernel<T, VEC, NV>, ((long long)(a.chunks - 1) * a.slabs + 7) / 8, 256, 0, stream, a);
}

template <typename T, int VEC>
int launch_fwd(const void* tokens, int wide, long long n, const void* weight, long long ld, long long vocab, int dim, float scale,
               void* out, int* status, cudaStream_t stream) {
    const int n_vec = dim / VEC;
    const int per = 32 * lookup_unroll(VEC * (int)sizeof(T)), segments = (n_vec + per - 1) / per;
    const long long blocks = (n * segments + 7) / 8;
    const unsigned grid = (unsigned)(blocks < 148LL * 64 ? blocks : 148LL * 64);
    embedding_fwd_kernel<T, VEC><<<grid, 256, 0, stream>>>(tokens, wide, n, static_cast<const T*>(weight), ld, vocab, dim, scale,
                                                           static_cast<T*>(out), segments, status);
    MGW_CUDA_CHECK(cudaGetLastError());
    return MGW_OK;
}

bool bad_sizes(long long n, long long vocab, int dim, int dtype) {
    return n < 0 || n > 0x7fffffffLL || vocab < 1 || vocab > 0x7ffffffeLL || dim < 1 || dtype < MGW_F32 || dtype > MGW_BF16;
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

extern "C" int mgw_embedding_fwd(const void* tokens, int wide, long long n, const void* weight, long long ld, long long vocab,
                                 int dim, int dtype, float scale, void* out, int* status, void* stream) {
    if (bad_sizes(n, vocab, dim, dtype) || ld < dim) return MGW_ERR_ARG;
    if (n == 0) return MGW_OK;
    if (tokens == nullptr || weight == nullptr || out == nullptr || status == nullptr) return MGW_ERR_ARG;
    const int wb = access_bytes(weight, ld, dim, dtype), ob = access_bytes(out, dim, dim, dtype);
    const int bytes = wb < ob ? wb : ob;
    cudaStream_t s = (cudaStream_t)stream;
#define MGW_FWD(T, V) launch_fwd<T, V>(tokens, wide, n, weight, ld, vocab, dim, scale, out, status, s)
    if (dtype == MGW_F32) return bytes == 16 ? MGW_FWD(float, 4) : MGW_FWD(float, 1);
    if (dtype == MGW_F16) return bytes == 16 ? MGW_FWD(__half, 8) : bytes == 4 ? MGW_FWD(__half, 2) : MGW_FWD(__half, 1);
    return bytes == 16 ? MGW_FWD(__nv_bfloat16, 8) : bytes == 4 ? MGW_FWD(__nv_bfloat16, 2) : MGW_FWD(__nv_bfloat16, 1);
#undef MGW_FWD
}

extern "C" size_t mgw_embedding_grad_bytes(long long n, long long vocab, int dim, int dtype) {
    if (bad_sizes(n, vocab, dim, dtype) || n == 0) return 0;
    const SortPlan p = sort_plan(n, vocab);
    size_t most = 0;                                                  // whatever access width the call ends up with
    const int es = element_size(dtype);
    for (int bytes : {16, 4, es}) {
        if ((long long)dim * es % bytes) continue;
        const SumPlan s = sum_plan(n, dim, dtype, bytes);
        if (s.partial_bytes > most) most = s.partial_bytes;
    }
    return 2 * p.list_bytes + p.counts_bytes + p.totals_bytes + most;
}

extern "C" int mgw_embedding_grad(const void* dy, long long dy_ld, const void* tokens, int wide, long long n, long long vocab, int dim,
                                  int dtype, float scale, long long padding, void* dw, void* work, size_t work_bytes, int* status,
                                  void* stream) {
    if (bad_sizes(n, vocab, dim, dtype) || dw == nullptr) return MGW_ERR_ARG;
    cudaStream_t s = (cudaStream_t)stream;
    if (n == 0) {
        MGW_CUDA_CHECK(cudaMemsetAsync(dw, 0, (size_t)vocab * dim * element_size(dtype), s));
        return MGW_OK;
    }
    if (dy == nullptr || tokens == nullptr || work == nullptr || status == nullptr || (n > 1 && dy_ld < dim)) return MGW_ERR_ARG;
    if (work_bytes < mgw_embedding_grad_bytes(n, vocab, dim, dtype) || ((uintptr_t)work & 15)) return MGW_ERR_ARG;
    const SortPlan p = sort_plan(n, vocab);
    const int db = access_bytes(dy, dy_ld, dim, dtype), wb = access_bytes(dw, dim, dim, dtype);
    const int bytes = db < wb ? db : wb;
    const SumPlan q = sum_plan(n, dim, dtype, bytes);
    char* at = static_cast<char*>(work);
    uint2* list[2];
    for (int i = 0; i < 2; ++i) {
        list[i] = reinterpret_cast<uint2*>(at);
        at += p.list_bytes;
    }
    uint32_t* counts = reinterpret_cast<uint32_t*>(at); at += p.counts_bytes;
    uint32_t* totals = reinterpret_cast<uint32_t*>(at); at += p.totals_bytes;
    // Rows without tokens: at most n rows have one.  With n below the vocabulary everything is filled with zeros while the
    // one cluster sorts (rows with tokens are written twice); with more tokens most rows have one, and the launch that adds
    // up looks for those that have none.
    const bool zero_first = n <= kClusterList && n < vocab;
    SortPass a = {};
    a.tokens = tokens; a.wide = wide; a.out = list[0];
    a.counts = counts; a.totals = totals;
    a.n = n; a.tiles = p.tiles; a.bits = p.bits;
    a.vocab = vocab; a.padding = padding; a.status = status;
    if (n <= kClusterList) {
        MGW_CUDA_CHECK(cudaFuncSetAttribute(sort_cluster_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(ClusterSmem)));
        sort_cluster_kernel<<<zero_first ? 16 * kCluster : kCluster, kClusterThreads, sizeof(ClusterSmem), s>>>(
            a, p.passes, static_cast<char*>(dw), (long long)vocab * dim * element_size(dtype));
        MGW_CUDA_CHECK(cudaGetLastError());
    } else {
        const int bins = 1 << p.bits;
        const size_t hist_smem = (size_t)bins * 4, scatter_smem = (size_t)bins * 4 + (size_t)bins * 2 * (kSortThreads / 32);
        for (int k = 0; k < p.passes; ++k) {
            a.in = k == 0 ? nullptr : list[(k + 1) & 1];
            a.out = list[k & 1];
            a.shift = k * p.bits;
            int rc = launch_dependent(sort_hist_kernel, p.tiles, kSortThreads, hist_smem, s, a);
            if (rc == MGW_OK) rc = launch_dependent(sort_scan_kernel, (bins + 7) / 8, 256, 0, s, counts, totals, bins, p.tiles);
            if (rc == MGW_OK) rc = launch_dependent(sort_scatter_kernel, p.tiles, kSortThreads, scatter_smem, s, a);
            if (rc != MGW_OK) return rc;
        }
    }
    GradArgs g;
    g.list = list[n > kClusterList ? (p.passes - 1) & 1 : 0];
    g.n = n; g.dy = dy; g.dy_ld = dy_ld; g.dw = dw; g.vocab = vocab; g.dim = dim; g.scale = scale;
    g.chunk = q.chunk; g.chunks = q.chunks; g.slabs = q.slabs;
    g.partial = reinterpret_cast<float*>(at);
    g.zero_blocks = zero_first ? 0 : (int)((vocab + 8 * kZeroRows - 1) / (8 * kZeroRows));
    if (dtype == MGW_F32) return bytes == 16 ? launch_sums<float, 4, 1>(g, s) : launch_sums<float, 1, 4>(g, s);
    if (dtype == MGW_F16)
        return bytes == 16 ? launch_sums<__half, 8, 1>(g, s) : bytes == 4 ? launch_sums<__half, 2, 4>(g, s) : launch_sums<__half, 1, 8>(g, s);
    return bytes == 16 ? launch_sums<__nv_bfloat16, 8, 1>(g, s)
                       : bytes == 4 ? launch_sums<__nv_bfloat16, 2, 4>(g, s) : launch_sums<__nv_bfloat16, 1, 8>(g, s);
}
