// Token tables in training: lookup of scaled rows, and the gradient of the table.
//
//   lookup     out[i, :] = scale * W[tok[i], :]
//   gradient   dW[v, :]  = scale * sum of dy[i, :] over the i with tok[i] = v
//
// Both are bounded by HBM bandwidth, a product or a sum per element moved: 6.5 TB/s where as much is read as written, 4.0 TB/s for
// writing alone (a plain fill: 3.9), which is what the whole gradient of a large table mostly is.  No counterparts in the
// reference.
#include "tbe_elements.cuh"
#include "tbe_token_plan.h"

namespace tbe {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;

__device__ __forceinline__ int64_t load_token(const void* tokens, bool wide, int64_t i)
{
    return wide ? __ldg(reinterpret_cast<const long long*>(tokens) + i) : static_cast<int64_t>(__ldg(reinterpret_cast<const int*>(tokens) + i));
}

// ---- lookup ---------------------------------------------------------------------------------------------------
//
// `lanes` threads (a power of two, at most the block) share a row and walk its pieces of VEC elements; a thread holds ROWS
// rows' pieces at a time, so that a block has ROWS * 16 bytes per thread in flight.  16384 rows of 4096 bf16 of a table of
// 131072: 31 us, 5.8 TB/s of what has to be moved.
__device__ __forceinline__ const char* row_of_token(const void* weight, int64_t row_bytes, int64_t num_embeddings, const void* tokens, int wide, int64_t i,
                                                    bool report, int32_t* error_flag)
{
    const int64_t t = load_token(tokens, wide, i);
    if (t >= 0 && t < num_embeddings) return static_cast<const char*>(weight) + t * row_bytes;
    if (t != -1 && error_flag && report) atomicOr(error_flag, 4);
    return nullptr;
}

template <typename TI, typename TO, int VEC, int ROWS>
__global__ void __launch_bounds__(kThreads)
token_embedding_kernel(const TI* __restrict__ weight, int64_t num_embeddings, int D, int64_t weight_stride, const void* __restrict__ tokens, int wide,
                       int64_t n, float scale, TO* __restrict__ out, int64_t out_stride, int lanes_log2, int32_t* error_flag)
{
    const int lanes = 1 << lanes_log2, k = threadIdx.x & (lanes - 1), pieces = D / VEC;
    const int rows_at_once = kThreads >> lanes_log2;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (rows_at_once * ROWS) + (threadIdx.x >> lanes_log2);
    const TI* src[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int64_t i = first + static_cast<int64_t>(j) * rows_at_once;
        src[j] = i < n ? reinterpret_cast<const TI*>(row_of_token(weight, weight_stride * sizeof(TI), num_embeddings, tokens, wide, i, k == 0, error_flag)) : nullptr;
    }
    for (int p = k; p < pieces; p += lanes) {
        Piece<TI, VEC> in[ROWS];
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            if (src[j]) load_piece<TI, VEC>(in[j], src[j] + static_cast<int64_t>(p) * VEC);
            else clear_piece(in[j]);
        }
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            const int64_t i = first + static_cast<int64_t>(j) * rows_at_once;
            if (i >= n) continue;
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = src[j] ? scale * element(in[j], e) : 0.0f;
            store_piece<TO, VEC>(out + i * out_stride + static_cast<int64_t>(p) * VEC, v);
        }
    }
}

// Rows that cannot be moved in pieces.  Cut by the result's 16-byte borders, all but the ends of a row is still written in whole
// pieces, and what goes into them is read in aligned words and shifted; a lane has kSplitAtOnce of them in flight.  The ends go
// element by element.  At most a warp shares a row: what a row costs beside its pieces is a good part of the instructions, which
// bound this form.  [65536, 1001] bf16: 43 us, 3.1 TB/s written (80 us element by element).
constexpr int kSplitAtOnce = 4;

template <typename TI, typename TO>
__global__ void __launch_bounds__(kThreads)
token_embedding_split_kernel(const TI* __restrict__ weight, int64_t num_embeddings, int D, int64_t weight_stride, const void* __restrict__ tokens, int wide,
                             int64_t n, float scale, TO* __restrict__ out, int64_t out_stride, int lanes_log2, int32_t* error_flag)
{
    constexpr int VEC = 16 / static_cast<int>(sizeof(TO));
    const int lanes = 1 << lanes_log2, k = threadIdx.x & (lanes - 1);
    const int64_t i = (static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x) >> lanes_log2;
    if (i >= n) return;
    const TI* src = reinterpret_cast<const TI*>(row_of_token(weight, weight_stride * sizeof(TI), num_embeddings, tokens, wide, i, k == 0, error_flag));
    TO* to = out + i * out_stride;
    int head = static_cast<int>(((16 - (reinterpret_cast<uintptr_t>(to) & 15)) & 15) / sizeof(TO));
    head = head < D ? head : D;
    const int whole = (D - head) / VEC, ends = D - whole * VEC;
    SplitRow split;
    split.of(src, D);
    for (int p = k; p < whole; p += kSplitAtOnce * lanes) {
        SplitPiece<TI, VEC> in[kSplitAtOnce];
#pragma unroll
        for (int j = 0; j < kSplitAtOnce; ++j)
            if (src && p + j * lanes < whole) in[j].load(split, head + (p + j * lanes) * VEC);
#pragma unroll
        for (int j = 0; j < kSplitAtOnce; ++j) {
            if (p + j * lanes >= whole) break;
            float v[VEC] = {};
            if (src) {
                const Piece<TI, VEC> r = in[j].piece();
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[e] = scale * element(r, e);
            }
            store_piece<TO, VEC>(to + head + (p + j * lanes) * VEC, v);
        }
    }
    for (int e = k; e < ends; e += lanes) {
        const int c = e < head ? e : whole * VEC + e;
        Piece<TI, 1> r;
        clear_piece(r);
        if (src) load_piece<TI, 1>(r, src + c);
        const float v[1] = {src ? scale * element(r, 0) : 0.0f};
        store_piece<TO, 1>(to + c, v);
    }
}

template <typename TI, typename TO, int VEC>
int launch_token_embedding(const TI* weight, int64_t num_embeddings, int64_t D, int64_t weight_stride, const void* tokens, int wide, int64_t n,
                           float scale, TO* out, int64_t out_stride, int32_t* error_flag, cudaStream_t s)
{
    const int64_t pieces = VEC ? D / (VEC ? VEC : 1) : D / (16 / static_cast<int64_t>(sizeof(TO)));
    const bool few = n <= static_cast<int64_t>(sm_count()) * 8;      // rows: as many threads to each as there are
    const int most = VEC || few ? kThreads : 32, share = VEC || few ? 1 : kSplitAtOnce;
    int lanes_log2 = 0;
    while ((share << lanes_log2) < pieces && (1 << lanes_log2) < most) ++lanes_log2;
    const int at_once = kThreads >> lanes_log2;
    const bool many = VEC && n >= static_cast<int64_t>(sm_count()) * 8 * at_once * 4;
    const int64_t per = static_cast<int64_t>(at_once) * (many ? 4 : 1), blocks = (n + per - 1) / per;
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "token_embedding: too many tokens");
    auto launch = [&](auto* kernel) {
        kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(weight, num_embeddings, static_cast<int>(D), weight_stride, tokens, wide, n, scale, out,
                                                                  out_stride, lanes_log2, error_flag);
        return check_launch("token_embedding_kernel");
    };
    if constexpr (VEC == 0) return launch(token_embedding_split_kernel<TI, TO>);
    else return many ? launch(token_embedding_kernel<TI, TO, VEC, 4>) : launch(token_embedding_kernel<TI, TO, VEC, 1>);
}

// ---- gradient: sort by token ----------------------------------------------------------------------------------
//
// Keys are tokens (num_embeddings stands for one that takes no part and sorts last), values their positions.  A stable
// radix sort from the lowest digit up keeps the positions of equal tokens in order, which fixes the order of every sum.
// A warp owns neighbouring keys and takes them 32 at a time: lanes with the same digit find one another, and a running
// count per warp and digit gives each its rank.
constexpr int kMaxBins = 512;

struct SortInput {
    const void* tokens;
    int wide;
    int64_t n, num_embeddings, padding_idx;
};

__device__ __forceinline__ uint32_t token_key(const SortInput& in, int64_t i)
{
    const int64_t t = load_token(in.tokens, in.wide, i);
    return static_cast<uint32_t>((t < 0 || t >= in.num_embeddings || t == in.padding_idx) ? in.num_embeddings : t);
}

// The rank of this lane's key among those of its warp with the same digit so far; `count` is the warp's.
template <typename C>
__device__ __forceinline__ uint32_t warp_rank(uint32_t digit, bool live, C* count)
{
    const int lane = threadIdx.x & 31;
    const uint32_t peers = __match_any_sync(kFull, live ? digit : 0xffffffffu);
    const uint32_t before = live ? count[digit] : 0u;
    __syncwarp();
    if (live && lane == 31 - __clz(peers)) count[digit] = static_cast<C>(before + __popc(peers));
    __syncwarp();
    return before + __popc(peers & ((1u << lane) - 1u));
}

// Exclusive running sum over a block of 1024 threads; `total` is everything.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t* warp_tot, uint32_t& total)
{
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t incl = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(kFull, incl, d);
        if (lane >= d) incl += up;
    }
    __syncthreads();      // warp_tot may still be read from an earlier call
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    uint32_t w = warp_tot[lane], run = w;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(kFull, run, d);
        if (lane >= d) run += up;
    }
    total = __shfl_sync(kFull, run, 31);
    return __shfl_sync(kFull, run - w, warp) + incl - v;
}

// ---- up to kClusterKeys tokens: one cluster sorts in shared memory, the other blocks clear the gradient meanwhile ------
//
// A block of the cluster holds items (at most ITEMS) * 1024 neighbouring places.  Per digit: ranks in registers, digit counts exchanged
// between the blocks, then every key straight to its place in whichever block's shared memory that is.  Bound by latency: the
// barriers, and a warp's ranks one after the other.  13 us for 8192 tokens of 128000 (two digits), 17 us for 32768, 24 us for
// 65537; clusters of eight blocks took 21 and 37 us, three kernels per digit through global memory 27 us for 8192.
constexpr int kSortWarps = kSortThreads / 32;

struct FillArgs {
    char* out;
    int64_t rows, row_bytes, stride_bytes;      // rows == 0: nothing to clear
    int64_t early;                              // so many are cleared beside the sort, the others beside the sums
    uint32_t* met;                              // a bit per row: tokens name it (null: early == rows)
};

// Shared memory that a clearing block keeps at zero and copies out, beside the sort and beside the sums.
constexpr int kZeroBytes = 32 * 1024, kFewZeroBytes = 8 * 1024;

// Clears `bytes` at p: thread `thread` of `threads` takes every threads-th run of ZEROS bytes, by bulk copies from `zeros`; what
// lies in front of the first 16-byte border and behind the last goes element by element.
template <int ZEROS>
__device__ __forceinline__ void clear_run(char* p, int64_t bytes, int64_t thread, int64_t threads, int unit, const void* zeros)
{
    const int64_t head = min((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15, bytes), body = (bytes - head) & ~int64_t(15);
    for (int64_t at = thread * ZEROS; at < body; at += threads * ZEROS) {
        const uint32_t run = static_cast<uint32_t>(body - at < ZEROS ? body - at : ZEROS);
        asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(p + head + at), "r"(static_cast<uint32_t>(__cvta_generic_to_shared(zeros))),
                     "r"(run) : "memory");
        asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    const int64_t edge = (bytes - body) >> (unit == 4 ? 2 : 1);
    for (int64_t i = thread; i < edge; i += threads) {
        char* q = i * unit < head ? p + i * unit : p + body + i * unit;
        if (unit == 4) *reinterpret_cast<uint32_t*>(q) = 0u;
        else *reinterpret_cast<unsigned short*>(q) = 0;
    }
}

template <int ZEROS>
__device__ __forceinline__ void make_zeros(unsigned char* zeros)
{
    for (int i = threadIdx.x; i < ZEROS / 16; i += blockDim.x) reinterpret_cast<uint4*>(zeros)[i] = make_uint4(0u, 0u, 0u, 0u);
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
}

// A block's share of the first `early` rows; `zeros`: kZeroBytes of shared memory, 16-byte aligned.
__device__ __forceinline__ void clear_rows(const FillArgs& f, int unit, int64_t block, int64_t blocks, unsigned char* zeros)
{
    make_zeros<kZeroBytes>(zeros);
    if (f.stride_bytes == f.row_bytes) {
        if (threadIdx.x == 0) clear_run<kZeroBytes>(f.out, f.early * f.row_bytes, block, blocks, unit, zeros);
    } else {
        for (int64_t r = block * blockDim.x + threadIdx.x; r < f.early; r += blocks * blockDim.x)
            clear_run<kZeroBytes>(f.out + r * f.stride_bytes, f.row_bytes, 0, 1, unit, zeros);
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

// Of the rows 32 w0 .. 32 w1 those that no token names (a bit of `met` each, which begins with row 32 w0): a thread takes 32 rows
// at a time.
__device__ __forceinline__ void clear_unmet_rows(const FillArgs& f, int unit, int64_t w0, int64_t w1, const uint32_t* met, int64_t thread, int64_t threads,
                                                 const void* zeros)
{
    for (int64_t w = w0 + thread; w < w1; w += threads) {
        const int64_t left = f.rows - w * 32;
        uint32_t clear = ~met[w - w0] & (left < 32 ? (1u << left) - 1u : kFull);
        while (clear) {
            const int first = __ffs(clear) - 1;
            const uint32_t behind = ~(clear >> first);
            int run = behind ? __ffs(behind) - 1 : 32 - first;
            if (f.stride_bytes != f.row_bytes) run = 1;
            clear_run<kFewZeroBytes>(f.out + (w * 32 + first) * f.stride_bytes, run * f.row_bytes, 0, 1, unit, zeros);
            clear &= run == 32 ? 0u : ~(((1u << run) - 1u) << first);
        }
    }
    asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
// The address of `p` of this block's shared memory in block `rank` of the cluster.
__device__ __forceinline__ uint32_t shared_of(const void* p, uint32_t rank)
{
    uint32_t a;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
    return a;
}

__host__ __device__ constexpr int64_t sort_shared_bytes(int items) { return int64_t(items) * kSortThreads * 8 + kSortWarps * kMaxBins * 2 + kSortBlocks * kMaxBins * 4 + kMaxBins * 4 + 128; }

// Sorts; block `mine` of `cluster` (1: alone) is left with places mine * items * 1024 on, (token << 32 | position) each, in the
// memory that is returned, the first of `shared`.  Ends with a barrier of all.
template <int ITEMS>
__device__ __forceinline__ unsigned long long* sort_in_shared(const SortInput& in, int cluster, uint32_t mine, int items, int passes, int width, unsigned char* shared)
{
    unsigned long long* buf = reinterpret_cast<unsigned long long*>(shared);
    unsigned short(*count)[kMaxBins] = reinterpret_cast<unsigned short(*)[kMaxBins]>(buf + ITEMS * kSortThreads);
    uint32_t(*table)[kMaxBins] = reinterpret_cast<uint32_t(*)[kMaxBins]>(count + kSortWarps);
    uint32_t* base = reinterpret_cast<uint32_t*>(table + kSortBlocks);
    uint32_t* warp_tot = base + kMaxBins;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, bins = 1 << width;
    const int per = items * kSortThreads;
    const int64_t first = static_cast<int64_t>(mine) * per;
    const int at = warp * (32 * items) + lane;
    // to / per: a quotient below 256 of numbers below 256 by one of at most 16, by its inverse in 1 / 65536
    const uint32_t inverse = (65536u + items - 1) / items;
    auto rank_of = [&](uint32_t to) { return ((to / kSortThreads) * inverse) >> 16; };
    auto sync_all = [&] {
        if (cluster > 1) cluster_sync();
        else __syncthreads();
    };
    if (cluster > 1) cluster_sync();      // every block has begun: its shared memory may be written
    for (int p = 0; p < passes; ++p) {
        uint32_t key[ITEMS], pos[ITEMS], rank[ITEMS];
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int64_t i = first + at + j * 32;
            key[j] = pos[j] = 0u;
            if (j < items && i < in.n) {
                if (p == 0) {
                    key[j] = token_key(in, i);
                    pos[j] = static_cast<uint32_t>(i);
                } else {
                    const unsigned long long both = buf[at + j * 32];
                    key[j] = static_cast<uint32_t>(both >> 32);
                    pos[j] = static_cast<uint32_t>(both);
                }
            }
        }
        for (int b = threadIdx.x; b < kSortWarps * kMaxBins / 2; b += kSortThreads) reinterpret_cast<uint32_t*>(count)[b] = 0u;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
            if (j < items) rank[j] = warp_rank((key[j] >> (p * width)) & (bins - 1), first + at + j * 32 < in.n, count[warp]);
        __syncthreads();
        if (threadIdx.x < bins) {
            uint32_t run = 0;
#pragma unroll
            for (int w0 = 0; w0 < kSortWarps; w0 += 16) {      // reads first: a write between them would hold up the next
                uint32_t c[16];
#pragma unroll
                for (int w = 0; w < 16; ++w) c[w] = count[w0 + w][threadIdx.x];
#pragma unroll
                for (int w = 0; w < 16; ++w) {
                    count[w0 + w][threadIdx.x] = static_cast<unsigned short>(run);
                    run += c[w];
                }
            }
            if (cluster > 1) {
                for (int r = 0; r < cluster; ++r)
                    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(shared_of(&table[mine][threadIdx.x], r)), "r"(run) : "memory");
            } else {
                table[0][threadIdx.x] = run;
            }
        }
        sync_all();      // every block's counts are here, and every block holds its keys in registers
        uint32_t all = 0, below = 0, total;
        if (threadIdx.x < bins)
            for (int r = 0; r < cluster; ++r) {
                const uint32_t c = table[r][threadIdx.x];
                all += c;
                if (r < mine) below += c;
            }
        const uint32_t before = block_exclusive(all, warp_tot, total);
        if (threadIdx.x < bins) base[threadIdx.x] = before + below;
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            if (j >= items || first + at + j * 32 >= in.n) continue;
            const uint32_t d = (key[j] >> (p * width)) & (bins - 1), to = base[d] + count[warp][d] + rank[j];
            const unsigned long long both = (static_cast<unsigned long long>(key[j]) << 32) | pos[j];
            if (cluster > 1)
                asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(shared_of(buf + (to - rank_of(to) * per), rank_of(to))), "l"(both) : "memory");
            else
                buf[to] = both;
        }
        sync_all();
    }
    return buf;
}

template <int ITEMS>
__global__ void __launch_bounds__(kSortThreads, 1)
sort_tokens_kernel(const SortInput in, int cluster, int items, int passes, int width, uint2* __restrict__ sorted, const FillArgs fill, int unit)
{
    extern __shared__ __align__(16) unsigned char sort_smem[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (blockIdx.x >= cluster) {
        clear_rows(fill, unit, blockIdx.x - cluster, gridDim.x - cluster, sort_smem);
        return;
    }
    const uint32_t mine = cluster > 1 ? cluster_rank() : 0u;
    const int per = items * kSortThreads;
    const int64_t first = static_cast<int64_t>(mine) * per;
    if (fill.met)
        for (int64_t w = mine * kSortThreads + threadIdx.x; w < (fill.rows + 31) / 32; w += cluster * kSortThreads) fill.met[w] = 0u;
    const unsigned long long* buf = sort_in_shared<ITEMS>(in, cluster, mine, items, passes, width, sort_smem);
    for (int i = threadIdx.x; i < per && first + i < in.n; i += kSortThreads) {
        const unsigned long long both = buf[i];
        const uint32_t key = static_cast<uint32_t>(both >> 32);
        sorted[first + i] = make_uint2(key, static_cast<uint32_t>(both));
        // once per token and block at least; the words were cleared two barriers ago or more
        if (fill.met && key < in.num_embeddings && (i == 0 || static_cast<uint32_t>(buf[i - 1] >> 32) != key)) atomicOr(fill.met + key / 32, 1u << (key & 31));
    }
}

// ---- more tokens than a cluster holds, or no cluster to be had: per digit tile histograms, their running sums tile by tile, and the
// scatter ----------------------------------------------------------------------------------
constexpr int kWarps = kThreads / 32;
constexpr int kSortItems = 16;
constexpr int kSortTile = kThreads * kSortItems;

template <bool FIRST>
__device__ __forceinline__ uint2 sort_entry(const SortInput& in, const uint2* from, int64_t i)
{
    if constexpr (FIRST) return make_uint2(token_key(in, i), static_cast<uint32_t>(i));
    else return __ldg(from + i);
}

template <bool FIRST>
__global__ void __launch_bounds__(kThreads)
sort_histogram_kernel(const SortInput in, const uint2* __restrict__ from, int shift, int bins, uint32_t* __restrict__ hist)
{
    __shared__ uint32_t count[kMaxBins];
    for (int b = threadIdx.x; b < bins; b += kThreads) count[b] = 0;
    __syncthreads();
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile;
#pragma unroll 4
    for (int j = 0; j < kSortItems; ++j) {
        const int64_t i = base + j * kThreads + threadIdx.x;
        if (i < in.n) atomicAdd(&count[(sort_entry<FIRST>(in, from, i).x >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) hist[static_cast<int64_t>(b) * gridDim.x + blockIdx.x] = count[b];
}

// One warp per digit: the counts of its tiles become exclusive running sums, `totals` their sum.
__global__ void __launch_bounds__(kThreads) sort_places_kernel(uint32_t* __restrict__ hist, int64_t tiles, int bins, uint32_t* __restrict__ totals)
{
    const int lane = threadIdx.x & 31, bin = blockIdx.x * kWarps + (threadIdx.x >> 5);
    if (bin >= bins) return;
    uint32_t* row = hist + bin * tiles;
    uint32_t carry = 0;
    for (int64_t base = 0; base < tiles; base += 32) {
        const uint32_t c = base + lane < tiles ? row[base + lane] : 0u;
        uint32_t incl = c;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t up = __shfl_up_sync(kFull, incl, d);
            if (lane >= d) incl += up;
        }
        if (base + lane < tiles) row[base + lane] = carry + incl - c;
        carry += __shfl_sync(kFull, incl, 31);
    }
    if (lane == 0) totals[bin] = carry;
}

template <bool FIRST>
__global__ void __launch_bounds__(kThreads)
sort_scatter_kernel(const SortInput in, const uint2* __restrict__ from, int shift, int bins, const uint32_t* __restrict__ places,
                    const uint32_t* __restrict__ totals, uint2* __restrict__ to)
{
    __shared__ uint32_t count[kWarps][kMaxBins];
    __shared__ uint32_t warp_tot[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = threadIdx.x; b < kWarps * kMaxBins; b += kThreads) (&count[0][0])[b] = 0;
    __syncthreads();
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * (32 * kSortItems) + lane;
    uint2 entry[kSortItems];
    uint32_t rank[kSortItems];
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        const int64_t i = base + j * 32;
        entry[j] = i < in.n ? sort_entry<FIRST>(in, from, i) : make_uint2(0u, 0u);
    }
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) rank[j] = warp_rank((entry[j].x >> shift) & (bins - 1), base + j * 32 < in.n, count[warp]);
    // digits of this thread: two neighbouring ones, behind all of the threads before it
    const int b0 = 2 * threadIdx.x;
    const uint32_t t0 = b0 < bins ? __ldg(totals + b0) : 0u, t1 = b0 + 1 < bins ? __ldg(totals + b0 + 1) : 0u;
    uint32_t incl = t0 + t1;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t up = __shfl_up_sync(kFull, incl, d);
        if (lane >= d) incl += up;
    }
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    uint32_t smaller = incl - t0 - t1;
    for (int w = 0; w < warp; ++w) smaller += warp_tot[w];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int b = b0 + i;
        if (b >= bins) break;
        uint32_t run = smaller + (i ? t0 : 0u) + places[static_cast<int64_t>(b) * gridDim.x + blockIdx.x];
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = count[w][b];
            count[w][b] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j)
        if (base + j * 32 < in.n) to[count[warp][(entry[j].x >> shift) & (bins - 1)] + rank[j]] = entry[j];
}

__global__ void __launch_bounds__(kThreads) clear_rows_kernel(const FillArgs fill, int unit)
{
    __shared__ __align__(16) unsigned char zeros[kZeroBytes];
    clear_rows(fill, unit, blockIdx.x, gridDim.x, zeros);
}

// ---- gradient: sums ---------------------------------------------------------------------------------------------
//
// The sorted positions are cut into tiles; a group of lanes (a warp where rows are wide) walks a tile over eight columns per
// lane and writes a row when its token ends.  A token that goes on past the tile leaves its piece in `parts`: slot 0 of a
// tile holds the sum of the token that came in from the tile before (the whole tile, if it goes on), slot 1 that of one that
// starts here and goes on.  join_parts_kernel adds the pieces in the order of the tiles.
constexpr int kColumns = 8;                 // per lane
constexpr int kAhead = 4;                   // rows whose loads are in flight together

// What the kernel before writes, `sorted` and `parts`, is read by plain loads: a block may have begun before that kernel ended,
// and the read-only path may be taken before the wait for it.
struct SumArgs {
    const uint2* sorted;
    int64_t n;
    uint32_t none;
    int64_t grad_stride, out_stride;
    int D, padded_D;                        // padded_D: of a row of `parts`
    int tile_rows, slices, lanes_log2;      // slices: of a row, lanes * 8 columns each
    int64_t tiles;
    float scale;
    float* parts;
};

// Such a load that stays behind the wait (volatile), but that the stores of sums do not hold up, as they would one that may alias.
__device__ __forceinline__ uint2 entry(const uint2* p)
{
    uint2 v;
    asm volatile("ld.global.v2.u32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}

// A lane's eight columns lie in runs of kRun neighbours, `lanes` runs apart: of 16 bytes where rows are aligned, else of 4, so that
// the lanes' loads and stores lie side by side wherever a row begins.  (With 16 bytes to a lane there too, read in two aligned words
// each and shifted, and stored element by element, the gradient of 65537 tokens of 1001 fp16 takes 100 us, not 90.)
template <typename T> constexpr int kVec = 16 / static_cast<int>(sizeof(T));
template <typename T, bool ALIGNED> constexpr int kRun = (ALIGNED ? 16 : 4) / static_cast<int>(sizeof(T));

template <typename T, bool ALIGNED>
struct Columns {
    static constexpr int VEC = kVec<T>, kPieces = kColumns / VEC;
    Piece<T, VEC> p[kPieces];

    __device__ __forceinline__ void load(const T* row, int column, int step, int D)
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            if (column + i * step < D) load_piece<T, VEC>(p[i], row + column + i * step);
            else clear_piece(p[i]);
        }
    }
    __device__ __forceinline__ void add_to(float (&acc)[kColumns]) const
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i)
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[i * VEC + e] += element(p[i], e);
    }
};

template <>
struct Columns<float, false> {
    float v[kColumns];

    __device__ __forceinline__ void load(const float* row, int column, int step, int D)
    {
#pragma unroll
        for (int i = 0; i < kColumns; ++i) v[i] = column + i * step < D ? __ldg(row + column + i * step) : 0.0f;
    }
    __device__ __forceinline__ void add_to(float (&acc)[kColumns]) const
    {
#pragma unroll
        for (int i = 0; i < kColumns; ++i) acc[i] += v[i];
    }
};

// Two 16-bit elements of a row that starts between the words lie in two: the word that holds the first, and the one that holds
// the second.  No word is read that holds nothing of the row.
template <typename T>
struct Columns<T, false> {
    static constexpr int kPieces = kColumns / 2;
    uint32_t first[kPieces], second[kPieces], off;      // off: bits in front of the first element

    __device__ __forceinline__ void load(const T* row, int column, int step, int D)
    {
        const uintptr_t at = reinterpret_cast<uintptr_t>(row + column);
        const uint32_t* p = reinterpret_cast<const uint32_t*>(at & ~uintptr_t(3));
        const uint32_t* q = reinterpret_cast<const uint32_t*>((at + 2) & ~uintptr_t(3));
        off = static_cast<uint32_t>(at & 2) * 8;
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            first[i] = column + i * step < D ? __ldg(p + i * (step / 2)) : 0u;
            second[i] = column + i * step + 1 < D ? __ldg(q + i * (step / 2)) : 0u;
        }
    }
    __device__ __forceinline__ void add_to(float (&acc)[kColumns]) const
    {
#pragma unroll
        for (int i = 0; i < kPieces; ++i) {
            Piece<T, 2> r;
            r.w[0] = __funnelshift_r(first[i], second[i], off);
            acc[2 * i] += element(r, 0);
            acc[2 * i + 1] += element(r, 1);
        }
    }
};

// The same columns, in runs of RUN, of a row of another type, kOne at a time.
template <int RUN, typename TO, int kOne>
__device__ __forceinline__ void load_row(float (&v)[kColumns], const TO* row, int column, int step, int D)
{
#pragma unroll
    for (int i = 0; i < kColumns / kOne; ++i) {
        const int c = column + (i * kOne / RUN) * step + (i * kOne) % RUN;
        Piece<TO, kOne> p;
        if (c < D) load_piece<TO, kOne, false>(p, row + c);
        else clear_piece(p);
#pragma unroll
        for (int e = 0; e < kOne; ++e) v[i * kOne + e] = element(p, e);
    }
}

template <int RUN, typename TO, int kOne>
__device__ __forceinline__ void store_row(TO* row, const float (&v)[kColumns], int column, int step, int D)
{
#pragma unroll
    for (int i = 0; i < kColumns / kOne; ++i) {
        const int c = column + (i * kOne / RUN) * step + (i * kOne) % RUN;
        float one[kOne];
#pragma unroll
        for (int e = 0; e < kOne; ++e) one[e] = v[i * kOne + e];
        if (c < D) store_piece<TO, kOne>(row + c, one);
    }
}

// ALIGNED: rows of `grad` are; OUT: elements of a row of the gradient that can be moved together.
// Blocks per multiprocessor: 16-bit rows that are aligned need the loads that four have in flight (101589 tokens of 528 fp16: 74 us,
// 84 with three); else two, whose registers let the loads of four rows go out together (65537 tokens of 1001 fp16: 90 us, 95 with
// three); one where old rows are moved element by element as well (16384 tokens into 50000 x 1001 fp32: 54 us, 56 with two).
template <typename TI, bool ALIGNED, int OUT, bool INTO>
constexpr int kSumBlocks = ALIGNED && !INTO && sizeof(TI) == 2 ? 4 : !ALIGNED && INTO && OUT == 1 ? 1 : 2;

template <typename TI, typename TO, bool ALIGNED, int OUT, bool INTO>
__global__ void __launch_bounds__(kThreads, (kSumBlocks<TI, ALIGNED, OUT, INTO>))
sum_tiles_kernel(const SumArgs a, const TI* __restrict__ grad, TO* out, const FillArgs fill, int fillers)
{
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    if (blockIdx.x < fillers) {
        __shared__ __align__(16) unsigned char zeros[INTO ? 16 : kFewZeroBytes];
        if constexpr (!INTO) {
            make_zeros<kFewZeroBytes>(zeros);
            const int64_t w0 = fill.early / 32;
            clear_unmet_rows(fill, sizeof(TO), w0, (fill.rows + 31) / 32, fill.met + w0, blockIdx.x + static_cast<int64_t>(threadIdx.x) * fillers,
                             static_cast<int64_t>(kThreads) * fillers, zeros);
        }
        return;
    }
    const int lanes = 1 << a.lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int64_t group = (static_cast<int64_t>(blockIdx.x - fillers) * kThreads + threadIdx.x) >> a.lanes_log2;
    const int64_t tile = group / a.slices;
    const int slice = static_cast<int>(group - tile * a.slices);
    if (tile >= a.tiles) return;
    constexpr int RUN = kRun<TI, ALIGNED>;
    const int step = lanes * RUN, column = slice * (lanes * kColumns) + lane * RUN, D = a.D;
    const int64_t first = tile * a.tile_rows;
    const int rows = static_cast<int>(a.n - first < a.tile_rows ? a.n - first : a.tile_rows);
    const uint2* entries = a.sorted + first;
    uint32_t cur = entry(entries).x;
    bool head = first > 0 && entry(entries - 1).x == cur;
    float acc[kColumns] = {}, kept[kColumns] = {};
    auto put_part = [&](int slot) {
        float* part = a.parts + (tile * 2 + slot) * a.padded_D;
        store_row<RUN, float, RUN>(part, acc, column, step, a.padded_D);
    };
    auto put_row = [&] {
        float v[kColumns];
#pragma unroll
        for (int e = 0; e < kColumns; ++e) v[e] = INTO ? fmaf(a.scale, acc[e], kept[e]) : a.scale * acc[e];
        TO* row = out + static_cast<int64_t>(cur) * a.out_stride;
        store_row<RUN, TO, OUT>(row, v, column, step, D);
    };
    bool fresh = !head;        // the row in the buffer has still to be fetched
    uint2 next[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) next[k] = k < rows ? entry(entries + k) : make_uint2(a.none, 0u);
    bool over = false;
    for (int r = 0; r < rows && !over; r += kAhead) {
        uint2 now[kAhead];
        Columns<TI, ALIGNED> row[kAhead];
        float old[INTO ? kAhead : 1][kColumns];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            now[k] = next[k];
            if (now[k].x != a.none) row[k].load(grad + static_cast<int64_t>(now[k].y) * a.grad_stride, column, step, D);
            if constexpr (INTO) {
                const uint32_t before = k == 0 ? cur : now[k == 0 ? 0 : k - 1].x;
                if (now[k].x != a.none && (now[k].x != before || (r + k == 0 && fresh)))
                    load_row<RUN, TO, OUT>(old[k], out + static_cast<int64_t>(now[k].x) * a.out_stride, column, step, D);
            }
        }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) next[k] = r + kAhead + k < rows ? entry(entries + r + kAhead + k) : make_uint2(a.none, 0u);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            if (over) continue;
            const bool starts = now[k].x != cur;
            if (starts) {
                if (r + k >= rows) {       // behind the tile
                    over = true;
                    continue;
                }
                if (head) put_part(0);
                else put_row();
                head = false;
                cur = now[k].x;
#pragma unroll
                for (int e = 0; e < kColumns; ++e) acc[e] = 0.0f;
            }
            if (cur == a.none) {           // they sort last
                over = true;
                continue;
            }
            if (r + k >= rows) {
                over = true;
                continue;
            }
            if constexpr (INTO)
                if (starts || (r + k == 0 && fresh)) {
#pragma unroll
                    for (int e = 0; e < kColumns; ++e) kept[e] = old[k][e];
                }
            row[k].add_to(acc);
        }
    }
    if (cur == a.none) return;
    const bool goes_on = first + rows < a.n && entry(entries + rows).x == cur;
    if (head || goes_on) put_part(head ? 0 : 1);
    else put_row();
}

// A token that starts in tile t and goes on: its piece in slot 1 of t and slot 0 of the tiles that it reaches, added in order.
// A warp looks at a tile and 128 columns, and adds up a token of up to kFewPieces pieces alone.  A longer one occupies as many
// tiles, whose blocks have nothing else to do: each takes 128 columns in turn, with its warps' sums of equal runs of the pieces
// added in order.
constexpr int kJoinColumns = 128;
constexpr int kFewPieces = 64;

// How many of the tiles t0, t0 + direction, ... begin with `key`, one after the other.  Of the first kThreads of them this thread's
// begins with `here`.
__device__ __forceinline__ uint32_t begin_of(const SumArgs& a, int64_t t) { return t >= 0 && t < a.tiles ? a.sorted[t * a.tile_rows].x : a.none; }
__device__ __forceinline__ int64_t tiles_that_begin_with(const SumArgs& a, uint32_t key, int64_t t0, int direction, uint32_t here)
{
    int64_t found = 0;
    for (;;) {
        const int more = __syncthreads_count(here == key);
        found += more;
        if (more < kThreads) return found;
        here = begin_of(a, t0 + direction * (found + threadIdx.x));
    }
}

__device__ __forceinline__ float4 add_pieces(const SumArgs& a, int64_t tile, int64_t from, int64_t to, int c)
{
    constexpr int kTogether = 8;      // loads in flight, whether there are as many pieces or not
    float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int64_t k0 = from; k0 < to; k0 += kTogether) {
        float4 v[kTogether];
#pragma unroll
        for (int k = 0; k < kTogether; ++k)
            if (k0 + k < to) v[k] = *reinterpret_cast<const float4*>(a.parts + ((tile + k0 + k) * 2 + (k0 + k == 0 ? 1 : 0)) * a.padded_D + c);
#pragma unroll
        for (int k = 0; k < kTogether; ++k)
            if (k0 + k < to) {
                sum.x += v[k].x; sum.y += v[k].y; sum.z += v[k].z; sum.w += v[k].w;
            }
    }
    return sum;
}

template <typename TO, bool INTO>
__device__ __forceinline__ void put_sum(const SumArgs& a, TO* row, float4 sum, int c)
{
    const float v[4] = {sum.x, sum.y, sum.z, sum.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        if (c + e >= a.D) continue;
        Piece<TO, 1> old;
        clear_piece(old);
        if constexpr (INTO) load_piece<TO, 1, false>(old, row + c + e);
        const float one[1] = {INTO ? fmaf(a.scale, v[e], element(old, 0)) : a.scale * v[e]};
        store_piece<TO, 1>(row + c + e, one);
    }
}

// `share_log2`: log2 of the warps that share a tile's columns; a block looks at as many tiles as its warps allow.
template <typename TO, bool INTO>
__global__ void __launch_bounds__(kThreads, 4) join_parts_kernel(const SumArgs a, TO* out, int share_log2)
{
    __shared__ float4 partial[kWarps][32];
    __shared__ int is_long[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, here_tiles = kWarps >> share_log2;
    const int64_t first_tile = static_cast<int64_t>(blockIdx.x) * here_tiles, tile = first_tile + (warp >> share_log2);
    const int64_t first = tile * a.tile_rows, next = first + a.tile_rows;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    // everything that an ordinary tile has to know at once
    auto key_at = [&](int64_t i) { return i >= 0 && i < a.n ? a.sorted[i].x : a.none; };
    const uint32_t begins = key_at(first), before = key_at(first - 1), ends = key_at(next - 1), after = key_at(next);
    const uint32_t far_back = begin_of(a, tile - kFewPieces / 2), far_on = begin_of(a, tile + kFewPieces / 2);
    const uint32_t here0 = begin_of(a, tile + 1 + lane), here1 = begin_of(a, tile + 33 + lane);
    const bool came_in = begins != a.none && before == begins;
    // more than kFewPieces pieces reach half as many tiles on one side at least
    if (lane == 0) is_long[warp] = came_in && (far_back == begins || far_on == begins);
    const bool onward = next < a.n && ends != a.none && after == ends && !(came_in && begins == ends);
    if (onward) {
        const int pieces = 1 + __popc(__ballot_sync(kFull, here0 == ends)) + __popc(__ballot_sync(kFull, here1 == ends));      // or more than kFewPieces
        const int c = ((static_cast<int>(blockIdx.y) << share_log2) + (warp & ((1 << share_log2) - 1))) * kJoinColumns + lane * 4;
        if (pieces <= kFewPieces && c < a.D) put_sum<TO, INTO>(a, out + static_cast<int64_t>(ends) * a.out_stride, add_pieces(a, tile, 0, pieces, c), c);
    }
    __syncthreads();
    uint32_t key = a.none;      // neighbouring tiles mostly belong to one long token: it is measured once
    int64_t lead = 0, pieces = 0;
    for (int i = 0; i < here_tiles; ++i) {
        if (!is_long[i << share_log2]) continue;
        const int64_t t = first_tile + i;
        const uint32_t begins_here = key_at(t * a.tile_rows);
        if (begins_here != key) {
            key = begins_here;
            const int64_t back = tiles_that_begin_with(a, key, t - 1, -1, begin_of(a, t - 1 - threadIdx.x)),
                          reach = tiles_that_begin_with(a, key, t + 1, 1, begin_of(a, t + 1 + threadIdx.x));
            // the first of the `back` tiles may be where the token starts
            const int64_t far = t - back;
            lead = key_at(far * a.tile_rows - 1) == key ? far - 1 : far;
            pieces = t + reach - lead + 1;
        }
        if (pieces <= kFewPieces) continue;
        const int64_t run = (pieces + kWarps - 1) / kWarps, from = warp * run < pieces ? warp * run : pieces, to = from + run < pieces ? from + run : pieces;
        // the tile where it starts has blocks of its own only if it begins with it; the others share the columns
        const int64_t helpers = (pieces - 1) * gridDim.y, me = (t - lead - 1) * gridDim.y + blockIdx.y;
        for (int64_t chunk = me; chunk * kJoinColumns < a.D; chunk += helpers) {
            const int c = static_cast<int>(chunk) * kJoinColumns + lane * 4;
            partial[warp][lane] = c < a.D ? add_pieces(a, lead, from, to, c) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            __syncthreads();
            if (warp == 0 && c < a.D) {
                float4 sum = partial[0][lane];
                for (int w = 1; w < kWarps; ++w) {
                    const float4 v = partial[w][lane];
                    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
                }
                put_sum<TO, INTO>(a, out + static_cast<int64_t>(key) * a.out_stride, sum, c);
            }
            __syncthreads();
        }
    }
}

// ---- gradient of a few tokens: one launch -------------------------------------------------------------------------
//
// Where launches are most of the time, every block that sums sorts all tokens for itself; it takes two to eight lanes' columns of
// all rows, a tile of the sorted positions to each group of lanes, and joins the pieces of the tiles in shared memory.  The
// blocks behind those clear the rows that no token names, which each finds for its own rows.
constexpr int kFewTokens = 2048, kFewItems = kFewTokens / kSortThreads;
constexpr int kMostClearWords = 8 * 1024;      // of rows that one block clears
constexpr int kMostFewColumns = 8192;

// two pieces, of every lane's columns
template <typename T> __host__ __device__ constexpr int64_t few_shared_bytes() { return sort_shared_bytes(kFewItems) + int64_t(kSortThreads) * 2 * kVec<T> * 4; }

template <typename TI, typename TO, bool ALIGNED, bool INTO>
__global__ void __launch_bounds__(kSortThreads, 1)
grad_of_few_kernel(const SortInput in, int passes, int width, const TI* __restrict__ grad, int64_t grad_stride, int D, float scale, TO* out, int64_t out_stride,
                   int lanes_log2, int sum_blocks, const FillArgs fill, int64_t words_per_block)
{
    constexpr int VEC = kVec<TI>, kOne = ALIGNED ? VEC : 1;
    const int lanes = 1 << lanes_log2, groups = kSortThreads >> lanes_log2, row_floats = VEC << lanes_log2;
    extern __shared__ __align__(16) unsigned char sort_smem[];
    if (blockIdx.x >= sum_blocks) {
        uint32_t* met = reinterpret_cast<uint32_t*>(sort_smem + kFewZeroBytes);
        const int64_t w0 = (blockIdx.x - sum_blocks) * words_per_block, last = (fill.rows + 31) / 32, w1 = w0 + words_per_block < last ? w0 + words_per_block : last;
        for (int64_t w = threadIdx.x; w < w1 - w0; w += kSortThreads) met[w] = 0u;
        make_zeros<kFewZeroBytes>(sort_smem);
        for (int i = threadIdx.x; i < in.n; i += kSortThreads) {
            const int64_t key = token_key(in, i), w = key / 32;
            if (key < in.num_embeddings && w >= w0 && w < w1) atomicOr(met + (w - w0), 1u << (key & 31));
        }
        __syncthreads();
        clear_unmet_rows(fill, sizeof(TO), w0, w1, met, threadIdx.x, kSortThreads, sort_smem);
        asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        return;
    }
    const int n = static_cast<int>(in.n), items = (n + kSortThreads - 1) / kSortThreads;
    const unsigned long long* sorted = sort_in_shared<kFewItems>(in, 1, 0u, items, passes, width, sort_smem);
    float* parts = reinterpret_cast<float*>(sort_smem + sort_shared_bytes(kFewItems));
    const uint32_t none = static_cast<uint32_t>(in.num_embeddings);
    auto key_of = [&](int i) { return static_cast<uint32_t>(sorted[i] >> 32); };
    const int group = threadIdx.x >> lanes_log2, lane = threadIdx.x & (lanes - 1);
    const int tile_rows = (n + groups - 1) / groups, first = group * tile_rows, rows = min(tile_rows, n - first);
    const int c = blockIdx.x * row_floats + lane * VEC;
    float acc[VEC] = {};
    auto put_part = [&](int slot) {
#pragma unroll
        for (int e = 0; e < VEC; ++e) parts[(group * 2 + slot) * row_floats + lane * VEC + e] = acc[e];
    };
    auto put_row = [&](uint32_t token) {
        TO* row = out + static_cast<int64_t>(token) * out_stride;
        Piece<TO, kOne> old[INTO ? VEC / kOne : 1];
        if constexpr (INTO) {
#pragma unroll
            for (int i = 0; i < VEC / kOne; ++i)
                if (c + i * kOne < D) load_piece<TO, kOne, false>(old[i], row + c + i * kOne);
        }
#pragma unroll
        for (int i = 0; i < VEC / kOne; ++i) {
            if (c + i * kOne >= D) break;
            float v[kOne];
#pragma unroll
            for (int e = 0; e < kOne; ++e) {
                if constexpr (INTO) v[e] = fmaf(scale, acc[i * kOne + e], element(old[i], e));
                else v[e] = scale * acc[i * kOne + e];
            }
            store_piece<TO, kOne>(row + c + i * kOne, v);
        }
    };
    uint32_t cur = none;
    bool onward = false;      // a token starts in this tile and goes on behind it
    if (rows > 0) {
        cur = key_of(first);
        bool head = first > 0 && key_of(first - 1) == cur;
        for (int r = 0; r < rows && cur != none; r += kAhead) {
            typename std::conditional<ALIGNED, Piece<TI, VEC>, SplitPiece<TI, VEC>>::type in_row[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const unsigned long long both = r + k < rows ? sorted[first + r + k] : static_cast<unsigned long long>(none) << 32;
                if (static_cast<uint32_t>(both >> 32) == none || c >= D) continue;
                const TI* row = grad + static_cast<int64_t>(static_cast<uint32_t>(both)) * grad_stride;
                if constexpr (ALIGNED) {
                    load_piece<TI, VEC>(in_row[k], row + c);
                } else {
                    SplitRow split;
                    split.of(row, D);
                    in_row[k].load(split, c);
                }
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                if (r + k >= rows || cur == none) break;
                const uint32_t key = key_of(first + r + k);
                if (key != cur) {
                    if (head) put_part(0);
                    else put_row(cur);
                    head = false;
                    cur = key;
#pragma unroll
                    for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
                    if (cur == none) break;
                }
                Piece<TI, VEC> one;
                if constexpr (ALIGNED) one = in_row[k];
                else one = in_row[k].piece();
#pragma unroll
                for (int e = 0; e < VEC; ++e) acc[e] += element(one, e);
            }
        }
        if (cur != none) {
            const bool goes_on = first + rows < n && key_of(first + rows) == cur;
            onward = goes_on && !head;
            if (head || goes_on) put_part(head ? 0 : 1);
            else put_row(cur);
        }
    }
    __syncthreads();
    if (!onward) return;
    for (int g = group + 1; g * tile_rows < n && key_of(g * tile_rows) == cur; ++g)
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += parts[g * 2 * row_floats + lane * VEC + e];
    put_row(cur);
}

int64_t align16(int64_t b) { return (b + 15) / 16 * 16; }

// Where things lie in the scratch, and how the sums are cut: about as many groups of lanes as the GPU holds, each with a tile
// and a slice of the columns.
struct GradPlan {
    int64_t sorted[2], hist, met, parts, total;
    int64_t tiles, sort_tiles;
    int tile_rows, slices, lanes_log2, padded_D;
    bool few;      // one launch, no scratch
};

// Of a whole GPU, whatever part of it there is: how sums are cut, and so their bits and the scratch, is the same on any.
constexpr int64_t kResidentWarps = 148 * 32;

bool plan_grad(int64_t n, int64_t num_embeddings, int64_t D, GradPlan& l)
{
    if (n < 0 || n > 0x7fffffff || num_embeddings < 1 || num_embeddings > 0x7fffffff || D < 1 || D > (1 << 20)) return false;
    // (every block sorts again: not for more blocks than two or three to a multiprocessor)
    l.few = n <= kFewTokens && D <= kMostFewColumns && (num_embeddings + 31) / 32 <= int64_t(kMostClearWords) * 64;
    l.total = 0;
    if (l.few) return true;
    l.lanes_log2 = 2;
    while (l.lanes_log2 < 5 && (kColumns << l.lanes_log2) < D) ++l.lanes_log2;
    l.slices = static_cast<int>((D + (kColumns << l.lanes_log2) - 1) / (kColumns << l.lanes_log2));
    const int64_t groups = kResidentWarps << (5 - l.lanes_log2), want = (n * l.slices + groups - 1) / groups;
    // Short tiles for few tokens, whose rows come one after the other; long tokens leave a piece per tile: not too many of them.
    // Where rows are wide `want` decides.  Measured over tables of 32000 bf16 rows (us a gradient, with tiles of 8 / 16 / 32 / 64):
    // 2500 tokens of 128 17.5 / 17.9 / 20.7 / 27.2, 12000 of 256 with a hot token 26.2 / 24.3 / 23.5 / 30.7, 32768 of 128 29.5 / 27.5 /
    // 30.5 / 35.6, 49152 of 128 37.3 / 32.8 / 32.9 / 39.0, 65537 of 128 47.8 / 42.1 / 41.5 / 46.1, 131072 of 256 with a hot token
    // 85.5 / 85.5 / 90.2 / 82.7, 300000 of 64 92.6 / 92.6 / 77.2 / 76.8.
    const int64_t least = n <= 8192 ? 8 : n <= 49152 ? 16 : n < 131072 ? 32 : 64;
    l.tile_rows = static_cast<int>(want < least ? least : want > 256 ? 256 : (want + kAhead - 1) / kAhead * kAhead);
    l.tiles = (n + l.tile_rows - 1) / l.tile_rows;
    l.padded_D = static_cast<int>((D + 7) / 8 * 8);
    l.sort_tiles = sort_form(n, false) == SortForm::kTiles ? (n + kSortTile - 1) / kSortTile : 0;      // whether the device needs it or not
    int64_t at = 0;
    l.sorted[0] = at; at += align16(8 * n);
    l.sorted[1] = at; at += l.sort_tiles ? align16(8 * n) : 0;
    l.hist = at; at += l.sort_tiles ? align16(4 * kMaxBins * (l.sort_tiles + 1)) : 0;
    l.met = at; at += align16((num_embeddings + 31) / 32 * 4);
    l.parts = at; at += l.tiles * 2 * l.padded_D * 4;
    l.total = at;
    return true;
}

// Digits of equal width, at most nine bits, that cover the keys 0 .. num_embeddings.
void digits_of(int64_t num_embeddings, int& passes, int& width)
{
    int bits = 1;
    while ((num_embeddings >> bits) != 0) ++bits;
    passes = (bits + 8) / 9;
    width = (bits + passes - 1) / passes;
}

template <typename TI, typename TO, bool INTO>
int launch_few(const SortInput& in, const TI* grad, int64_t grad_stride, int D, float scale, TO* out, int64_t out_stride, const FillArgs& fill, cudaStream_t s)
{
    constexpr int kWhole = kVec<TI>, shared = static_cast<int>(few_shared_bytes<TI>());
    const bool aligned = D % kWhole == 0 && rows_aligned(grad, grad_stride, sizeof(TI), kWhole) && rows_aligned(out, out_stride, sizeof(TO), kWhole);
    auto* kernel = aligned ? grad_of_few_kernel<TI, TO, true, INTO> : grad_of_few_kernel<TI, TO, false, INTO>;
    static std::atomic<uint64_t> allowed[2] = {};
    if (const int rc = allow_shared(reinterpret_cast<const void*>(kernel), shared, allowed[aligned])) return rc;
    int passes, width;
    digits_of(in.num_embeddings, passes, width);
    // as many lanes to a row, up to eight, as leave every second multiprocessor a block and a tile four rows
    int lanes_log2 = 1;
    auto blocks_of = [&](int l) { return (D + (kWhole << l) - 1) / (kWhole << l); };
    while (lanes_log2 < 3 && (2 * blocks_of(lanes_log2) > sm_count() || (in.n << lanes_log2) < 4 * kSortThreads)) ++lanes_log2;
    const int64_t words = (fill.rows + 31) / 32, sums = blocks_of(lanes_log2);
    // blocks that clear: 64 KB each at least, one per multiprocessor that sums leave free at most (half of all, if
    // those are fewer), and as many as their bits of rows take
    const int64_t room = sums < sm_count() / 2 ? sm_count() - sums : sm_count() / 2;
    int64_t fillers = (fill.rows * fill.row_bytes + 65535) / 65536;
    fillers = fillers < room ? fillers : room;
    fillers = fillers < words ? fillers : words;
    const int64_t least = (words + kMostClearWords - 1) / kMostClearWords;
    fillers = fillers > least ? fillers : least;
    const int64_t each = fillers ? (words + fillers - 1) / fillers : 0;
    kernel<<<static_cast<unsigned>((in.n ? sums : 0) + fillers), kSortThreads, shared, s>>>(in, passes, width, grad, grad_stride, D, scale, out, out_stride,
                                                                                           lanes_log2, static_cast<int>(in.n ? sums : 0), fill, each);
    return check_launch("grad_of_few_kernel");
}

// A launch of the sort by clusters of `cluster` blocks; `together` has to outlive it.
template <int ITEMS>
int sort_config(int cluster, int64_t fillers, cudaStream_t s, cudaLaunchAttribute& together, cudaLaunchConfig_t& config)
{
    auto* kernel = sort_tokens_kernel<ITEMS>;
    const int shared = static_cast<int>(sort_shared_bytes(ITEMS));
    static std::atomic<uint64_t> allowed{0};
    if (const int rc = allow_shared(reinterpret_cast<const void*>(kernel), shared, allowed)) return rc;
    together = {};
    together.id = cudaLaunchAttributeClusterDimension;
    together.val.clusterDim.x = cluster;
    together.val.clusterDim.y = together.val.clusterDim.z = 1;
    config = {};
    config.gridDim = dim3(static_cast<unsigned>(cluster + fillers));
    config.blockDim = dim3(kSortThreads);
    config.dynamicSmemBytes = shared;
    config.stream = s;
    config.attrs = &together;
    config.numAttrs = 1;
    static std::atomic<uint64_t> large{0};      // clusters of more than 8 blocks, once per device
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 64 || !(large.load(std::memory_order_relaxed) >> dev & 1)) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)
            return fail(TBE_B200_ERR_CUDA, "sort_tokens_kernel: clusters of %d blocks are not allowed", kSortBlocks);
        if (dev < 64) large.fetch_or(uint64_t(1) << dev, std::memory_order_relaxed);
    }
    return TBE_B200_OK;
}

// Whether the current device can hold a cluster that sorts; the driver is asked once per device.
bool sort_cluster_fits()
{
    static std::atomic<uint64_t> asked{0}, fits{0};
    int dev = 0;
    const bool kept = cudaGetDevice(&dev) == cudaSuccess && dev < 64;
    const uint64_t bit = kept ? uint64_t(1) << dev : 0;
    if (asked.load(std::memory_order_acquire) & bit) return fits.load(std::memory_order_relaxed) & bit;
    cudaLaunchAttribute together;
    cudaLaunchConfig_t config;
    int clusters = 0;
    if (sort_config<kMostItems>(kSortBlocks, 0, nullptr, together, config) != TBE_B200_OK ||
        cudaOccupancyMaxActiveClusters(&clusters, sort_tokens_kernel<kMostItems>, &config) != cudaSuccess) {
        cudaGetLastError();      // an answer, not a failure
        clusters = 0;
    }
    if (clusters > 0) fits.fetch_or(bit, std::memory_order_relaxed);
    asked.fetch_or(bit, std::memory_order_release);
    return clusters > 0;
}

template <int ITEMS>
int launch_sort(const SortInput& in, int cluster, int items, int passes, int width, uint2* sorted, const FillArgs& fill, int unit, int64_t fillers, cudaStream_t s)
{
    auto* kernel = sort_tokens_kernel<ITEMS>;
    cudaLaunchAttribute together;
    cudaLaunchConfig_t config;
    if (const int rc = sort_config<ITEMS>(cluster, fillers, s, together, config)) return rc;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, in, cluster, items, passes, width, sorted, fill, unit);
    if (e != cudaSuccess) return fail(TBE_B200_ERR_CUDA, "sort_tokens_kernel: %s", cudaGetErrorString(e));
    return check_launch("sort_tokens_kernel");
}

// Sorted (token, position) pairs into one of the two halves of the scratch, whose number is returned in `half`; the
// gradient cleared on the way.
int sort_and_clear(const SortInput& in, SortForm form, const GradPlan& l, char* scratch, const FillArgs& fill, int unit, int& half, cudaStream_t s)
{
    half = 0;
    const int sms = sm_count(), cluster = form == SortForm::kBlock ? 1 : kSortBlocks;
    const int64_t bytes = fill.early * fill.row_bytes;
    const int64_t fillers = in.n == 0 || form == SortForm::kTiles ? 0 : clearing_blocks(bytes, sms, cluster);
    if (bytes && !fillers) {
        const int64_t blocks = (bytes + 65535) / 65536;
        clear_rows_kernel<<<static_cast<unsigned>(blocks < 4 * sms ? blocks : 4 * sms), kThreads, 0, s>>>(fill, unit);
        if (const int rc = check_launch("clear_rows_kernel")) return rc;
    }
    if (in.n == 0) return TBE_B200_OK;
    int passes, width;
    digits_of(in.num_embeddings, passes, width);
    const int bins = 1 << width;
    if (form != SortForm::kTiles) {
        const int items = static_cast<int>((in.n + cluster * kSortThreads - 1) / (cluster * kSortThreads));
        uint2* sorted = reinterpret_cast<uint2*>(scratch + l.sorted[0]);
        if (items <= 2) return launch_sort<2>(in, cluster, items, passes, width, sorted, fill, unit, fillers, s);
        if (items <= 6) return launch_sort<6>(in, cluster, items, passes, width, sorted, fill, unit, fillers, s);
        return launch_sort<kMostItems>(in, cluster, items, passes, width, sorted, fill, unit, fillers, s);
    }
    uint32_t* hist = reinterpret_cast<uint32_t*>(scratch + l.hist);
    uint32_t* totals = hist + kMaxBins * l.sort_tiles;
    const unsigned tiles = static_cast<unsigned>(l.sort_tiles);
    for (int p = 0; p < passes; ++p) {
        const uint2* from = reinterpret_cast<const uint2*>(scratch + l.sorted[half]);
        uint2* to = reinterpret_cast<uint2*>(scratch + l.sorted[half ^ 1]);
        if (p == 0) sort_histogram_kernel<true><<<tiles, kThreads, 0, s>>>(in, from, p * width, bins, hist);
        else sort_histogram_kernel<false><<<tiles, kThreads, 0, s>>>(in, from, p * width, bins, hist);
        sort_places_kernel<<<static_cast<unsigned>((bins + kWarps - 1) / kWarps), kThreads, 0, s>>>(hist, tiles, bins, totals);
        if (p == 0) sort_scatter_kernel<true><<<tiles, kThreads, 0, s>>>(in, from, p * width, bins, hist, totals, to);
        else sort_scatter_kernel<false><<<tiles, kThreads, 0, s>>>(in, from, p * width, bins, hist, totals, to);
        if (const int rc = check_launch("sort kernels")) return rc;
        half ^= 1;
    }
    return TBE_B200_OK;
}

// early: its blocks may come up while the kernel before it ends; they wait for it themselves.
template <typename... Params, typename... Args>
int launch_behind(const char* what, bool can_be_early, void (*kernel)(Params...), dim3 grid, cudaStream_t s, Args... args)
{
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(kThreads);
    config.stream = s;
    config.attrs = &early;
    config.numAttrs = can_be_early ? 1 : 0;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, args...);
    return e == cudaSuccess ? check_launch(what) : fail(TBE_B200_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
}

template <typename TI, typename TO, bool INTO>
int launch_sums(const SumArgs& a, const TI* grad, TO* out, const FillArgs& fill, cudaStream_t s)
{
    const int fillers = fill.early < fill.rows ? sm_count() : 0;
    const int64_t blocks = ((a.tiles * a.slices << a.lanes_log2) + kThreads - 1) / kThreads;
    if (blocks > 0x7fffffff - fillers) return fail(TBE_B200_ERR_UNSUPPORTED, "token_embedding_grad: too many tokens");
    constexpr int kWhole = kVec<TI>;
    const bool aligned = a.D % kWhole == 0 && rows_aligned(grad, a.grad_stride, sizeof(TI), kWhole) && rows_aligned(out, a.out_stride, sizeof(TO), kWhole);
    auto* sums = sum_tiles_kernel<TI, TO, true, kWhole, INTO>;
    if (!aligned) {
        sums = sum_tiles_kernel<TI, TO, false, 1, INTO>;
        if constexpr (sizeof(TI) == 2)
            if (a.D % 2 == 0 && rows_aligned(out, a.out_stride, sizeof(TO), 2)) sums = sum_tiles_kernel<TI, TO, false, 2, INTO>;
    }
    if (const int rc = launch_behind("sum_tiles_kernel", fillers == 0, sums, dim3(static_cast<unsigned>(blocks + fillers)), s, a, grad, out, fill, fillers)) return rc;
    // (clearing blocks that come up early would crowd on the few multiprocessors that have room: 197 instead of 161 us)
    int share_log2 = 0;
    while ((kJoinColumns << share_log2) < a.D && (1 << share_log2) < kWarps) ++share_log2;
    const int64_t here = kWarps >> share_log2, columns = kJoinColumns << share_log2;
    const dim3 grid(static_cast<unsigned>((a.tiles + here - 1) / here), static_cast<unsigned>((a.D + columns - 1) / columns));
    return launch_behind("join_parts_kernel", true, join_parts_kernel<TO, INTO>, grid, s, a, out, share_log2);
}

}  // namespace
}  // namespace tbe

using namespace tbe;

extern "C" int tbe_b200_token_embedding(const void* weight, int32_t weight_dtype, int64_t num_embeddings, int64_t D, int64_t weight_stride,
                                        const void* tokens, int32_t token_bits, int64_t n, float scale, void* output, int32_t output_dtype,
                                        int64_t output_stride, int32_t* error_flag, tbe_b200_stream_t stream)
{
    const int ib = element_bytes(weight_dtype), ob = element_bytes(output_dtype);
    if (!ib || !ob) return fail(TBE_B200_ERR_UNSUPPORTED, "token_embedding: element types FP32, FP16 and BF16, got %d and %d", weight_dtype, output_dtype);
    if (token_bits != 32 && token_bits != 64) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding: token_bits must be 32 or 64, got %d", token_bits);
    if (n < 0 || D < 0 || num_embeddings < 0 || D > 0x10000000) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding: size out of range");
    if (weight_stride < D || output_stride < D) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding: row strides must be at least D");
    if (n == 0 || D == 0) return TBE_B200_OK;
    if (!tokens || !output || (num_embeddings > 0 && !weight)) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding: NULL pointer");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(weight_dtype, [&](auto* ti) {
        return with_element(output_dtype, [&](auto* to) {
            using TI = std::remove_pointer_t<decltype(ti)>;
            using TO = std::remove_pointer_t<decltype(to)>;
            const TI* w = static_cast<const TI*>(weight);
            TO* o = static_cast<TO*>(output);
            const int wide = token_bits == 64;
            auto fits = [&](int vec) { return D % vec == 0 && rows_aligned(w, weight_stride, ib, vec) && rows_aligned(o, output_stride, ob, vec); };
            if (fits(8)) return launch_token_embedding<TI, TO, 8>(w, num_embeddings, D, weight_stride, tokens, wide, n, scale, o, output_stride, error_flag, s);
            if (fits(4)) return launch_token_embedding<TI, TO, 4>(w, num_embeddings, D, weight_stride, tokens, wide, n, scale, o, output_stride, error_flag, s);
            return launch_token_embedding<TI, TO, 0>(w, num_embeddings, D, weight_stride, tokens, wide, n, scale, o, output_stride, error_flag, s);
        });
    });
}

extern "C" int64_t tbe_b200_token_embedding_grad_scratch_bytes(int64_t n, int64_t num_embeddings, int64_t D)
{
    GradPlan l;
    return plan_grad(n, num_embeddings, D, l) ? l.total : -1;
}

extern "C" int tbe_b200_token_embedding_grad(const void* grad, int32_t grad_dtype, int64_t grad_stride, const void* tokens, int32_t token_bits,
                                             int64_t n, int64_t num_embeddings, int64_t D, float scale, int64_t padding_idx, int32_t accumulate,
                                             void* grad_weight, int32_t grad_weight_dtype, int64_t grad_weight_stride, void* scratch,
                                             int64_t scratch_bytes, tbe_b200_stream_t stream)
{
    const int ib = element_bytes(grad_dtype), ob = element_bytes(grad_weight_dtype);
    if (!ib || !ob) return fail(TBE_B200_ERR_UNSUPPORTED, "token_embedding_grad: element types FP32, FP16 and BF16, got %d and %d", grad_dtype, grad_weight_dtype);
    if (token_bits != 32 && token_bits != 64) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: token_bits must be 32 or 64, got %d", token_bits);
    GradPlan l;
    if (!plan_grad(n, num_embeddings, D, l))
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: n and num_embeddings must be below 2^31, D at most 2^20, the last two positive");
    if (padding_idx < -1 || padding_idx >= num_embeddings) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: padding_idx %lld is no row", (long long)padding_idx);
    if (grad_stride < 0 || grad_weight_stride < D) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: bad row stride");
    if (!grad_weight || (n > 0 && (!grad || !tokens || (l.total > 0 && !scratch)))) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: NULL pointer");
    if (l.total > 0 && (scratch_bytes < l.total || (reinterpret_cast<uintptr_t>(scratch) & 15)))
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: scratch must be %lld bytes, 16-byte aligned", (long long)l.total);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    char* base = static_cast<char*>(scratch);
    const SortInput in{tokens, token_bits == 64, n, num_embeddings, padding_idx};
    FillArgs fill{static_cast<char*>(grad_weight), accumulate ? 0 : num_embeddings, D * ob, grad_weight_stride * ob, 0, nullptr};
    fill.early = fill.rows;
    const SortForm form = sort_form(n, n > kOneBlockKeys && !l.few && sort_cluster_fits());
    if (!l.few && n > 0 && form != SortForm::kTiles) {
        // Writing alone runs at 4 TB/s, beside reads at most of what a copy writes: the sums' reads cost little then.  As many rows
        // are cleared beside the sort as that takes; where little is left, all.  Measured (us, 16384 tokens into 131072 x 2048 bf16 /
        // 131072 tokens into 500000 x 512): this rule 158 / 173, without its 32 MB 162 / 184, with 128 MB 162 / 168, with 32 MB however
        // many tokens there are 155 / 204, everything beside the sort 172 / 184.
        const int64_t beside_sort = ((int64_t(32) << 20) + n * 1100) / fill.row_bytes / 32 * 32;
        if (beside_sort + beside_sort / 4 < fill.rows) {
            fill.early = beside_sort;
            fill.met = reinterpret_cast<uint32_t*>(base + l.met);
        }
    }
    if (l.few) {
        if (accumulate && n == 0) return TBE_B200_OK;
        return with_element(grad_weight_dtype, [&](auto* to) {
            return with_element(grad_dtype, [&](auto* ti) {
                using TO = std::remove_pointer_t<decltype(to)>;
                using TI = std::remove_pointer_t<decltype(ti)>;
                const TI* g = static_cast<const TI*>(grad);
                TO* o = static_cast<TO*>(grad_weight);
                if (accumulate) return launch_few<TI, TO, true>(in, g, grad_stride, static_cast<int>(D), scale, o, grad_weight_stride, fill, s);
                return launch_few<TI, TO, false>(in, g, grad_stride, static_cast<int>(D), scale, o, grad_weight_stride, fill, s);
            });
        });
    }
    int half;
    if (const int rc = sort_and_clear(in, form, l, base, fill, ob, half, s)) return rc;
    if (n == 0) return TBE_B200_OK;
    const SumArgs a{reinterpret_cast<const uint2*>(base + l.sorted[half]), n, static_cast<uint32_t>(num_embeddings), grad_stride, grad_weight_stride,
                    static_cast<int>(D), l.padded_D, l.tile_rows, l.slices, l.lanes_log2, l.tiles, scale, reinterpret_cast<float*>(base + l.parts)};
    return with_element(grad_weight_dtype, [&](auto* to) {
        return with_element(grad_dtype, [&](auto* ti) {
            using TO = std::remove_pointer_t<decltype(to)>;
            using TI = std::remove_pointer_t<decltype(ti)>;
            if (accumulate) return launch_sums<TI, TO, true>(a, static_cast<const TI*>(grad), static_cast<TO*>(grad_weight), fill, s);
            return launch_sums<TI, TO, false>(a, static_cast<const TI*>(grad), static_cast<TO*>(grad_weight), fill, s);
        });
    });
}
