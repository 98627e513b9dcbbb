// Token tables in training: lookup of scaled rows, and the gradient of the table.
//
//   lookup     out[i, :] = scale * W[tok[i], :]
//   gradient   dW[v, :]  = scale * sum of dy[i, :] over the i with tok[i] = v
//
// Both are bounded by HBM bandwidth: a product or a sum per element moved.  No counterparts in the reference.
#include "tbe_elements.cuh"

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
// `lanes` threads (a power of two, at most the block) share a row and walk its pieces; a thread holds ROWS rows' pieces
// at a time, so that a block has ROWS * 16 bytes per thread in flight.
template <typename TI, typename TO, int VEC, int ROWS>
__global__ void __launch_bounds__(kThreads)
token_embedding_kernel(const TI* __restrict__ weight, int64_t num_embeddings, int pieces, int64_t weight_stride, const void* __restrict__ tokens,
                       int wide, int64_t n, float scale, TO* __restrict__ out, int64_t out_stride, int lanes_log2, int32_t* error_flag)
{
    const int lanes = 1 << lanes_log2, k = threadIdx.x & (lanes - 1);
    const int rows_at_once = kThreads >> lanes_log2;
    const int64_t first = static_cast<int64_t>(blockIdx.x) * (rows_at_once * ROWS) + (threadIdx.x >> lanes_log2);
    const TI* src[ROWS];
#pragma unroll
    for (int j = 0; j < ROWS; ++j) {
        const int64_t i = first + static_cast<int64_t>(j) * rows_at_once;
        src[j] = nullptr;
        if (i < n) {
            const int64_t t = load_token(tokens, wide, i);
            if (t >= 0 && t < num_embeddings) src[j] = weight + t * weight_stride;
            else if (t != -1 && error_flag && k == 0) atomicOr(error_flag, 4);
        }
    }
    for (int c = k; c < pieces; c += lanes) {
        Piece<TI, VEC> p[ROWS];
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            if (src[j]) load_piece<TI, VEC>(p[j], src[j] + static_cast<int64_t>(c) * VEC);
            else clear_piece(p[j]);
        }
#pragma unroll
        for (int j = 0; j < ROWS; ++j) {
            const int64_t i = first + static_cast<int64_t>(j) * rows_at_once;
            if (i >= n) continue;
            float v[VEC];
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = src[j] ? scale * element(p[j], e) : 0.0f;
            store_piece<TO, VEC>(out + i * out_stride + static_cast<int64_t>(c) * VEC, v);
        }
    }
}

template <typename TI, typename TO, int VEC>
int launch_token_embedding(const TI* weight, int64_t num_embeddings, int64_t D, int64_t weight_stride, const void* tokens, int wide, int64_t n,
                           float scale, TO* out, int64_t out_stride, int32_t* error_flag, cudaStream_t s)
{
    const int pieces = static_cast<int>(D / VEC);
    int lanes_log2 = 0;
    while ((1 << lanes_log2) < pieces && (1 << lanes_log2) < kThreads) ++lanes_log2;
    const int at_once = kThreads >> lanes_log2;
    const bool many = n >= static_cast<int64_t>(sm_count()) * 8 * at_once * 4;
    const int64_t per = static_cast<int64_t>(at_once) * (many ? 4 : 1);
    const int64_t blocks = (n + per - 1) / per;
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "token_embedding: too many tokens");
    if (many)
        token_embedding_kernel<TI, TO, VEC, 4><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(
            weight, num_embeddings, pieces, weight_stride, tokens, wide, n, scale, out, out_stride, lanes_log2, error_flag);
    else
        token_embedding_kernel<TI, TO, VEC, 1><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(
            weight, num_embeddings, pieces, weight_stride, tokens, wide, n, scale, out, out_stride, lanes_log2, error_flag);
    return check_launch("token_embedding_kernel");
}

// ---- gradient: sort by token ----------------------------------------------------------------------------------
//
// Keys are tokens (num_embeddings stands for one that takes no part and sorts last), values their positions.  A stable
// radix sort from the lowest digit up keeps the positions of equal tokens in order, which fixes the order of every sum.
// Per digit: tile histograms, one block that turns them into places (digit by digit, tile by tile), and the scatter.
constexpr int kSortItems = 16;
constexpr int kSortTile = kThreads * kSortItems;
constexpr int kMaxBins = 512;
constexpr int kWarps = kThreads / 32;

__device__ __forceinline__ uint32_t token_key(const void* tokens, bool wide, int64_t i, int64_t num_embeddings, int64_t padding_idx)
{
    const int64_t t = load_token(tokens, wide, i);
    return static_cast<uint32_t>((t < 0 || t >= num_embeddings || t == padding_idx) ? num_embeddings : t);
}

template <bool FIRST>
__device__ __forceinline__ uint32_t sort_key(const void* tokens, const uint32_t* keys, int wide, int64_t i, int64_t num_embeddings, int64_t padding_idx)
{
    if constexpr (FIRST) return token_key(tokens, wide, i, num_embeddings, padding_idx);
    else return __ldg(keys + i);
}

template <bool FIRST>
__global__ void __launch_bounds__(kThreads)
sort_histogram_kernel(const void* __restrict__ tokens, const uint32_t* __restrict__ keys, int wide, int64_t n, int64_t num_embeddings,
                      int64_t padding_idx, int shift, int bins, uint32_t* __restrict__ hist)
{
    __shared__ uint32_t count[kMaxBins];
    for (int b = threadIdx.x; b < bins; b += kThreads) count[b] = 0;
    __syncthreads();
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile;
#pragma unroll 4
    for (int j = 0; j < kSortItems; ++j) {
        const int64_t i = base + j * kThreads + threadIdx.x;
        if (i < n) atomicAdd(&count[(sort_key<FIRST>(tokens, keys, wide, i, num_embeddings, padding_idx) >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) hist[static_cast<int64_t>(b) * gridDim.x + blockIdx.x] = count[b];
}

// Exclusive running sum of `count` numbers in place, by one block.
__global__ void __launch_bounds__(1024) sort_places_kernel(uint32_t* __restrict__ hist, int64_t count)
{
    __shared__ uint32_t warp_tot[32];
    __shared__ uint32_t total;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t carry = 0;
    for (int64_t base = 0; base < count; base += 4096) {
        const int64_t first = base + threadIdx.x * 4;
        uint32_t v[4], mine = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            v[j] = first + j < count ? hist[first + j] : 0u;
            mine += v[j];
        }
        uint32_t incl = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t up = __shfl_up_sync(kFull, incl, d);
            if (lane >= d) incl += up;
        }
        __syncthreads();
        if (lane == 31) warp_tot[warp] = incl;
        __syncthreads();
        uint32_t run = carry + incl - mine;
        for (int w = 0; w < warp; ++w) run += warp_tot[w];
        if (threadIdx.x == 1023) total = run + mine;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (first + j < count) hist[first + j] = run;
            run += v[j];
        }
        __syncthreads();
        carry = total;
    }
}

// A warp owns 32 * kSortItems consecutive keys of the tile and takes them 32 at a time: lanes with the same digit find
// one another, and a running count per warp and digit gives each its rank.
template <bool FIRST>
__global__ void __launch_bounds__(kThreads)
sort_scatter_kernel(const void* __restrict__ tokens, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, int wide, int64_t n,
                    int64_t num_embeddings, int64_t padding_idx, int shift, int bins, const uint32_t* __restrict__ places,
                    uint32_t* __restrict__ keys_out, uint32_t* __restrict__ vals_out)
{
    __shared__ uint32_t count[kWarps][kMaxBins];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int b = threadIdx.x; b < kWarps * bins; b += kThreads) count[b / bins][b % bins] = 0;
    __syncthreads();
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kSortTile + warp * (32 * kSortItems) + lane;
    uint32_t key[kSortItems], rank[kSortItems];
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        const int64_t i = base + j * 32;
        key[j] = i < n ? sort_key<FIRST>(tokens, keys, wide, i, num_embeddings, padding_idx) : 0u;
    }
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        const bool live = base + j * 32 < n;
        const uint32_t d = live ? (key[j] >> shift) & (bins - 1) : static_cast<uint32_t>(bins);
        const uint32_t peers = __match_any_sync(kFull, d);
        const uint32_t before = live ? count[warp][d] : 0u;
        __syncwarp();
        if (live && lane == 31 - __clz(peers)) count[warp][d] = before + __popc(peers);
        __syncwarp();
        rank[j] = before + __popc(peers & ((1u << lane) - 1u));
    }
    __syncthreads();
    for (int b = threadIdx.x; b < bins; b += kThreads) {
        uint32_t run = places[static_cast<int64_t>(b) * gridDim.x + blockIdx.x];
        for (int w = 0; w < kWarps; ++w) {
            const uint32_t c = count[w][b];
            count[w][b] = run;
            run += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < kSortItems; ++j) {
        const int64_t i = base + j * 32;
        if (i >= n) continue;
        const uint32_t at = count[warp][(key[j] >> shift) & (bins - 1)] + rank[j];
        keys_out[at] = key[j];
        vals_out[at] = FIRST ? static_cast<uint32_t>(i) : __ldg(vals + i);
    }
}

// ---- gradient: sums ---------------------------------------------------------------------------------------------
//
// The sorted positions are cut into tiles of kTileRows; a warp walks a tile over 32 * VEC columns and writes a row when its
// token ends.  A token that goes on past the tile leaves its piece in `parts`: slot 0 of a tile holds the sum of the token
// that came in from the tile before (the whole tile, if it goes on), slot 1 that of one that starts here and goes on.
// join_parts_kernel adds the pieces in the order of the tiles.
constexpr int kTileRows = 32;

template <typename TO, int VEC>
__device__ __forceinline__ void write_sum(TO* out, float (&acc)[VEC], float scale, int accumulate)
{
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] *= scale;
    if (accumulate) {
        Piece<TO, VEC> old;
        load_piece<TO, VEC, false>(old, out);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += element(old, e);
    }
    store_piece<TO, VEC>(out, acc);
}

template <typename TI, typename TO, int VEC>
__global__ void __launch_bounds__(kThreads)
sum_tiles_kernel(const TI* __restrict__ grad, int64_t grad_stride, const uint32_t* __restrict__ keys, const uint32_t* __restrict__ vals, int64_t n,
                 uint32_t none, int64_t pieces, float scale, int accumulate, TO* out, int64_t out_stride, float* __restrict__ parts)
{
    const int lane = threadIdx.x & 31;
    const int64_t tile = static_cast<int64_t>(blockIdx.x) * kWarps + (threadIdx.x >> 5);
    const int64_t c = static_cast<int64_t>(blockIdx.y) * 32 + lane;
    const int64_t first = tile * kTileRows;
    if (first >= n || c >= pieces) return;
    const int rows = static_cast<int>(n - first < kTileRows ? n - first : kTileRows);
    const int64_t D = pieces * VEC;
    uint32_t cur = __ldg(keys + first);
    const bool came_in = first > 0 && __ldg(keys + first - 1) == cur;
    bool head = came_in;
    float acc[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
    for (int r = 0; r < rows; ++r) {
        const uint32_t key = __ldg(keys + first + r);
        if (key != cur) {
            if (head) {
#pragma unroll
                for (int e = 0; e < VEC; ++e) parts[(tile * 2) * D + c * VEC + e] = acc[e];
            } else {
                write_sum<TO, VEC>(out + static_cast<int64_t>(cur) * out_stride + c * VEC, acc, scale, accumulate);
            }
            head = false;
            cur = key;
#pragma unroll
            for (int e = 0; e < VEC; ++e) acc[e] = 0.0f;
        }
        if (cur == none) return;      // they sort last
        Piece<TI, VEC> p;
        load_piece<TI, VEC>(p, grad + static_cast<int64_t>(__ldg(vals + first + r)) * grad_stride + c * VEC);
#pragma unroll
        for (int e = 0; e < VEC; ++e) acc[e] += element(p, e);
    }
    const bool goes_on = first + rows < n && __ldg(keys + first + rows) == cur;
    if (head || goes_on) {
        const int64_t slot = tile * 2 + (head ? 0 : 1);
#pragma unroll
        for (int e = 0; e < VEC; ++e) parts[slot * D + c * VEC + e] = acc[e];
    } else {
        write_sum<TO, VEC>(out + static_cast<int64_t>(cur) * out_stride + c * VEC, acc, scale, accumulate);
    }
}

// A token that starts in tile t and goes on: its piece in slot 1 of t and slot 0 of the tiles that it reaches.
template <typename TO>
__global__ void __launch_bounds__(kThreads)
join_parts_kernel(const uint32_t* __restrict__ keys, int64_t n, uint32_t none, int64_t D, float scale, int accumulate, TO* out, int64_t out_stride,
                  const float* __restrict__ parts)
{
    const int64_t tile = blockIdx.x, first = tile * kTileRows, next = first + kTileRows;
    if (next >= n) return;
    const uint32_t cur = __ldg(keys + next - 1);
    if (cur == none || __ldg(keys + next) != cur) return;
    if (__ldg(keys + first) == cur && first > 0 && __ldg(keys + first - 1) == cur) return;      // came in: another tile's
    const int64_t c = static_cast<int64_t>(blockIdx.y) * kThreads + threadIdx.x;
    if (c >= D) return;
    float sum[1] = {parts[(tile * 2 + 1) * D + c]};
    for (int64_t t = tile + 1; t * kTileRows < n && __ldg(keys + t * kTileRows) == cur; ++t) sum[0] += parts[(t * 2) * D + c];
    write_sum<TO, 1>(out + static_cast<int64_t>(cur) * out_stride + c, sum, scale, accumulate);
}

template <typename TO, int VEC>
__global__ void __launch_bounds__(kThreads) zero_rows_kernel(TO* __restrict__ out, int64_t rows, int64_t pieces, int64_t stride)
{
    const float zero[VEC] = {};
    const int64_t step = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * kThreads + threadIdx.x; i < rows * pieces; i += step)
        store_piece<TO, VEC>(out + (i / pieces) * stride + (i % pieces) * VEC, zero);
}

int64_t align16(int64_t b) { return (b + 15) / 16 * 16; }

struct GradLayout {
    int64_t keys[2], vals[2], hist, parts, total;
    int64_t tiles, sort_tiles;
};

bool grad_layout(int64_t n, int64_t num_embeddings, int64_t D, GradLayout& l)
{
    if (n < 0 || n > 0x7fffffff || num_embeddings < 1 || num_embeddings > 0x7fffffff || D < 1 || D > (1 << 20)) return false;
    l.tiles = (n + kTileRows - 1) / kTileRows;
    l.sort_tiles = (n + kSortTile - 1) / kSortTile;
    int64_t at = 0;
    for (int i = 0; i < 2; ++i) {
        l.keys[i] = at; at += align16(4 * n);
        l.vals[i] = at; at += align16(4 * n);
    }
    l.hist = at; at += align16(4 * kMaxBins * l.sort_tiles);
    l.parts = at; at += align16(l.tiles * 2 * D * 4);
    l.total = at;
    return true;
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
    if (n < 0 || D < 0 || num_embeddings < 0 || D > 0x7fffffff) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding: size out of range");
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
            return launch_token_embedding<TI, TO, 1>(w, num_embeddings, D, weight_stride, tokens, wide, n, scale, o, output_stride, error_flag, s);
        });
    });
}

extern "C" int64_t tbe_b200_token_embedding_grad_scratch_bytes(int64_t n, int64_t num_embeddings, int64_t D)
{
    GradLayout l;
    return grad_layout(n, num_embeddings, D, l) ? l.total : -1;
}

extern "C" int tbe_b200_token_embedding_grad(const void* grad, int32_t grad_dtype, int64_t grad_stride, const void* tokens, int32_t token_bits,
                                             int64_t n, int64_t num_embeddings, int64_t D, float scale, int64_t padding_idx, int32_t accumulate,
                                             void* grad_weight, int32_t grad_weight_dtype, int64_t grad_weight_stride, void* scratch,
                                             int64_t scratch_bytes, tbe_b200_stream_t stream)
{
    const int ib = element_bytes(grad_dtype), ob = element_bytes(grad_weight_dtype);
    if (!ib || !ob) return fail(TBE_B200_ERR_UNSUPPORTED, "token_embedding_grad: element types FP32, FP16 and BF16, got %d and %d", grad_dtype, grad_weight_dtype);
    if (token_bits != 32 && token_bits != 64) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: token_bits must be 32 or 64, got %d", token_bits);
    GradLayout l;
    if (!grad_layout(n, num_embeddings, D, l))
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: n and num_embeddings must be below 2^31, D at most 2^20, the last two positive");
    if (padding_idx < -1 || padding_idx >= num_embeddings) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: padding_idx %lld is no row", (long long)padding_idx);
    if (grad_stride < 0 || grad_weight_stride < D) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: bad row stride");
    if (!grad_weight || (n > 0 && (!grad || !tokens || !scratch))) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: NULL pointer");
    if (n > 0 && (scratch_bytes < l.total || (reinterpret_cast<uintptr_t>(scratch) & 15)))
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "token_embedding_grad: scratch must be %lld bytes, 16-byte aligned", (long long)l.total);
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    char* base = static_cast<char*>(scratch);
    return with_element(grad_weight_dtype, [&](auto* to) {
        using TO = std::remove_pointer_t<decltype(to)>;
        TO* o = static_cast<TO*>(grad_weight);
        if (!accumulate) {
            const bool v8 = D % 8 == 0 && rows_aligned(o, grad_weight_stride, ob, 8);
            const int64_t pieces = v8 ? D / 8 : D, want = (num_embeddings * pieces + kThreads - 1) / kThreads, most = sm_count() * 32;
            const unsigned blocks = static_cast<unsigned>(want < most ? want : most);
            if (v8) zero_rows_kernel<TO, 8><<<blocks, kThreads, 0, s>>>(o, num_embeddings, pieces, grad_weight_stride);
            else zero_rows_kernel<TO, 1><<<blocks, kThreads, 0, s>>>(o, num_embeddings, pieces, grad_weight_stride);
            if (const int rc = check_launch("zero_rows_kernel")) return rc;
        }
        if (n == 0) return static_cast<int>(TBE_B200_OK);
        // digits of equal width, at most nine bits, that cover the keys 0 .. num_embeddings
        int bits = 1;
        while ((num_embeddings >> bits) != 0) ++bits;
        const int passes = (bits + 8) / 9, width = (bits + passes - 1) / passes, bins = 1 << width, wide = token_bits == 64;
        uint32_t* hist = reinterpret_cast<uint32_t*>(base + l.hist);
        const unsigned tiles = static_cast<unsigned>(l.sort_tiles);
        int cur = 0;
        for (int p = 0; p < passes; ++p) {
            const uint32_t* k_in = reinterpret_cast<const uint32_t*>(base + l.keys[cur]);
            const uint32_t* v_in = reinterpret_cast<const uint32_t*>(base + l.vals[cur]);
            uint32_t* k_out = reinterpret_cast<uint32_t*>(base + l.keys[cur ^ 1]);
            uint32_t* v_out = reinterpret_cast<uint32_t*>(base + l.vals[cur ^ 1]);
            if (p == 0) sort_histogram_kernel<true><<<tiles, kThreads, 0, s>>>(tokens, k_in, wide, n, num_embeddings, padding_idx, p * width, bins, hist);
            else sort_histogram_kernel<false><<<tiles, kThreads, 0, s>>>(tokens, k_in, wide, n, num_embeddings, padding_idx, p * width, bins, hist);
            sort_places_kernel<<<1, 1024, 0, s>>>(hist, static_cast<int64_t>(bins) * tiles);
            if (p == 0) sort_scatter_kernel<true><<<tiles, kThreads, 0, s>>>(tokens, k_in, v_in, wide, n, num_embeddings, padding_idx, p * width, bins, hist, k_out, v_out);
            else sort_scatter_kernel<false><<<tiles, kThreads, 0, s>>>(tokens, k_in, v_in, wide, n, num_embeddings, padding_idx, p * width, bins, hist, k_out, v_out);
            if (const int rc = check_launch("sort kernels")) return rc;
            cur ^= 1;
        }
        const uint32_t* keys = reinterpret_cast<const uint32_t*>(base + l.keys[cur]);
        const uint32_t* vals = reinterpret_cast<const uint32_t*>(base + l.vals[cur]);
        float* parts = reinterpret_cast<float*>(base + l.parts);
        const uint32_t none = static_cast<uint32_t>(num_embeddings);
        const int rc = with_element(grad_dtype, [&](auto* ti) {
            using TI = std::remove_pointer_t<decltype(ti)>;
            const TI* g = static_cast<const TI*>(grad);
            const unsigned gx = static_cast<unsigned>((l.tiles + kWarps - 1) / kWarps);
            auto fits = [&](int vec) { return D % vec == 0 && rows_aligned(g, grad_stride, ib, vec) && rows_aligned(o, grad_weight_stride, ob, vec); };
            auto grid = [&](int vec) { return dim3(gx, static_cast<unsigned>((D / vec + 31) / 32)); };
            if (fits(8)) sum_tiles_kernel<TI, TO, 8><<<grid(8), kThreads, 0, s>>>(g, grad_stride, keys, vals, n, none, D / 8, scale, accumulate, o, grad_weight_stride, parts);
            else if (fits(4)) sum_tiles_kernel<TI, TO, 4><<<grid(4), kThreads, 0, s>>>(g, grad_stride, keys, vals, n, none, D / 4, scale, accumulate, o, grad_weight_stride, parts);
            else sum_tiles_kernel<TI, TO, 1><<<grid(1), kThreads, 0, s>>>(g, grad_stride, keys, vals, n, none, D, scale, accumulate, o, grad_weight_stride, parts);
            return check_launch("sum_tiles_kernel");
        });
        if (rc) return rc;
        join_parts_kernel<TO><<<dim3(static_cast<unsigned>(l.tiles), static_cast<unsigned>((D + kThreads - 1) / kThreads)), kThreads, 0, s>>>(
            keys, n, none, D, scale, accumulate, o, grad_weight_stride, parts);
        return check_launch("join_parts_kernel");
    });
}
