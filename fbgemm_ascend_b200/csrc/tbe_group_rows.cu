// 4-bit rows with group scales: [D / 2 bytes of codes][fp16 scale, fp16 bias per group][zeros], rows a multiple of 16 bytes.
//
//   quantize   per group: bias = fp16(min), scale = fp16((max - bias) / 15), code = round((x - bias) / scale) in 0 .. 15
//   lookup     out[i, :] = s * (code * scale + bias), of row tokens[i] or of row i
//
// The arithmetic of a group is that of the 4-bit row quantizer (tbe_quant.cu), step by step: a table that one group spans gets
// the same bytes.  Both are HBM-bound streams.  No counterparts in the reference.
#include "tbe_elements.cuh"

namespace tbe {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;

template <typename T, bool WIDE>
__device__ __forceinline__ Piece<T, 8> load_eight(const T* p)
{
    Piece<T, 8> r;
    if constexpr (WIDE) {
        load_piece<T, 8>(r, p);
    } else {
#pragma unroll
        for (int i = 0; i < Piece<T, 8>::kWords; ++i) {
            if constexpr (sizeof(T) == 4) {
                r.w[i] = ldg4(p + i);
            } else {
                const unsigned short* q = reinterpret_cast<const unsigned short*>(p) + 2 * i;
                r.w[i] = static_cast<uint32_t>(__ldg(q)) | (static_cast<uint32_t>(__ldg(q + 1)) << 16);
            }
        }
    }
    return r;
}

// How warps share rows: a wide row (more than a warp's lanes hold at once) takes `shares` warps, narrow rows 1 << lanes_log2 lanes
// each, and a warp as many of them side by side as fit, some times over.
struct Sharing {
    int lanes_log2, shares;
};
inline Sharing sharing_of(int64_t D, int per_lane, int at_once)
{
    Sharing s{0, 1};
    while (s.lanes_log2 < 5 && (static_cast<int64_t>(per_lane) << s.lanes_log2) < D) ++s.lanes_log2;
    if (D > 32 * per_lane) s.shares = static_cast<int>((D + 32 * per_lane * at_once - 1) / (32 * per_lane * at_once));
    return s;
}
// Warps that rows of D elements need.
inline int64_t warps_for(int64_t nrows, const Sharing& s, int64_t D, int per_lane, int at_once)
{
    const int64_t rows_per_warp = static_cast<int64_t>(32 >> s.lanes_log2) * at_once;
    return D > 32 * per_lane ? nrows * s.shares : (nrows + rows_per_warp - 1) / rows_per_warp;
}

// The row and the first column of this lane's k-th piece.
template <bool NARROW, int PER_LANE, int AT_ONCE>
struct Places {
    int64_t row;
    int column, rows_apart;

    __device__ __forceinline__ Places(int64_t unit, const Sharing& s)
    {
        const int lane = threadIdx.x & 31;
        if constexpr (NARROW) {
            rows_apart = 32 >> s.lanes_log2;
            row = unit * (rows_apart * AT_ONCE) + (lane >> s.lanes_log2);
            column = (lane & ((1 << s.lanes_log2) - 1)) * PER_LANE;
        } else {
            rows_apart = 0;
            row = (unit >> 32) ? unit / s.shares : static_cast<int64_t>(static_cast<uint32_t>(unit) / static_cast<uint32_t>(s.shares));
            column = static_cast<int>(unit - row * s.shares) * (32 * PER_LANE * AT_ONCE) + lane * PER_LANE;
        }
    }
    __device__ __forceinline__ int64_t row_of(int k) const { return NARROW ? row + k * rows_apart : row; }
    __device__ __forceinline__ int column_of(int k) const { return NARROW ? column : column + k * (32 * PER_LANE); }
};

// ---- quantize -------------------------------------------------------------------------------------------------------
//
// Bound by the issue of instructions (86 % of the slots; HBM at half its rate): a lane takes 16 neighbouring elements, which halves what a group costs beside its
// elements (its two divisions, the exchange of its smallest and largest), twice.  The ends of 16-bit
// rows are found two elements at a time, and the smallest travels between lanes with the largest's negative in one word.
// 65536 rows of 4096 bf16 in groups of 128: 150 us, 4.5 TB/s (345 us with eight elements a lane).
constexpr int kQuantLane = 16, kQuantAtOnce = 2;

// The smallest and largest of the words' elements.
template <typename T, int W>
struct Ends {
    float mn, mx;
    __device__ __forceinline__ void of(const uint32_t (&w)[W], bool second)
    {
        if constexpr (sizeof(T) == 4) {
            mn = mx = __uint_as_float(w[0]);
#pragma unroll
            for (int i = 1; i < W; ++i)
                if (i < W / 2 || second) {
                    mn = fminf(mn, __uint_as_float(w[i]));
                    mx = fmaxf(mx, __uint_as_float(w[i]));
                }
        } else {
            using V = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            auto pair = [&](int i) { return *reinterpret_cast<const V*>(&w[i]); };
            V lo = pair(0), hi = pair(0);
#pragma unroll
            for (int i = 1; i < W; ++i)
                if (i < W / 2 || second) {
                    lo = __hmin2(lo, pair(i));
                    hi = __hmax2(hi, pair(i));
                }
            mn = fminf(__low2float(lo), __high2float(lo));
            mx = fmaxf(__low2float(hi), __high2float(hi));
        }
    }
    // over `sharing` lanes
    __device__ __forceinline__ void join(int sharing)
    {
        if constexpr (sizeof(T) == 4) {
            for (int d = sharing / 2; d >= 1; d >>= 1) {
                mn = fminf(mn, __shfl_xor_sync(kFull, mn, d));
                mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, d));
            }
        } else {
            using V = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
            V both;
            if constexpr (std::is_same<T, __half>::value) both = __floats2half2_rn(mn, -mx);
            else both = __floats2bfloat162_rn(mn, -mx);
            for (int d = sharing / 2; d >= 1; d >>= 1) {
                const uint32_t other = __shfl_xor_sync(kFull, *reinterpret_cast<const uint32_t*>(&both), d);
                both = __hmin2(both, *reinterpret_cast<const V*>(&other));
            }
            mn = __low2float(both);
            mx = -__high2float(both);
        }
    }
};

template <typename T, bool WIDE, bool NARROW>
__global__ void __launch_bounds__(kThreads)
quantize_group_rows_kernel(const T* __restrict__ in, int64_t in_stride, int64_t nrows, int D, int group_log2, Sharing share, int64_t row_bytes,
                           uint8_t* __restrict__ rows)
{
    constexpr int W = 2 * Piece<T, 8>::kWords;
    const int lane = threadIdx.x & 31;
    // lanes that hold one group; a row shorter than a group is one by itself
    const int sharing = 1 << (NARROW && share.lanes_log2 < group_log2 - 4 ? share.lanes_log2 : group_log2 - 4);
    const Places<NARROW, kQuantLane, kQuantAtOnce> places(static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5), share);
    if (places.row - (NARROW ? lane >> share.lanes_log2 : 0) >= nrows) return;      // the same for the whole warp
    uint32_t w[kQuantAtOnce][W];
#pragma unroll
    for (int k = 0; k < kQuantAtOnce; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Piece<T, 8> p;
            clear_piece(p);
            const int c = places.column_of(k) + 8 * h;
            if (places.row_of(k) < nrows && c < D) p = load_eight<T, WIDE>(in + places.row_of(k) * in_stride + c);
#pragma unroll
            for (int i = 0; i < W / 2; ++i) w[k][h * (W / 2) + i] = p.w[i];
        }
#pragma unroll
    for (int k = 0; k < kQuantAtOnce; ++k) {
        const int c = places.column_of(k);
        const int64_t r = places.row_of(k);
        const bool live = c < D && r < nrows, second = live && c + 8 < D;      // the lane has elements; it has all 16
        if (!__any_sync(kFull, live)) break;
        uint8_t* row = rows + r * row_bytes;
        Ends<T, W> ends;
        ends.of(w[k], second);
        if (!live) {
            ends.mn = __int_as_float(0x7f800000);
            ends.mx = __int_as_float(0xff800000);
        }
        ends.join(sharing);
        Piece<T, 16> all;
#pragma unroll
        for (int i = 0; i < W; ++i) all.w[i] = w[k][i];
        float mn = ends.mn;
        if (__any_sync(kFull, live && mn == 0.0f)) {
            // Of zeros of both signs a scan for the smallest keeps the first: its sign is the bias's.
            uint32_t zero = 0;
#pragma unroll
            for (int e = 15; e >= 0; --e)
                if (live && (e < 8 || second) && element(all, e) == 0.0f) zero = 1u + (__float_as_uint(element(all, e)) >> 31);
            const uint32_t mine = ((1u << sharing) - 1u) << (lane & ~(sharing - 1));
            const uint32_t with_zero = __ballot_sync(kFull, zero != 0) & mine;
            const uint32_t first = __shfl_sync(kFull, zero, with_zero ? __ffs(with_zero) - 1 : lane);
            if (mn == 0.0f) mn = first == 2u ? -0.0f : 0.0f;
        }
        if (!live) continue;
        const __half bias_h = __float2half_rn(mn);
        const float bias = __half2float(bias_h);
        const float range = __fsub_rn(ends.mx, bias);
        __half scale_h = __float2half_rn(range == 0.0f ? 1.0f : __fdiv_rn(range, 15.0f));
        if (__half2float(scale_h) == 0.0f) scale_h = __float2half_rn(1.0f);
        float inv = __fdiv_rn(1.0f, __half2float(scale_h));
        if (isinf(inv)) {
            scale_h = __float2half_rn(1.0f);
            inv = 1.0f;
        }
        // In sixteenths (a power of two changes no rounding) a code is cut off below by the multiplication itself, rounded to a
        // whole sixteenth by adding 2^19, and the low bits of that; what 2^19 leaves in the word is taken off at the end.
        const float inv16 = inv * 0.0625f;
        uint32_t codes[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            codes[h] = 0;
#pragma unroll
            for (int e = 7; e >= 0; --e)
                codes[h] = codes[h] * 16u +
                           __float_as_uint(__fadd_rn(fminf(__saturatef(__fmul_rn(__fsub_rn(element(all, 8 * h + e), bias), inv16)), 0.9375f), 524288.0f));
            codes[h] -= 0xd9000000u;
        }
        uint8_t* to = row + c / 2;
        if (second && (D & 15) == 0) *reinterpret_cast<uint2*>(to) = make_uint2(codes[0], codes[1]);
        else {
            *reinterpret_cast<uint32_t*>(to) = codes[0];
            if (second) *reinterpret_cast<uint32_t*>(to + 4) = codes[1];
        }
        if ((lane & (sharing - 1)) == 0)
            *reinterpret_cast<uint32_t*>(row + D / 2 + 4 * (c >> group_log2)) =
                static_cast<uint32_t>(__half_as_ushort(scale_h)) | (static_cast<uint32_t>(__half_as_ushort(bias_h)) << 16);
    }
    // what lies behind the groups
    const int lanes = 1 << share.lanes_log2;
    const int64_t used = D / 2 + 4 * ((D + (1 << group_log2) - 1) >> group_log2);
#pragma unroll
    for (int k = 0; k < (NARROW ? kQuantAtOnce : 1); ++k) {
        if (places.row_of(k) >= nrows || (!NARROW && places.column >= 32 * kQuantLane)) break;
        for (int64_t b = used + 4 * (lane & (lanes - 1)); b < row_bytes; b += 4 * lanes) *reinterpret_cast<uint32_t*>(rows + places.row_of(k) * row_bytes + b) = 0u;
    }
}

// ---- lookup ---------------------------------------------------------------------------------------------------------
//
// A lane takes eight elements, one word of codes, four times over: of a wide row 256 elements apart, so that stores are whole
// 16-byte pieces side by side, or of four rows.  Bound by the result's bytes (writing alone runs at 4 TB/s) and by instructions.
// 16384 rows of 4096 in groups of 128 as bf16: 24 us, 6.0 TB/s of what has to be moved.
constexpr int kLookupLane = 8, kLookupAtOnce = 4;

__device__ __forceinline__ void codes_of(uint32_t w, float (&q)[8])
{
    uint32_t p[4];
    decode_codes(w, p);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&p[i]));
        q[i] = f.x;
        q[i + 4] = f.y;
    }
}

template <typename T, bool WIDE, bool NARROW>
__global__ void __launch_bounds__(kThreads)
group_row_embedding_kernel(const uint8_t* __restrict__ rows, int64_t num_embeddings, int64_t row_bytes, int D, int group_log2, Sharing share,
                           const void* __restrict__ tokens, int wide, int64_t n, float scale, T* __restrict__ out, int64_t out_stride,
                           int32_t* error_flag)
{
    const Places<NARROW, kLookupLane, kLookupAtOnce> places(static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5), share);
    constexpr int kRows = NARROW ? kLookupAtOnce : 1;
    const uint8_t* row[kRows];
#pragma unroll
    for (int k = 0; k < kRows; ++k) {
        const int64_t i = places.row_of(k);
        int64_t t = i;
        if (tokens && i < n) t = wide ? __ldg(reinterpret_cast<const long long*>(tokens) + i) : static_cast<int64_t>(__ldg(reinterpret_cast<const int*>(tokens) + i));
        const bool met = i < n && t >= 0 && t < num_embeddings;
        if (!met && i < n && t != -1 && error_flag && places.column == 0) atomicOr(error_flag, 4);
        row[k] = met ? rows + t * row_bytes : nullptr;
    }
    uint32_t codes[kLookupAtOnce], head[kLookupAtOnce];
#pragma unroll
    for (int k = 0; k < kLookupAtOnce; ++k) {
        const uint8_t* from = row[NARROW ? k : 0];
        const int c = places.column_of(k);
        codes[k] = head[k] = 0u;
        if (from && c < D) {
            codes[k] = ldg4(from + c / 2);
            head[k] = ldg4(from + D / 2 + 4 * (c >> group_log2));
        }
    }
#pragma unroll
    for (int k = 0; k < kLookupAtOnce; ++k) {
        const int c = places.column_of(k);
        if (c >= D || places.row_of(k) >= n) break;
        // of a row that is none codes, scale and bias are 0
        const __half2 ab = *reinterpret_cast<const __half2*>(&head[k]);
        const float a = __low2float(ab), b = __high2float(ab);
        float v[8];
        codes_of(codes[k], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e], a, b);
        if (scale != 1.0f && row[NARROW ? k : 0]) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= scale;
        }
        T* to = out + places.row_of(k) * out_stride + c;
        if constexpr (WIDE) store_piece<T, 8>(to, v);
        else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float one[1] = {v[e]};
                store_piece<T, 1>(to + e, one);
            }
        }
    }
}

}  // namespace

int group_log2_of(int group_size)
{
    return group_size == 32 ? 5 : group_size == 64 ? 6 : group_size == 128 ? 7 : group_size == 256 ? 8 : -1;
}

// The checks that all entry points over such rows make.
int check_group_rows(const char* op, int64_t D, int group_size, int64_t row_bytes, const void* rows, int64_t nrows)
{
    if (group_log2_of(group_size) < 0) return fail(TBE_B200_ERR_UNSUPPORTED, "%s: group_size must be 32, 64, 128 or 256, got %d", op, group_size);
    if (nrows < 0 || D < 0 || D > 0x40000000) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "%s: size out of range", op);
    if (D % 8) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "%s: D must be a multiple of 8, got %lld", op, (long long)D);
    const int64_t need = D / 2 + 4 * ((D + group_size - 1) / group_size);
    if (row_bytes < need || row_bytes % 16)
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "%s: row_bytes must be a multiple of 16 and at least %lld, got %lld", op, (long long)need, (long long)row_bytes);
    if (reinterpret_cast<uintptr_t>(rows) & 15) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "%s: rows must be 16-byte aligned", op);
    return TBE_B200_OK;
}

}  // namespace tbe

using namespace tbe;

extern "C" int tbe_b200_quantize_to_group_rows(const void* input, int32_t input_dtype, int64_t input_stride, int64_t nrows, int64_t D,
                                               int32_t group_size, int64_t row_bytes, uint8_t* rows, tbe_b200_stream_t stream)
{
    const int ib = element_bytes(input_dtype);
    if (!ib) return fail(TBE_B200_ERR_UNSUPPORTED, "quantize_to_group_rows: element types FP32, FP16 and BF16, got %d", input_dtype);
    if (const int rc = check_group_rows("quantize_to_group_rows", D, group_size, row_bytes, rows, nrows)) return rc;
    if (input_stride < 0) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "quantize_to_group_rows: negative row stride");
    if (nrows == 0 || D == 0) return TBE_B200_OK;
    if (!input || !rows) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "quantize_to_group_rows: NULL pointer");
    const Sharing share = sharing_of(D, kQuantLane, kQuantAtOnce);
    const int64_t blocks = (warps_for(nrows, share, D, kQuantLane, kQuantAtOnce) + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "quantize_to_group_rows: too many rows");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(input_dtype, [&](auto* ti) {
        using T = std::remove_pointer_t<decltype(ti)>;
        const T* in = static_cast<const T*>(input);
        const bool wide = rows_aligned(in, input_stride, ib, 8), narrow = D <= 32 * kQuantLane;
        auto* kernel = wide ? (narrow ? quantize_group_rows_kernel<T, true, true> : quantize_group_rows_kernel<T, true, false>)
                            : (narrow ? quantize_group_rows_kernel<T, false, true> : quantize_group_rows_kernel<T, false, false>);
        kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(in, input_stride, nrows, static_cast<int>(D), group_log2_of(group_size), share, row_bytes, rows);
        return check_launch("quantize_group_rows_kernel");
    });
}

extern "C" int tbe_b200_group_row_embedding(const uint8_t* rows, int64_t num_embeddings, int64_t row_bytes, int64_t D, int32_t group_size,
                                            const void* tokens, int32_t token_bits, int64_t n, float scale, void* output, int32_t output_dtype,
                                            int64_t output_stride, int32_t* error_flag, tbe_b200_stream_t stream)
{
    const int ob = element_bytes(output_dtype);
    if (!ob) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_embedding: element types FP32, FP16 and BF16, got %d", output_dtype);
    if (const int rc = check_group_rows("group_row_embedding", D, group_size, row_bytes, rows, num_embeddings)) return rc;
    if (tokens && token_bits != 32 && token_bits != 64) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_embedding: token_bits must be 32 or 64, got %d", token_bits);
    if (n < 0 || output_stride < D) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_embedding: n must not be negative, the output's row stride at least D");
    if (!tokens && n > num_embeddings) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_embedding: %lld rows wanted of %lld", (long long)n, (long long)num_embeddings);
    if (n == 0 || D == 0) return TBE_B200_OK;
    if (!output || (num_embeddings > 0 && !rows)) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_embedding: NULL pointer");
    const Sharing share = sharing_of(D, kLookupLane, kLookupAtOnce);
    const int64_t blocks = (warps_for(n, share, D, kLookupLane, kLookupAtOnce) + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_embedding: too many tokens");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(output_dtype, [&](auto* to) {
        using T = std::remove_pointer_t<decltype(to)>;
        T* o = static_cast<T*>(output);
        const bool whole = rows_aligned(o, output_stride, ob, 8), narrow = D <= 32 * kLookupLane;
        auto* kernel = whole ? (narrow ? group_row_embedding_kernel<T, true, true> : group_row_embedding_kernel<T, true, false>)
                             : (narrow ? group_row_embedding_kernel<T, false, true> : group_row_embedding_kernel<T, false, false>);
        kernel<<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(rows, num_embeddings, row_bytes, static_cast<int>(D), group_log2_of(group_size), share, tokens,
                                                                  token_bits == 64, n, scale, o, output_stride, error_flag);
        return check_launch("group_row_embedding_kernel");
    });
}
