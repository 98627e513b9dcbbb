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

// A warp's row and its share of it: `shares` warps to a row.
__device__ __forceinline__ void place_of(int64_t unit, int shares, int64_t& row, int& share)
{
    row = (unit >> 32) ? unit / shares : static_cast<int64_t>(static_cast<uint32_t>(unit) / static_cast<uint32_t>(shares));
    share = static_cast<int>(unit - row * shares);
}

// ---- quantize -------------------------------------------------------------------------------------------------------
//
// Bound by instructions as much as by HBM: a lane takes 16 neighbouring elements, which halves what a group costs beside its
// elements (its two divisions, the exchange of its smallest and largest), a warp two times 512 of a row.  The ends of 16-bit
// rows are found two elements at a time, and the smallest travels between lanes with the largest's negative in one word.
constexpr int kQuantSpan = 512, kQuantAtOnce = 2;

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

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
quantize_group_rows_kernel(const T* __restrict__ in, int64_t in_stride, int64_t nrows, int D, int group_log2, int shares, int64_t row_bytes,
                           uint8_t* __restrict__ rows)
{
    constexpr int W = 2 * Piece<T, 8>::kWords;
    const int lane = threadIdx.x & 31, sharing = 1 << (group_log2 - 4);
    int64_t r;
    int share;
    place_of(static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5), shares, r, share);
    if (r >= nrows) return;
    const int c0 = share * (kQuantAtOnce * kQuantSpan) + lane * 16;
    const T* from = in + r * in_stride + c0;
    uint8_t* row = rows + r * row_bytes;
    uint32_t w[kQuantAtOnce][W];
#pragma unroll
    for (int k = 0; k < kQuantAtOnce; ++k)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            Piece<T, 8> p;
            clear_piece(p);
            if (c0 + k * kQuantSpan + 8 * h < D) p = load_eight<T, WIDE>(from + k * kQuantSpan + 8 * h);
#pragma unroll
            for (int i = 0; i < W / 2; ++i) w[k][h * (W / 2) + i] = p.w[i];
        }
#pragma unroll
    for (int k = 0; k < kQuantAtOnce; ++k) {
        const int c = c0 + k * kQuantSpan;
        if (c - lane * 16 >= D) break;                            // the same for the whole warp
        const bool live = c < D, second = c + 8 < D;              // the lane has elements; it has all 16
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
    if (share == 0) {
        const int64_t used = D / 2 + 4 * ((D + (1 << group_log2) - 1) >> group_log2);
        for (int64_t b = used + 4 * lane; b < row_bytes; b += 128) *reinterpret_cast<uint32_t*>(row + b) = 0u;
    }
}

// ---- lookup ---------------------------------------------------------------------------------------------------------
//
// A lane takes eight elements, one word of codes, of each of four times 256 of a row: stores are whole 16-byte pieces side by
// side.  Bound by the result's bytes (writing alone runs at 4 TB/s) and by instructions.
constexpr int kSpan = 256, kLookupAtOnce = 4;

// Eight codes as numbers: a nibble or'ed into the low bits of 1024 in fp16 (16 steps apart for the upper nibble of a byte) is that
// plus the code, and taking it off leaves the code exactly.
__device__ __forceinline__ void codes_of(uint32_t w, float (&q)[8])
{
    const __half2 even = __float2half2_rn(1024.0f), sixteenth = __float2half2_rn(0.0625f), odd = __float2half2_rn(-64.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint32_t bits;
        asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(bits) : "r"(i < 2 ? w : w >> 8), "r"((i & 1) ? 0x00f000f0u : 0x000f000fu), "r"(0x64006400u));
        const __half2 h = *reinterpret_cast<const __half2*>(&bits);
        const float2 f = __half22float2((i & 1) ? __hfma2(h, sixteenth, odd) : __hsub2(h, even));
        q[i] = f.x;
        q[i + 4] = f.y;
    }
}

template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
group_row_embedding_kernel(const uint8_t* __restrict__ rows, int64_t num_embeddings, int64_t row_bytes, int D, int group_log2, int shares,
                           const void* __restrict__ tokens, int wide, int64_t n, float scale, T* __restrict__ out, int64_t out_stride,
                           int32_t* error_flag)
{
    const int lane = threadIdx.x & 31;
    int64_t i;
    int share;
    place_of(static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5), shares, i, share);
    if (i >= n) return;
    int64_t t = i;
    if (tokens) t = wide ? __ldg(reinterpret_cast<const long long*>(tokens) + i) : static_cast<int64_t>(__ldg(reinterpret_cast<const int*>(tokens) + i));
    const bool met = t >= 0 && t < num_embeddings;
    if (!met && t != -1 && error_flag && share == 0 && lane == 0) atomicOr(error_flag, 4);
    const int c0 = share * (kLookupAtOnce * kSpan) + lane * 8;
    const uint8_t* row = rows + (met ? t : 0) * row_bytes;
    const uint8_t* words = row + c0 / 2;
    const uint8_t* heads = row + D / 2 + 4 * (c0 >> group_log2);
    uint32_t codes[kLookupAtOnce], head[kLookupAtOnce];
#pragma unroll
    for (int k = 0; k < kLookupAtOnce; ++k) {
        codes[k] = head[k] = 0u;
        if (met && c0 + k * kSpan < D) {
            codes[k] = ldg4(words + k * (kSpan / 2));
            head[k] = ldg4(heads + k * (4 * kSpan >> group_log2));
        }
    }
    T* to = out + i * out_stride + c0;
#pragma unroll
    for (int k = 0; k < kLookupAtOnce; ++k) {
        if (c0 + k * kSpan >= D) break;
        // of a row that is none codes, scale and bias are 0
        const __half2 ab = *reinterpret_cast<const __half2*>(&head[k]);
        const float a = __low2float(ab), b = __high2float(ab);
        float v[8];
        codes_of(codes[k], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = fmaf(v[e], a, b);
        if (scale != 1.0f && met) {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= scale;
        }
        if constexpr (WIDE) store_piece<T, 8>(to + k * kSpan, v);
        else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float one[1] = {v[e]};
                store_piece<T, 1>(to + k * kSpan + e, one);
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
    const int64_t shares = (D + kQuantAtOnce * kQuantSpan - 1) / (kQuantAtOnce * kQuantSpan), blocks = (nrows * shares + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "quantize_to_group_rows: too many rows");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(input_dtype, [&](auto* ti) {
        using T = std::remove_pointer_t<decltype(ti)>;
        const T* in = static_cast<const T*>(input);
        const int g = group_log2_of(group_size);
        if (rows_aligned(in, input_stride, ib, 8))
            quantize_group_rows_kernel<T, true><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(in, input_stride, nrows, static_cast<int>(D), g, static_cast<int>(shares), row_bytes, rows);
        else
            quantize_group_rows_kernel<T, false><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(in, input_stride, nrows, static_cast<int>(D), g, static_cast<int>(shares), row_bytes, rows);
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
    const int64_t shares = (D + kLookupAtOnce * kSpan - 1) / (kLookupAtOnce * kSpan), blocks = (n * shares + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_embedding: too many tokens");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(output_dtype, [&](auto* to) {
        using T = std::remove_pointer_t<decltype(to)>;
        T* o = static_cast<T*>(output);
        const int g = group_log2_of(group_size);
        if (rows_aligned(o, output_stride, ob, 8))
            group_row_embedding_kernel<T, true><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(
                rows, num_embeddings, row_bytes, static_cast<int>(D), g, static_cast<int>(shares), tokens, token_bits == 64, n, scale, o, output_stride, error_flag);
        else
            group_row_embedding_kernel<T, false><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(
                rows, num_embeddings, row_bytes, static_cast<int>(D), g, static_cast<int>(shares), tokens, token_bits == 64, n, scale, o, output_stride, error_flag);
        return check_launch("group_row_embedding_kernel");
    });
}
