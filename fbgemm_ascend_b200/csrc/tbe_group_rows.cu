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
constexpr int kSpan = 256;      // elements that a warp takes at once: eight to a lane, one word of codes; whole groups

template <typename T, bool WIDE>
__device__ __forceinline__ void load_eight(float (&v)[8], const T* p)
{
    if constexpr (WIDE) {
        Piece<T, 8> r;
        load_piece<T, 8>(r, p);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = element(r, e);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            Piece<T, 1> r;
            load_piece<T, 1>(r, p + e);
            v[e] = element(r, 0);
        }
    }
}

// One warp per (row, span).  `sharing` lanes hold one group.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
quantize_group_rows_kernel(const T* __restrict__ in, int64_t in_stride, int64_t nrows, int64_t D, int group_log2, int64_t spans, int64_t row_bytes,
                           uint8_t* __restrict__ rows)
{
    const int lane = threadIdx.x & 31, sharing = 1 << (group_log2 - 3);
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
    if (unit >= nrows * spans) return;
    const int64_t r = unit / spans, c = (unit % spans) * kSpan + lane * 8;
    const bool live = c < D;
    float v[8];
    float mn = __int_as_float(0x7f800000), mx = __int_as_float(0xff800000);
    if (live) {
        load_eight<T, WIDE>(v, in + r * in_stride + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            mn = fminf(mn, v[e]);
            mx = fmaxf(mx, v[e]);
        }
    }
    for (int d = sharing / 2; d >= 1; d >>= 1) {
        mn = fminf(mn, __shfl_xor_sync(kFull, mn, d));
        mx = fmaxf(mx, __shfl_xor_sync(kFull, mx, d));
    }
    if (__any_sync(kFull, live && mn == 0.0f)) {
        // Of zeros of both signs a scan for the smallest keeps the first: its sign is the bias's.
        uint32_t zero = 0;
        for (int e = 7; live && e >= 0; --e)
            if (v[e] == 0.0f) zero = 1u + (__float_as_uint(v[e]) >> 31);
        const uint32_t mine = (sharing == 32 ? kFull : (1u << sharing) - 1u) << (lane & ~(sharing - 1));
        const uint32_t with_zero = __ballot_sync(kFull, zero != 0) & mine;
        const uint32_t first = __shfl_sync(kFull, zero, with_zero ? __ffs(with_zero) - 1 : lane);
        if (mn == 0.0f) mn = first == 2u ? -0.0f : 0.0f;
    }
    uint8_t* row = rows + r * row_bytes;
    if (live) {
        const __half bias_h = __float2half_rn(mn);
        const float bias = __half2float(bias_h);
        const float range = __fsub_rn(mx, bias);
        __half scale_h = __float2half_rn(range == 0.0f ? 1.0f : __fdiv_rn(range, 15.0f));
        if (__half2float(scale_h) == 0.0f) scale_h = __float2half_rn(1.0f);
        float inv = __fdiv_rn(1.0f, __half2float(scale_h));
        if (isinf(inv)) {
            scale_h = __float2half_rn(1.0f);
            inv = 1.0f;
        }
        uint32_t codes = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int q = max(0, min(15, __float2int_rn(__fmul_rn(__fsub_rn(v[e], bias), inv))));
            codes |= static_cast<uint32_t>(q) << (4 * e);
        }
        *reinterpret_cast<uint32_t*>(row + c / 2) = codes;
        if ((lane & (sharing - 1)) == 0)
            *reinterpret_cast<uint32_t*>(row + D / 2 + 4 * (c >> group_log2)) =
                static_cast<uint32_t>(__half_as_ushort(scale_h)) | (static_cast<uint32_t>(__half_as_ushort(bias_h)) << 16);
    }
    if (unit % spans == 0) {
        const int64_t used = D / 2 + 4 * ((D + (1 << group_log2) - 1) >> group_log2);
        for (int64_t b = used + 4 * lane; b < row_bytes; b += 128) *reinterpret_cast<uint32_t*>(row + b) = 0u;
    }
}

// One warp per (output row, span).
template <typename T, bool WIDE>
__global__ void __launch_bounds__(kThreads)
group_row_embedding_kernel(const uint8_t* __restrict__ rows, int64_t num_embeddings, int64_t row_bytes, int64_t D, int group_log2, int64_t spans,
                           const void* __restrict__ tokens, int wide, int64_t n, float scale, T* __restrict__ out, int64_t out_stride,
                           int32_t* error_flag)
{
    const int lane = threadIdx.x & 31;
    const int64_t unit = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
    if (unit >= n * spans) return;
    const int64_t i = unit / spans, c = (unit % spans) * kSpan + lane * 8;
    int64_t t = i;
    if (tokens) t = wide ? __ldg(reinterpret_cast<const long long*>(tokens) + i) : static_cast<int64_t>(__ldg(reinterpret_cast<const int*>(tokens) + i));
    const bool met = t >= 0 && t < num_embeddings;
    if (!met && t != -1 && error_flag && lane == 0) atomicOr(error_flag, 4);
    if (c >= D) return;
    float v[8] = {};
    if (met) {
        const uint8_t* row = rows + t * row_bytes;
        const uint32_t codes = ldg4(row + c / 2), head = ldg4(row + D / 2 + 4 * (c >> group_log2));
        const float a = half_bits_to_float(head & 0xffffu), b = half_bits_to_float(head >> 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = scale * fmaf(static_cast<float>((codes >> (4 * e)) & 15u), a, b);
    }
    T* o = out + i * out_stride + c;
    if constexpr (WIDE) store_piece<T, 8>(o, v);
    else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float one[1] = {v[e]};
            store_piece<T, 1>(o + e, one);
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
    if (nrows < 0 || D < 0 || D > 0x7fffffff) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "%s: size out of range", op);
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
    const int64_t spans = (D + kSpan - 1) / kSpan, blocks = (nrows * spans + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "quantize_to_group_rows: too many rows");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(input_dtype, [&](auto* ti) {
        using T = std::remove_pointer_t<decltype(ti)>;
        const T* in = static_cast<const T*>(input);
        const int g = group_log2_of(group_size);
        if (rows_aligned(in, input_stride, ib, 8))
            quantize_group_rows_kernel<T, true><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(in, input_stride, nrows, D, g, spans, row_bytes, rows);
        else
            quantize_group_rows_kernel<T, false><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(in, input_stride, nrows, D, g, spans, row_bytes, rows);
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
    const int64_t spans = (D + kSpan - 1) / kSpan, blocks = (n * spans + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_embedding: too many tokens");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(output_dtype, [&](auto* to) {
        using T = std::remove_pointer_t<decltype(to)>;
        T* o = static_cast<T*>(output);
        const int g = group_log2_of(group_size);
        if (rows_aligned(o, output_stride, ob, 8))
            group_row_embedding_kernel<T, true><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(
                rows, num_embeddings, row_bytes, D, g, spans, tokens, token_bits == 64, n, scale, o, output_stride, error_flag);
        else
            group_row_embedding_kernel<T, false><<<static_cast<unsigned>(blocks), kThreads, 0, s>>>(
                rows, num_embeddings, row_bytes, D, g, spans, tokens, token_bits == 64, n, scale, o, output_stride, error_flag);
        return check_launch("group_row_embedding_kernel");
    });
}
