// Products of a few vectors with 4-bit rows that carry group scales:
//
//   out[m, r] = sum over c of x[m, c] * (code[r, c] * scale[r, g(c)] + bias[r, g(c)])   (+ b[r])
//
// A decoding step's states times a weight matrix or a token table.  Bounded by the rows' bytes.
#include "tbe_elements.cuh"

namespace tbe {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kThreads = 256;

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i)
{
    if (dtype == TBE_B200_FP32) return __ldg(static_cast<const float*>(p) + i);
    if (dtype == TBE_B200_FP16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

// One warp per row and four vectors; a lane takes words of eight codes.
template <typename TI, typename TO>
__global__ void __launch_bounds__(kThreads)
group_row_linear_kernel(const TI* __restrict__ x, int64_t x_stride, int64_t m, const uint8_t* __restrict__ rows, int64_t num_rows, int64_t row_bytes,
                        int64_t D, int group_log2, const void* __restrict__ bias, int bias_dtype, TO* __restrict__ out, int64_t out_stride)
{
    const int lane = threadIdx.x & 31;
    const int64_t r = static_cast<int64_t>(blockIdx.x) * (kThreads / 32) + (threadIdx.x >> 5);
    if (r >= num_rows) return;
    const uint8_t* row = rows + r * row_bytes;
    for (int64_t m0 = static_cast<int64_t>(blockIdx.y) * 4; m0 < m; m0 += static_cast<int64_t>(gridDim.y) * 4) {
        const int live = static_cast<int>(m - m0 < 4 ? m - m0 : 4);
        float acc[4] = {};
        for (int64_t c = lane * 8; c < D; c += 256) {
            const uint32_t codes = ldg4(row + c / 2), head = ldg4(row + D / 2 + 4 * (c >> group_log2));
            const float a = half_bits_to_float(head & 0xffffu), b = half_bits_to_float(head >> 16);
            float w[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) w[e] = fmaf(static_cast<float>((codes >> (4 * e)) & 15u), a, b);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (j >= live) break;
                Piece<TI, 8> p;
                load_piece<TI, 8>(p, x + (m0 + j) * x_stride + c);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[j] = fmaf(element(p, e), w[e], acc[j]);
            }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int d = 16; d >= 1; d >>= 1) acc[j] += __shfl_xor_sync(kFull, acc[j], d);
        if (lane < live) {
            float y[1] = {lane == 0 ? acc[0] : lane == 1 ? acc[1] : lane == 2 ? acc[2] : acc[3]};
            if (bias) y[0] += load_any(bias, bias_dtype, r);
            store_piece<TO, 1>(out + (m0 + lane) * out_stride + r, y);
        }
    }
}

}  // namespace
}  // namespace tbe

using namespace tbe;

extern "C" int tbe_b200_group_row_linear(const void* input, int32_t input_dtype, int64_t input_stride, int64_t m, const uint8_t* rows,
                                         int64_t num_rows, int64_t row_bytes, int64_t D, int32_t group_size, const void* bias, int32_t bias_dtype,
                                         void* output, int32_t output_dtype, int64_t output_stride, tbe_b200_stream_t stream)
{
    const int ib = element_bytes(input_dtype), ob = element_bytes(output_dtype);
    if (!ib || !ob || (bias && !element_bytes(bias_dtype))) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: element types FP32, FP16 and BF16");
    if (const int rc = check_group_rows("group_row_linear", D, group_size, row_bytes, rows, num_rows)) return rc;
    if (m < 0 || D == 0 || input_stride < D || output_stride < num_rows)
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: D must be positive, row strides at least D and num_rows");
    if (m == 0 || num_rows == 0) return TBE_B200_OK;
    if (!input || !rows || !output) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: NULL pointer");
    if (!rows_aligned(input, input_stride, ib, 8)) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: input rows must be 16-byte aligned");
    const int64_t blocks = (num_rows + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffff) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: too many rows");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    return with_element(input_dtype, [&](auto* ti) {
        return with_element(output_dtype, [&](auto* to) {
            using TI = std::remove_pointer_t<decltype(ti)>;
            using TO = std::remove_pointer_t<decltype(to)>;
            const int64_t quads = (m + 3) / 4;
            const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(quads < 65535 ? quads : 65535));
            group_row_linear_kernel<TI, TO><<<grid, kThreads, 0, s>>>(static_cast<const TI*>(input), input_stride, m, rows, num_rows, row_bytes, D,
                                                                        group_log2_of(group_size), bias, bias_dtype, static_cast<TO*>(output), output_stride);
            return check_launch("group_row_linear_kernel");
        });
    });
}
