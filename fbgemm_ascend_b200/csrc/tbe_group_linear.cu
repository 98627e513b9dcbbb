// Products of a few vectors with 4-bit rows that carry group scales:
//
//   out[m, r] = sum over c of x[m, c] * (code[r, c] * scale[r, g(c)] + bias[r, g(c)])   (+ b[r])
//             = sum over groups of scale * sum (code - 8) x  +  (bias + 8 scale) * sum x
//
// A decoding step's states times a weight matrix or a token table.  Bounded by the rows' bytes: each is read once for up to
// 16 vectors, straight into registers, and only the codes (exact in fp16 and bf16) meet the tensor core.
#include "tbe_elements.cuh"

namespace tbe {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 16;
constexpr int kThreads = 32 * kWarps;
constexpr int kUnit = 128;                      // elements of a row that a warp takes at once: 16 bytes to each of four lanes
constexpr int kMostShared = 224 * 1024;

__device__ __forceinline__ float load_any(const void* p, int dtype, int64_t i)
{
    if (dtype == TBE_B200_FP32) return __ldg(static_cast<const float*>(p) + i);
    if (dtype == TBE_B200_FP16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ void store_any(void* p, int dtype, int64_t i, float v)
{
    if (dtype == TBE_B200_FP32) static_cast<float*>(p)[i] = v;
    else if (dtype == TBE_B200_FP16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// How states of type T meet the codes: the operand type, and into how many pieces a state's element is cut.  fp32 has 24
// significant bits, which three bf16 pieces hold exactly over the whole range.
template <typename T> struct Operand { static constexpr int kPieces = 1; static constexpr bool kHalf = std::is_same<T, __half>::value; };
template <> struct Operand<float> { static constexpr int kPieces = 3; static constexpr bool kHalf = false; };

// One word of codes (elements 0 .. 7, low nibble first) as four pairs (0,4) (1,5) (2,6) (3,7) of code - 8.  A nibble or'ed into
// the low bits of 1024 (fp16: 16 steps apart for the upper nibble of a byte) or 128 (bf16) makes that number plus the
// code; what is taken off again leaves it exact.
template <bool HALF>
__device__ __forceinline__ void decode(uint32_t w, uint32_t (&p)[4])
{
    if constexpr (HALF) {
        const uint32_t v = w >> 8;
        const uint32_t lo[4] = {(w & 0x000f000fu) | 0x64006400u, (w & 0x00f000f0u) | 0x64006400u, (v & 0x000f000fu) | 0x64006400u, (v & 0x00f000f0u) | 0x64006400u};
        const __half2 even = __float2half2_rn(1032.0f), sixteenth = __float2half2_rn(0.0625f), odd = __float2half2_rn(-72.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __half2 h = *reinterpret_cast<const __half2*>(&lo[i]);
            const __half2 r = (i & 1) ? __hfma2(h, sixteenth, odd) : __hsub2(h, even);
            p[i] = *reinterpret_cast<const uint32_t*>(&r);
        }
    } else {
        const __nv_bfloat162 off = __float2bfloat162_rn(136.0f);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t b = ((w >> (4 * i)) & 0x000f000fu) | 0x43004300u;
            const __nv_bfloat162 r = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&b), off);
            p[i] = *reinterpret_cast<const uint32_t*>(&r);
        }
    }
}

template <bool HALF>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (HALF)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight elements of a state as pairs (0,4) (1,5) (2,6) (3,7), one set per piece; zeros where `live` is false.
template <typename T>
__device__ __forceinline__ void state_pairs(const T* p, bool live, uint4 (&out)[Operand<T>::kPieces])
{
    Piece<T, 8> r;
    if (live) load_piece<T, 8>(r, p);
    else clear_piece(r);
    if constexpr (sizeof(T) == 2) {
        out[0] = make_uint4(__byte_perm(r.w[0], r.w[2], 0x5410), __byte_perm(r.w[0], r.w[2], 0x7632), __byte_perm(r.w[1], r.w[3], 0x5410),
                            __byte_perm(r.w[1], r.w[3], 0x7632));
    } else {
        // cut off, not rounded: fp32's largest numbers stay finite, and the remainders are exact
        uint32_t top[3][8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = __uint_as_float(r.w[e]);
            const bool finite = (r.w[e] & 0x7f800000u) != 0x7f800000u;
            const float hi = __uint_as_float(r.w[e] & 0xffff0000u), rest = v - hi;
            const float mid = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
            top[0][e] = (v != v) ? 0x7fc0u : r.w[e] >> 16;
            top[1][e] = finite ? __float_as_uint(mid) >> 16 : 0u;
            top[2][e] = finite ? __float_as_uint(rest - mid) >> 16 : 0u;
        }
#pragma unroll
        for (int q = 0; q < 3; ++q)
            out[q] = make_uint4(top[q][0] | (top[q][4] << 16), top[q][1] | (top[q][5] << 16), top[q][2] | (top[q][6] << 16), top[q][3] | (top[q][7] << 16));
    }
}

struct LinearArgs {
    const void* x;
    int64_t x_stride, m;
    const uint8_t* rows;
    int64_t num_rows, row_bytes;
    int D, group_log2;
    const void* bias;
    int bias_dtype, out_dtype;
    void* out;
    int64_t out_stride;
    int slices_log2;                            // warps that share a row's elements
    int64_t tiles;
};

// A warp holds RT * 16 rows by NT * 8 states.  The warps of a block are `slices` shares of the elements times 16 / slices
// groups of rows; units of 128 elements go round the slices.  In a unit lane (g, t) = (lane / 4, lane % 4) holds 16 bytes of
// rows g and g + 8 of every 16: elements 32 t .. 32 t + 31, so that one matrix instruction takes 4 of each lane's (TURNED
// false; a group is at least the unit).  Groups of 32 and 64 need an instruction's elements side by side: TURNED exchanges the
// words among the four lanes, and lane t then holds elements 32 s + 8 t .. + 7 of the four steps s.
// SHARED: the states lie in shared memory in the order that the instructions take them, else they are read as they are.
template <typename T, int RT, int NT, bool TURNED, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1) group_row_linear_kernel(const LinearArgs a)
{
    constexpr int P = Operand<T>::kPieces;
    constexpr bool HALF = Operand<T>::kHalf;
    constexpr int kPitch = RT * 16 + 4;         // of a state's sums in shared memory: a warp's stores meet no bank twice
    extern __shared__ __align__(16) unsigned char smem[];
    float* red = reinterpret_cast<float*>(smem);
    uint4* xs = reinterpret_cast<uint4*>(smem + kWarps * NT * 8 * kPitch * 4);

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int slices = 1 << a.slices_log2, slice = warp & (slices - 1), band = warp >> a.slices_log2, bands = kWarps >> a.slices_log2;
    const int units = (a.D + kUnit - 1) / kUnit, groups = (a.D + (1 << a.group_log2) - 1) >> a.group_log2;
    const int mine = (units - slice + slices - 1) >> a.slices_log2;           // units of a tile that are this warp's; at least one
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (NT * 8);
    const int cols = static_cast<int>(a.m - m0 < NT * 8 ? a.m - m0 : NT * 8);
    const int tile_rows = bands * RT * 16;
    const T* x = static_cast<const T*>(a.x) + m0 * a.x_stride;

    struct Held {
        uint4 w[RT][2];
        uint32_t head[RT][2];
    };
    Held buf[2];
    // what is fetched next, and what is worked on: tile and place among this warp's units
    int64_t f_tile = blockIdx.x, c_tile = blockIdx.x;
    int f_i = 0, c_i = 0;

    auto fetch = [&](Held& h) {
        if (f_tile >= a.tiles) return;
        const int u = slice + (f_i << a.slices_log2);
        const int64_t at = static_cast<int64_t>(u) * (kUnit / 2) + t * 16;
        int gi = (u * kUnit + (TURNED ? 32 * t : 0)) >> a.group_log2;
        gi = gi < groups ? gi : groups - 1;
        const int64_t head = a.D / 2 + 4 * gi;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                int64_t r = f_tile * tile_rows + band * (RT * 16) + i * 16 + j * 8 + g;
                r = r < a.num_rows ? r : a.num_rows - 1;
                const uint8_t* row = a.rows + r * a.row_bytes;
                if (at < a.row_bytes) asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(h.w[i][j].x), "=r"(h.w[i][j].y), "=r"(h.w[i][j].z), "=r"(h.w[i][j].w) : "l"(row + at));
                else h.w[i][j] = make_uint4(0u, 0u, 0u, 0u);
                h.head[i][j] = ldg4(row + head);
            }
        if (++f_i == mine) {
            f_i = 0;
            f_tile += gridDim.x;
        }
    };
    fetch(buf[0]);
    fetch(buf[1]);

    if constexpr (SHARED) {
        const int words = units * (kUnit / 8);
        for (int i = threadIdx.x; i < words * cols; i += kThreads) {
            const int j = i / words, wd = i % words;
            const int u = wd / 16, q = wd % 16;
            const int step = TURNED ? q / 4 : q % 4, lt = TURNED ? q % 4 : q / 4;
            uint4 v[P];
            state_pairs<T>(x + j * a.x_stride + wd * 8, wd * 8 < a.D, v);
#pragma unroll
            for (int p = 0; p < P; ++p) xs[(static_cast<int64_t>(p) * words + (u * 4 + step) * 4 + lt) * cols + j] = v[p];
        }
        __syncthreads();
    }

    float y[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][n][e] = 0.0f;

    auto work = [&](Held& h) {
        const int u = slice + (c_i << a.slices_log2);
        if constexpr (TURNED) {
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    uint32_t w[4] = {h.w[i][j].x, h.w[i][j].y, h.w[i][j].z, h.w[i][j].w};
                    // 4 x 4 words turned about the diagonal: first single words between neighbours, then pairs
#pragma unroll
                    for (int d = 1; d <= 2; d <<= 1)
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            if (k & d) continue;
                            const bool up = t & d;
                            const uint32_t got = __shfl_xor_sync(kFull, up ? w[k] : w[k | d], d);
                            if (up) w[k] = got;
                            else w[k | d] = got;
                        }
                    h.w[i][j] = make_uint4(w[0], w[1], w[2], w[3]);
                }
        }
        float acc[RT][NT][4], sum[NT][4];
        const int steps = TURNED ? 1 << (a.group_log2 - 5) : 4;      // per group
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            if (s == 0 || (TURNED && (s & (steps - 1)) == 0)) {
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        sum[n][e] = 0.0f;
#pragma unroll
                        for (int i = 0; i < RT; ++i) acc[i][n][e] = 0.0f;
                    }
            }
            uint32_t p[RT][2][4];
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j) decode<HALF>(s == 0 ? h.w[i][j].x : s == 1 ? h.w[i][j].y : s == 2 ? h.w[i][j].z : h.w[i][j].w, p[i][j]);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int j = n * 8 + g;
                uint4 b[P];
                if constexpr (SHARED) {
#pragma unroll
                    for (int q = 0; q < P; ++q)
                        b[q] = j < cols ? xs[(static_cast<int64_t>(q) * units * (kUnit / 8) + (u * 4 + s) * 4 + t) * cols + j] : make_uint4(0u, 0u, 0u, 0u);
                } else {
                    const int c = u * kUnit + (TURNED ? 32 * s + 8 * t : 32 * t + 8 * s);
                    state_pairs<T>(x + j * a.x_stride + c, j < cols && c < a.D, b);
                }
                constexpr uint32_t one = HALF ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
                for (int q = 0; q < P; ++q) {
#pragma unroll
                    for (int i = 0; i < RT; ++i) {
                        mma<HALF>(acc[i][n], p[i][0][0], p[i][1][0], p[i][0][1], p[i][1][1], b[q].x, b[q].y);
                        mma<HALF>(acc[i][n], p[i][0][2], p[i][1][2], p[i][0][3], p[i][1][3], b[q].z, b[q].w);
                    }
                    // the states' own sums, in every row of the result: a row of ones
                    mma<HALF>(sum[n], one, one, one, one, b[q].x, b[q].y);
                    mma<HALF>(sum[n], one, one, one, one, b[q].z, b[q].w);
                }
            }
            if (s == 3 || (TURNED && ((s + 1) & (steps - 1)) == 0)) {
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const uint32_t head = TURNED ? __shfl_sync(kFull, h.head[i][j], (lane & ~3) | s) : h.head[i][j];
                        const float sc = half_bits_to_float(head & 0xffffu), bi = fmaf(8.0f, sc, half_bits_to_float(head >> 16));
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e)
                                y[i][n][2 * j + e] = fmaf(sc, acc[i][n][2 * j + e], fmaf(bi, sum[n][e], y[i][n][2 * j + e]));
                    }
            }
        }
        fetch(h);
        if (++c_i < mine) return;
        // the tile's end: the slices' sums are added in their order
        c_i = 0;
        float* part = red + warp * (NT * 8 * kPitch);
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    part[(n * 8 + 2 * t + (e & 1)) * kPitch + i * 16 + (e >> 1) * 8 + g] = y[i][n][e];
                    y[i][n][e] = 0.0f;
                }
        __syncthreads();
        for (int i = threadIdx.x; i < tile_rows * cols; i += kThreads) {
            const int col = i / tile_rows, row = i % tile_rows, b = row / (RT * 16);
            const int64_t r = c_tile * tile_rows + row;
            if (r >= a.num_rows) continue;
            const float* from = red + (b << a.slices_log2) * (NT * 8 * kPitch) + col * kPitch + row % (RT * 16);
            float v = 0.0f;
            for (int k = 0; k < slices; ++k) v += from[k * (NT * 8 * kPitch)];
            if (a.bias) v += load_any(a.bias, a.bias_dtype, r);
            store_any(a.out, a.out_dtype, (m0 + col) * a.out_stride + r, v);
        }
        __syncthreads();
        c_tile += gridDim.x;
    };
    while (c_tile < a.tiles) {
        work(buf[0]);
        if (c_tile >= a.tiles) break;
        work(buf[1]);
    }
}

template <typename T, int RT, int NT, bool TURNED, bool SHARED>
int launch_linear(const LinearArgs& a, int64_t shared, cudaStream_t s)
{
    auto* kernel = group_row_linear_kernel<T, RT, NT, TURNED, SHARED>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared));
    if (e != cudaSuccess) return fail(TBE_B200_ERR_CUDA, "group_row_linear: %s", cudaGetErrorString(e));
    const int64_t blocks = a.tiles < sm_count() ? a.tiles : sm_count();
    kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>((a.m + NT * 8 - 1) / (NT * 8))), kThreads, shared, s>>>(a);
    return check_launch("group_row_linear_kernel");
}

template <typename T, int RT, int NT>
int launch_linear(LinearArgs a, cudaStream_t s)
{
    const int units = (a.D + kUnit - 1) / kUnit;
    // Warps share the elements of a row rather than take rows of their own where there are few rows.
    a.slices_log2 = 0;
    while (a.slices_log2 < 4 && (2 << a.slices_log2) <= units &&
           a.num_rows < static_cast<int64_t>(RT * 16) * (kWarps >> a.slices_log2) * 4 * sm_count())
        ++a.slices_log2;
    const int tile_rows = RT * 16 * (kWarps >> a.slices_log2);
    a.tiles = (a.num_rows + tile_rows - 1) / tile_rows;
    const int64_t sums = static_cast<int64_t>(kWarps) * NT * 8 * (RT * 16 + 4) * 4;
    const int64_t states = static_cast<int64_t>(a.m < NT * 8 ? a.m : NT * 8) * units * kUnit * 2 * Operand<T>::kPieces;
    const bool turned = a.group_log2 < 7;
    if (sums + states <= kMostShared)
        return turned ? launch_linear<T, RT, NT, true, true>(a, sums + states, s) : launch_linear<T, RT, NT, false, true>(a, sums + states, s);
    return turned ? launch_linear<T, RT, NT, true, false>(a, sums, s) : launch_linear<T, RT, NT, false, false>(a, sums, s);
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
    if (D > (1 << 24) || m > (1 << 19)) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: D at most 2^24 and m at most 2^19");
    if (m == 0 || num_rows == 0) return TBE_B200_OK;
    if (!input || !rows || !output) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: NULL pointer");
    if (!rows_aligned(input, input_stride, ib, 8)) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: input rows must be 16-byte aligned");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    LinearArgs a{input, input_stride, m, rows, num_rows, row_bytes, static_cast<int>(D), group_log2_of(group_size), bias, bias_dtype, output_dtype,
                 output, output_stride, 0, 0};
    return with_element(input_dtype, [&](auto* ti) {
        using T = std::remove_pointer_t<decltype(ti)>;
        // Rows 32 to a warp use every state twice; 16 where that leaves multiprocessors without any.
        const bool many = num_rows >= static_cast<int64_t>(64) * sm_count();
        if (m <= 8) return many ? launch_linear<T, 2, 1>(a, s) : launch_linear<T, 1, 1>(a, s);
        return many ? launch_linear<T, 2, 2>(a, s) : launch_linear<T, 1, 2>(a, s);
    });
}
