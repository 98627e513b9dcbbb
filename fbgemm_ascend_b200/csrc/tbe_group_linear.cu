// Products of a few vectors with 4-bit rows that carry group scales:
//
//   out[m, r] = sum over c of x[m, c] * (code[r, c] * scale[r, g(c)] + bias[r, g(c)])   (+ b[r])
//             = sum over groups of scale * sum (code - 8) x  +  (bias + 8 scale) * sum x
//
// A decoding step's states times a weight matrix or a token table.  Bounded by the rows' bytes: each is read once for up to
// 16 vectors, by bulk copies into shared memory, and only the codes (exact in fp16 and bf16) meet the tensor core.
#include <cuda.h>

#include <atomic>

#include "tbe_elements.cuh"

namespace tbe {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 16;
constexpr int kWorkers = 32 * kWarps;
constexpr int kThreads = kWorkers + 32;
constexpr int kParts = kWarps / 2;              // warps whose sums lie in shared memory at a time
constexpr int kMostStages = 4;
constexpr int kUnit = 128;                      // elements of a row that a warp takes at once: 16 bytes to each of four lanes
constexpr int kMostShared = 227 * 1024;

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
    int32_t* error_flag;
    int slices_log2;                            // warps that share a row's elements
    int stages, head_bytes;                     // of a stage; of a row's scales and biases in it
    int64_t tiles;
};

// ---- bulk copies and their barriers -----------------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded: false if the phase is not over after the better part of a second.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity)
{
    for (int polls = 0; polls < (1 << 20); ++polls) {
        uint32_t done;
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                     : "=r"(done) : "r"(bar), "r"(parity) : "memory");
        if (done) return true;
    }
    return false;
}
// A box of the matrix that `map` describes, at word `x` of row `y`, into shared memory.
__device__ __forceinline__ void box_copy(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x),
                 "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

// Bytes of a row's scales and biases that `units` units of it need, as they are fetched: from a 16-byte border on, in whole
// 16-byte pieces, an odd number of them (so that eight rows' words lie in different banks).
int head_window(int units, int group_log2)
{
    const int groups = ((units * kUnit - 1) >> group_log2) + 2;
    return (((groups * 4 + 15) / 16 + 1) | 1) * 16;
}

// The row that lane group g stands for among eight.  Copies put 16-byte piece p of row r at place p ^ (r % 8) of its 128 bytes:
// lanes that load 16 bytes at a time, two rows of four pieces each, meet no bank twice if the rows differ in bit 2.
__device__ __forceinline__ int row_of(int g) { return (g >> 1) | ((g & 1) << 2); }

// A block is kWarps warps that work and one that fetches.  A warp holds RT * 16 rows by NT * 8 states; the warps are `slices`
// shares of the elements times `bands` groups of rows.  A stage holds a unit of 128 elements of its rows for every warp: the
// codes of slices * 128 neighbouring elements of bands * RT * 16 rows, in boxes of 128 bytes by all rows, and one box of the
// scales and biases of their groups.
//
// In a unit lane (g, t) = (lane / 4, lane % 4) takes two rows of every 16.  One matrix instruction takes 4 elements of each lane,
// and one group: where a group is at least a unit, lane t takes elements 32 t .. 32 t + 31 with one 16-byte load; SMALL
// groups (32 and 64) need an instruction's elements side by side, so that lane t takes elements 32 s + 8 t .. + 7 in step
// s, a word at a time.
// SHARED: the states lie in shared memory in the order that the instructions take them, else they are read as they are.
template <typename T, int RT, int NT, bool SMALL, bool SHARED>
__global__ void __launch_bounds__(kThreads, 1)
group_row_linear_kernel(const LinearArgs a, const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap head_map)
{
    constexpr int P = Operand<T>::kPieces;
    constexpr bool HALF = Operand<T>::kHalf;
    constexpr int kPitch = RT * 16 + 4;         // of a state's sums in shared memory: a warp's stores meet no bank twice
    constexpr int kPart = NT * 8 * kPitch;      // one warp's sums
    extern __shared__ __align__(1024) unsigned char smem[];
    const int bands = kWarps >> a.slices_log2, slices = 1 << a.slices_log2, tile_rows = bands * RT * 16;
    const int code_bytes = tile_rows * slices * (kUnit / 2), head_bytes = tile_rows * a.head_bytes;
    // boxes of codes first (1024-byte aligned), then those of heads, sums, states, barriers
    unsigned char* heads_at = smem + a.stages * code_bytes;
    float* red = reinterpret_cast<float*>(heads_at + a.stages * head_bytes);
    const uint32_t full = shared_address(red + kParts * kPart), empty = full + 8 * kMostStages;
    uint4* xs = reinterpret_cast<uint4*>(red + kParts * kPart + 4 * kMostStages);

    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int units = (a.D + kUnit - 1) / kUnit, groups = (a.D + (1 << a.group_log2) - 1) >> a.group_log2;
    const int chunks = (units + slices - 1) >> a.slices_log2;
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (NT * 8);
    const int cols = static_cast<int>(a.m - m0 < NT * 8 ? a.m - m0 : NT * 8);

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            barrier_init(full + 8 * i, 1);
            barrier_init(empty + 8 * i, kWarps);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    if (warp == kWarps) {
        // ---- the warp that fetches ------------------------------------------------------------------------------------
        if (lane != 0) return;
        int stage = 0;
        uint32_t round = 0;
        for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
            const int first = static_cast<int>(tile * tile_rows);
            for (int c = 0; c < chunks; ++c) {
                if (round > 0 && !barrier_wait(empty + 8 * stage, (round - 1) & 1)) {
                    if (a.error_flag) atomicOr(a.error_flag, 16);
                    return;
                }
                const uint32_t bar = full + 8 * stage;
                barrier_expect(bar, code_bytes + head_bytes);
                // what lies outside the matrix arrives as zeros
                for (int k = 0; k < slices / 2; ++k)
                    box_copy(shared_address(smem + stage * code_bytes + k * (tile_rows * 128)), &code_map, (c * (slices / 2) + k) * 32, first, bar);
                const int g0 = (c * slices * kUnit) >> a.group_log2;
                box_copy(shared_address(heads_at + stage * head_bytes), &head_map, ((a.D / 2 + 4 * g0) & ~15) / 4, first, bar);
                if (++stage == a.stages) {
                    stage = 0;
                    ++round;
                }
            }
        }
        return;      // the workers wait for every copy
    }

    // ---- the warps that work ---------------------------------------------------------------------------------------
    const int g = row_of(lane >> 2), t = lane & 3, slice = warp & (slices - 1), band = warp >> a.slices_log2;
    const T* x = static_cast<const T*>(a.x) + m0 * a.x_stride;
    const int words = units * (kUnit / 8);
    if constexpr (SHARED) {
        for (int i = threadIdx.x; i < words * cols; i += kWorkers) {
            const int j = i / words, wd = i - j * words, u = wd / 16, q = wd % 16;
            const int step = SMALL ? q / 4 : q % 4, lt = SMALL ? q % 4 : q / 4;
            uint4 v[P];
            state_pairs<T>(x + j * a.x_stride + wd * 8, wd * 8 < a.D, v);
#pragma unroll
            for (int p = 0; p < P; ++p) xs[(p * words + (u * 4 + step) * 4 + lt) * cols + j] = v[p];
        }
        workers_sync();
    }
    float y[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][n][e] = 0.0f;

    int stage = 0;
    uint32_t round = 0;
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        for (int c = 0; c < chunks; ++c) {
            if (!barrier_wait(full + 8 * stage, round & 1) && a.error_flag) atomicOr(a.error_flag, 16);
            const int u = (c << a.slices_log2) + slice;
            if (u < units) {
                const unsigned char* code_rows = smem + stage * code_bytes + (slice >> 1) * (tile_rows * 128) + (band * RT * 16 + g) * 128;
                const int half = (slice & 1) * 4;
                const int g0 = (c * slices * kUnit) >> a.group_log2;
                const unsigned char* head_rows = heads_at + stage * head_bytes + (band * RT * 16 + g) * a.head_bytes + ((a.D / 2 + 4 * g0) & 15) - 4 * g0;
                uint4 w[RT][2];
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const unsigned char* row = code_rows + (i * 16 + j * 8) * 128;
                        if constexpr (SMALL) {
                            auto word = [&](int s) { return *reinterpret_cast<const uint32_t*>(row + (((half + s) ^ g) * 16 + t * 4)); };
                            w[i][j] = make_uint4(word(0), word(1), word(2), word(3));
                        } else {
                            w[i][j] = *reinterpret_cast<const uint4*>(row + ((half + t) ^ g) * 16);
                        }
                    }
                float acc[RT][NT][4], sum[NT][4];
                const int steps = SMALL ? 1 << (a.group_log2 - 5) : 4;      // per group
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    if (s == 0 || (SMALL && (s & (steps - 1)) == 0)) {
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
                        for (int j = 0; j < 2; ++j) decode<HALF>(s == 0 ? w[i][j].x : s == 1 ? w[i][j].y : s == 2 ? w[i][j].z : w[i][j].w, p[i][j]);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        // a column that no state stands in takes another's: what comes of it is not stored
                        const int j = n * 8 + (lane >> 2) < cols ? n * 8 + (lane >> 2) : cols - 1;
                        uint4 b[P];
                        if constexpr (SHARED) {
#pragma unroll
                            for (int q = 0; q < P; ++q) b[q] = xs[(q * words + (u * 4 + s) * 4 + t) * cols + j];
                        } else {
                            const int k = u * kUnit + (SMALL ? 32 * s + 8 * t : 32 * t + 8 * s);
                            state_pairs<T>(x + j * a.x_stride + k, k < a.D, b);
                        }
                        constexpr uint32_t one = HALF ? 0x3c003c00u : 0x3f803f80u;
#pragma unroll
                        for (int q = 0; q < P; ++q) {
#pragma unroll
                            for (int i = 0; i < RT; ++i) {
                                mma<HALF>(acc[i][n], p[i][0][0], p[i][1][0], p[i][0][1], p[i][1][1], b[q].x, b[q].y);
                                mma<HALF>(acc[i][n], p[i][0][2], p[i][1][2], p[i][0][3], p[i][1][3], b[q].z, b[q].w);
                            }
                            // the states' own sums, in every row of the result: rows of ones
                            mma<HALF>(sum[n], one, one, one, one, b[q].x, b[q].y);
                            mma<HALF>(sum[n], one, one, one, one, b[q].z, b[q].w);
                        }
                    }
                    if (s == 3 || (SMALL && ((s + 1) & (steps - 1)) == 0)) {
                        int gi = (u * kUnit + 32 * s) >> a.group_log2;
                        gi = gi < groups ? gi : groups - 1;
#pragma unroll
                        for (int i = 0; i < RT; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const uint32_t head = *reinterpret_cast<const uint32_t*>(head_rows + (i * 16 + j * 8) * a.head_bytes + 4 * gi);
                                const float sc = half_bits_to_float(head & 0xffffu), bi = fmaf(8.0f, sc, half_bits_to_float(head >> 16));
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int e = 0; e < 2; ++e)
                                        y[i][n][2 * j + e] = fmaf(sc, acc[i][n][2 * j + e], fmaf(bi, sum[n][e], y[i][n][2 * j + e]));
                            }
                    }
                }
            }
            __syncwarp();
            if (lane == 0) barrier_arrive(empty + 8 * stage);
            if (++stage == a.stages) {
                stage = 0;
                ++round;
            }
        }
        // The tile's end: the slices' sums are added in their order, half the warps' at a time.
        const int fold = a.slices_log2 == 4 ? 1 : 0;      // all warps share one band: the upper half is added to the lower first
        for (int half = 0; half < 2; ++half) {
            const bool give = fold ? (half == 0) == (warp >= kParts) : (warp / kParts) == half;
            if (give) {
                float* part = red + (warp % kParts) * kPart;
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) part[(n * 8 + 2 * t + (e & 1)) * kPitch + i * 16 + (e >> 1) * 8 + g] = y[i][n][e];
            }
            workers_sync();
            if (fold && half == 0) {
                if (warp < kParts) {
                    const float* part = red + warp * kPart;
#pragma unroll
                    for (int i = 0; i < RT; ++i)
#pragma unroll
                        for (int n = 0; n < NT; ++n)
#pragma unroll
                            for (int e = 0; e < 4; ++e) y[i][n][e] += part[(n * 8 + 2 * t + (e & 1)) * kPitch + i * 16 + (e >> 1) * 8 + g];
                }
            } else {
                const int depth = fold ? kParts : slices, here = fold ? tile_rows : tile_rows / 2, from_row = fold ? 0 : half * here;
                for (int i = threadIdx.x; i < here * cols; i += kWorkers) {
                    const int col = i / here, row = i - col * here, b = row / (RT * 16);
                    const int64_t r = tile * tile_rows + from_row + row;
                    if (r >= a.num_rows) continue;
                    const float* from = red + b * depth * kPart + col * kPitch + row % (RT * 16);
                    float v = 0.0f;
                    for (int k = 0; k < depth; ++k) v += from[k * kPart];
                    if (a.bias) v += load_any(a.bias, a.bias_dtype, r);
                    store_any(a.out, a.out_dtype, (m0 + col) * a.out_stride + r, v);
                }
            }
            workers_sync();
        }
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) y[i][n][e] = 0.0f;
    }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                 const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// The driver's encoder of tensor maps, looked up once.
EncodeTiled tensor_map_encoder()
{
    static std::atomic<void*> cached{nullptr};
    void* f = cached.load(std::memory_order_relaxed);
    if (!f) {
        cudaDriverEntryPointQueryResult found;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess || found != cudaDriverEntryPointSuccess) return nullptr;
        cached.store(f, std::memory_order_relaxed);
    }
    return reinterpret_cast<EncodeTiled>(f);
}

// The rows as a matrix of 32-bit words, fetched in boxes of box_words by box_rows.
bool encode_rows(CUtensorMap* map, const LinearArgs& a, int box_words, int box_rows, bool swizzled)
{
    const EncodeTiled encode = tensor_map_encoder();
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(a.row_bytes / 4), static_cast<cuuint64_t>(a.num_rows)}, strides[1] = {static_cast<cuuint64_t>(a.row_bytes)};
    const cuuint32_t box[2] = {static_cast<cuuint32_t>(box_words), static_cast<cuuint32_t>(box_rows)}, step[2] = {1, 1};
    return encode && encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 2, const_cast<uint8_t*>(a.rows), dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            swizzled ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int RT, int NT, bool SMALL, bool SHARED>
int launch_linear(const LinearArgs& a, int64_t shared, cudaStream_t s)
{
    auto* kernel = group_row_linear_kernel<T, RT, NT, SMALL, SHARED>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(shared));
    if (e != cudaSuccess) return fail(TBE_B200_ERR_CUDA, "group_row_linear: %s", cudaGetErrorString(e));
    const int tile_rows = RT * 16 * (kWarps >> a.slices_log2);
    CUtensorMap codes, heads;
    if (!encode_rows(&codes, a, 32, tile_rows, true) || !encode_rows(&heads, a, a.head_bytes / 4, tile_rows, false))
        return fail(TBE_B200_ERR_CUDA, "group_row_linear: the rows could not be described to the copy engine");
    const int64_t blocks = a.tiles < sm_count() ? a.tiles : sm_count();
    kernel<<<dim3(static_cast<unsigned>(blocks), static_cast<unsigned>((a.m + NT * 8 - 1) / (NT * 8))), kThreads, shared, s>>>(a, codes, heads);
    return check_launch("group_row_linear_kernel");
}

template <typename T, int RT, int NT>
int launch_linear(LinearArgs a, cudaStream_t s)
{
    const int units = (a.D + kUnit - 1) / kUnit;
    // Shares of the elements: as few as keep every multiprocessor at work to the end, counted in units that a warp goes
    // through (tiles per block times chunks of a tile); a tile's end is worth about one more.
    int64_t best = 0;
    for (int l = 1; l <= 4 && (l == 1 || (1 << l) <= units); ++l) {
        const int64_t tiles = (a.num_rows + RT * 16 * (kWarps >> l) - 1) / (RT * 16 * (kWarps >> l));
        const int64_t cost = ((tiles + sm_count() - 1) / sm_count()) * ((units + (1 << l) - 1) / (1 << l) + 1);
        if (l == 1 || cost < best) {
            best = cost;
            a.slices_log2 = l;
            a.tiles = tiles;
        }
    }
    const bool small = a.group_log2 < 7;
    const int slices = 1 << a.slices_log2, tile_rows = RT * 16 * (kWarps >> a.slices_log2);
    a.head_bytes = head_window(slices, a.group_log2);
    const int64_t stage = static_cast<int64_t>(tile_rows) * (slices * (kUnit / 2) + a.head_bytes);
    const int64_t fixed = static_cast<int64_t>(kParts) * NT * 8 * (RT * 16 + 4) * 4 + 16 * kMostStages;
    const int64_t states = static_cast<int64_t>(a.m < NT * 8 ? a.m : NT * 8) * units * kUnit * 2 * Operand<T>::kPieces;
    const bool shared = fixed + states + 2 * stage <= kMostShared;
    const int64_t stages = (kMostShared - fixed - (shared ? states : 0)) / stage;
    a.stages = static_cast<int>(stages < kMostStages ? stages : kMostStages);
    const int64_t bytes = fixed + a.stages * stage + (shared ? states : 0);
    if (shared) return small ? launch_linear<T, RT, NT, true, true>(a, bytes, s) : launch_linear<T, RT, NT, false, true>(a, bytes, s);
    return small ? launch_linear<T, RT, NT, true, false>(a, bytes, s) : launch_linear<T, RT, NT, false, false>(a, bytes, s);
}

}  // namespace
}  // namespace tbe

using namespace tbe;

extern "C" int tbe_b200_group_row_linear(const void* input, int32_t input_dtype, int64_t input_stride, int64_t m, const uint8_t* rows,
                                         int64_t num_rows, int64_t row_bytes, int64_t D, int32_t group_size, const void* bias, int32_t bias_dtype,
                                         void* output, int32_t output_dtype, int64_t output_stride, int32_t* error_flag, tbe_b200_stream_t stream)
{
    const int ib = element_bytes(input_dtype), ob = element_bytes(output_dtype);
    if (!ib || !ob || (bias && !element_bytes(bias_dtype))) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: element types FP32, FP16 and BF16");
    if (const int rc = check_group_rows("group_row_linear", D, group_size, row_bytes, rows, num_rows)) return rc;
    if (num_rows > 0x7fffffff - 512) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: too many rows");
    if (m < 0 || D == 0 || input_stride < D || output_stride < num_rows)
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: D must be positive, row strides at least D and num_rows");
    if (D > (1 << 20) || m > (1 << 19)) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: D at most 2^20 and m at most 2^19");
    if (m == 0 || num_rows == 0) return TBE_B200_OK;
    if (!input || !rows || !output) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: NULL pointer");
    if (!rows_aligned(input, input_stride, ib, 8)) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: input rows must be 16-byte aligned");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    LinearArgs a{input, input_stride, m, rows, num_rows, row_bytes, static_cast<int>(D), group_log2_of(group_size), bias, bias_dtype, output_dtype,
                 output, output_stride, error_flag, 0, 0, 0, 0};
    return with_element(input_dtype, [&](auto* ti) {
        using T = std::remove_pointer_t<decltype(ti)>;
        // Rows 32 to a warp use every state twice; 16 where that leaves multiprocessors without any.
        const bool many = num_rows >= static_cast<int64_t>(64) * sm_count();
        if (m <= 8) return many ? launch_linear<T, 2, 1>(a, s) : launch_linear<T, 1, 1>(a, s);
        return many ? launch_linear<T, 2, 2>(a, s) : launch_linear<T, 1, 2>(a, s);
    });
}
