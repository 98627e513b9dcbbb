// Products of a few vectors with 4-bit rows that carry group scales:
//
//   out[m, r] = sum over c of x[m, c] * (code[r, c] * scale[r, g(c)] + bias[r, g(c)])   (+ b[r])
//             = sum over groups of scale * sum code x  +  bias * sum x
//
// Codes stay 0 .. 15: where all of a group's are 0 (elements that are alike, zeros among them: its scale is 1 whatever its
// elements are) nothing but the bias is left.  Taken around their middle such a group would be a difference of two sums of
// the scale's size, each with its own roundings.
//
// A decoding step's states times a weight matrix or a token table.  No counterpart in the reference.
//
// The rows' bytes are the floor.  Each row is read once for up to 16 states, by copies into shared memory that a warp of its own
// issues some stages ahead, and only the codes (exact in fp16) meet the tensor core: what a group's scale and bias multiply are
// sums over the group.  The matrix instruction is the warp's (16 rows by 8 states by 16 elements, one per 8 clocks and SM quarter):
// operands must come out of registers, where codes become numbers, and at 16 states or fewer its rate is no limit (26 % of it is
// used at eight).  What the codes cost is decoding: four masks and four subtractions for eight of them, and the loads; 315 warp
// instructions per 4096 codes in all, at eight states by groups of 128.
//
// Large tables: no unit is saturated (8 states by 131072 x 4096: 64 % of the issue slots, 54 % of the DRAM peak); four working warps
// to a scheduler do not hide the chain from a code to the scaled sum.  Layers: what every block does once, arranging all states
// before its first product and a tile's end.
//
// Measured, bf16 states, rows of 4096 in groups of 128, within a graph: 131072 rows (285 MB) by one state 53 us, 5.4 TB/s; by
// eight 61 us, 4.7 TB/s; by 16 80 us, 3.6 TB/s; groups of 32, whose sums are scaled four times as often, by eight 77 us (336 MB,
// 4.4 TB/s).  16384 rows by one state 10.7 us, 3.3 TB/s; 4096 rows 5.1 us, of which the launch and the first stage's way are the most.
#include <cuda.h>

#include <atomic>

#include "tbe_elements.cuh"

namespace tbe {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 16;
constexpr int kWorkers = 32 * kWarps;
constexpr int kThreads = kWorkers + 32;
constexpr int kMostStages = 4;
constexpr int kUnit = 128;                      // elements of a row that a warp takes at once: 16 bytes to each of four lanes
constexpr int kBoxUnits = 2;                    // the 128 bytes of a row of a box
// Units that a warp takes between two barriers: its share of a stage is 4096 codes either way.
__host__ __device__ constexpr int units_at_once(int RT) { return 2 / RT; }
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

// c = a * b, or c += a * b.
template <bool FIRST>
__device__ __forceinline__ void mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1)
{
    if constexpr (FIRST)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- the states, in the order that the matrix instructions take them --------------------------------------------
//
// A state's elements become fp16: as they are, or times the power of two that brings the state's largest into 2^14 .. 2^15
// (bf16 keeps its 8 bits then down to 2^-31 of the largest; elements below that are off by 2^-39 of the largest at most); fp32
// in two pieces, off by 2^-23 of the element down to 2^-16 of the largest, below that by 2^-39 of the largest, since the second
// piece is subnormal there.  (A state below 2^-112 is brought up by 2^126, and off by 2^-151.)  The sums are scaled back.
//
// For a unit of 128 elements: four steps, in each 64 bytes per state and piece, 16 to each of four lanes; then the sums of the
// states over every group of the unit.  A block that arranges the states itself (LOCAL) keeps only those that there are; else
// there is room for NT * 8.
template <typename T> constexpr int kPieces = sizeof(T) == 4 ? 2 : 1;

__host__ __device__ constexpr int sums_bytes(int NT, int steps) { return 4 / steps * NT * 32; }
__host__ __device__ constexpr int unit_bytes(int NT, int P, int steps) { return P * NT * 2048 + sums_bytes(NT, steps); }
__host__ __device__ constexpr int local_unit_bytes(int cols, int NT, int P, int steps) { return P * cols * 256 + sums_bytes(NT, steps); }

__device__ __forceinline__ int largest_bits(float v) { return static_cast<int>(__float_as_uint(v) & 0x7fffffffu); }      // magnitudes order like their bits

// 2^e with 14 - e the exponent of the largest, both ways within fp32's normal numbers.
__device__ __forceinline__ int scale_exponent(int largest) { return min(126, 14 - ((largest >> 23) - 127)); }
__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(127 + e) << 23); }

// The largest magnitude among elements `first` on, 8 at a time and `stride` words of 8 apart, of a row of D.
template <typename T>
__device__ __forceinline__ int largest_of(const T* row, int D, int first, int stride)
{
    int most = 0;
    for (int i = first; i < D / 8; i += stride) {
        Piece<T, 8> r;
        load_piece<T, 8>(r, row + i * 8);
#pragma unroll
        for (int e = 0; e < 8; ++e) most = max(most, largest_bits(element(r, e)));
    }
    return __reduce_max_sync(kFull, most);
}

// Words of 8 elements `first`, `first` + stride ... of a state (whole warps, neighbouring lanes neighbouring words).  Where word
// (step, t) of unit u goes: at(u, step, piece, t); where the sum of the unit's group k goes: sum_at(u, k).
template <typename T, int STEPS, typename At, typename SumAt>
__device__ __forceinline__ void arrange_words(const T* row, int D, float scale, int first, int stride, At at, SumAt sum_at)
{
    constexpr int P = kPieces<T>;
    const int words = (D + kUnit - 1) / kUnit * (kUnit / 8);
    for (int i = first; i < (words + 31) / 32 * 32; i += stride) {
        Piece<T, 8> r;
        if (i * 8 < D) load_piece<T, 8>(r, row + i * 8);
        else clear_piece(r);
        const int u = i / 16, q = i % 16, step = STEPS < 4 ? q / 4 : q % 4, t = STEPS < 4 ? q % 4 : q / 4;
        __half h[P][8];
        float sum = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float v = element(r, e) * scale;
            h[0][e] = __float2half_rn(v);
            if constexpr (P == 2) {
                const float rest = v - __half2float(h[0][e]);
                h[1][e] = __float2half_rn(isfinite(rest) ? rest : 0.0f);      // of an infinite element nothing is left
                sum += __half2float(h[1][e]);
            }
            sum += __half2float(h[0][e]);
        }
        for (int d = 1; d < 4 * STEPS; d <<= 1) sum += __shfl_xor_sync(kFull, sum, d);
        if (i >= words) continue;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const __half2 pair[4] = {__halves2half2(h[p][0], h[p][4]), __halves2half2(h[p][1], h[p][5]), __halves2half2(h[p][2], h[p][6]), __halves2half2(h[p][3], h[p][7])};
            *at(u, step, p, t) = *reinterpret_cast<const uint4*>(pair);
        }
        if (q % (4 * STEPS) == 0) *sum_at(u, q / (4 * STEPS)) = sum;
    }
}

constexpr int kStateThreads = 512;

// One block per state.
template <typename T, int STEPS>
__global__ void __launch_bounds__(kStateThreads)
arrange_states_kernel(const T* __restrict__ x, int64_t x_stride, int D, int NT, unsigned char* __restrict__ arranged, float* __restrict__ back)
{
    constexpr int P = kPieces<T>;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int m = blockIdx.x, units = (D + kUnit - 1) / kUnit;
    const T* row = x + m * x_stride;
    float scale = 1.0f;
    if constexpr (!std::is_same<T, __half>::value) {
        __shared__ int largest;
        if (threadIdx.x == 0) largest = 0;
        __syncthreads();
        const int most = largest_of(row, D, threadIdx.x, kStateThreads);
        if ((threadIdx.x & 31) == 0) atomicMax(&largest, most);
        __syncthreads();
        const int e = scale_exponent(largest);
        scale = power_of_two(e);
        if (threadIdx.x == 0) back[m] = power_of_two(-e);
    } else if (threadIdx.x == 0) {
        back[m] = 1.0f;
    }
    const int n = (m % (NT * 8)) / 8, col = m % 8, unit_size = unit_bytes(NT, P, STEPS);
    unsigned char* to = arranged + static_cast<int64_t>(m / (NT * 8)) * units * unit_size;
    arrange_words<T, STEPS>(
        row, D, scale, threadIdx.x, kStateThreads,
        [&](int u, int step, int p, int t) {
            return reinterpret_cast<uint4*>(to + static_cast<int64_t>(u) * unit_size + ((step * NT + n) * P + p) * 512 + (col * 4 + t) * 16);
        },
        [&](int u, int k) { return reinterpret_cast<float*>(to + static_cast<int64_t>(u) * unit_size + P * NT * 2048 + (k * NT * 8 + n * 8 + col) * 4); });
}

struct LinearArgs {
    const unsigned char* arranged;              // states as arrange_states_kernel leaves them, and what undoes their scales
    const float* back;
    const void* x;                              // LOCAL: as they are
    int64_t x_stride, m;
    const uint8_t* rows;
    int64_t num_rows, row_bytes;
    int D, group_log2;
    const void* bias;
    int bias_dtype, out_dtype;
    void* out;
    int64_t out_stride;
    int32_t* error_flag;
    int slices, bands;                          // warps that share a row's elements; groups of rows
    int stages, head_bytes;                     // head_bytes: of a row's scales and biases in a stage
    int buffers;                                // of the warps' sums, two where they do not cost a stage
    int polls;                                  // after which a wait for a stage is given up
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
// Whether the barrier's phase of that parity is over (the hardware may look on for a while).
__device__ __forceinline__ bool barrier_passed(uint32_t bar, uint32_t parity)
{
    uint32_t done;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(done) : "r"(bar), "r"(parity) : "memory");
    return done;
}
// Bounded: false if the phase is not over after so many polls; kPolls of them are the better part of a second.  Polls after the
// first are out of the way of what follows (8 states by 131072 x 4096: 61.3 us, 62.3 with them in line).
constexpr int kPolls = 1 << 20;
__device__ __noinline__ bool barrier_wait_on(uint32_t bar, uint32_t parity, int polls)
{
    for (; polls > 0; --polls)
        if (barrier_passed(bar, parity)) return true;
    return false;
}
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, int polls)
{
    return (barrier_passed(bar, parity) && polls > 0) || barrier_wait_on(bar, parity, polls);
}
// A box of the matrix that `map` describes, at word `x` of row `y`, into shared memory.
__device__ __forceinline__ void box_copy(uint32_t to, const CUtensorMap* map, int x, int y, uint32_t bar)
{
    asm volatile("cp.async.bulk.tensor.2d.shared::cta.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(to), "l"(map), "r"(x),
                 "r"(y), "r"(bar) : "memory");
}
// A run of bytes, all 16-byte aligned.
__device__ __forceinline__ void bulk_copy(uint32_t to, const void* from, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to), "l"(from), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void workers_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kWorkers) : "memory"); }

// Bytes of a row's scales and biases that a chunk of `units` (an even number) needs, as they are fetched: from the 16-byte
// border in front of them on, in whole 16-byte pieces, an odd number of them (so that eight rows' words lie in different
// banks).  A chunk begins with a group, and where in 16 bytes repeats after four chunks at most.
int head_window(int D, int units, int group_log2)
{
    const int step = 4 * (units * kUnit >> group_log2), bytes = step > 4 ? step : 4;
    int most = 0;
    for (int c = 0; c < 4; ++c) {
        const int pieces = ((D / 2 + c * bytes) % 16 + bytes + 15) / 16;
        most = pieces > most ? pieces : most;
    }
    return (most | 1) * 16;
}

// The row that lane group g stands for among eight.  Copies put 16-byte piece p of row r at place p ^ (r % 8) of its 128 bytes:
// lanes that load 16 bytes at a time, two rows of four pieces each, meet no bank twice if the rows differ in bit 2.
__device__ __forceinline__ int row_of(int g) { return (g >> 1) | ((g & 1) << 2); }

// A block is kWarps warps that work and one that fetches.  A warp holds RT * 16 rows by NT * 8 states; the warps are `slices`
// shares of the elements times `bands` groups of rows.  A stage holds U units of 128 elements of its rows for every warp:
// the codes of slices * U neighbouring units of bands * RT * 16 rows, in boxes of 128 bytes by all rows, one box of the scales
// and biases of their groups, and the states' elements.
//
// In a unit lane (g, t) = (lane / 4, lane % 4) takes two rows of every 16.  One matrix instruction takes 4 elements of each lane,
// and one group: where a group is at least a unit, lane t takes elements 32 t .. 32 t + 31 with one 16-byte load; small
// groups (32 and 64) need an instruction's elements side by side, so that lane t takes elements 32 s + 8 t .. + 7 in step
// s, a word at a time.
// STEPS: how many steps of a unit a group spans.  P: pieces of a state's element.  T: the states' type, where the workers arrange
// them themselves before they begin and keep them in shared memory (LOCAL); void: they come with every stage.
template <typename T, int RT, int NT, int P, int STEPS>
__global__ void __launch_bounds__(kThreads, 1)
group_row_linear_kernel(const LinearArgs a, const __grid_constant__ CUtensorMap code_map, const __grid_constant__ CUtensorMap head_map)
{
    constexpr int kPitch = RT * 16 + 4;         // of a state's sums in shared memory: a warp's stores meet no bank twice
    constexpr int kPart = NT * 8 * kPitch;      // one warp's sums
    constexpr int U = units_at_once(RT), kStates = unit_bytes(NT, P, STEPS);
    constexpr bool LOCAL = !std::is_void<T>::value;
    extern __shared__ __align__(1024) unsigned char smem[];
    const int bands = a.bands, slices = a.slices, tile_rows = bands * RT * 16, boxes = (slices * U + 1) / kBoxUnits;
    const int code_bytes = boxes * tile_rows * 128, head_bytes = tile_rows * a.head_bytes, state_bytes = LOCAL ? 0 : slices * U * kStates;
    // boxes of codes first (1024-byte aligned), then those of heads, the states, sums, barriers
    unsigned char* heads_at = smem + a.stages * code_bytes;
    unsigned char* states_at = heads_at + a.stages * head_bytes;
    float* red = reinterpret_cast<float*>(states_at + a.stages * state_bytes);
    const uint32_t full = shared_address(red + a.buffers * kWarps * kPart), empty = full + 8 * kMostStages;
    // LOCAL: what undoes the states' scales, the largest of each, the states
    float* backs = red + a.buffers * kWarps * kPart + 4 * kMostStages;
    int* largest = reinterpret_cast<int*>(backs + 16);
    unsigned char* local = reinterpret_cast<unsigned char*>(largest + 16);

    const int lane = threadIdx.x & 31, warp = __shfl_sync(kFull, threadIdx.x >> 5, 0);      // known to be the same for all lanes
    const int units = (a.D + kUnit - 1) / kUnit, groups = (a.D + (1 << a.group_log2) - 1) >> a.group_log2;
    const int chunks = (units + U * slices - 1) / (U * slices);
    const int64_t m0 = static_cast<int64_t>(blockIdx.y) * (NT * 8);
    const int cols = static_cast<int>(a.m - m0 < NT * 8 ? a.m - m0 : NT * 8);

    if (threadIdx.x == 0) {
        for (int i = 0; i < a.stages; ++i) {
            barrier_init(full + 8 * i, 1);
            barrier_init(empty + 8 * i, bands * slices);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();

    if (warp == kWarps) {
        // ---- the warp that fetches ------------------------------------------------------------------------------------
        if (lane != 0) return;
        const unsigned char* arranged = a.arranged + static_cast<int64_t>(blockIdx.y) * units * kStates;
        int64_t tile = blockIdx.x;
        int chunk = 0;
        auto next = [&] {
            if (++chunk == chunks) {
                chunk = 0;
                tile += gridDim.x;
            }
        };
        auto states_of = [&](int c) { return LOCAL ? 0 : (units - c * U * slices < U * slices ? units - c * U * slices : U * slices) * kStates; };
        auto fetch_rows = [&](int stage) {
            const uint32_t bar = full + 8 * stage;
            const int first = static_cast<int>(tile * tile_rows);
            barrier_expect(bar, code_bytes + head_bytes + states_of(chunk));
            // what lies outside the matrix arrives as zeros
            for (int k = 0; k < boxes; ++k)
                box_copy(shared_address(smem + stage * code_bytes + k * (tile_rows * 128)), &code_map, (chunk * slices * U + k * kBoxUnits) * (kUnit / 8), first, bar);
            const int g0 = (chunk * slices * U * kUnit) >> a.group_log2;
            box_copy(shared_address(heads_at + stage * head_bytes), &head_map, ((a.D / 2 + 4 * g0) & ~15) / 4, first, bar);
        };
        auto fetch_states = [&](int stage) {
            bulk_copy(shared_address(states_at + stage * state_bytes), arranged + static_cast<int64_t>(chunk) * state_bytes, states_of(chunk), full + 8 * stage);
        };
        // The first stages' rows are on their way before the states are ready.
        int filled = 0;
        for (; filled < a.stages && tile < a.tiles; ++filled) {
            fetch_rows(filled);
            next();
        }
        if constexpr (!LOCAL) {
            asm volatile("griddepcontrol.wait;" ::: "memory");
            tile = blockIdx.x;
            chunk = 0;
            for (int i = 0; i < filled; ++i) {
                fetch_states(i);
                next();
            }
        }
        int stage = 0;
        uint32_t round = 0;
        int64_t fills = filled;
        while (tile < a.tiles) {
            if (!barrier_wait(empty + 8 * stage, round & 1, a.polls)) {
                if (a.error_flag) atomicOr(a.error_flag, 16);
                break;
            }
            fetch_rows(stage);
            if constexpr (!LOCAL) fetch_states(stage);
            next();
            ++fills;
            if (++stage == a.stages) {
                stage = 0;
                ++round;
            }
        }
        // a block stays until its copies have arrived, also where a worker gave one up
        for (int64_t k = fills > a.stages ? fills - a.stages : 0; k < fills; ++k)
            barrier_wait(full + 8 * static_cast<int>(k % a.stages), static_cast<uint32_t>(k / a.stages) & 1, kPolls);
        return;
    }

    // ---- the warps that work ---------------------------------------------------------------------------------------
    const int local_unit = local_unit_bytes(cols, NT, P, STEPS);
    if constexpr (LOCAL) {
        // as many warps to each state
        int share_log2 = 4;
        while ((kWarps >> share_log2) < cols) --share_log2;
        const int j = warp >> share_log2, first = (warp & ((1 << share_log2) - 1)) * 32 + lane, stride = 32 << share_log2;
        const T* row = static_cast<const T*>(a.x) + (m0 + j) * a.x_stride;
        float scale = 1.0f;
        if constexpr (!std::is_same<T, __half>::value) {
            if (threadIdx.x < 16) largest[threadIdx.x] = 0;
            workers_sync();
            if (j < cols) {
                const int most = largest_of(row, a.D, first, stride);
                if (lane == 0) atomicMax(&largest[j], most);
            }
            workers_sync();
            const int e = scale_exponent(largest[j]);
            scale = power_of_two(e);
            if (j < cols && first == 0) backs[j] = power_of_two(-e);
        } else if (threadIdx.x < 16) {
            backs[threadIdx.x] = 1.0f;
        }
        if (j < cols)
            arrange_words<T, STEPS>(
                row, a.D, scale, first, stride,
                [&](int u, int step, int p, int t) { return reinterpret_cast<uint4*>(local + u * local_unit + ((step * P + p) * cols + j) * 64 + t * 16); },
                [&](int u, int k) { return reinterpret_cast<float*>(local + u * local_unit + P * cols * 256 + (k * NT * 8 + j) * 4); });
        workers_sync();
    } else {
        asm volatile("griddepcontrol.wait;" ::: "memory");      // `back` is read at a tile's end
    }
    const int g = row_of(lane >> 2), t = lane & 3, slice = warp % slices, band = warp / slices;
    const bool working = band < bands;          // the others only help at a tile's end
    float y[RT][NT][4];
#pragma unroll
    for (int i = 0; i < RT; ++i)
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) y[i][n][e] = 0.0f;

    // this lane's places in a stage
    const unsigned char* code_rows = smem + slice * U / kBoxUnits * (tile_rows * 128) + (band * RT * 16 + g) * 128;      // not used where band >= bands
    const int half = U == 1 ? slice & 1 : 0;
    const int row8 = 8 * a.head_bytes;
    const unsigned char* head_rows = heads_at + (band * RT * 16 + g) * a.head_bytes;
    // a column that no state stands in takes another's: what comes of it is not stored
    int column[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) column[n] = (n * 8 + (lane >> 2) < cols ? n * 8 + (lane >> 2) : cols - 1) * 64 + t * 16;
    int buffer = 0;
    int stage = 0;
    uint32_t round = 0;
    float lost = 0.0f;                          // NaN once a stage was given up
    for (int64_t tile = blockIdx.x; tile < a.tiles; tile += gridDim.x) {
        for (int c = working && lost == 0.0f ? 0 : chunks; c < chunks; ++c) {
            const bool arrived = barrier_wait(full + 8 * stage, round & 1, a.polls);
            if (!__all_sync(kFull, arrived)) {
                // This warp's sums cannot be had: no stage is read or given back from here on, so that the fetching warp stops too.
                if (a.error_flag) atomicOr(a.error_flag, 16);
                lost = __int_as_float(0x7fc00000);
                break;
            }
            const int g0 = (c * slices * U * kUnit) >> a.group_log2;
            const unsigned char* heads = head_rows + stage * head_bytes + ((a.D / 2 + 4 * g0) & 15) - 4 * g0;
            const unsigned char* codes = code_rows + stage * code_bytes;
#pragma unroll
            for (int k = 0; k < U; ++k) {
                const int u = U * (c * slices + slice) + k;
                if (u >= units) break;
                const unsigned char* states = LOCAL ? local + u * local_unit : states_at + stage * state_bytes + (slice * U + k) * kStates;
                const unsigned char* sums_of_states = states + (LOCAL ? P * cols * 256 : P * NT * 2048);
                uint4 w[RT][2];
#pragma unroll
                for (int i = 0; i < RT; ++i)
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const unsigned char* row = codes + (i * 16 + j * 8) * 128;
                        if constexpr (STEPS < 4) {
                            auto word = [&](int s) { return *reinterpret_cast<const uint32_t*>(row + ((((k + half) * 4 + s) ^ g) * 16 + t * 4)); };
                            w[i][j] = make_uint4(word(0), word(1), word(2), word(3));
                        } else {
                            w[i][j] = *reinterpret_cast<const uint4*>(row + (((k + half) * 4 + t) ^ g) * 16);
                        }
                    }
                // The second pieces of fp32 states have sums of their own: a matrix instruction cuts off what it adds to a large sum, and
                // they would double how often.  (Worst error of 4 states of 8192 by groups of 256, over the product of the norms: 1.4e-8, 2.5e-8
                // with one sum for both; the registers cost 16 states 4 %.)
                float acc[P][RT][NT][4];
#pragma unroll
                for (int s = 0; s < 4; ++s) {
                    const bool first = s % STEPS == 0, last = s % STEPS == STEPS - 1;
                    uint32_t p[RT][2][4];
#pragma unroll
                    for (int i = 0; i < RT; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j) decode_codes(s == 0 ? w[i][j].x : s == 1 ? w[i][j].y : s == 2 ? w[i][j].z : w[i][j].w, p[i][j]);
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int q = 0; q < P; ++q) {
                            const uint4 b = *reinterpret_cast<const uint4*>(states + (LOCAL ? (s * P + q) * (cols * 64) + column[n] : ((s * NT + n) * P + q) * 512 + lane * 16));
#pragma unroll
                            for (int i = 0; i < RT; ++i) {
                                if (first) mma<true>(acc[q][i][n], p[i][0][0], p[i][1][0], p[i][0][1], p[i][1][1], b.x, b.y);
                                else mma<false>(acc[q][i][n], p[i][0][0], p[i][1][0], p[i][0][1], p[i][1][1], b.x, b.y);
                                mma<false>(acc[q][i][n], p[i][0][2], p[i][1][2], p[i][0][3], p[i][1][3], b.z, b.w);
                            }
                        }
                    if (last) {
                        // groups behind the last have states of zero: any scale and bias will do
                        int gi = (u * kUnit + 32 * s) >> a.group_log2;
                        gi = gi < groups ? gi : groups - 1;
                        float2 sum[NT];
#pragma unroll
                        for (int n = 0; n < NT; ++n) sum[n] = *reinterpret_cast<const float2*>(sums_of_states + (s / STEPS * NT * 8 + n * 8 + 2 * t) * 4);
#pragma unroll
                        for (int i = 0; i < RT; ++i)
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const __half2 head = *reinterpret_cast<const __half2*>(heads + (i * 2 + j) * row8 + 4 * gi);
                                const float sc = __low2float(head), bi = __high2float(head);
#pragma unroll
                                for (int n = 0; n < NT; ++n)
#pragma unroll
                                    for (int e = 0; e < 2; ++e) {
                                        float total = acc[0][i][n][2 * j + e];
                                        if constexpr (P == 2) total += acc[1][i][n][2 * j + e];
                                        y[i][n][2 * j + e] = fmaf(bi, e ? sum[n].y : sum[n].x, fmaf(sc, total, y[i][n][2 * j + e]));
                                    }
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
        // The tile's end: the slices' sums are added in their order.
        float* sums = red + buffer * (kWarps * kPart);
        float* part = sums + warp * kPart;
#pragma unroll
        for (int i = 0; i < RT; ++i)
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    part[(n * 8 + 2 * t + (e & 1)) * kPitch + i * 16 + (e >> 1) * 8 + g] = y[i][n][e] + lost;
                    y[i][n][e] = 0.0f;
                }
        workers_sync();
        for (int i = threadIdx.x; i < cols * tile_rows; i += kWorkers) {
            const int col = i / tile_rows, row = i - col * tile_rows;
            const int64_t r = tile * tile_rows + row;
            if (r >= a.num_rows) continue;
            const float* from = sums + row / (RT * 16) * slices * kPart + col * kPitch + row % (RT * 16);
            float v = 0.0f;
            for (int k = 0; k < slices; ++k) v += from[k * kPart];
            v *= LOCAL ? backs[col] : __ldcg(a.back + m0 + col);
            if (a.bias) v += load_any(a.bias, a.bias_dtype, r);
            store_any(a.out, a.out_dtype, (m0 + col) * a.out_stride + r, v);
        }
        // the next tile's sums go to the other buffer, where there is one: its own barrier parts the two after it
        if (a.buffers == 1) workers_sync();
        else buffer ^= 1;
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

int states_per_block(int64_t m) { return m <= 8 ? 1 : 2; }      // in eights
int pieces_of(int dtype) { return dtype == TBE_B200_FP32 ? 2 : 1; }
int steps_of(int group_log2) { return group_log2 == 5 ? 1 : group_log2 == 6 ? 2 : 4; }
int64_t units_of(int64_t D) { return (D + kUnit - 1) / kUnit; }

// Whether a block keeps all states in shared memory: it then arranges them itself, which saves a launch and the scratch.  What
// is left holds two stages of any shape.
constexpr int64_t kMostLocal = 96 * 1024;
int64_t local_bytes(int64_t m, int64_t D, int dtype, int group_log2)
{
    return units_of(D) * local_unit_bytes(static_cast<int>(m), states_per_block(m), pieces_of(dtype), steps_of(group_log2));
}
bool is_local(int64_t m, int64_t D, int dtype, int group_log2) { return m <= 16 && local_bytes(m, D, dtype, group_log2) <= kMostLocal; }

int64_t arranged_bytes(int64_t m, int64_t D, int dtype, int group_log2)
{
    const int NT = states_per_block(m);
    return (m + NT * 8 - 1) / (NT * 8) * units_of(D) * unit_bytes(NT, pieces_of(dtype), steps_of(group_log2));
}

// How the warps of a block share rows and elements, and what that costs.
struct Shape {
    int slices, bands, stages, head_bytes, buffers;
    int64_t tiles, shared, cost;
};

// Of all shapes the one whose blocks are done first: counted in shares of a stage (4096 codes) that a warp goes through (tiles of
// a block times chunks of a tile), twice, and one for every tile's end.  Two stages have to fit, and a box is at most 256 rows.
Shape shape_for(const LinearArgs& a, int RT, int NT, int P, int steps, bool local)
{
    const int U = units_at_once(RT), sms = sm_count(), shares = (a.D + U * kUnit - 1) / (U * kUnit);
    const int64_t sums = static_cast<int64_t>(kWarps) * NT * 8 * (RT * 16 + 4) * 4;
    const int64_t fixed = sums + 16 * kMostStages + (local ? 128 + units_of(a.D) * local_unit_bytes(static_cast<int>(a.m), NT, P, steps) : 0);
    auto fitting = [&](int64_t bytes, int64_t stage) { return static_cast<int>((kMostShared - bytes) / stage < kMostStages ? (kMostShared - bytes) / stage : kMostStages); };
    Shape best{};
    for (int slices = kBoxUnits / U; slices <= kWarps; slices += kBoxUnits / U) {      // whole boxes
        const int most = 256 / (RT * 16), bands = kWarps / slices < most ? kWarps / slices : most, rows = bands * RT * 16;
        const int heads = head_window(a.D, U * slices, a.group_log2);
        const int64_t stage = static_cast<int64_t>(rows) * (slices * U * (kUnit / 2) + heads) + (local ? 0 : slices * U * unit_bytes(NT, P, steps));
        const int64_t tiles = (a.num_rows + rows - 1) / rows;
        const int stages = fitting(fixed, stage), buffers = fitting(fixed + sums, stage) == stages ? 2 : 1;
        const int64_t cost = ((tiles + sms - 1) / sms) * (2 * ((shares + slices - 1) / slices) + 1);
        if (best.slices && (stages < 2 || cost >= best.cost)) continue;
        best = Shape{slices, bands, stages, heads, buffers, tiles, fixed + (buffers - 1) * sums + stages * stage, cost};
    }
    return best;
}

template <typename T, int RT, int NT, int P, int STEPS>
int launch_linear(LinearArgs a, const Shape& shape, cudaStream_t s)
{
    constexpr bool LOCAL = !std::is_void<T>::value;
    a.slices = shape.slices;
    a.bands = shape.bands;
    a.stages = shape.stages;
    a.head_bytes = shape.head_bytes;
    a.buffers = shape.buffers;
    a.tiles = shape.tiles;
    const int tile_rows = RT * 16 * a.bands, sms = sm_count();
    CUtensorMap codes, heads;
    if (!encode_rows(&codes, a, 32, tile_rows, true) || !encode_rows(&heads, a, a.head_bytes / 4, tile_rows, false))
        return fail(TBE_B200_ERR_CUDA, "group_row_linear: the rows could not be described to the copy engine");
    auto* kernel = group_row_linear_kernel<T, RT, NT, P, STEPS>;
    static std::atomic<uint64_t> allowed{0};
    if (const int rc = allow_shared(reinterpret_cast<const void*>(kernel), kMostShared, allowed)) return rc;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(a.tiles < sms ? a.tiles : sms), static_cast<unsigned>((a.m + NT * 8 - 1) / (NT * 8)));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = shape.shared;
    config.stream = s;
    config.attrs = &early;
    config.numAttrs = LOCAL ? 0 : 1;
    const cudaError_t e = cudaLaunchKernelEx(&config, kernel, a, codes, heads);
    if (e != cudaSuccess) return fail(TBE_B200_ERR_CUDA, "group_row_linear_kernel: %s", cudaGetErrorString(e));
    return check_launch("group_row_linear_kernel");
}

// T: the states' type where blocks arrange them themselves, else void.
template <typename T, int P>
int launch_linear(const LinearArgs& a, cudaStream_t s)
{
    constexpr bool LOCAL = !std::is_void<T>::value;
    const int NT = states_per_block(a.m), steps = steps_of(a.group_log2);
    // 32 rows to a warp use every state twice, which makes a stage about a tenth shorter; 16 fit more numbers of rows.  Measured over
    // 1024 to 131072 rows of 1024 to 8192 by 1, 8 and 16 states (us, 32 / 16): at equal cost 61.5 / 65.5 (8 states by 131072 x 4096) and
    // 28.2 / 30.6 (1 by 28672 x 5000), seldom behind; at a cost 1.13 times as high 10.7 / 10.0 (1 by 5000 x 8192) and 38.4 / 34.8 (16 by
    // 20000 x 8192).
    const Shape wide = shape_for(a, 2, NT, P, steps, LOCAL), narrow = shape_for(a, 1, NT, P, steps, LOCAL);
    const bool two = NT == 2, many = 10 * wide.cost <= 11 * narrow.cost;
    auto by_group = [&](auto rt, auto nt) {
        constexpr int RT = decltype(rt)::value, N = decltype(nt)::value;
        const Shape& shape = RT == 2 ? wide : narrow;
        switch (steps) {
            case 1: return launch_linear<T, RT, N, P, 1>(a, shape, s);
            case 2: return launch_linear<T, RT, N, P, 2>(a, shape, s);
            default: return launch_linear<T, RT, N, P, 4>(a, shape, s);
        }
    };
    const std::integral_constant<int, 1> one{};
    const std::integral_constant<int, 2> both{};
    if (many) return two ? by_group(both, both) : by_group(both, one);
    return two ? by_group(one, both) : by_group(one, one);
}

template <typename T>
int launch_arrange(const T* x, int64_t x_stride, int64_t m, int D, int group_log2, unsigned char* arranged, float* back, cudaStream_t s)
{
    auto* kernel = group_log2 == 5 ? arrange_states_kernel<T, 1> : group_log2 == 6 ? arrange_states_kernel<T, 2> : arrange_states_kernel<T, 4>;
    kernel<<<static_cast<unsigned>(m), kStateThreads, 0, s>>>(x, x_stride, D, states_per_block(m), arranged, back);
    return check_launch("arrange_states_kernel");
}

}  // namespace
}  // namespace tbe

using namespace tbe;

extern "C" int64_t tbe_b200_group_row_linear_scratch_bytes(int64_t m, int64_t D, int32_t group_size, int32_t input_dtype)
{
    const int group_log2 = group_log2_of(group_size);
    if (m < 0 || m > (1 << 19) || D < 1 || D > (1 << 20) || group_log2 < 0 || !element_bytes(input_dtype)) return -1;
    return is_local(m, D, input_dtype, group_log2) ? 0 : arranged_bytes(m, D, input_dtype, group_log2) + (4 * m + 15) / 16 * 16;
}

extern "C" int tbe_b200_group_row_linear(const void* input, int32_t input_dtype, int64_t input_stride, int64_t m, const uint8_t* rows,
                                         int64_t num_rows, int64_t row_bytes, int64_t D, int32_t group_size, const void* bias, int32_t bias_dtype,
                                         void* output, int32_t output_dtype, int64_t output_stride, int32_t* error_flag, void* scratch,
                                         int64_t scratch_bytes, tbe_b200_stream_t stream)
{
    return tbe_b200_group_row_linear_bounded(input, input_dtype, input_stride, m, rows, num_rows, row_bytes, D, group_size, bias, bias_dtype, output, output_dtype,
                                             output_stride, error_flag, scratch, scratch_bytes, kPolls, stream);
}

extern "C" int tbe_b200_group_row_linear_bounded(const void* input, int32_t input_dtype, int64_t input_stride, int64_t m, const uint8_t* rows,
                                                 int64_t num_rows, int64_t row_bytes, int64_t D, int32_t group_size, const void* bias, int32_t bias_dtype,
                                                 void* output, int32_t output_dtype, int64_t output_stride, int32_t* error_flag, void* scratch,
                                                 int64_t scratch_bytes, int64_t max_polls, tbe_b200_stream_t stream)
{
    const int ib = element_bytes(input_dtype), ob = element_bytes(output_dtype);
    if (!ib || !ob || (bias && !element_bytes(bias_dtype))) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: element types FP32, FP16 and BF16");
    if (const int rc = check_group_rows("group_row_linear", D, group_size, row_bytes, rows, num_rows)) return rc;
    if (num_rows > 0x7fffffff - 512) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: too many rows");
    if (m < 0 || D == 0 || input_stride < D || output_stride < num_rows)
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: D must be positive, row strides at least D and num_rows");
    if (D > (1 << 20) || m > (1 << 19)) return fail(TBE_B200_ERR_UNSUPPORTED, "group_row_linear: D at most 2^20 and m at most 2^19");
    if (max_polls < 0) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: max_polls must not be negative");
    if (m == 0 || num_rows == 0) return TBE_B200_OK;
    if (!input || !rows || !output) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: NULL pointer");
    if (!rows_aligned(input, input_stride, ib, 8)) return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: input rows must be 16-byte aligned");
    cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
    const int group_log2 = group_log2_of(group_size);
    LinearArgs a{nullptr, nullptr, input, input_stride, m, rows, num_rows, row_bytes, static_cast<int>(D), group_log2, bias, bias_dtype, output_dtype, output,
                 output_stride, error_flag, 0, 0, 0, 0, 0, static_cast<int>(max_polls < INT32_MAX ? max_polls : INT32_MAX), 0};
    if (is_local(m, D, input_dtype, group_log2))
        return with_element(input_dtype, [&](auto* ti) {
            using T = std::remove_pointer_t<decltype(ti)>;
            return launch_linear<T, kPieces<T>>(a, s);
        });
    const int64_t need = tbe_b200_group_row_linear_scratch_bytes(m, D, group_size, input_dtype);
    if (!scratch || scratch_bytes < need || (reinterpret_cast<uintptr_t>(scratch) & 15))
        return fail(TBE_B200_ERR_INVALID_ARGUMENT, "group_row_linear: scratch must be %lld bytes, 16-byte aligned", (long long)need);
    unsigned char* states = static_cast<unsigned char*>(scratch);
    float* back = reinterpret_cast<float*>(states + arranged_bytes(m, D, input_dtype, group_log2));
    a.arranged = states;
    a.back = back;
    const int rc = with_element(input_dtype, [&](auto* ti) {
        using T = std::remove_pointer_t<decltype(ti)>;
        return launch_arrange<T>(static_cast<const T*>(input), input_stride, m, static_cast<int>(D), group_log2, states, back, s);
    });
    if (rc) return rc;
    return pieces_of(input_dtype) == 1 ? launch_linear<void, 1>(a, s) : launch_linear<void, 2>(a, s);
}
