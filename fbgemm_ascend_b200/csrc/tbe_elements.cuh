// Rows of fp32 / fp16 / bf16 elements, moved in pieces of VEC elements: shared by the token-table kernels.
#pragma once

#include <type_traits>

#include "tbe_common.cuh"

namespace tbe {

// VEC consecutive elements of type T as they lie in memory (at most 32 bytes).
template <typename T, int VEC>
struct Piece {
    static constexpr int kBytes = VEC * static_cast<int>(sizeof(T));
    static constexpr int kWords = (kBytes + 3) / 4;
    uint32_t w[kWords];
};

// CONSTANT: nothing writes this memory while the kernel runs (read-only loads).
template <typename U, bool CONSTANT>
__device__ __forceinline__ U load_as(const void* p)
{
    if constexpr (CONSTANT) return __ldg(static_cast<const U*>(p));
    else return *static_cast<const U*>(p);
}

template <typename T, int VEC, bool CONSTANT = true>
__device__ __forceinline__ void load_piece(Piece<T, VEC>& r, const T* p)
{
    constexpr int B = Piece<T, VEC>::kBytes;
    if constexpr (B >= 16) {
#pragma unroll
        for (int i = 0; i < B / 16; ++i) {
            const uint4 q = load_as<uint4, CONSTANT>(reinterpret_cast<const char*>(p) + 16 * i);
            r.w[4 * i] = q.x; r.w[4 * i + 1] = q.y; r.w[4 * i + 2] = q.z; r.w[4 * i + 3] = q.w;
        }
    } else if constexpr (B == 8) {
        const uint2 q = load_as<uint2, CONSTANT>(p);
        r.w[0] = q.x; r.w[1] = q.y;
    } else if constexpr (B == 4) {
        r.w[0] = load_as<uint32_t, CONSTANT>(p);
    } else {
        r.w[0] = load_as<unsigned short, CONSTANT>(p);
    }
}

template <typename T, int VEC>
__device__ __forceinline__ void clear_piece(Piece<T, VEC>& r)
{
#pragma unroll
    for (int i = 0; i < Piece<T, VEC>::kWords; ++i) r.w[i] = 0u;
}

// A row (of one element at least) that starts at any element: the 16-byte border in front of it, where it begins behind that, and
// the last 16-byte word that holds some of it, bytes.
struct SplitRow {
    const char* base;
    int begin, last;

    template <typename T>
    __device__ __forceinline__ void of(const T* row, int D)
    {
        const uintptr_t a = reinterpret_cast<uintptr_t>(row);
        base = reinterpret_cast<const char*>(a & ~uintptr_t(15));
        begin = static_cast<int>(a & 15);
        last = (begin + D * static_cast<int>(sizeof(T)) - 1) & ~15;
    }
};

// A piece of such a row, which may reach past its end: read in aligned 16-byte words, none of which lies wholly outside the
// row (past the end the last one stands in), and shifted into place.  What is not the row's is whatever lies there.
template <typename T, int VEC>
struct SplitPiece {
    static constexpr int kBytes = Piece<T, VEC>::kBytes;
    static constexpr int kQuads = (kBytes + 15) / 16 + 1;
    uint4 q[kQuads];
    int offset;      // of the first element in the first word, bytes

    // from element c on
    __device__ __forceinline__ void load(const SplitRow& row, int c)
    {
        const int at = row.begin + c * static_cast<int>(sizeof(T)), first = at & ~15;
        offset = at & 15;
#pragma unroll
        for (int i = 0; i < kQuads; ++i) q[i] = ldg16(row.base + min(first + 16 * i, row.last));
    }
    __device__ __forceinline__ Piece<T, VEC> piece() const
    {
        constexpr int W = Piece<T, VEC>::kWords;
        uint32_t w[4 * kQuads];
#pragma unroll
        for (int i = 0; i < kQuads; ++i) {
            w[4 * i] = q[i].x; w[4 * i + 1] = q[i].y; w[4 * i + 2] = q[i].z; w[4 * i + 3] = q[i].w;
        }
#pragma unroll
        for (int i = 0; i < W + 2; ++i) w[i] = (offset & 8) ? w[i + 2 < 4 * kQuads ? i + 2 : i] : w[i];
#pragma unroll
        for (int i = 0; i < W + 1; ++i) w[i] = (offset & 4) ? w[i + 1] : w[i];
        Piece<T, VEC> r;
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = sizeof(T) == 2 ? __funnelshift_r(w[i], w[i + 1], (offset & 2) * 8) : w[i];
        return r;
    }
};

// 16-bit types come two to a word; bf16 is the upper half of an fp32.
template <typename T, int VEC>
__device__ __forceinline__ float element(const Piece<T, VEC>& r, int i)
{
    if constexpr (sizeof(T) == 4) return __uint_as_float(r.w[i]);
    else {
        const uint32_t w = r.w[i / 2];
        if constexpr (std::is_same<T, __half>::value) return half_bits_to_float((i & 1) ? w >> 16 : w & 0xffffu);
        else return __uint_as_float((i & 1) ? w & 0xffff0000u : w << 16);
    }
}

// Rounds VEC fp32 numbers to T (to nearest even) and stores them; streaming, since a result is not read again here.
template <typename T, int VEC>
__device__ __forceinline__ void store_piece(T* p, const float (&v)[VEC])
{
    if constexpr (VEC == 1) {
        if constexpr (sizeof(T) == 4) *p = v[0];
        else if constexpr (std::is_same<T, __half>::value) *p = __float2half_rn(v[0]);
        else *p = __float2bfloat16_rn(v[0]);
    } else {
        constexpr int W = Piece<T, VEC>::kWords;
        uint32_t w[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
            if constexpr (sizeof(T) == 4) w[i] = __float_as_uint(v[i]);
            else if constexpr (std::is_same<T, __half>::value) {
                const __half2 h = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            } else {
                const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&h);
            }
        }
        if constexpr (W >= 4) {
#pragma unroll
            for (int i = 0; i < W / 4; ++i)
                st_stream16(reinterpret_cast<char*>(p) + 16 * i, make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]));
        } else if constexpr (W == 2) {
            st_stream8(p, make_uint2(w[0], w[1]));
        } else {
            st_stream4(p, w[0]);
        }
    }
}

// (v & mask) | bits in one instruction; written out with two constants it becomes two.
__device__ __forceinline__ uint32_t mask_or(uint32_t v, uint32_t mask, uint32_t bits)
{
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(r) : "r"(v), "r"(mask), "r"(bits));
    return r;
}

// One word of 4-bit codes (elements 0 .. 7, low nibble first) as four pairs (0,4) (1,5) (2,6) (3,7) of fp16 numbers.  A nibble
// or'ed into the low bits of 1024 (16 steps apart for the upper nibble of a byte) makes that number plus the code; what is
// taken off again leaves it exact.
__device__ __forceinline__ void decode_codes(uint32_t w, uint32_t (&p)[4])
{
    const uint32_t v = w >> 8;
    const uint32_t in[4] = {mask_or(w, 0x000f000fu, 0x64006400u), mask_or(w, 0x00f000f0u, 0x64006400u), mask_or(v, 0x000f000fu, 0x64006400u),
                            mask_or(v, 0x00f000f0u, 0x64006400u)};
    const __half2 even = __float2half2_rn(1024.0f), sixteenth = __float2half2_rn(0.0625f), odd = __float2half2_rn(-64.0f);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __half2 h = *reinterpret_cast<const __half2*>(&in[i]);
        const __half2 r = (i & 1) ? __hfma2(h, sixteenth, odd) : __hsub2(h, even);
        p[i] = *reinterpret_cast<const uint32_t*>(&r);
    }
}

inline int element_bytes(int dtype) { return dtype == TBE_B200_FP32 ? 4 : (dtype == TBE_B200_FP16 || dtype == TBE_B200_BF16) ? 2 : 0; }

// Whether rows that start at p, stride elements apart, can be moved in pieces of vec elements.
inline bool rows_aligned(const void* p, int64_t stride, int elem_bytes, int vec)
{
    const int64_t b = static_cast<int64_t>(vec) * elem_bytes < 16 ? static_cast<int64_t>(vec) * elem_bytes : 16;
    return reinterpret_cast<uintptr_t>(p) % b == 0 && (stride * elem_bytes) % b == 0;
}

// Calls f with a null pointer to the element type that `dtype` (checked before) names.
template <typename F>
int with_element(int dtype, F&& f)
{
    switch (dtype) {
        case TBE_B200_FP32: return f(static_cast<float*>(nullptr));
        case TBE_B200_FP16: return f(static_cast<__half*>(nullptr));
        default: return f(static_cast<__nv_bfloat16*>(nullptr));
    }
}

// 4-bit rows with group scales (tbe_group_rows.cu): log2 of a group size, -1 if it is none; and the argument checks that every
// entry point over such rows makes.
int group_log2_of(int group_size);
int check_group_rows(const char* op, int64_t D, int group_size, int64_t row_bytes, const void* rows, int64_t nrows);

}  // namespace tbe
