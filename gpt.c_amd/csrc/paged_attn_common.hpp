// Pieces that the attention kernels over pages share: row loads, exact sums of bf16 values, products.
#pragma once

#include "attn_common.hpp"
#include "paged_plan.hpp"

namespace gptc {

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// What is known of the rows: D is the tile's width; every row starts at a multiple of 16 bytes and holds whole
// vectors; or nothing.
enum Rows { kFull, kVec, kAny };

// N consecutive 32-bit words of T values from row + d; values at or past D are zeros (the load then takes the
// row's first values instead, so that no branch parts the loads).
template <typename T, int N, Rows R>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const T *row, int d, int D) {
    if constexpr (R != kAny) {
        static_assert(N == 1 || N == 2 || N == 4, "one load");
        const bool in = R == kFull || d < D;
        const T *from = row + (in ? d : 0);
        if constexpr (N == 1) {
            const uint32_t x = *reinterpret_cast<const uint32_t *>(from);
            w[0] = in ? x : 0;
        } else {
            typedef uint32_t vec __attribute__((ext_vector_type(N)));
            const vec x = *reinterpret_cast<const vec *>(from);
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = in ? x[i] : 0;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = d + i < D ? __builtin_bit_cast(uint32_t, row[d + i]) : 0u;
    } else {
        const uint16_t *r = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const uint32_t lo = d + 2 * i < D ? r[d + 2 * i] : 0u, hi = d + 2 * i + 1 < D ? r[d + 2 * i + 1] : 0u;
            w[i] = lo | hi << 16;
        }
    }
}

// x, y as sums of three bf16 values, packed in pairs.
__device__ __forceinline__ void split3(float x, float y, uint32_t (&p)[3]) {
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const f32x2 v = {x, y};
        p[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, bf16x2));
        x -= __builtin_bit_cast(float, p[i] << 16);
        y -= __builtin_bit_cast(float, p[i] & 0xffff0000u);
    }
}

__device__ __forceinline__ f32x4 mfma_bf16(const uint32_t (&a)[4], const uint32_t (&b)[4], f32x4 c) {
    const u32x4 x = {a[0], a[1], a[2], a[3]}, y = {b[0], b[1], b[2], b[3]};
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, x), __builtin_bit_cast(bf16x8, y), c, 0, 0,
                                                   0);
}

// A matrix instruction's result may be read 11 cycles after it at the earliest.  The compiler counts them inside
// a block; across a branch it was seen to read the last two registers at once (wrong sums at every second step of
// bf16 pages).  So results are taken over in the block of the product, or after a wait of 16.
__device__ __forceinline__ void settled(f32x4 &x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void finished(f32x4 &x) { asm volatile("s_nop 15" : "+a"(x)); }

}  // namespace gptc
