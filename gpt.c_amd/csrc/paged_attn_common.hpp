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

// N consecutive 32-bit words of T values from row + d.  Values at or past D come from the row itself, so that no branch
// parts the loads; with kZero (queries) they are zeros.  Keys and values go without: the query is 0 there and results
// past D are not stored, and a selection between load and use would have to wait for the load.
template <typename T, int N, Rows R, bool kZero>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const T *row, int d, int D) {
    if constexpr (R != kAny) {
        static_assert(N == 1 || N == 2 || N == 4, "one load");
        const bool in = R == kFull || d < D;
        const T *from = row + (in ? d : 0);
        if constexpr (N == 1) {
            w[0] = *reinterpret_cast<const uint32_t *>(from);
        } else {
            typedef uint32_t vec __attribute__((ext_vector_type(N)));
            const vec x = *reinterpret_cast<const vec *>(from);
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = x[i];
        }
        if (kZero && !in)
#pragma unroll
            for (int i = 0; i < N; ++i) w[i] = 0;
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            w[i] = __builtin_bit_cast(uint32_t, row[min(d + i, D - 1)]);
            if (kZero && d + i >= D) w[i] = 0;
        }
    } else {
        static_assert(!kZero, "queries are floats");
        const uint16_t *r = reinterpret_cast<const uint16_t *>(row);
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = r[min(d + 2 * i, D - 1)] | static_cast<uint32_t>(r[min(d + 2 * i + 1, D - 1)]) << 16;
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

// A matrix instruction's result may be touched 8 instruction slots after it at the earliest (16x16x32 bf16), or 10
// (16x16x4 fp32), and the hardware does not wait.  The compiler counts them inside a block; across a branch it was seen
// to read the last two registers at once (wrong sums at every second step of bf16 pages), and a slot too soon where a
// branch was turned round after the count.  So results are taken over in the block of the product (settled), or after
// a wait (drain) that nothing is moved across; tests/test_kernel_code.py looks at every path of the built kernels.
__device__ __forceinline__ void settled(f32x4 &x) { asm volatile("" : "+v"(x)); }
__device__ __forceinline__ void drain() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_nop 15");
    __builtin_amdgcn_sched_barrier(0);
}

// ---- values that are no numbers, in the tokens that some rows of a tile must not see ----
//
// A hidden key's weight is 0, but 0 times NaN or infinity is not.  So in the tiles where keys are hidden from some
// rows, values that are not finite are taken out of the products, and an item where there was one is done again, one
// key after the other.

// A 32-bit word of T values without those that are not finite; with kSplit also without the floats that split3 rounds to
// infinity, from half a step past the largest bf16 value on.
template <typename T, bool kSplit = false>
__device__ __forceinline__ uint32_t finite_part(uint32_t w) {
    if constexpr (sizeof(T) == 4) return (w & 0x7fffffffu) >= (kSplit ? 0x7f7f8000u : 0x7f800000u) ? 0 : w;
    if ((w & 0x7f80u) == 0x7f80u) w &= 0xffff0000u;
    if ((w & 0x7f800000u) == 0x7f800000u) w &= 0xffffu;
    return w;
}

// Query rows row0 .. row0 + count - 1 of an item by one wave, whose lanes hold two values of a head each.  `slot`:
// the workspace row of row0.
template <typename T>
__device__ __forceinline__ void rows_by_key(const PagedAttnParams &a, const PagedItem &it, int kv, int row0, int count,
                                            int64_t slot) {
    const int d0 = threadIdx.x & 63, d1 = d0 + 64;
    const bool in0 = d0 < a.D, in1 = d1 < a.D;
    const int *table = a.table + it.table;
    for (int i = 0; i < count; ++i) {
        const int row = row0 + i, token = row / a.group;
        if (row >= it.rows || it.tok0 + token >= a.rows) return;
        const int head = kv * a.group + row - token * a.group;
        const float *q = a.q + static_cast<int64_t>(it.tok0 + token) * a.q_stride + static_cast<int64_t>(head) * a.D;
        const float q0 = in0 ? q[d0] : 0.0f, q1 = in1 ? q[d1] : 0.0f;
        float m = -INFINITY, l = 0.0f, o0 = 0.0f, o1 = 0.0f;
        const int end = min(it.past + token + 1, it.key1);
        for (int key = it.key0; key < end; ++key) {
            const int64_t page = table[key >> a.page_shift];
            const int64_t at = (((page * a.KV + kv) << a.page_shift) + (key & ((1 << a.page_shift) - 1))) * a.D;
            const T *k = static_cast<const T *>(a.k) + at, *v = static_cast<const T *>(a.v) + at;
            float s = in0 ? q0 * static_cast<float>(k[d0]) : 0.0f;
            if (in1) s = fmaf(q1, static_cast<float>(k[d1]), s);
            s = wave_sum(s) * a.scale_log2;
            const float top = fmaxf(m, s), base = top == -INFINITY ? 0.0f : top;
            const float f = fast_exp2(m - base), p = fast_exp2(s - base);
            l = fmaf(l, f, p);
            if (in0) o0 = fmaf(o0, f, p * static_cast<float>(v[d0]));
            if (in1) o1 = fmaf(o1, f, p * static_cast<float>(v[d1]));
            m = top;
        }
        float *dst = a.part_o + (slot + i) * a.D, scale = 1.0f;
        if (it.part < 0) {
            dst = a.out + (static_cast<int64_t>(it.tok0 + token) * a.H + head) * a.D;
            scale = 1.0f / l;
        } else if (d0 == 0) {
            a.part_ml[2 * (slot + i)] = m;
            a.part_ml[2 * (slot + i) + 1] = l;
        }
        if (in0) dst[d0] = o0 * scale;
        if (in1) dst[d1] = o1 * scale;
    }
}

}  // namespace gptc
