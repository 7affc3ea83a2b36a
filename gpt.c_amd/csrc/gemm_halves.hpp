// Products of fp32 operands that are laid out beforehand as sums of two fp16
// values, three matrix instructions a product (gemm_halves.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>

namespace gptc {

typedef float hf32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t hu32x4 __attribute__((ext_vector_type(4)));

// An operand of `rows` (of the product's M or N) by `terms` (of its reduction),
// padded with zeros to 128 rows and 64 terms.  Row r's values are held
// times 2^shift[r], which puts the largest below 2^15: value = high + low to
// 2^-24 of it, or to 2^-40 of the row's largest for values below its 2^-17th.
// Blocks of 32 rows x 16 terms, block (r / 32, k / 16) after block, high part
// (1 KB) then low part: lane l of a wave holds row l % 32 and the terms
// 4 (l / 32) + {0, 1, 2, 3, 8, 9, 10, 11}, as the 32x32x16 instruction takes them
// (in an order of terms that suits fp32 results as the next product's operand).
struct Halves {
    hu32x4 *data;
    int *shift;  // (padded rows), or null: every row's is `shift_all`
    int shift_all;
    int rows, terms;
    __host__ __device__ int row_blocks() const { return (rows + 127) / 128 * 4; }
    __host__ __device__ int term_blocks() const { return (terms + 63) / 64 * 4; }
    __host__ __device__ int64_t bytes() const { return static_cast<int64_t>(row_blocks()) * term_blocks() * 2048; }
};

// The cache hint of stores whose values are not read again soon: dW's, beside which W stays in the caches (100 rows of 768
// on 50257: 183 us without it, 174 with it; 1024 rows: 872, 868).
constexpr int kStreamed = 2;

constexpr int kHalvesTop = 14;  // the largest value of a row is held below 2^(kHalvesTop + 1)

// The shift of a row whose largest magnitude is m (0, infinities and NaN: as they are).
__device__ __forceinline__ int halves_shift(float m) {
    const int e = static_cast<int>((__float_as_uint(m) >> 23) & 0xff);
    if (e == 0xff || m == 0.0f) return 0;
    return kHalvesTop - (e == 0 ? -127 : e - 127);  // subnormal values end up to 2^23 lower, still exact
}

// Two values as high parts and low parts (packed): each part the nearest fp16 of what is left.
__device__ __forceinline__ void halves_split(float x, float y, uint32_t &high, uint32_t &low) {
    const _Float16 hx = static_cast<_Float16>(x), hy = static_cast<_Float16>(y);
    const _Float16 lx = static_cast<_Float16>(x - static_cast<float>(hx));
    const _Float16 ly = static_cast<_Float16>(y - static_cast<float>(hy));
    high = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, hx)) |
           static_cast<uint32_t>(__builtin_bit_cast(uint16_t, hy)) << 16;
    low = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, lx)) |
          static_cast<uint32_t>(__builtin_bit_cast(uint16_t, ly)) << 16;
}

// Negating every other 64 terms of one of a product's operands keeps the matrix core's truncation
// from adding up: the kernels subtract those sums.
__device__ __forceinline__ bool halves_negated(int term) { return ((term >> 6) & 1) != 0; }

// x (rows x terms without gaps; with weights, rows of weight 0 as zeros) into h.data and h.shift, as a second operand;
// `zeros` words at `zero` to 0.
void launch_halves_rows(const float *x, const float *weights, const Halves &h, uint32_t *zero, int zeros, hipStream_t s);
// The same for other paddings, or (in_lines) as the operand whose terms are negated, with another order of a block's terms:
// lane l of blocks 2 j and 2 j + 1 holds 32 j + 16 (l / 32) + {0 .. 7} and {8 .. 15}, a step's 64 consecutive bytes for
// either half of the lanes.
struct HalvesRows {
    hu32x4 *data;
    int *shift;
    int row_blocks, term_blocks;  // of 32 and of 16
    bool in_lines;
    uint32_t *zero;  // the same launch sets `zeros` words here to 0
    int zeros;
};
void launch_rows(const float *x, const float *weights, int rows, int terms, const HalvesRows &t, hipStream_t s);
// x (rows x terms without gaps) as a first operand, 64 rows each by the shift of their largest magnitude (up to 126).
void launch_halves_table(const float *x, const Halves &h, hipStream_t s);
// x (terms x rows, rows of ld floats; with weights, times weights[k] / divisor by term k, and zeros where it is 0),
// as a second operand, or as the one that is negated.  largest: the bits of each column's largest magnitude, which the
// first call raises from what it holds and which may count further terms too; null with up to
// kColumnTerms terms, whose largest the second call finds by itself.
constexpr int kColumnTerms = 128;
void launch_column_largest(const float *x, int ld, const float *weights, float divisor, int terms, int cols,
                           uint32_t *largest, hipStream_t s);
void launch_halves_columns(const float *x, int ld, const float *weights, float divisor, const Halves &h,
                           bool negate, const uint32_t *largest, hipStream_t s);

// In products A has one shift, B one a row.
// C (A.rows x B.rows, rows of ldc) = A B^T times row_factor[m] / divisor (+ C); rows of factor 0 are 0.
struct HalvesProduct {
    float *C;
    int ldc;
    const float *row_factor;  // or null for ones
    float divisor;
    bool add;
};
void launch_halves_product(const Halves &A, const Halves &B, const HalvesProduct &p, hipStream_t s);
// C (A.terms x B.rows) = A^T B^T for A as in another product, where it was the first operand, with one shift; B is
// negated.  C (A.rows x B.terms) = A B for such a B, with a shift for 64 rows each.  What is read across is readable up
// to 8 KB past its end.
void launch_product_across_a(const Halves &A, const Halves &B, const HalvesProduct &p, hipStream_t s);
void launch_product_across_b(const Halves &A, const Halves &B, const HalvesProduct &p, hipStream_t s);
// C from the sums of `slices` parts of the reduction, (M, N) each, in their order.
void launch_join_slices(const float *part, int M, int N, int slices, const HalvesProduct &p, hipStream_t s);

}  // namespace gptc
