// The pieces of the cross entropy without logits (head_loss.hip) that its two
// kinds of products share: gemm_halves.hip for many rows, head_few.hip for few.
#pragma once

#include "gemm_halves.hpp"
#include "ops_common.hpp"

namespace gptc {

// A token held in a float, truncated; -1 for what is not in [0, V).
__device__ __forceinline__ int token_of(float f, int V) {
    return f > -1.0f && f < static_cast<float>(V) ? static_cast<int>(f) : -1;
}

// Where the logits of a piece go.
struct LogitsArgs {
    float *logits;         // blocks of 32 rows x 32 tokens in the order of the accumulators, or null
    float2 *stats;         // (parts of the tokens, rows): largest logit and the sum of exp of the distances from it
    const float *targets;  // (rows)
    float *target_logits;  // (rows), written where the target is
    int vocabulary, rows;
    int token_blocks, row_stride;  // blocks of 32 tokens of `logits`, rows of `stats`
};

// A wave's logits of 32 rows x 32 NI tokens from token0 on: lane l holds row l % 32 of row block
// `row_block` and, at 4 q + e of x[i], token token0 + 32 i + 8 q + 4 (l / 32) + e.  So a row's
// largest logit and sum (of exp of the distances from it) need two lanes only; both lanes return them.  STREAMED: the
// logits of many rows, which leave the caches before they are read (8192 rows' step 6.15 ms without the hint, 6.12 with
// it; 100 rows' 174.7 us without, 176.5 with it).
template <int NI, bool STREAMED>
__device__ __forceinline__ float2 put_logits(const LogitsArgs &l, hf32x16 (&x)[NI], int token0, int row_block) {
    constexpr float kLog2e = 1.4426950408889634f;
    const int lane = threadIdx.x & 63, hf = lane >> 5, row = row_block * 32 + (lane & 31);
    const int mine = token0 + 4 * hf;  // this lane's tokens: mine + 32 i + 8 q + e
    if (token0 + 32 * NI > l.vocabulary) {
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (mine + 32 * i + 8 * (r >> 2) + (r & 3) >= l.vocabulary) x[i][r] = -INFINITY;
    }
    if (l.logits != nullptr) {
        f32x4_t *out = reinterpret_cast<f32x4_t *>(l.logits) +
                       (static_cast<int64_t>(row_block) * l.token_blocks + (token0 >> 5)) * 256 + lane;
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4_t four = {x[i][4 * q], x[i][4 * q + 1], x[i][4 * q + 2], x[i][4 * q + 3]};
                if (STREAMED)
                    __builtin_nontemporal_store(four, out + i * 256 + q * 64);
                else
                    out[i * 256 + q * 64] = four;
            }
    }
    const int target = (row < l.rows ? token_of(l.targets[row], l.vocabulary) : -1) - mine;
    float m = -INFINITY, t = 0.0f;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            m = fmaxf(m, x[i][r]);
            t = target == 32 * i + 8 * (r >> 2) + (r & 3) ? x[i][r] : t;
        }
    if (target >= 0 && target < 32 * NI && (target & 4) == 0) l.target_logits[row] = t;
    m = fmaxf(m, __shfl_xor(m, 32, 64));
    const float ref = m == -INFINITY ? 0.0f : m;
    float s = 0.0f;
    // The distance first, which is as exact as the logits: m times log2(e), rounded, would be off by 2^-24 of m itself.
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s += __builtin_amdgcn_exp2f((x[i][r] - ref) * kLog2e);
    s += __shfl_xor(s, 32, 64);
    return make_float2(m, s);
}

// A = W (vocabulary x features), B = x (rows x features).  Returns the tokens of each of the stats' parts.
int launch_logits(const Halves &A, const Halves &B, const LogitsArgs &l, hipStream_t s);

// An operand of few rows in two fp16 parts, as Halves, but padded to row_blocks of 32 rows and 32 terms.  d's terms lie as
// there, x's as head_few.hip reads W's rows.
struct FewRows {
    hu32x4 *data;
    int *shift;  // (padded rows), or null: every row's is `shift_all`
    int shift_all;
    int row_blocks, terms;
    __host__ __device__ int term_blocks() const { return (terms + 31) / 32 * 2; }
    __host__ __device__ int64_t bytes() const { return static_cast<int64_t>(row_blocks) * term_blocks() * 2048; }
};

// Blocks of 32 rows that launch_few_logits and launch_few_dx take for this many rows.
int few_row_blocks(int rows);
// x (rows x terms without gaps) into t, rows of weight 0 as zeros; `zeros` words at `zero` to 0.
void launch_few_rows(const float *x, const float *weights, int rows, const FewRows &t, uint32_t *zero, int zeros,
                     hipStream_t s);
// The logits of x (V x C floats W as they come).  Returns the tokens of each of the stats' parts.
int launch_few_logits(const float *W, int V, int C, const FewRows &x, const LogitsArgs &l, hipStream_t s);
// p.C (rows x C) = d W by the rows' factors.
void launch_few_dx(const FewRows &d, const float *W, int V, int C, int rows, const HalvesProduct &p, hipStream_t s);

// p.C (dt.rows x xt.rows) = d^T x (+ p.C) for up to kFewDwTerms rows; p without factors.
constexpr int kFewDwTerms = 128;
void launch_few_dw(const Halves &dt, const Halves &xt, const HalvesProduct &p, hipStream_t s);

}  // namespace gptc
