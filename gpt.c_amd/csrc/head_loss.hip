// Cross entropy of softmax(x W^T) and its gradients without keeping the logits.
// No counterpart in gpt.c, whose GPT2 keeps the logits, their log-softmax and
// their gradient (src/transformer.c:69-158, src/loss.c:19-148):
//   l[r, j] = x[r] . W[j],  lse[r] = log sum_j exp l[r, j],  loss[r] = lse[r] - l[r, t[r]],
//   d[r, j] = w[r] / R (exp(l[r, j] - lse[r]) - [j = t[r]]),  dx = d W,  dW (+)= d^T x.
// The rows go through in pieces, so that a piece's logits fit the scratch: its
// logits are formed once, turned into d, and used for both gradients.
#include <algorithm>
#include "gpu_kernels.h"
#include "head_loss.hpp"

namespace gptc {

namespace {

constexpr int kThreads = 256;
constexpr float kLog2eF = 1.4426950408889634f;
constexpr int kMaxVocabulary = 1 << 22;  // a product's tile offsets fit 32 bits
constexpr int kMaxRows = 1000000000;     // 2^24 workgroups of column_largest_kernel; a piece more still fits an int

__device__ __forceinline__ float weight_of(const float *weights, int row) {
    return weights != nullptr ? weights[row] : 1.0f;
}

struct MeanArgs {
    const float *losses, *weights;
    float *out;
    int rows;
};

// out[0] = sum of w[r] loss[r] / rows in a fixed order, in 64 bits; one workgroup.
template <int THREADS>
__device__ __forceinline__ void mean_loss(const MeanArgs &a) {
    __shared__ double part[THREADS / kWave];
    double t = 0.0;
#pragma unroll 8
    for (int r = threadIdx.x; r < a.rows; r += THREADS)
        t += static_cast<double>(a.losses[r]) * weight_of(a.weights, r);  // rows of weight 0: 0 * 0
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) t += __shfl_xor(t, off, kWave);
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = t;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < THREADS / kWave; ++i) t += part[i];
    a.out[0] = static_cast<float>(t / a.rows);
}

constexpr int kMeanThreads = 1024;
__global__ __launch_bounds__(kMeanThreads) void mean_loss_kernel(const MeanArgs a) { mean_loss<kMeanThreads>(a); }

constexpr int kMeanRows = 32;  // up to here, the kernel that forms the rows' losses forms their mean; else the shares' does

struct HeadLoss {
    const float *x, *W, *targets, *weights;
    float *losses, *mean, *dx, *dW;
    int rows, V, C;
    bool add;
};

void launch_mean(const HeadLoss &h, hipStream_t s) {
    mean_loss_kernel<<<dim3(1), dim3(kMeanThreads), 0, s>>>({h.losses, h.weights, h.mean, h.rows});
    hipCheck(hipGetLastError());
}

// ---- many rows: products of operands laid out as two fp16 parts ----

struct JoinArgs {
    const float2 *stats;
    int parts;
    const float *targets, *target_logits, *weights;
    float2 *shares;  // what a row's shares are taken by: the largest logit and 1 / sum
    int *whole;      // the targets, -1 for none
    float *losses;
    int rows, padded, V;
    float *mean;  // MEAN: of all rows, which are the first workgroup's
};

// A row's loss, largest logit m, 1 / sum and target from the parts of its tokens: ROWS rows a workgroup, whose slices of
// the parts are joined in a fixed order.  m and the sum stay apart: their join, lse = m + log(sum), would be rounded to
// 2^-24 of itself, and every share of the row with it.  Rows that take no part, those past the last one among them: 1 / sum
// is 0 and the target -1.  Latency bound (100 rows: 5.6 us).
constexpr int kJoinThreads = 1024;

// What sums are taken relative to: without a logit but minus infinity they are 0, or NaN where there is one.
__device__ __forceinline__ float reference(float largest) { return largest == -INFINITY ? 0.0f : largest; }

__device__ __forceinline__ void join_sums(float &m, float &s, float m2, float s2) {
    const float top = fmaxf(m, m2), ref = reference(top);
    s = s * __builtin_amdgcn_exp2f((m - ref) * kLog2eF) + s2 * __builtin_amdgcn_exp2f((m2 - ref) * kLog2eF);
    m = top;
}

template <int ROWS, bool MEAN>
__global__ __launch_bounds__(kJoinThreads) void join_stats_kernel(const JoinArgs a) {
    constexpr int kAhead = 16, kWaves = kJoinThreads / kWave, kSlices = kJoinThreads / ROWS;
    __shared__ float2 red[kWaves][ROWS];
    const int r = threadIdx.x % ROWS, slice = threadIdx.x / ROWS, row = blockIdx.x * ROWS + r;
    float m = -INFINITY, s = 0.0f;
    for (int p0 = slice; p0 < a.parts; p0 += kAhead * kSlices) {
        float2 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int p = p0 + k * kSlices;
            v[k] = a.stats[static_cast<int64_t>(min(p, a.parts - 1)) * a.padded + row];
            if (p >= a.parts) v[k] = make_float2(-INFINITY, 0.0f);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) top = fmaxf(top, v[k].x);
        const float ref = reference(top);
        s *= __builtin_amdgcn_exp2f((m - ref) * kLog2eF);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) s += v[k].y * __builtin_amdgcn_exp2f((v[k].x - ref) * kLog2eF);
        m = top;
    }
#pragma unroll
    for (int off = ROWS; off < kWave; off <<= 1) {
        const float m2 = __shfl_xor(m, off, kWave), s2 = __shfl_xor(s, off, kWave);
        join_sums(m, s, m2, s2);
    }
    if ((threadIdx.x & (kWave - 1)) < ROWS) red[threadIdx.x / kWave][r] = make_float2(m, s);
    __syncthreads();
    if (threadIdx.x >= kWave) return;
    constexpr int kGroups = kWave / ROWS;  // of the first wave, each with an equal part of the waves' sums
    m = red[slice][r].x;
    s = red[slice][r].y;
#pragma unroll
    for (int k = kGroups; k < kWaves; k += kGroups) {
        const float2 b = red[slice + k][r];
        join_sums(m, s, b.x, b.y);
    }
#pragma unroll
    for (int off = ROWS; off < kWave; off <<= 1) {
        const float m2 = __shfl_xor(m, off, kWave), s2 = __shfl_xor(s, off, kWave);
        join_sums(m, s, m2, s2);
    }
    if (threadIdx.x >= ROWS) return;
    const float weight = row < a.rows ? weight_of(a.weights, row) : 0.0f;
    const bool live = weight != 0.0f;
    const int target = live ? token_of(a.targets[row], a.V) : -1;
    const float logsum = logf(s);
    const float loss = !live ? 0.0f : target >= 0 ? logsum - (a.target_logits[row] - m) : NAN;
    a.shares[row] = live ? make_float2(m, 1.0f / s) : make_float2(0.0f, 0.0f);
    a.whole[row] = target;
    if (row < a.rows) a.losses[row] = loss;
    if (!MEAN || blockIdx.x > 0) return;
    double t = static_cast<double>(loss) * weight;
#pragma unroll
    for (int off = 1; off < ROWS; off <<= 1) t += __shfl_xor(t, off, ROWS);
    if (threadIdx.x == 0) a.mean[0] = static_cast<float>(t / a.rows);
}

void launch_join_stats(const JoinArgs &a, hipStream_t s) {
    if (a.mean != nullptr)
        join_stats_kernel<kMeanRows, true><<<dim3(a.padded / kMeanRows), dim3(kJoinThreads), 0, s>>>(a);
    else
        join_stats_kernel<8, false><<<dim3(a.padded / 8), dim3(kJoinThreads), 0, s>>>(a);
    hipCheck(hipGetLastError());
}

struct ShareArgs {
    const float *logits;
    const float2 *shares;  // of the rows
    const int *targets;
    hu32x4 *d, *dt;  // as first operands of d W and d^T x; either may be null
    int row_blocks, token_blocks;  // of the logits
    int rows_used, tokens_used;    // blocks that the products' reductions reach
    int per_wave;                  // blocks of tokens a wave
    MeanArgs mean;                 // by one more workgroup, unless `out` is null
};

// Shares are held times 2^15, as both products take the one copy: to 24 bits from 2^-16 on, below that to 2^-40 of a row's
// whole.  A token that is no row's target has smaller shares alone; its row of dW is off by up to 2^-40 mean |w x|, which is
// 5e-5 of it at shares of 2^-28 and all of it at 2^-42.  An AdamW step (eps 1e-8) takes that for 1e-4 |x| of the rate at
// most.  A scale for each token would need their largest share before d is written, and a copy of d for either product
// (8192 rows: shares 880 us instead of 587).
constexpr int kShareShift = 15;
constexpr int kShareStride = 36;  // words of LDS a token: 16-byte rows, no two in the same banks

// d' = exp(l - m) / sum - [target] of a block of 32 rows x 32 tokens, in two fp16 parts, as the
// operand of either product.  The logits come in the order of the accumulators: a lane holds row
// l % 32 and tokens 8 q + 4 (l / 32) + {0 .. 3}, which is also its share of d's block; d^T's goes
// through LDS.  Memory bound: 4 bytes in, 4 out for each operand (8192 rows, 50257 tokens, d alone: 575 us, 5.7 TB/s).
__global__ __launch_bounds__(kThreads) void shares_kernel(const ShareArgs a) {
    if (a.mean.out != nullptr && blockIdx.x == gridDim.x - 1) {
        if (blockIdx.y == 0) mean_loss<kThreads>(a.mean);
        return;
    }
    __shared__ uint32_t lds[4][32 * kShareStride];
    const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rb = blockIdx.y;
    const int first = (blockIdx.x * 4 + w) * a.per_wave;
    const int row = rb * 32 + l32;
    const float m = a.shares[row].x, by_sum = a.shares[row].y;
    const int target = a.targets[row];
    const bool live = by_sum != 0.0f;  // else there may be no logits
    uint32_t *mine = lds[w];
    for (int jb = first; jb < min(first + a.per_wave, a.token_blocks); ++jb) {
        const f32x4_t *x = reinterpret_cast<const f32x4_t *>(a.logits) +
                           (static_cast<int64_t>(rb) * a.token_blocks + jb) * 256 + lane;
        f32x4_t v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = x[q * 64];
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = live ? __builtin_amdgcn_exp2f((v[q][e] - m) * kLog2eF) * by_sum : 0.0f;
                v[q][e] = p - (jb * 32 + 8 * q + 4 * hf + e == target ? 1.0f : 0.0f);
            }
        uint32_t high[4][2], low[4][2];
        constexpr float kUp = static_cast<float>(1 << kShareShift);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            halves_split(v[q][0] * kUp, v[q][1] * kUp, high[q][0], low[q][0]);
            halves_split(v[q][2] * kUp, v[q][3] * kUp, high[q][1], low[q][1]);
        }
        if (a.d != nullptr && jb < a.tokens_used) {
            const uint32_t flip = halves_negated(jb * 32) ? 0x80008000u : 0;
            hu32x4 *out = a.d + (static_cast<int64_t>(rb) * a.tokens_used + jb) * 256 + lane;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                out[(2 * k) * 64] = hu32x4{high[2 * k][0], high[2 * k][1], high[2 * k + 1][0], high[2 * k + 1][1]} ^ flip;
                out[(2 * k + 1) * 64] = hu32x4{low[2 * k][0], low[2 * k][1], low[2 * k + 1][0], low[2 * k + 1][1]} ^ flip;
            }
        }
        if (a.dt == nullptr || rb >= a.rows_used) continue;
        const uint32_t flip = halves_negated(rb * 32) ? 0x80008000u : 0;
#pragma unroll
        for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                uint32_t *at = mine + (8 * q + 4 * hf + 2 * e) * kShareStride + l32;
                at[0] = ((high[q][e] & 0xffffu) | (low[q][e] << 16)) ^ flip;
                at[kShareStride] = ((high[q][e] >> 16) | (low[q][e] & 0xffff0000u)) ^ flip;
            }
        wave_lds_order();
        hu32x4 *out = a.dt + (static_cast<int64_t>(jb) * a.rows_used + rb) * 256 + lane;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const hu32x4 *at = reinterpret_cast<const hu32x4 *>(mine + l32 * kShareStride + 16 * k + 4 * hf);
            const hu32x4 one = at[0], two = at[2];
            const uint32_t word[8] = {one[0], one[1], one[2], one[3], two[0], two[1], two[2], two[3]};
            hu32x4 hi, lo;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                hi[e] = (word[2 * e] & 0xffffu) | (word[2 * e + 1] << 16);
                lo[e] = (word[2 * e] >> 16) | (word[2 * e + 1] & 0xffff0000u);
            }
            out[(2 * k) * 64] = hi;
            out[(2 * k + 1) * 64] = lo;
        }
        wave_lds_order();
    }
}

void launch_shares(ShareArgs a, hipStream_t s) {
    // Four blocks a wave, fewer where that leaves less than eight waves a CU.
    const int64_t blocks = static_cast<int64_t>(a.row_blocks) * a.token_blocks;
    a.per_wave = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(4, blocks / 2048)));
    const int per = 4 * a.per_wave;
    const int across = (a.token_blocks + per - 1) / per + (a.mean.out != nullptr);
    shares_kernel<<<dim3(across, a.row_blocks), dim3(kThreads), 0, s>>>(a);
    hipCheck(hipGetLastError());
}

constexpr int kPastEnd = 8192;  // bytes behind an operand that products across may read

// Blocks of the pool for the length of a call.
struct Scratch {
    static constexpr int kMax = 24;
    void *blocks[kMax];
    int n = 0;
    template <typename T>
    T *take(int64_t count) {
        CHECK_ERROR(n == kMax, "Too many blocks of scratch.");
        blocks[n] = alloc_cuda(static_cast<size_t>(std::max<int64_t>(count, 1)) * sizeof(T));
        return static_cast<T *>(blocks[n++]);
    }
    Halves halves(int rows, int terms) {
        Halves h{nullptr, nullptr, 0, rows, terms};
        h.data = take<hu32x4>((h.bytes() + kPastEnd) / 16);
        h.shift = take<int>(h.row_blocks() * 32);
        return h;
    }
    void release() {
        while (n > 0) free_cuda(blocks[--n]);
    }
};

constexpr int64_t kPieceBytes = 5ll << 28;  // logits and d of a piece
constexpr int kLossPiece = 16384;           // rows of a piece whose logits are not written

void run_halves(const HeadLoss &h, hipStream_t s) {
    const bool grad = h.dx != nullptr || h.dW != nullptr;
    const int tokens = (h.V + 127) / 128 * 128;
    const int64_t fit = std::max<int64_t>(1, kPieceBytes / (8ll * tokens) / 128) * 128;
    const int piece = static_cast<int>(std::min<int64_t>(h.rows, grad ? fit : kLossPiece));
    const int padded = (piece + 127) / 128 * 128;
    Scratch scratch;
    Halves x = scratch.halves(piece, h.C), xt{}, d{nullptr, nullptr, kShareShift, piece, h.V};
    uint32_t *largest_x = scratch.take<uint32_t>(h.C);  // magnitudes of x's columns
    launch_halves_rows(h.x, h.weights, x, largest_x, h.C, s);
    // W is held by a shift for 64 rows each, as its rows are the terms of dx, whose product takes 64 of them at a time: to
    // 2^-40 of their largest value where it is below the 2^-17th of that, which counts for features of dx that small.  Laid
    // out by rows and, for dx, a second time by columns it would be held to 2^-40 of each row's and column's largest, and
    // cost 171 us instead of 69 (50257 x 768) and 371 instead of 166 (50257 x 1600).
    const Halves W = scratch.halves(h.V, h.C);
    launch_halves_table(h.W, W, s);
    if (h.dW != nullptr) {
        xt = scratch.halves(h.C, piece);
        launch_column_largest(h.x, h.C, h.weights, static_cast<float>(h.rows), h.rows, h.C, largest_x, s);
    }
    if (grad) d.data = scratch.take<hu32x4>((d.bytes() + kPastEnd) / 16);
    float *logits = grad ? scratch.take<float>(static_cast<int64_t>(padded) * tokens) : nullptr;
    float2 *stats = scratch.take<float2>(static_cast<int64_t>(padded) * (tokens / 64));
    int *targets = scratch.take<int>(padded);
    float *target_logits = scratch.take<float>(padded);
    float2 *shares = scratch.take<float2>(padded);
    for (int r = 0; r < h.rows; r += piece) {
        const int n = std::min(piece, h.rows - r), n_padded = (n + 127) / 128 * 128;
        const float *xr = h.x + static_cast<int64_t>(r) * h.C;
        const float *weights = h.weights != nullptr ? h.weights + r : nullptr;
        x.rows = d.rows = xt.terms = n;
        if (r > 0) launch_halves_rows(xr, weights, x, nullptr, 0, s);
        const int part = launch_logits(
            W, x, {logits, stats, h.targets + r, target_logits, h.V, n, tokens / 32, n_padded}, s);
        launch_join_stats({stats, tokens / part, h.targets + r, target_logits, weights, shares, targets, h.losses + r,
                           n, n_padded, h.V, nullptr},
                          s);
        if (!grad) continue;
        const ShareArgs a{logits, shares, targets, d.data, nullptr, n_padded / 32, tokens / 32, 0,
                          (h.V + 63) / 64 * 2, 0, {h.losses, h.weights, r + piece >= h.rows ? h.mean : nullptr, h.rows}};
        launch_shares(a, s);
        if (h.dx != nullptr)
            launch_product_across_b(d, W, {h.dx + static_cast<int64_t>(r) * h.C, h.C, weights,
                                          static_cast<float>(h.rows), false},
                                  s);
        if (h.dW != nullptr) {
            launch_halves_columns(xr, h.C, weights, static_cast<float>(h.rows), xt, true, largest_x, s);
            launch_product_across_a(d, xt, {h.dW, h.C, nullptr, 1.0f, h.add || r > 0}, s);
        }
    }
    if (!grad) launch_mean(h, s);
    scratch.release();
}

// ---- few rows: W as it comes (head_few.hip) ----

void run_few(const HeadLoss &h, hipStream_t s) {
    const bool grad = h.dx != nullptr || h.dW != nullptr;
    const int tokens = (h.V + 127) / 128 * 128;
    // Blocks of 32 rows; dt's terms are whole pairs of them, whose second one may hold no row and have no logits.
    const int own = few_row_blocks(h.rows), blocks = std::max(own, h.dW != nullptr ? 2 : 1), padded = blocks * 32;
    Scratch scratch;
    FewRows x{nullptr, scratch.take<int>(padded), 0, own, h.C}, d{nullptr, nullptr, kShareShift, own, tokens};
    x.data = scratch.take<hu32x4>(x.bytes() / 16);
    uint32_t *largest = scratch.take<uint32_t>(h.C);  // of x's columns
    launch_few_rows(h.x, h.weights, h.rows, x, largest, h.C, s);
    float *logits = grad ? scratch.take<float>(static_cast<int64_t>(padded) * tokens) : nullptr;
    float2 *stats = scratch.take<float2>(static_cast<int64_t>(padded) * (tokens / 32));
    int *targets = scratch.take<int>(padded);
    float *target_logits = scratch.take<float>(padded);
    float2 *shares = scratch.take<float2>(padded);
    const int part = launch_few_logits(
        h.W, h.V, h.C, x, {logits, stats, h.targets, target_logits, h.V, h.rows, tokens / 32, padded}, s);
    const bool mean = h.rows <= kMeanRows;
    launch_join_stats({stats, tokens / part, h.targets, target_logits, h.weights, shares, targets, h.losses, h.rows,
                       padded, h.V, mean ? h.mean : nullptr},
                      s);
    if (!grad && !mean) launch_mean(h, s);
    if (grad) {
        Halves dt{nullptr, nullptr, kShareShift, h.V, h.rows}, xt{};
        if (h.dx != nullptr) d.data = scratch.take<hu32x4>(d.bytes() / own * blocks / 16);
        if (h.dW != nullptr) dt.data = scratch.take<hu32x4>(dt.bytes() / 16);
        launch_shares({logits, shares, targets, d.data, dt.data, blocks, tokens / 32, dt.term_blocks() / 2,
                       tokens / 32, 0, {h.losses, h.weights, mean ? nullptr : h.mean, h.rows}},
                      s);
        if (h.dx != nullptr)
            launch_few_dx(d, h.W, h.V, h.C, h.rows,
                          {h.dx, h.C, h.weights, static_cast<float>(h.rows), false}, s);
        if (h.dW != nullptr) {
            xt = scratch.halves(h.C, h.rows);
            if (h.rows <= kColumnTerms) {
                launch_halves_columns(h.x, h.C, h.weights, static_cast<float>(h.rows), xt, false, nullptr, s);
            } else {
                launch_column_largest(h.x, h.C, h.weights, static_cast<float>(h.rows), h.rows, h.C, largest, s);
                launch_halves_columns(h.x, h.C, h.weights, static_cast<float>(h.rows), xt, false, largest, s);
            }
            if (h.rows <= kFewDwTerms)
                launch_few_dw(dt, xt, {h.dW, h.C, nullptr, 1.0f, h.add}, s);
            else
                launch_halves_product(dt, xt, {h.dW, h.C, nullptr, 1.0f, h.add}, s);
        }
    }
    scratch.release();
}

// Whether W is read as it comes, again for every 128 rows and with a split of each float, instead of laid out first.
// A row of products costs more there (the split, W again), the call less (W's layout, wider launches).  us as it comes / laid
// out, features x vocabulary: rows (taken from 900 sizes of 16 to 1600 x 128 to 130000, 96 to 4096 rows, all with both ways:
// the rule's side is the quicker one or within 3 % of it for 871 of them, within 12 % for all, at a mean of 0.2 %).
// With gradients, up to 240 rows and 1.6e9 / (V (C + 500)) more:
//   768 x 50257   96: 179 / 227    200: 320 / 312    384: 476 / 405
//   200 x 50257  200: 152 / 166    384: 206 / 202    512: 267 / 239
//   16 x 50257   200: 104 / 122    384: 129 / 142    512: 168 / 168    640: 218 / 192
//   768 x 5003   384: 84 / 89      512: 107 / 98     768: 128 / 114
//   200 x 5003   384: 60 / 63      640: 74 / 76      768: 83 / 81      1024: 92 / 88
//   768 x 1000   1024: 83 / 96     1280: 87 / 91     1536: 102 / 98
//   200 x 1000   2048: 62 / 67     2944: 73 / 76     4096: 86 / 82
// and 2^21 values of x, past which dx takes W again too often:
//   768 x 300    1536: 75 / 79     2048: 80 / 82     2944: 105 / 91    4096: 134 / 99
//   768 x 128    1536: 75 / 77     2048: 78 / 78     2944: 91 / 84
// The loss alone, up to 512 rows and 5e9 / (V (C + 4)) more:
//   768 x 50257  512: 184 / 195    640: 215 / 217    768: 269 / 248
//   200 x 50257  512: 74 / 79      768: 100 / 98     1024: 127 / 119
//   64 x 50257   1024: 64 / 68     1280: 74 / 73     2048: 112 / 107   2944: 156 / 138
//   16 x 50257   2944: 112 / 126   4096: 149 / 164
//   768 x 5003   1024: 55 / 55     1536: 66 / 66     2048: 90 / 82
//   200 x 5003   2048: 40 / 40     2944: 49 / 48     4096: 60 / 62
//   1600 x 1000  2048: 60 / 79     2944: 78 / 85     4096: 86 / 92
bool few_rows(int rows, int V, int C, bool grad) {
    const int64_t read = (rows + 127) / 128 * 128, values = static_cast<int64_t>(rows) * C;
    if (rows > 4096 || values >= 1 << 28) return false;  // offsets of 32 bits, and no size past 4096 that was measured
    if (!grad) return read <= 512 + 5000000000 / (V * (C + 4ll));
    return rows <= 128 || (read <= 240 + 1600000000 / (V * (C + 500ll)) && values <= 1 << 21);
}

}  // namespace

}  // namespace gptc

using namespace gptc;

extern "C" void gptc_linear_cross_entropy_cuda(const tensor_t *x, const tensor_t *W, const tensor_t *targets,
                                               const tensor_t *weights, tensor_t *output, tensor_t *row_losses,
                                               tensor_t *dx, tensor_t *dW, const int accumulate) {
    check_gpu(x, "x");
    check_gpu(W, "W");
    check_gpu(targets, "targets");
    check_gpu(output, "output");
    CHECK_ERROR(W->ndims != 2, "Expected W to be (vocabulary, features), but got %d dims.", W->ndims);
    const int V = W->shape[0], C = W->shape[1];
    CHECK_ERROR(V < 1 || V >= kMaxVocabulary || C < 1 || C >= kMaxVocabulary,
                "Expected W to be up to %d on either side, but got %d x %d.", kMaxVocabulary - 1, V, C);
    CHECK_ERROR(last_dim(x) != C, "Expected x's last dimension to be %d, but got %d.", C, last_dim(x));
    const int rows = x->length / C;
    CHECK_ERROR(rows < 1, "Expected at least one row of x.");
    CHECK_ERROR(rows > kMaxRows, "Expected up to %d rows of x, but got %d.", kMaxRows, rows);
    CHECK_ERROR(targets->length != rows, "Expected %d targets, but got %d.", rows, targets->length);
    CHECK_ERROR(output->length < 1, "Expected output to hold the loss.");
    const tensor_t *in[4] = {x, W, targets, weights};
    const tensor_t *out[4] = {output, row_losses, dx, dW};
    if (weights != NULL) {
        check_gpu(weights, "weights");
        CHECK_ERROR(weights->length != rows, "Expected %d weights, but got %d.", rows, weights->length);
    }
    if (row_losses != NULL) {
        check_gpu(row_losses, "row_losses");
        CHECK_ERROR(row_losses->length != rows, "Expected row_losses to hold %d elements, but it holds %d.", rows,
                    row_losses->length);
    }
    if (dx != NULL) {
        check_gpu(dx, "dx");
        CHECK_ERROR(dx->length != x->length, "Expected dx to match x's %d elements, but got %d.", x->length, dx->length);
    }
    if (dW != NULL) {
        check_gpu(dW, "dW");
        CHECK_ERROR(dW->length != W->length, "Expected dW to match W's %d elements, but got %d.", W->length, dW->length);
    }
    for (int i = 0; i < 4; ++i)
        for (int j = 0; j < 4 && out[i] != NULL; ++j) {
            CHECK_ERROR(in[j] != NULL && overlap(out[i], in[j]), "Results may not overlap another tensor of the call.");
            CHECK_ERROR(j != i && out[j] != NULL && overlap(out[i], out[j]),
                        "Results may not overlap another tensor of the call.");
        }
    CHECK_ERROR(gptc_stream_capturing(), "gptc_linear_cross_entropy_cuda takes scratch: not under graph capture.");
    hipStream_t s = gptc_stream_checked();
    float *losses = row_losses != NULL ? row_losses->t : static_cast<float *>(alloc_cuda(sizeof(float) * rows));
    const HeadLoss h{x->t, W->t, targets->t, weights != NULL ? weights->t : nullptr, losses, output->t,
                     dx != NULL ? dx->t : nullptr, dW != NULL ? dW->t : nullptr, rows, V, C, accumulate != 0};
    if (few_rows(rows, V, C, dx != NULL || dW != NULL))
        run_few(h, s);
    else
        run_halves(h, s);
    if (row_losses == NULL) free_cuda(losses);
}
