// Cross entropy of softmax(x W^T) and its gradients without keeping the logits.
// No counterpart in gpt.c, whose GPT2 keeps the logits, their log-softmax and
// their gradient (src/transformer.c:69-158, src/loss.c:19-148):
//   l[r, j] = x[r] . W[j],  lse[r] = log sum_j exp l[r, j],  loss[r] = lse[r] - l[r, t[r]],
//   d[r, j] = w[r] / R (exp(l[r, j] - lse[r]) - [j = t[r]]),  dx = d W,  dW (+)= d^T x.
// The rows go through in pieces, so that a piece's logits fit the scratch: its
// logits are formed once, turned into d, and used for both gradients.
#include <algorithm>
#include "gemm_halves.hpp"
#include "gemm_split.hpp"
#include "gpu_kernels.h"
#include "ops_common.hpp"

namespace gptc {

namespace {

constexpr int kThreads = 256;
constexpr int kRowThreads = 512;
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int64_t kPieceFloats = 1ll << 27;  // logits of a piece
constexpr int kHalvesRows = 128;             // from here on the operands are laid out first
constexpr int kMaxVocabulary = 1 << 22;      // a product's tile offsets fit 32 bits

__device__ __forceinline__ float weight_of(const float *weights, int row) {
    return weights != nullptr ? weights[row] : 1.0f;
}

// One row a workgroup: its loss, and with `grad` its logits become d.
__global__ __launch_bounds__(kRowThreads) void loss_row_kernel(float *__restrict__ logits,
                                                              const float *__restrict__ targets,
                                                              const float *__restrict__ weights,
                                                              float *__restrict__ losses, int V, float rows,
                                                              bool grad) {
    __shared__ float sm[kRowWaves], ss[kRowWaves];
    const int row = blockIdx.x;
    float *x = logits + static_cast<int64_t>(row) * V;
    const float weight = weight_of(weights, row);
    if (weight == 0.0f) {
        if (threadIdx.x == 0) losses[row] = 0.0f;
        if (grad)
            for (int j = threadIdx.x; j < V; j += kRowThreads) x[j] = 0.0f;
        return;
    }
    float m = -INFINITY, s = 0.0f;
    for (int j = threadIdx.x; j < V; j += kRowThreads) {
        const float v = x[j];
        if (v > m) {
            s = s * expf(m - v) + 1.0f;
            m = v;
        } else if (v != -INFINITY) {
            s += expf(v - m);
        }
    }
    wave_online(m, s);
    const int w = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) {
        sm[w] = m;
        ss[w] = s;
    }
    __syncthreads();
    m = sm[0];
    s = ss[0];
#pragma unroll
    for (int i = 1; i < kRowWaves; ++i) online_merge(m, s, sm[i], ss[i]);
    const float logsum = logf(s);
    const int t = token_of(targets[row], V);
    if (threadIdx.x == 0) losses[row] = t >= 0 ? logsum - (x[t] - m) : NAN;
    if (!grad) return;
    __syncthreads();  // the target's logit has been read
    const float factor = weight / rows;
    for (int j = threadIdx.x; j < V; j += kRowThreads) x[j] = factor * (expf(x[j] - m - logsum) - (j == t ? 1.0f : 0.0f));
}

// out[0] = sum of w[r] loss[r] / rows in a fixed order, in 64 bits.
constexpr int kMeanThreads = 1024;
__global__ __launch_bounds__(kMeanThreads) void mean_loss_kernel(const float *__restrict__ losses,
                                                                const float *__restrict__ weights,
                                                                float *__restrict__ out, int rows) {
    __shared__ double part[kMeanThreads / kWave];
    double t = 0.0;
#pragma unroll 8
    for (int r = threadIdx.x; r < rows; r += kMeanThreads)
        t += static_cast<double>(losses[r]) * weight_of(weights, r);  // rows of weight 0: 0 * 0
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) t += __shfl_xor(t, off, kWave);
    if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = t;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int i = 1; i < kMeanThreads / kWave; ++i) t += part[i];
    out[0] = static_cast<float>(t / rows);
}

// y = x with rows of weight 0 as zeros.
__global__ __launch_bounds__(kThreads) void live_rows_kernel(const float *__restrict__ x,
                                                            const float *__restrict__ weights, float *__restrict__ y,
                                                            int C) {
    const int row = blockIdx.x;
    const int64_t base = static_cast<int64_t>(row) * C;
    const bool live = weights[row] != 0.0f;
    for (int c = threadIdx.x; c < C; c += kThreads) y[base + c] = live ? x[base + c] : 0.0f;
}

struct HeadLoss {
    const float *x, *W, *targets, *weights;
    float *losses, *dx, *dW;
    int rows, V, C;
    bool add;
};

// ---- many rows: products of operands laid out as two fp16 parts ----

// A row's loss, lse and target from the parts of its tokens: 32 rows a workgroup, whose
// 32 slices of the parts are joined in order.  Rows that take no part, those past the
// last one among them: lse is infinite, which makes their shares 0, and the target -1.
constexpr int kJoinThreads = 1024;
__global__ __launch_bounds__(kJoinThreads) void join_stats_kernel(const float2 *__restrict__ stats, int parts,
                                                                 const float *__restrict__ targets,
                                                                 const float *__restrict__ target_logits,
                                                                 const float *__restrict__ weights,
                                                                 float *__restrict__ lse, int *__restrict__ whole,
                                                                 float *__restrict__ losses, int rows, int padded,
                                                                 int V) {
    constexpr int kAhead = 8;
    __shared__ float2 red[32][33];
    const int r = threadIdx.x & 31, slice = threadIdx.x >> 5, row = blockIdx.x * 32 + r;
    const int per = (parts + 31) / 32, end = min(parts, (slice + 1) * per);
    float m = -INFINITY, s = 0.0f;
    for (int p0 = slice * per; p0 < end; p0 += kAhead) {
        float2 v[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            v[k] = stats[static_cast<int64_t>(min(p0 + k, end - 1)) * padded + row];
            if (p0 + k >= end) v[k] = make_float2(-INFINITY, 0.0f);
        }
        float top = m;
#pragma unroll
        for (int k = 0; k < kAhead; ++k) top = fmaxf(top, v[k].x);
        if (top == -INFINITY) continue;  // nothing but parts without a logit
        s *= expf(m - top);
#pragma unroll
        for (int k = 0; k < kAhead; ++k) s += v[k].y * expf(v[k].x - top);
        m = top;
    }
    red[slice][r] = make_float2(m, s);
    __syncthreads();
    if (slice != 0) return;
    for (int i = 1; i < 32; ++i) online_merge(m, s, red[i][r].x, red[i][r].y);
    const bool live = row < rows && weight_of(weights, row) != 0.0f;
    const int target = live ? token_of(targets[row], V) : -1;
    const float logsum = logf(s);
    lse[row] = live ? m + logsum : INFINITY;
    whole[row] = target;
    if (row < rows) losses[row] = !live ? 0.0f : target >= 0 ? logsum - (target_logits[row] - m) : NAN;
}

struct ShareArgs {
    const float *logits, *lse;
    const int *targets;
    hu32x4 *d, *dt;  // as first operands of d W and d^T x; either may be null
    int row_blocks, token_blocks;  // of the logits
    int rows_used, tokens_used;    // blocks that the products' reductions reach
};

constexpr int kShareShift = 15;  // shares are held times 2^15
constexpr float kLog2eF = 1.4426950408889634f;
constexpr int kShareStride = 36;  // words of LDS a token: 16-byte rows, no two in the same banks
constexpr int kShareTokens = 4;   // blocks of 32 tokens a wave

// d' = exp(l - lse) - [target] of a block of 32 rows x 32 tokens, in two fp16 parts, as the
// operand of either product.  The logits come in the order of the accumulators: a lane holds row
// l % 32 and tokens 8 q + 4 (l / 32) + {0 .. 3}, which is also its share of d's block; d^T's goes
// through LDS.  Memory bound: 4 bytes in, 8 out.
__global__ __launch_bounds__(kThreads) void shares_kernel(const ShareArgs a) {
    __shared__ uint32_t lds[4][32 * kShareStride];
    const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int rb = blockIdx.y;
    const int first = (blockIdx.x * 4 + w) * kShareTokens;
    const int row = rb * 32 + l32;
    const float lse = a.lse[row];
    const int target = a.targets[row];
    uint32_t *mine = lds[w];
    for (int jb = first; jb < min(first + kShareTokens, a.token_blocks); ++jb) {
        const f32x4_t *x = reinterpret_cast<const f32x4_t *>(a.logits) +
                           (static_cast<int64_t>(rb) * a.token_blocks + jb) * 256 + lane;
        f32x4_t v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = x[q * 64];
        uint32_t high[4][2], low[4][2];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float d[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float p = __builtin_amdgcn_exp2f((v[q][e] - lse) * kLog2eF);
                d[e] = (p - (jb * 32 + 8 * q + 4 * hf + e == target ? 1.0f : 0.0f)) *
                       static_cast<float>(1 << kShareShift);
            }
            halves_split(d[0], d[1], high[q][0], low[q][0]);
            halves_split(d[2], d[3], high[q][1], low[q][1]);
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
        h.data = take<hu32x4>(h.bytes() / 16);
        h.shift = take<int>(h.row_blocks() * 32);
        return h;
    }
    void release() {
        while (n > 0) free_cuda(blocks[--n]);
    }
};

constexpr int64_t kPieceBytes = 5ll << 28;  // logits, d and d^T of a piece
constexpr int kLossPiece = 16384;           // rows of a piece whose logits are not written

void run_halves(const HeadLoss &h, hipStream_t s) {
    const bool grad = h.dx != nullptr || h.dW != nullptr;
    const int tokens = (h.V + 127) / 128 * 128;
    const int64_t fit = std::max<int64_t>(1, kPieceBytes / (12ll * tokens) / 128) * 128;
    const int piece = static_cast<int>(std::min<int64_t>(h.rows, grad ? fit : kLossPiece));
    const int padded = (piece + 127) / 128 * 128;
    Scratch scratch;
    const Halves W = scratch.halves(h.V, h.C);
    launch_halves_rows(h.W, h.C, nullptr, W, true, s);
    // The largest magnitudes of the columns of W and x.
    uint32_t *largest = scratch.take<uint32_t>(2 * h.C), *largest_x = largest + h.C;
    if (grad) launch_zero_words(largest, 2 * h.C, s);
    Halves Wt{};
    if (h.dx != nullptr) {
        Wt = scratch.halves(h.C, h.V);
        launch_column_largest(h.W, h.C, nullptr, 1.0f, h.V, h.C, largest, s);
        launch_halves_columns(h.W, h.C, nullptr, 1.0f, Wt, largest, s);
    }
    Halves x = scratch.halves(piece, h.C), xt{}, d{nullptr, nullptr, kShareShift, piece, h.V},
           dt{nullptr, nullptr, kShareShift, h.V, piece};
    if (h.dW != nullptr) {
        xt = scratch.halves(h.C, piece);
        dt.data = scratch.take<hu32x4>(dt.bytes() / 16);
        launch_column_largest(h.x, h.C, h.weights, static_cast<float>(h.rows), h.rows, h.C, largest_x, s);
    }
    if (h.dx != nullptr) d.data = scratch.take<hu32x4>(d.bytes() / 16);
    float *logits = grad ? scratch.take<float>(static_cast<int64_t>(padded) * tokens) : nullptr;
    float2 *stats = scratch.take<float2>(static_cast<int64_t>(padded) * (tokens / 64));
    int *targets = scratch.take<int>(padded);
    float *target_logits = scratch.take<float>(padded), *lse = scratch.take<float>(padded);
    for (int r = 0; r < h.rows; r += piece) {
        const int n = std::min(piece, h.rows - r), n_padded = (n + 127) / 128 * 128;
        const float *xr = h.x + static_cast<int64_t>(r) * h.C;
        const float *weights = h.weights != nullptr ? h.weights + r : nullptr;
        x.rows = d.rows = xt.terms = dt.terms = n;
        launch_halves_rows(xr, h.C, weights, x, false, s);
        const int part = launch_logits(
            W, x, {logits, stats, h.targets + r, target_logits, h.V, n, tokens / 32, n_padded}, s);
        join_stats_kernel<<<dim3(n_padded / 32), dim3(kJoinThreads), 0, s>>>(
            stats, tokens / part, h.targets + r, target_logits, weights, lse, targets, h.losses + r, n, n_padded, h.V);
        hipCheck(hipGetLastError());
        if (!grad) continue;
        const ShareArgs a{logits, lse, targets, d.data, dt.data, n_padded / 32, tokens / 32, (n + 63) / 64 * 2, (h.V + 63) / 64 * 2};
        shares_kernel<<<dim3((a.token_blocks + 4 * kShareTokens - 1) / (4 * kShareTokens), a.row_blocks),
                        dim3(kThreads), 0, s>>>(a);
        hipCheck(hipGetLastError());
        if (h.dx != nullptr)
            launch_halves_product(d, Wt, {h.dx + static_cast<int64_t>(r) * h.C, h.C, weights,
                                          static_cast<float>(h.rows), false},
                                  s);
        if (h.dW != nullptr) {
            launch_halves_columns(xr, h.C, weights, static_cast<float>(h.rows), xt, largest_x, s);
            launch_halves_product(dt, xt, {h.dW, h.C, nullptr, 1.0f, h.add || r > 0}, s);
        }
    }
    scratch.release();
}

// ---- few rows: products that split the floats as they come ----

void run_pieces(const HeadLoss &h, hipStream_t s) {
    const bool grad = h.dx != nullptr || h.dW != nullptr;
    const int64_t fit = std::max<int64_t>(1, kPieceFloats / h.V);
    const int piece = static_cast<int>(std::min<int64_t>(h.rows, fit));
    float *logits = static_cast<float *>(alloc_cuda(sizeof(float) * static_cast<size_t>(piece) * h.V));
    const float *x = h.x;
    float *live = nullptr;
    if (h.weights != nullptr) {
        live = static_cast<float *>(alloc_cuda(sizeof(float) * static_cast<size_t>(h.rows) * h.C));
        live_rows_kernel<<<dim3(h.rows), dim3(kThreads), 0, s>>>(h.x, h.weights, live, h.C);
        hipCheck(hipGetLastError());
        x = live;
    }
    for (int r = 0; r < h.rows; r += piece) {
        const int n = std::min(piece, h.rows - r);
        const float *xr = x + static_cast<int64_t>(r) * h.C;
        launch_split_gemm({xr, h.W, logits, nullptr, nullptr, n, h.V, h.C, h.C, h.C, h.V, false, true}, s);
        loss_row_kernel<<<dim3(n), dim3(kRowThreads), 0, s>>>(
            logits, h.targets + r, h.weights != nullptr ? h.weights + r : nullptr, h.losses + r, h.V,
            static_cast<float>(h.rows), grad);
        hipCheck(hipGetLastError());
        if (h.dx != nullptr)
            launch_split_gemm({logits, h.W, h.dx + static_cast<int64_t>(r) * h.C, nullptr, nullptr, n, h.C, h.V, h.V, h.C,
                               h.C, false, false},
                              s);
        if (h.dW != nullptr)
            launch_split_gemm({logits, xr, h.dW, nullptr, h.add || r > 0 ? h.dW : nullptr, h.V, h.C, n, h.V, h.C, h.C,
                               true, false},
                              s);
    }
    free_cuda(live);
    free_cuda(logits);
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
    const HeadLoss h{x->t, W->t, targets->t, weights != NULL ? weights->t : nullptr, losses, dx != NULL ? dx->t : nullptr,
                     dW != NULL ? dW->t : nullptr, rows, V, C, accumulate != 0};
    if (rows >= kHalvesRows)
        run_halves(h, s);
    else
        run_pieces(h, s);
    mean_loss_kernel<<<dim3(1), dim3(kMeanThreads), 0, s>>>(losses, weights != NULL ? weights->t : nullptr, output->t, rows);
    hipCheck(hipGetLastError());
    if (row_losses == NULL) free_cuda(losses);
}
