// Cross entropy of softmax(x W^T) and its gradients without keeping the logits.
// No counterpart in gpt.c, whose GPT2 keeps the logits, their log-softmax and
// their gradient (src/transformer.c:69-158, src/loss.c:19-148):
//   l[r, j] = x[r] . W[j],  lse[r] = log sum_j exp l[r, j],  loss[r] = lse[r] - l[r, t[r]],
//   d[r, j] = w[r] / R (exp(l[r, j] - lse[r]) - [j = t[r]]),  dx = d W,  dW (+)= d^T x.
// The rows go through in pieces, so that a piece's logits fit the scratch: its
// logits are formed once, turned into d, and used for both gradients.
#include <algorithm>
#include "gemm_split.hpp"
#include "gpu_kernels.h"
#include "ops_common.hpp"

namespace gptc {

namespace {

constexpr int kThreads = 256;
constexpr int kRowThreads = 512;
constexpr int kRowWaves = kRowThreads / kWave;
constexpr int64_t kPieceFloats = 1ll << 27;  // logits of a piece
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
    const float f = targets[row];
    const int t = f > -1.0f && f < static_cast<float>(V) ? static_cast<int>(f) : -1;
    if (threadIdx.x == 0) losses[row] = t >= 0 ? logsum - (x[t] - m) : NAN;
    if (!grad) return;
    __syncthreads();  // the target's logit has been read
    const float factor = weight / rows;
    for (int j = threadIdx.x; j < V; j += kRowThreads) x[j] = factor * (expf(x[j] - m - logsum) - (j == t ? 1.0f : 0.0f));
}

// out[0] = sum of w[r] loss[r] / rows in a fixed order, in 64 bits.
__global__ __launch_bounds__(kThreads) void mean_loss_kernel(const float *__restrict__ losses,
                                                            const float *__restrict__ weights, float *__restrict__ out,
                                                            int rows) {
    __shared__ double part[kThreads];
    double t = 0.0;
    for (int r = threadIdx.x; r < rows; r += kThreads)
        t += static_cast<double>(losses[r]) * weight_of(weights, r);  // rows of weight 0: 0 * 0
    part[threadIdx.x] = t;
    __syncthreads();
    for (int off = kThreads / 2; off > 0; off >>= 1) {
        if (static_cast<int>(threadIdx.x) < off) part[threadIdx.x] += part[threadIdx.x + off];
        __syncthreads();
    }
    if (threadIdx.x == 0) out[0] = static_cast<float>(part[0] / rows);
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
    run_pieces({x->t, W->t, targets->t, weights != NULL ? weights->t : nullptr, losses, dx != NULL ? dx->t : nullptr,
                dW != NULL ? dW->t : nullptr, rows, V, C, accumulate != 0},
               s);
    mean_loss_kernel<<<dim3(1), dim3(kThreads), 0, s>>>(losses, weights != NULL ? weights->t : nullptr, output->t, rows);
    hipCheck(hipGetLastError());
    if (row_losses == NULL) free_cuda(losses);
}
