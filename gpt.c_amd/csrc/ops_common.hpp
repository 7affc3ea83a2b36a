// Shared pieces of the model-op kernels (Linear, LayerNorm, GELU, Softmax,
// CrossEntropy, Embedding, AdamW): 64-lane wave reductions, launch sizing
// and the host-side tensor checks every entry point runs before a launch.
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>
#include "hip_check.hpp"
#include "tensor.h"
#include "utils.h"
#include "wave_reduce.hpp"

namespace gptc {

typedef float f32x4_t __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;

// Online (max, sum of exp(x - max)) pair merge; an empty side has m = -inf, s = 0.
__device__ __forceinline__ void online_merge(float &m, float &s, float m2, float s2) {
    const float mn = fmaxf(m, m2);
    if (mn == -INFINITY) return;  // both empty
    s = s * expf(m - mn) + s2 * expf(m2 - mn);
    m = mn;
}

__device__ __forceinline__ void wave_online(float &m, float &s) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
        const float m2 = __shfl_xor(m, off, kWave), s2 = __shfl_xor(s, off, kWave);
        online_merge(m, s, m2, s2);
    }
}

// Workgroups for a grid-stride loop over `work` items of `per_block` each,
// capped at 8 workgroups per CU of a 256-CU MI355X.
inline int blocks_for(int64_t work, int64_t per_block) {
    int64_t g = (work + per_block - 1) / per_block;
    if (g > 256 * 8) g = 256 * 8;
    return g < 1 ? 1 : static_cast<int>(g);
}

inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline bool overlap(const tensor_t *a, const tensor_t *b) {
    const auto x = reinterpret_cast<uintptr_t>(a->t), y = reinterpret_cast<uintptr_t>(b->t);
    return x < y + 4 * static_cast<uintptr_t>(b->length) && y < x + 4 * static_cast<uintptr_t>(a->length);
}

inline void check_gpu(const tensor_t *t, const char *name) {
    CHECK_ERROR(t == NULL, "missing tensor argument `%s` (NULL).", name);
    CHECK_ERROR(t->device != CUDA, "Expected %s to be a tensor on the GPU.", name);
    CHECK_ERROR(t->length > 0 && t->t == NULL, "%s has no device data.", name);
}

// Product of all dimensions but the last (the row count of a (..., C) tensor).
inline int leading_rows(const tensor_t *t) {
    int64_t r = 1;
    for (int i = 0; i + 1 < t->ndims; i++) r *= t->shape[i];
    return static_cast<int>(r);
}

inline int last_dim(const tensor_t *t) { return t->ndims > 0 ? t->shape[t->ndims - 1] : 1; }

// out[c] += sum over p < parts of partial[p * cols + c], added in a fixed
// order (deterministic), and with out2 the same of the next `parts` rows of
// partial into out2; defined in linear.hip.
void launch_add_column_partials(const float *partial, float *out, int parts, int cols, hipStream_t s,
                                float *out2 = nullptr);
// y (rows x cols) += b per column; out[c] += the column sums of g (rows x
// cols), in a fixed order.  Defined in linear.hip.
void launch_bias_add(float *y, const float *b, int64_t rows, int cols, hipStream_t s);
void launch_column_sum_add(const float *g, float *out, int rows, int cols, hipStream_t s);

// attention_decode_cuda_kernel over a caller-owned partials buffer, with
// the position from the host (pos_dev nullptr) or read from device memory
// (*pos_dev, checked against the cache length by the kernel): the form a
// captured graph can replay for every token.  `part` (D == 64 only; may be
// nullptr) is a buffer of attention_decode_part_floats(B, H, L) floats for
// the split-key kernels, allocated by the caller since nothing may be
// allocated inside a capture (and once per cache rather than once per
// call in the eager loop).  Defined in attention.hip.
void attention_decode_cached(const tensor_t *qkv, tensor_t *k_cache, tensor_t *v_cache, int pos, const int *pos_dev,
                             int n_heads, tensor_t *output, float *part);
size_t attention_decode_part_floats(int B, int H, int L);


// The rest of the device-position generation step (decode_ops.hip), for B
// sequences whose tokens are rows of a (B, stride) float buffer:
//   out (B, C) = wte[tokens[b, pos]] + wpe[pos];
//   tokens[b, pos + 1] = argmax of logits row b, when prompt <= pos + 1 < total;
//   pos += 1.
void launch_embed_tokens_devpos(const tensor_t *wte, const tensor_t *wpe, const float *tokens, int B, int stride,
                                const int *pos_dev, tensor_t *out);
void launch_argmax_next(const tensor_t *logits, float *tokens, int stride, const int *pos_dev, int prompt, int total);
void launch_advance_pos(int *pos_dev);

// gptc_linear_rows_cuda with an optional LayerNorm of x in front (ln_w set;
// ln_b may be null): y = act(LN(x) W^T + b) + residual for 1 .. 8 rows.
void ln_linear_rows(const tensor_t *ln_w, const tensor_t *ln_b, float eps, const tensor_t *W, const tensor_t *b,
                    const tensor_t *x, const tensor_t *residual, int act, tensor_t *y);

}  // namespace gptc
