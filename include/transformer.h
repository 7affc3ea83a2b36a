/*
 * transformer.h -- gpt.c's GPT-2 model, unchanged interface
 * (/root/reference/include/transformer.h:34-79).  forward(ids (B, T)) returns
 * logits (B, T, vocab_size); backward(dlogits) accumulates every parameter
 * gradient (lm_head shares wte's weight, and its gradient is added into
 * wte's).  parameters()/gradients() list _num_param_tensors tensors in the
 * order wte, wpe, layers[0..n), ln_f.
 */
#pragma once

#include "blocks.h"
#include "embedding.h"
#include "layer_norm.h"
#include "linear.h"
#include "loss.h"
#include "tensor.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct gpt2 {
    int n_embd;
    int n_heads;
    int n_layers;
    int block_size;
    int vocab_size;
    int _num_param_tensors;

    block_t **layers;
    embedding_t *wpe;
    embedding_t *wte;
    linear_t *lm_head;
    layer_norm_t *ln_f;

    tensor_t *(*forward)(struct gpt2 *, tensor_t *);
    tensor_t *(*backward)(struct gpt2 *, tensor_t *);
    void (*description)(const struct gpt2 *);
    int (*num_parameters)(const struct gpt2 *);
    void (*free_layer)(struct gpt2 *);
    void (*free_cache)(struct gpt2 *);
    tensor_t **(*parameters)(const struct gpt2 *);
    tensor_t **(*gradients)(const struct gpt2 *);
    void (*load_state_dict)(struct gpt2 *, tensor_t **);
    void (*fast_load_state_dict)(struct gpt2 *, tensor_t **);
    void (*to)(struct gpt2 *, const device_t);
} gpt2_t;

typedef struct {
    int block_size;
    int vocab_size;
    int n_layers;
    int n_heads;
    int n_embd;
} GPT2Config_t;

gpt2_t *GPT2(GPT2Config_t *config);

/*
 * A step without the logits: no counterpart in the reference, whose loop keeps
 * them, their log-softmax and their gradient (train_gpt.c:481-521).  On the GPU.
 *
 * gptc_gpt2_loss(gpt, x, targets, weights)
 *   The mean cross entropy of the model's predictions for ids x (B, T) against
 *   targets (B, T), a 1-element tensor: CrossEntropyLoss over forward(x).
 *   weights (B, T), or NULL for ones: the sum of weights times losses over B T;
 *   what a position of weight 0 is given as a target does not matter (the loss of
 *   gptc_linear_cross_entropy_cuda, gpu_kernels.h).  Leaves no caches behind.
 * gptc_gpt2_loss_backward(gpt, x, targets, weights)
 *   The same, and every parameter's gradient is added to: forward, loss, and the
 *   two backwards of gpt.c's loop for an upstream gradient of ones.
 * Both read x, targets and weights, which stay the caller's.  Both run forwards
 * of their own: a forward that still waits for its backward is dropped, and that
 * backward is refused.
 */
tensor_t *gptc_gpt2_loss(gpt2_t *gpt, const tensor_t *x, const tensor_t *targets, const tensor_t *weights);
tensor_t *gptc_gpt2_loss_backward(gpt2_t *gpt, const tensor_t *x, const tensor_t *targets, const tensor_t *weights);

#ifdef __cplusplus
}
#endif
