/*
 * GPT-2 model (/root/reference/src/transformer.c:23-456):
 *   logits = lm_head(ln_f(blocks(wte[ids] + wpe[0..T))))
 * with lm_head's weight tied to wte's.  The backward re-creates lm_head's
 * gradient each call and adds it into wte's after the embedding backward,
 * as the reference does.  parameters()/gradients() list wte, wpe, the
 * blocks and ln_f (_num_param_tensors counts lm_head's shared weight in
 * place of wte's, so the count matches the list).
 */
#include <stdio.h>
#include "layer_util.h"
#include "transformer.h"

/* (src/transformer.c:69-111) */
static tensor_t *forward_transformer(gpt2_t *gpt, tensor_t *x) {
    REQUIRE_ARG(gpt);
    REQUIRE_ARG(x);
    CHECK_ERROR(x->ndims != 2, "Expected ids of shape (B, T), but got %d dims.", x->ndims);
    const device_t device = x->device;
    const int B = x->shape[0], T = x->shape[1], C = gpt->n_embd;
    CHECK_ERROR(T > gpt->block_size, "Cannot forward a sequence of length %d, block size is %d.", T, gpt->block_size);
    tensor_t *tok_emb = gpt->wte->forward(gpt->wte, x);
    tensor_t *pos = arange(0, T, 1, device);
    tensor_t *pos_emb = gpt->wpe->forward(gpt->wpe, pos);
    for (int b = 0; b < B; b++) saxpy(T * C, 1.0f, pos_emb, 0, 1, tok_emb, b * T * C, 1);
    free_tensor(pos_emb);
    tensor_t *out = tok_emb;
    for (int i = 0; i < gpt->n_layers; i++) out = gpt->layers[i]->forward(gpt->layers[i], out);
    out = gpt->ln_f->forward(gpt->ln_f, out);
    return gpt->lm_head->forward(gpt->lm_head, out);
}

/* (src/transformer.c:113-158) */
static tensor_t *backward_transformer(gpt2_t *gpt, tensor_t *global_grad) {
    REQUIRE_ARG(gpt);
    REQUIRE_ARG(global_grad);
    const device_t device = global_grad->device;
    linear_t *lm_head = gpt->lm_head;
    free_tensor(lm_head->dW);
    lm_head->dW = NULL;
    tensor_t *out = lm_head->backward(lm_head, global_grad);
    out = gpt->ln_f->backward(gpt->ln_f, out);
    for (int i = gpt->n_layers - 1; i >= 0; i--) out = gpt->layers[i]->backward(gpt->layers[i], out);
    tensor_t *out2 = create_tensor(out->shape, out->ndims, device);
    tensor_copy(out2, out);
    gpt->wpe->backward(gpt->wpe, out2);
    tensor_t *d_tok_emb = gpt->wte->backward(gpt->wte, out);
    saxpy(gpt->wte->dW->length, 1.0f, lm_head->dW, 0, 1, gpt->wte->dW, 0, 1);
    return d_tok_emb;
}

/* ln_f's output for ids x: the embeddings in one lookup, then the blocks. */
static tensor_t *forward_hidden(gpt2_t *gpt, const tensor_t *x) {
    const int T = x->shape[1];
    int shape[3] = {x->shape[0], T, gpt->n_embd};
    CHECK_ERROR(T > gpt->block_size, "Cannot forward a sequence of length %d, block size is %d.", T, gpt->block_size);
    tensor_t *out = create_tensor(shape, 3, CUDA);
    gptc_embedding_forward_scaled_cuda(gpt->wte->W, gpt->wpe->W, x, 1.0f, out);
    for (int i = 0; i < gpt->n_layers; i++) out = gpt->layers[i]->forward(gpt->layers[i], out);
    return gpt->ln_f->forward(gpt->ln_f, out);
}

static void check_loss_args(const gpt2_t *gpt, const tensor_t *x, const tensor_t *targets, const tensor_t *weights) {
    CHECK_ERROR(x->ndims != 2, "Expected ids of shape (B, T), but got %d dims.", x->ndims);
    CHECK_ERROR(x->device != CUDA || targets->device != CUDA || gpt->wte->W->device != CUDA ||
                    (weights != NULL && weights->device != CUDA),
                "The loss without logits runs on the GPU: move the model, ids, targets and weights there.");
    CHECK_ERROR(x->length < 1 || targets->length != x->length, "Expected as many targets as ids, but got %d and %d.",
                targets->length, x->length);
    CHECK_ERROR(weights != NULL && weights->length != x->length, "Expected as many weights as ids, but got %d and %d.",
                weights != NULL ? weights->length : 0, x->length);
}

tensor_t *gptc_gpt2_loss(gpt2_t *gpt, const tensor_t *x, const tensor_t *targets, const tensor_t *weights) {
    REQUIRE_ARG(gpt);
    REQUIRE_ARG(x);
    REQUIRE_ARG(targets);
    check_loss_args(gpt, x, targets, weights);
    int one[1] = {1};
    tensor_t *loss = create_tensor(one, 1, CUDA);
    tensor_t *out = forward_hidden(gpt, x);
    gptc_linear_cross_entropy_cuda(out, gpt->wte->W, targets, weights, loss, NULL, NULL, NULL, 0);
    free_tensor(out);
    gpt->free_cache(gpt);
    return loss;
}

tensor_t *gptc_gpt2_loss_backward(gpt2_t *gpt, const tensor_t *x, const tensor_t *targets, const tensor_t *weights) {
    REQUIRE_ARG(gpt);
    REQUIRE_ARG(x);
    REQUIRE_ARG(targets);
    check_loss_args(gpt, x, targets, weights);
    embedding_t *wte = gpt->wte, *wpe = gpt->wpe;
    if (!wte->dW) wte->dW = zeros(wte->W->shape, wte->W->ndims, CUDA);
    if (!wpe->dW) wpe->dW = zeros(wpe->W->shape, wpe->W->ndims, CUDA);
    int one[1] = {1};
    tensor_t *loss = create_tensor(one, 1, CUDA);
    tensor_t *hidden = forward_hidden(gpt, x);
    tensor_t *out = create_tensor(hidden->shape, hidden->ndims, CUDA);
    gptc_linear_cross_entropy_cuda(hidden, wte->W, targets, weights, loss, NULL, out, wte->dW, 1);
    free_tensor(hidden);
    out = gpt->ln_f->backward(gpt->ln_f, out);
    for (int i = gpt->n_layers - 1; i >= 0; i--) out = gpt->layers[i]->backward(gpt->layers[i], out);
    gptc_embedding_backward_sorted_cuda(out, x, 1.0f, wte->dW, wpe->dW, 1);
    free_tensor(out);
    return loss;
}

static void description_transformer(const gpt2_t *gpt) {
    printf("GPT-2 model: %d layers, %d heads, width %d, context %d, vocabulary %d; %d parameters\n",
           gpt->n_layers, gpt->n_heads, gpt->n_embd, gpt->block_size, gpt->vocab_size, gpt->num_parameters(gpt));
}

/* wte's weight is lm_head's, counted once. */
static int num_parameters_transformer(const gpt2_t *gpt) {
    if (gpt == NULL) return 0;
    int n = gpt->wpe->num_parameters(gpt->wpe) + gpt->wte->num_parameters(gpt->wte);
    for (int i = 0; i < gpt->n_layers; i++) n += gpt->layers[i]->num_parameters(gpt->layers[i]);
    return n + gpt->ln_f->num_parameters(gpt->ln_f);
}

static void free_layer_transformer(gpt2_t *gpt) {
    if (gpt == NULL) return;
    gpt->lm_head->W = NULL;  // owned by wte
    gpt->lm_head->free_layer(gpt->lm_head);
    gpt->wte->free_layer(gpt->wte);
    gpt->wpe->free_layer(gpt->wpe);
    for (int i = 0; i < gpt->n_layers; i++) gpt->layers[i]->free_layer(gpt->layers[i]);
    free(gpt->layers);
    gpt->ln_f->free_layer(gpt->ln_f);
    free(gpt);
}

static void free_cache_transformer(gpt2_t *gpt) {
    gpt->wte->free_cache(gpt->wte);
    gpt->wpe->free_cache(gpt->wpe);
    for (int i = 0; i < gpt->n_layers; i++) gpt->layers[i]->free_cache(gpt->layers[i]);
    gpt->ln_f->free_cache(gpt->ln_f);
    gpt->lm_head->free_cache(gpt->lm_head);
}

static tensor_t **parameters_transformer(const gpt2_t *gpt) {
    tensor_t **p = (tensor_t **)mallocCheck(sizeof(tensor_t *) * gpt->_num_param_tensors);
    int idx = 0;
    append_list(p, &idx, gpt->wte->parameters(gpt->wte), gpt->wte->_num_param_tensors);
    append_list(p, &idx, gpt->wpe->parameters(gpt->wpe), gpt->wpe->_num_param_tensors);
    for (int i = 0; i < gpt->n_layers; i++)
        append_list(p, &idx, gpt->layers[i]->parameters(gpt->layers[i]), gpt->layers[i]->_num_param_tensors);
    append_list(p, &idx, gpt->ln_f->parameters(gpt->ln_f), gpt->ln_f->_num_param_tensors);
    return p;
}

static tensor_t **gradients_transformer(const gpt2_t *gpt) {
    tensor_t **g = (tensor_t **)mallocCheck(sizeof(tensor_t *) * gpt->_num_param_tensors);
    int idx = 0;
    append_list(g, &idx, gpt->wte->gradients(gpt->wte), gpt->wte->_num_param_tensors);
    append_list(g, &idx, gpt->wpe->gradients(gpt->wpe), gpt->wpe->_num_param_tensors);
    for (int i = 0; i < gpt->n_layers; i++)
        append_list(g, &idx, gpt->layers[i]->gradients(gpt->layers[i]), gpt->layers[i]->_num_param_tensors);
    append_list(g, &idx, gpt->ln_f->gradients(gpt->ln_f), gpt->ln_f->_num_param_tensors);
    return g;
}

static void load_state_dict_transformer(gpt2_t *gpt, tensor_t **state) {
    CHECK_ERROR(gpt == NULL || state == NULL, "load_state_dict: NULL model or state.");
    gpt->wte->load_state_dict(gpt->wte, state);
    state += gpt->wte->_num_param_tensors;
    gpt->wpe->load_state_dict(gpt->wpe, state);
    state += gpt->wpe->_num_param_tensors;
    for (int i = 0; i < gpt->n_layers; i++) {
        gpt->layers[i]->load_state_dict(gpt->layers[i], state);
        state += gpt->layers[i]->_num_param_tensors;
    }
    gpt->ln_f->load_state_dict(gpt->ln_f, state);
}

/* state[i] -> parameters()[i] for every i, lengths checked
 * (src/transformer.c:392-415); any devices. */
static void fast_load_state_dict_transformer(gpt2_t *gpt, tensor_t **state) {
    CHECK_ERROR(gpt == NULL || state == NULL, "fast_load_state_dict: NULL model or state.");
    tensor_t **params = gpt->parameters(gpt);
    for (int i = 0; i < gpt->_num_param_tensors; i++) {
        CHECK_ERROR(params[i]->length != state[i]->length,
                    "Expected both model parameters and state tensor length's to match at index %d. Got %d != %d", i,
                    params[i]->length, state[i]->length);
        load_param(params[i], state[i], "parameter");
    }
    free(params);
}

static void to_transformer(gpt2_t *gpt, const device_t device) {
    gpt->wpe->to(gpt->wpe, device);
    gpt->wte->to(gpt->wte, device);
    for (int i = 0; i < gpt->n_layers; i++) gpt->layers[i]->to(gpt->layers[i], device);
    gpt->ln_f->to(gpt->ln_f, device);
    gpt->lm_head->to(gpt->lm_head, device);
}

gpt2_t *GPT2(GPT2Config_t *config) {
    REQUIRE_ARG(config);
    gpt2_t *gpt = (gpt2_t *)mallocCheck(sizeof(gpt2_t));
    gpt->block_size = config->block_size;
    gpt->vocab_size = config->vocab_size;
    gpt->n_embd = config->n_embd;
    gpt->n_heads = config->n_heads;
    gpt->n_layers = config->n_layers;
    gpt->wte = Embedding(gpt->vocab_size, gpt->n_embd);
    gpt->wpe = Embedding(gpt->block_size, gpt->n_embd);
    gpt->layers = (block_t **)mallocCheck(sizeof(block_t *) * (gpt->n_layers > 0 ? gpt->n_layers : 1));
    for (int i = 0; i < gpt->n_layers; i++) gpt->layers[i] = Block(gpt->n_embd, gpt->n_heads, gpt->block_size, 1);
    gpt->ln_f = LayerNorm(gpt->n_embd, 1e-5f, 1);
    gpt->lm_head = Linear(gpt->n_embd, gpt->vocab_size, 0);
    free_tensor(gpt->lm_head->W);
    free_tensor(gpt->lm_head->dW);
    gpt->lm_head->W = gpt->wte->W;
    gpt->lm_head->dW = NULL;
    gpt->_num_param_tensors = gpt->wpe->_num_param_tensors + gpt->ln_f->_num_param_tensors +
                              gpt->lm_head->_num_param_tensors;
    for (int i = 0; i < gpt->n_layers; i++) gpt->_num_param_tensors += gpt->layers[i]->_num_param_tensors;
    gpt->forward = forward_transformer;
    gpt->backward = backward_transformer;
    gpt->description = description_transformer;
    gpt->num_parameters = num_parameters_transformer;
    gpt->free_layer = free_layer_transformer;
    gpt->free_cache = free_cache_transformer;
    gpt->parameters = parameters_transformer;
    gpt->gradients = gradients_transformer;
    gpt->load_state_dict = load_state_dict_transformer;
    gpt->fast_load_state_dict = fast_load_state_dict_transformer;
    gpt->to = to_transformer;
    return gpt;
}
