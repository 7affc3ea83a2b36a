/*
 * paged.h -- keys and values in pages, for many sequences at once.
 * No counterpart in gpt.c, whose inference loop (infer_gpt.c:339-351) has no
 * K/V cache at all; attention_decode_cuda_kernel (gpu_kernels.h) serves one
 * contiguous cache whose sequences all stand at one position.  Here every
 * sequence has its own length, a step may bring any number of new tokens for
 * each (a prompt, a chunk of one, a single token, none), and memory is given
 * out page by page.  One step of a model:
 *
 *   gptc_paged_plan_set(plan, ...)                      once: who has what
 *   per layer: qkv = the qkv Linear of all new tokens
 *              gptc_paged_append_cuda(plan, layer, qkv, ...)
 *              gptc_paged_attention_cuda(plan, layer, qkv, out)
 *   gptc_sample_cuda(logits, params, u, ids, prob)      (gpu_kernels.h)
 *
 * As everywhere in this library, work is ordered on gptc_stream(), and every
 * refused argument is a fatal error (print and exit) before anything runs.
 */
#pragma once

#include <stddef.h>
#include "tensor.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { GPTC_F32 = 0, GPTC_BF16 = 1 };

/*
 * The pool: per layer two device blocks, keys and values, each
 * (n_pages, n_kv_heads, page, head_dim) values of `dtype`.  Token t of a
 * sequence lies in slot t % page of the t / page-th page of that sequence.
 * Pages of GPTC_BF16 hold the values rounded to nearest even; products with
 * them are formed at fp32 accuracy.
 */
typedef struct gptc_paged_cache {
    int n_layers, n_pages, page, n_kv_heads, head_dim, dtype;
    int owned;  // the blocks were allocated here and go with the cache
    void **k;   // n_layers device pointers each
    void **v;
} gptc_paged_cache_t;

/*
 * gptc_paged_cache_create(n_layers, n_pages, page, n_kv_heads, head_dim, dtype, k, v)
 *   page: a power of two from 16 to 4096.  1 <= head_dim <= 128.  k, v: arrays
 *   of n_layers device pointers (memory of the caller, which outlives the
 *   cache; 16-byte aligned), or both NULL to allocate, uninitialised: slots
 *   that hold no token are never used.
 */
gptc_paged_cache_t *gptc_paged_cache_create(const int n_layers, const int n_pages, const int page,
                                            const int n_kv_heads, const int head_dim, const int dtype,
                                            void *const *k, void *const *v);
void gptc_paged_cache_free(gptc_paged_cache_t *cache);

/*
 * The plan of one step, shared by its layers: which tokens are new, where they
 * go, and how the attention's work is cut.
 *
 * gptc_paged_plan_create(cache, n_heads, max_seqs, max_tokens, max_len)
 *   For steps of up to max_seqs sequences with up to max_tokens new tokens in
 *   all, each sequence at most max_len tokens long with them.  n_heads is a
 *   multiple of the cache's n_kv_heads: query head h reads kv head
 *   h / (n_heads / n_kv_heads).  Its device memory is taken by the first
 *   gptc_paged_plan_set and never moves; the cache has to outlive the plan, and
 *   the plan the graphs captured with it.
 * gptc_paged_plan_create_single(cache, n_heads, max_seqs, max_len)
 *   For steps in which no sequence brings more than one token (others are
 *   refused).  Captured launches cover what a plan can hold: up to 63 query heads
 *   per kv head this one has no workspace for prompts, and graphs captured with it
 *   no launch for them.  A step's results are the same under every plan.
 * gptc_paged_plan_set(plan, n_seqs, past, fresh, table, stride)
 *   All arrays are host memory, read before the call returns.  Sequence s has
 *   past[s] >= 0 tokens in its pages and brings fresh[s] >= 0 new ones; its
 *   pages are table[s * stride + i], i < ceil((past[s] + fresh[s]) / page).
 *   Page numbers are checked, and so is that no page which receives a token is
 *   used by another sequence or twice: sequences may share pages that all of
 *   them only read.  The new tokens of all sequences are the rows
 *   0 .. sum(fresh) - 1 of the step's tensors, sequence by sequence.
 *   Not allowed while the stream is being captured.
 *
 * A plan holds the workspace of its calls too: two steps that overlap (graphs
 * launched on streams of the caller's) need a plan each.  A captured graph
 * reads the plan as it is when the graph runs: after another plan_set the same
 * graph serves the new step, as long as its tensors have the rows for it.
 * plan_set returns when its arrays have been read; the plan's device memory is
 * written by work queued on gptc_stream().  A graph launched on another stream
 * has to wait for an event recorded on gptc_stream() after plan_set, and
 * gptc_stream() for one recorded behind the graph before the next plan_set.
 */
typedef struct gptc_paged_plan gptc_paged_plan_t;

gptc_paged_plan_t *gptc_paged_plan_create(const gptc_paged_cache_t *cache, const int n_heads, const int max_seqs,
                                          const int max_tokens, const int max_len);
gptc_paged_plan_t *gptc_paged_plan_create_single(const gptc_paged_cache_t *cache, const int n_heads, const int max_seqs,
                                                 const int max_len);
void gptc_paged_plan_set(gptc_paged_plan_t *plan, const int n_seqs, const int *past, const int *fresh,
                         const int *table, const int stride);
void gptc_paged_plan_free(gptc_paged_plan_t *plan);  // during a capture: done by the first plan call after it

/*
 * gptc_rotary_table(rows, rot, theta)
 *   A (rows, rot) device tensor for gptc_paged_append_cuda, formed in 64 bits:
 *   row p holds cos(p theta^(-2i/rot)), i < rot/2, then the sines.
 *
 * gptc_paged_append_cuda(plan, layer, qkv, rotary, interleaved, q_out)
 *   qkv (rows, (n_heads + 2 n_kv_heads) * head_dim): q | k | v of the step's
 *   new tokens, rows >= sum(fresh) (rows past the last token are not read).
 *   Writes each token's keys and values into its pages.  rotary NULL: as they
 *   are, and q_out must be NULL.  Otherwise a (positions, rot) table, rot even
 *   and <= head_dim, of at least max_len rows: the first rot values of every q and k head are
 *   rotated by their token's position, in pairs (i, i + rot/2), or (2i, 2i+1)
 *   when `interleaved`, and q_out (rows, n_heads * head_dim) receives the
 *   queries; q_out may not overlap qkv.  Rows past the last token are left as
 *   they were.
 *
 * gptc_paged_attention_cuda(plan, layer, q, output)
 *   q (rows, n_heads * head_dim), or the qkv tensor itself (its first columns
 *   are read).  output (rows, n_heads * head_dim): token i of sequence s
 *   attends, scaled by 1/sqrt(head_dim), to that sequence's tokens
 *   0 .. past[s] + i, which have to be in their pages.  output rows past the
 *   last token are left as they were; output may not overlap q.
 *   Deterministic; no allocation.  Sums are fp32.  Keys and values of later
 *   tokens, and what unused slots hold, have no influence, finite or not.  Those
 *   of the tokens attended to are taken to be finite: infinities and NaN make
 *   the results that use them NaN or infinite.  Where a sequence brings 64 query
 *   rows per kv head or more, products are sums of bf16 parts: there fp32 values
 *   below 2^-110 count with fewer than 24 bits, and those past the largest bf16
 *   value may count as infinite.  So do queries with bf16 pages.
 */
tensor_t *gptc_rotary_table(const int rows, const int rot, const double theta);
void gptc_paged_append_cuda(gptc_paged_plan_t *plan, const int layer, const tensor_t *qkv, const tensor_t *rotary,
                            const int interleaved, tensor_t *q_out);
void gptc_paged_attention_cuda(gptc_paged_plan_t *plan, const int layer, const tensor_t *q, tensor_t *output);

/*
 * gptc_paged_schedule(n_seqs, past, fresh, n_heads, n_kv_heads, head_dim, dtype, items, cap)
 *   The work list that gptc_paged_plan_set makes for such a step (host
 *   computation only, for tests and tuning): item i is items[8i .. 8i+7] =
 *   (first token row, past, query rows of the sequence, first query row, first
 *   key, end key, part, kind): query rows are token * group + head for the
 *   group = n_heads / n_kv_heads heads of one kv head; kind 0: 16 rows, 1:
 *   64 of bf16 pages or 128 of fp32 ones; part -1 when the item covers all
 *   keys of its rows, else its place in the workspace (the first of rows / 16
 *   places).  Returns the number of items, or -1 when cap (in items) does not
 *   hold them.
 */
int gptc_paged_schedule(const int n_seqs, const int *past, const int *fresh, const int n_heads, const int n_kv_heads,
                        const int head_dim, const int dtype, int *items, const int cap);

#ifdef __cplusplus
}
#endif
