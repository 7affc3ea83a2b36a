// The plan of a paged step (include/paged.h) as the kernels and their launches see it (internal).
#pragma once

#include <hip/hip_runtime.h>
#include <cstdint>
#include "paged.h"

namespace gptc {

// One piece of attention work for one kv head: the query rows row0 .. of one sequence against the keys
// [key0, key1).  Everything a workgroup needs is in its item, so that it waits for one load only.
struct PagedItem {
    int tok0;   // the sequence's first row of the step's tensors
    int past;   // its tokens before the step
    int rows;   // its query rows of one kv head: new tokens * group, row = token * group + head of the group
    int row0;   // the item's first row
    int key0, key1;
    int part;   // -1: the item covers all keys of its rows; else its slot of the workspace
    int table;  // where the sequence's page numbers start; on the host side of the list, its sequence
};

// Up to 16 rows whose keys were cut into n items: their parts are part0, part0 + step, ...
struct PagedMerge {
    int tok0, rows, row0, part0, n, step, pad0, pad1;
};

constexpr int kPagedRows = 16;   // query rows of an item, and of a slot of the workspace
// Query rows of a wide item (csrc/paged_attn_wide.hip).
constexpr int paged_wide_rows(int dtype) { return dtype == GPTC_BF16 ? 64 : 128; }

// Keys that an item's kernel takes at a time, which its range is made of: a round of the four waves of a workgroup,
// 16 or 32 keys each (csrc/paged_attn.hip); an LDS tile of a wide item.
constexpr int paged_unit(int dtype) { return dtype == GPTC_BF16 ? 128 : 64; }
constexpr int paged_wide_keys(int dtype, int head_dim) {
    return dtype == GPTC_BF16 ? (head_dim <= 64 ? 128 : 64) : 32;
}

// Items that the keys of one step are cut into at most, over all kv heads: see paged_schedule.
constexpr int kPagedTarget = 1024;
constexpr int kPagedWideTarget = 512;

// Which merges take a workgroup for each row, see paged_merge_kernel.
constexpr bool paged_many(int parts, int rows) { return parts > (rows > 8 ? 32 : 4); }

// The lists of a step: items, wide items, and what is to be joined afterwards.
struct PagedLists {
    PagedItem *items, *wide;
    PagedMerge *merges;
    int item_cap, wide_cap, merge_cap, part_cap;
    int n_items, n_wide, n_merges;
    int n_many;      // merges of many parts, which come first
    int merge_rows;  // the rows of one of them, at most
};

// Fills the lists for a step (an item's table receives its sequence); false when one of them does not fit.
bool paged_schedule(int n_seqs, const int *past, const int *fresh, int group, int n_kv_heads, int head_dim, int dtype,
                    PagedLists &lists);

// What the attention kernels take.
struct PagedAttnParams {
    const float *q;
    float *out;
    const void *k, *v;
    const int *head;  // {tokens, items, merges, wide items, merges of many parts} of the plan, read on the device: a captured launch covers the
                      // plan's capacity and runs what the plan holds then
    const PagedItem *items, *wide;
    const PagedMerge *merges;
    const int *table;
    float *part_o, *part_ml;  // partial outputs [part][kv head][row][D], and their (max, sum) pairs
    int q_stride, rows;       // floats of a q row; rows of q and out
    int H, KV, group, D, page_shift;
    float scale_log2;
    int n_items, n_wide, merge_groups;  // of the launch
    int merge_rows;         // rows of a merge of many parts, at most
    bool bf16, vec;         // vec: every row starts at a multiple of 16 bytes and holds whole vectors
};

void launch_paged_attention(const PagedAttnParams &p, hipStream_t s);
void launch_paged_wide(const PagedAttnParams &p, hipStream_t s);

}  // namespace gptc
