// Paged K/V caches (include/paged.h): the pool, the plan of a step, and the kernel that puts a step's new
// keys and values into their pages with the position rotation applied on the way.
//
// The plan is made on the host, once per step, and read by all its layers.  There the lengths and page
// numbers are checked (nothing that reaches the GPU can point outside the pool), the attention's work is cut
// into items of about equal size (paged_schedule), and every new token's slot and position are written out, so
// that the kernels search nothing.  Its device memory is laid out for the plan's capacity and never moves.
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdlib>
#include <cstring>
#include <mutex>
#include <utility>
#include "gpu_kernels.h"
#include "ops_common.hpp"
#include "paged_plan.hpp"

using namespace gptc;

struct gptc_paged_plan {
    const gptc_paged_cache_t *cache;
    int n_heads, group, max_seqs, max_tokens, max_len, max_pages;
    int max_fresh;  // new tokens of a sequence
    int item_cap, wide_cap, merge_cap, part_cap;  // wide_cap 0: no sequence can have wide items
    // Device memory (taken by the first set): ints [head 8 | items | wide items | merges | slot | pos | table], then
    // the parts.
    int *dev;
    float *part_o, *part_ml;
    size_t at_items, at_wide, at_merges, at_slot, at_pos, at_table, ints;
    // Two pinned copies of it, so that the host may prepare a step while the one before is still queued.
    int *host[2];
    hipEvent_t copied[2];
    int turn;
    bool is_set;
    int n_tokens, n_items, n_wide, n_many, n_few, merge_rows;
    int *table_at;  // where each sequence's page numbers start
    // Who writes each page in this step: checked without clearing the array between steps.
    long long *writer;  // step * max_seqs + sequence
    long long step;
    gptc_paged_plan *next_freed;
};

namespace {

constexpr int kMaxHeads = 4096;

int64_t part_slots(const gptc_paged_plan *p) {
    return static_cast<int64_t>(p->part_cap) * p->cache->n_kv_heads;
}

// A sequence with this many query rows per kv head or more takes wide items.
constexpr int kWideFrom = 64;

// How a list's tiles of rows are cut.
int tile_keys(int past, int rows, int row0, int tile, int group) {
    const int end = row0 + tile < rows ? row0 + tile : rows;
    return past + (end - 1) / group + 1;
}

struct Cutting {
    bool wide;
    int tile, unit, target, least, whole;
    int64_t tiles, total, per;

    int rounds(int keys) const { return (keys + unit - 1) / unit; }
    int cuts(int rounds) const { return rounds <= whole ? 1 : static_cast<int>((rounds + per - 1) / per); }
    int64_t items(int n_seqs, const int *past, const int *fresh, int group) const {
        int64_t n = 0;
        for (int s = 0; s < n_seqs; ++s) {
            const int rows = fresh[s] * group;
            if ((rows >= kWideFrom) != wide) continue;
            for (int r = 0; r < rows; r += tile) n += cuts(rounds(tile_keys(past[s], rows, r, tile, group)));
        }
        return n;
    }
};

}  // namespace

bool gptc::paged_schedule(int n_seqs, const int *past, const int *fresh, int group, int n_kv_heads, int head_dim,
                          int dtype, PagedLists &lists) {
    // The work is counted in rounds: of a workgroup's four waves, or tiles of a wide item.  A tile of rows whose keys take
    // more than `per` rounds is cut evenly, into parts of `least` rounds at least; what takes no more than `whole` stays
    // whole.  Joining costs 3 to 4 us, a round 0.5 us up to heads of 64 and 1.4 us above: one token of 32 heads of 128
    // over 900 bf16 keys (8 rounds) takes 14.5 us whole and 11.3 us in four parts, of 12 heads of 64 over 364 fp32 keys
    // (6 rounds) 6.2 us and 7.9 us.
    const bool small = head_dim <= 64;
    const int wide_least = std::max(1, 64 / paged_wide_keys(dtype, head_dim));
    Cutting cut[2] = {{false, kPagedRows, paged_unit(dtype), kPagedTarget, small ? 4 : 2, small ? 8 : 4, 0, 0, 0},
                      {true, paged_wide_rows(dtype), paged_wide_keys(dtype, head_dim), kPagedWideTarget, wide_least,
                       wide_least, 0, 0, 0}};
    for (int s = 0; s < n_seqs; ++s) {
        const int rows = fresh[s] * group;
        Cutting &c = cut[rows >= kWideFrom];
        for (int r = 0; r < rows; r += c.tile) c.total += c.rounds(tile_keys(past[s], rows, r, c.tile, group));
        c.tiles += (rows + c.tile - 1) / c.tile;
    }
    for (Cutting &c : cut) c.per = std::max<int64_t>(c.least, (c.total * n_kv_heads + c.target - 1) / c.target);
    // Single tokens, or few.  `slots` workgroups run at once, two on a CU up to heads of 64 (the kernel's launch bounds
    // see to it) and one above; the work is done soonest when all of them get the same, and a few too many would run
    // alone.  So there are as many as that where the tiles can be cut in three, twice as many where they cannot, and where
    // there are more tiles than that, only the longest are cut.  Heads of 128, fp32: 8 contexts of 3200 of 8 kv heads 45 us
    // in 256 and 48 in 512 workgroups (59 us in 1024), 32 of 1700 107 and 92 us, 64 of 900 90 us whole, 104 us where every
    // one was cut in two.
    Cutting &few = cut[0];
    const int64_t slots = small ? 512 : 256, tiles = few.tiles * n_kv_heads;
    if (tiles >= 2 * slots) {
        few.per = std::max(few.per, (2 * few.total + few.tiles - 1) / few.tiles);
    } else {
        few.target = static_cast<int>(3 * tiles <= slots ? slots : 2 * slots);
        few.per = std::max(few.per, (few.total * n_kv_heads + few.target - 1) / few.target);
        while (few.items(n_seqs, past, fresh, group) * n_kv_heads > few.target) few.per += (few.per + 15) / 16;
    }
    // Wide ones differ too much in length for that (a prompt of 4096: 220 us became 244), but parts of less than 256 keys
    // pay only as long as every workgroup has a CU of its own: a prompt of 512 with 12 heads of 64 takes 22 us in parts of
    // 256 fp32 keys and 14 us in 240 workgroups of 64, one of 1024 26 us in 240 of 256 and 28 us in 432 of 128.
    const int wide_most = 256 / paged_wide_keys(dtype, head_dim);
    while (cut[1].per < wide_most && cut[1].items(n_seqs, past, fresh, group) * n_kv_heads > 256) ++cut[1].per;
    lists.n_items = lists.n_wide = lists.n_merges = lists.merge_rows = 0;
    int parts = 0, tok0 = 0;
    for (int s = 0; s < n_seqs; ++s) {
        const int rows = fresh[s] * group;
        const bool wide = rows >= kWideFrom;
        const Cutting &c = cut[wide];
        const int slots = c.tile / kPagedRows;
        for (int r = 0; r < rows; r += c.tile) {
            const int keys = tile_keys(past[s], rows, r, c.tile, group);
            const int rounds = c.rounds(keys), cuts = c.cuts(rounds);
            int &n = wide ? lists.n_wide : lists.n_items;
            if (n + cuts > (wide ? lists.wide_cap : lists.item_cap)) return false;
            if (cuts > 1 && (parts + cuts * slots > lists.part_cap || lists.n_merges + slots > lists.merge_cap)) return false;
            for (int i = 0; i < cuts; ++i) {
                const int64_t from = static_cast<int64_t>(rounds) * i / cuts, to = static_cast<int64_t>(rounds) * (i + 1) / cuts;
                const int key1 = to * c.unit < keys ? static_cast<int>(to * c.unit) : keys;
                (wide ? lists.wide : lists.items)[n++] = PagedItem{
                    tok0, past[s], rows, r, static_cast<int>(from * c.unit), key1, cuts > 1 ? parts + i * slots : -1, s};
            }
            if (cuts > 1) {
                for (int i = 0; i < slots && r + i * kPagedRows < rows; ++i)
                    lists.merges[lists.n_merges++] = PagedMerge{tok0, rows, r + i * kPagedRows, parts + i, cuts, slots, 0, 0};
                parts += cuts * slots;
            }
        }
        tok0 += fresh[s];
    }
    // The longest first: workgroups start in this order, and what starts last should be short.
    const auto longer = [](const PagedItem &x, const PagedItem &y) { return x.key1 - x.key0 > y.key1 - y.key0; };
    std::sort(lists.items, lists.items + lists.n_items, longer);
    std::sort(lists.wide, lists.wide + lists.n_wide, longer);
    const auto rows_of = [](const PagedMerge &x) { return std::min(x.rows - x.row0, kPagedRows); };
    lists.n_many = static_cast<int>(std::partition(lists.merges, lists.merges + lists.n_merges,
                                                   [&](const PagedMerge &x) { return paged_many(x.n, rows_of(x)); }) -
                                    lists.merges);
    for (int i = 0; i < lists.n_many; ++i) lists.merge_rows = std::max(lists.merge_rows, rows_of(lists.merges[i]));
    return true;
}

extern "C" int gptc_paged_schedule(const int n_seqs, const int *past, const int *fresh, const int n_heads,
                                   const int n_kv_heads, const int head_dim, const int dtype, int *items,
                                   const int cap) {
    REQUIRE_ARG(past);
    REQUIRE_ARG(fresh);
    REQUIRE_ARG(items);
    CHECK_ERROR(n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads != 0,
                "Expected n_heads = %d to be a multiple of n_kv_heads = %d.", n_heads, n_kv_heads);
    CHECK_ERROR(dtype != GPTC_F32 && dtype != GPTC_BF16, "Unknown page type %d.", dtype);
    CHECK_ERROR(head_dim < 1 || head_dim > 128, "Head size %d is not supported in pages (1 <= head_dim <= 128).",
                head_dim);
    CHECK_ERROR(cap > 1 << 24, "Expected room for up to 2^24 items, but got %d.", cap);
    for (int s = 0; s < n_seqs; ++s)
        CHECK_ERROR(past[s] < 0 || fresh[s] < 0 || static_cast<int64_t>(past[s]) + fresh[s] > (1 << 30) ||
                        static_cast<int64_t>(fresh[s]) * n_heads > (1 << 26),
                    "Sequence %d has %d tokens and %d new ones.", s, past[s], fresh[s]);
    if (n_seqs <= 0 || cap <= 0) return n_seqs <= 0 ? 0 : -1;
    PagedLists l{};
    l.items = reinterpret_cast<PagedItem *>(items);
    l.item_cap = l.wide_cap = cap;
    l.part_cap = INT32_MAX / 2;
    l.merge_cap = 8 * cap;  // a cut tile has at least two items, and at most one merge for each 16 of its 128 rows
    l.wide = static_cast<PagedItem *>(mallocCheck(sizeof(PagedItem) * static_cast<size_t>(cap)));
    l.merges = static_cast<PagedMerge *>(mallocCheck(sizeof(PagedMerge) * static_cast<size_t>(l.merge_cap)));
    int n = -1;
    if (paged_schedule(n_seqs, past, fresh, n_heads / n_kv_heads, n_kv_heads, head_dim, dtype, l) &&
        l.n_items + l.n_wide <= cap) {
        n = l.n_items + l.n_wide;
        for (int i = 0; i < l.n_items; ++i) l.items[i].table = 0;  // the item's kind
        for (int i = 0; i < l.n_wide; ++i) {
            l.items[l.n_items + i] = l.wide[i];
            l.items[l.n_items + i].table = 1;
        }
    }
    free(l.wide);
    free(l.merges);
    return n;
}

// ---- the pool ----

extern "C" gptc_paged_cache_t *gptc_paged_cache_create(const int n_layers, const int n_pages, const int page,
                                                       const int n_kv_heads, const int head_dim, const int dtype,
                                                       void *const *k, void *const *v) {
    CHECK_ERROR(n_layers < 1, "Expected at least one layer, but got %d.", n_layers);
    CHECK_ERROR(page < 16 || page > 4096 || (page & (page - 1)) != 0,
                "Expected the page to be a power of two from 16 to 4096, but got %d.", page);
    CHECK_ERROR(n_pages < 1 || static_cast<int64_t>(n_pages) * page > INT32_MAX,
                "Expected 1 .. %d pages of %d tokens, but got %d.", INT32_MAX / page, page, n_pages);
    CHECK_ERROR(n_kv_heads < 1 || n_kv_heads > kMaxHeads, "Expected 1 .. %d kv heads, but got %d.", kMaxHeads, n_kv_heads);
    CHECK_ERROR(head_dim < 1 || head_dim > 128, "Head size %d is not supported in pages (1 <= head_dim <= 128).",
                head_dim);
    CHECK_ERROR(dtype != GPTC_F32 && dtype != GPTC_BF16, "Unknown page type %d.", dtype);
    CHECK_ERROR((k == NULL) != (v == NULL), "Expected both k and v, or neither.");
    auto *c = static_cast<gptc_paged_cache_t *>(mallocCheck(sizeof(gptc_paged_cache_t)));
    *c = gptc_paged_cache_t{n_layers, n_pages, page, n_kv_heads, head_dim, dtype, k == NULL, nullptr, nullptr};
    c->k = static_cast<void **>(mallocCheck(sizeof(void *) * n_layers));
    c->v = static_cast<void **>(mallocCheck(sizeof(void *) * n_layers));
    const size_t bytes = static_cast<size_t>(n_pages) * page * n_kv_heads * head_dim * (dtype == GPTC_BF16 ? 2 : 4);
    for (int l = 0; l < n_layers; ++l) {
        if (c->owned) {
            c->k[l] = alloc_cuda(bytes);
            c->v[l] = alloc_cuda(bytes);
            continue;
        }
        CHECK_ERROR(k[l] == NULL || v[l] == NULL, "The pages of layer %d are NULL.", l);
        CHECK_ERROR(!aligned16(k[l]) || !aligned16(v[l]), "The pages of layer %d are not 16-byte aligned.", l);
        c->k[l] = k[l];
        c->v[l] = v[l];
    }
    return c;
}

extern "C" void gptc_paged_cache_free(gptc_paged_cache_t *cache) {
    if (cache == NULL) return;
    for (int l = 0; cache->owned && gptc_runtime_up() && l < cache->n_layers; ++l) {
        free_cuda(cache->k[l]);
        free_cuda(cache->v[l]);
    }
    free(cache->k);
    free(cache->v);
    free(cache);
}

// ---- the plan ----

namespace {

// What a step uses of the plan's memory, from the pinned copy to the device, at the same places.
constexpr int kSegments = 6;
struct Segments {
    size_t from[kSegments], count[kSegments];
};

__global__ __launch_bounds__(256) void send_plan_kernel(const Segments s, const int *src, int *dst) {
    const size_t from = s.from[blockIdx.y], count = s.count[blockIdx.y];
    for (size_t i = blockIdx.x * 256 + threadIdx.x; i < count; i += 256 * gridDim.x) dst[from + i] = src[from + i];
}

}  // namespace

// Plans that were freed while the stream was being captured.  They go with the next call that makes, sets or frees a
// plan when it is not.
static std::mutex g_freed_mu;
static gptc_paged_plan_t *g_freed = nullptr;

static void release_plan(gptc_paged_plan_t *plan) {
    if (plan->dev != nullptr) {
        if (gptc_runtime_up()) {
            free_cuda(plan->dev);
            free_cuda(plan->part_o);
            free_cuda(plan->part_ml);
        }
        // None of this touches a stream that somebody may be capturing in the mode that forbids such calls.
        hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
        hipCheck(hipThreadExchangeStreamCaptureMode(&mode));
        for (int i = 0; i < 2; ++i) {
            hipCheck(hipEventSynchronize(plan->copied[i]));  // its last copy may still read the host memory
            hipCheck(hipEventDestroy(plan->copied[i]));
            hipCheck(hipHostFree(plan->host[i]));
        }
        hipCheck(hipThreadExchangeStreamCaptureMode(&mode));
    }
    free(plan->writer);
    free(plan->table_at);
    free(plan);
}

static void release_freed() {
    gptc_paged_plan_t *plan = nullptr;
    {
        std::lock_guard<std::mutex> lock(g_freed_mu);
        if (g_freed == nullptr || (gptc_runtime_up() && gptc_stream_capturing())) return;
        std::swap(plan, g_freed);
    }
    while (plan != nullptr) {
        gptc_paged_plan_t *next = plan->next_freed;
        release_plan(plan);
        plan = next;
    }
}

static gptc_paged_plan_t *make_plan(const gptc_paged_cache_t *cache, int n_heads, int max_seqs, int max_tokens, int max_len,
                                    int max_fresh) {
    release_freed();
    CHECK_ERROR(n_heads < 1 || n_heads > kMaxHeads || n_heads % cache->n_kv_heads != 0,
                "Expected n_heads = %d to be a multiple of the cache's %d kv heads, up to %d.", n_heads,
                cache->n_kv_heads, kMaxHeads);
    CHECK_ERROR(max_seqs < 1 || max_tokens < 1 || max_len < 1,
                "Expected room for sequences, tokens and lengths, but got %d, %d, %d.", max_seqs, max_tokens, max_len);
    CHECK_ERROR(max_len > (1 << 30), "Sequences of up to 2^30 tokens are supported, but got max_len = %d.", max_len);
    const int group = n_heads / cache->n_kv_heads;
    // What the grids and the page lists can hold.
    CHECK_ERROR(max_tokens > (1 << 22) || static_cast<int64_t>(max_tokens) * n_heads > (1 << 26),
                "max_tokens = %d with %d heads is too large.", max_tokens, n_heads);
    CHECK_ERROR(max_seqs > (1 << 20) || static_cast<int64_t>(max_seqs) * ((max_len + cache->page - 1) / cache->page) > (1 << 28),
                "%d sequences of %d tokens have too many pages.", max_seqs, max_len);
    auto *p = static_cast<gptc_paged_plan_t *>(mallocCheck(sizeof(gptc_paged_plan_t)));
    memset(p, 0, sizeof(*p));
    p->cache = cache;
    p->n_heads = n_heads;
    p->group = group;
    p->max_seqs = max_seqs;
    p->max_tokens = max_tokens;
    p->max_len = max_len;
    p->max_fresh = max_fresh;
    p->max_pages = (max_len + cache->page - 1) / cache->page;
    // Every tile of rows is an item; cutting adds at most one item per `per` rounds, target / kv heads in all, and
    // cuts at most as many tiles, so it makes at most twice as many parts.
    const int64_t work = static_cast<int64_t>(max_tokens) * group, active = max_seqs < max_tokens ? max_seqs : max_tokens;
    // Where no sequence can have the rows for wide items, a graph captured with the plan has no launch for them.
    const bool wide = static_cast<int64_t>(max_fresh) * group >= kWideFrom;
    const int cut = kPagedTarget / cache->n_kv_heads + 1, wide_cut = wide ? kPagedWideTarget / cache->n_kv_heads + 1 : 0;
    const int wide_rows = paged_wide_rows(cache->dtype), slots = wide_rows / kPagedRows;
    p->item_cap = static_cast<int>(work / kPagedRows + active) + cut;
    p->wide_cap = wide ? static_cast<int>(work / wide_rows + std::min(active, work / kWideFrom)) + wide_cut : 0;
    p->merge_cap = cut + slots * wide_cut;
    p->part_cap = 2 * p->merge_cap;
    // A launch has fewer than 2^32 threads: 256 for each item and kv head, up to 512 for wide ones.
    CHECK_ERROR(static_cast<int64_t>(std::max(p->item_cap, 2 * p->wide_cap)) * cache->n_kv_heads >= 1 << 24,
                "The work of %d sequences and %d tokens with %d heads is too large.", max_seqs, max_tokens, n_heads);
    p->at_items = 8;
    p->at_wide = p->at_items + 8 * static_cast<size_t>(p->item_cap);
    p->at_merges = p->at_wide + 8 * static_cast<size_t>(p->wide_cap);
    p->at_slot = p->at_merges + 8 * static_cast<size_t>(p->merge_cap);
    p->at_pos = p->at_slot + max_tokens;
    p->at_table = p->at_pos + max_tokens;
    p->ints = p->at_table + static_cast<size_t>(max_seqs) * p->max_pages;
    const size_t n_pages = cache->n_pages;
    p->writer = static_cast<long long *>(mallocCheck(sizeof(long long) * n_pages));
    memset(p->writer, 0, sizeof(long long) * n_pages);
    p->table_at = static_cast<int *>(mallocCheck(sizeof(int) * static_cast<size_t>(max_seqs)));
    return p;
}

extern "C" gptc_paged_plan_t *gptc_paged_plan_create(const gptc_paged_cache_t *cache, const int n_heads,
                                                     const int max_seqs, const int max_tokens, const int max_len) {
    REQUIRE_ARG(cache);
    return make_plan(cache, n_heads, max_seqs, max_tokens, max_len, std::min(max_tokens, max_len));
}

extern "C" gptc_paged_plan_t *gptc_paged_plan_create_single(const gptc_paged_cache_t *cache, const int n_heads,
                                                            const int max_seqs, const int max_len) {
    REQUIRE_ARG(cache);
    return make_plan(cache, n_heads, max_seqs, max_seqs, max_len, 1);
}

extern "C" void gptc_paged_plan_free(gptc_paged_plan_t *plan) {
    if (plan == NULL) return;
    if (plan->dev != nullptr && gptc_runtime_up() && gptc_stream_capturing()) {
        std::lock_guard<std::mutex> lock(g_freed_mu);
        plan->next_freed = g_freed;
        g_freed = plan;
        return;
    }
    release_plan(plan);
    release_freed();
}

extern "C" void gptc_paged_plan_set(gptc_paged_plan_t *plan, const int n_seqs, const int *past, const int *fresh,
                                    const int *table, const int stride) {
    REQUIRE_ARG(plan);
    const gptc_paged_cache_t *c = plan->cache;
    CHECK_ERROR(n_seqs < 0 || n_seqs > plan->max_seqs, "The plan has room for %d sequences, but got %d.",
                plan->max_seqs, n_seqs);
    if (n_seqs > 0) {
        REQUIRE_ARG(past);
        REQUIRE_ARG(fresh);
        REQUIRE_ARG(table);
    }
    int64_t tokens = 0;
    for (int s = 0; s < n_seqs; ++s) {
        CHECK_ERROR(past[s] < 0 || fresh[s] < 0, "Sequence %d has %d tokens and %d new ones.", s, past[s], fresh[s]);
        const int64_t len = static_cast<int64_t>(past[s]) + fresh[s];
        CHECK_ERROR(len > plan->max_len, "Sequence %d grows to %lld tokens: the plan was made for %d.", s,
                    static_cast<long long>(len), plan->max_len);
        CHECK_ERROR((len + c->page - 1) / c->page > stride, "Sequence %d needs %lld pages, but the table has %d.", s,
                    static_cast<long long>((len + c->page - 1) / c->page), stride);
        CHECK_ERROR(fresh[s] > plan->max_fresh, "Sequence %d has %d new tokens: the plan was made for %d.", s, fresh[s],
                    plan->max_fresh);
        tokens += fresh[s];
    }
    CHECK_ERROR(tokens > plan->max_tokens, "The plan has room for %d new tokens, but got %lld.", plan->max_tokens,
                static_cast<long long>(tokens));
    // Page numbers, and who writes what.
    const long long base = ++plan->step * plan->max_seqs;
    for (int s = 0; s < n_seqs; ++s) {
        const int used = (past[s] + fresh[s] + c->page - 1) / c->page;
        const int *mine = table + static_cast<int64_t>(s) * stride;
        for (int i = 0; i < used; ++i)
            CHECK_ERROR(mine[i] < 0 || mine[i] >= c->n_pages, "Page %d of sequence %d is %d: the cache has %d pages.",
                        i, s, mine[i], c->n_pages);
        for (int i = fresh[s] > 0 ? past[s] / c->page : used; i < used; ++i) {
            CHECK_ERROR(plan->writer[mine[i]] >= base, "Page %d would receive tokens of sequences %lld and %d.",
                        mine[i], plan->writer[mine[i]] - base, s);
            plan->writer[mine[i]] = base + s;
        }
    }
    for (int s = 0; s < n_seqs; ++s) {
        const int used = (past[s] + fresh[s] + c->page - 1) / c->page, own = fresh[s] > 0 ? past[s] / c->page : used;
        const int *mine = table + static_cast<int64_t>(s) * stride;
        for (int i = 0; i < own; ++i)
            CHECK_ERROR(plan->writer[mine[i]] >= base, "Page %d, which sequence %d reads, would receive tokens of %lld.",
                        mine[i], s, plan->writer[mine[i]] - base);
    }

    hipStream_t stream = gptc_stream_checked();
    CHECK_ERROR(gptc_stream_capturing(), "A plan cannot be set while the stream is being captured.");
    release_freed();
    if (plan->dev == nullptr) {
        plan->dev = static_cast<int *>(alloc_cuda(sizeof(int) * plan->ints));
        plan->part_o = static_cast<float *>(alloc_cuda(sizeof(float) * part_slots(plan) * kPagedRows * c->head_dim));
        plan->part_ml = static_cast<float *>(alloc_cuda(sizeof(float) * part_slots(plan) * kPagedRows * 2));
        for (int i = 0; i < 2; ++i) {
            hipCheck(hipHostMalloc(reinterpret_cast<void **>(&plan->host[i]), sizeof(int) * plan->ints, 0));
            hipCheck(hipEventCreateWithFlags(&plan->copied[i], hipEventDisableTiming));
            hipCheck(hipEventRecord(plan->copied[i], stream));
        }
    }
    plan->turn ^= 1;
    hipCheck(hipEventSynchronize(plan->copied[plan->turn]));
    int *h = plan->host[plan->turn];
    PagedLists lists{};
    lists.items = reinterpret_cast<PagedItem *>(h + plan->at_items);
    lists.wide = reinterpret_cast<PagedItem *>(h + plan->at_wide);
    lists.merges = reinterpret_cast<PagedMerge *>(h + plan->at_merges);
    lists.item_cap = plan->item_cap;
    lists.wide_cap = plan->wide_cap;
    lists.merge_cap = plan->merge_cap;
    lists.part_cap = plan->part_cap;
    const bool fits = paged_schedule(n_seqs, past, fresh, plan->group, c->n_kv_heads, c->head_dim, c->dtype, lists);
    CHECK_ERROR(!fits, "The work of %d sequences does not fit the plan.", n_seqs);
    int t = 0, at = 0;
    for (int s = 0; s < n_seqs; ++s) {
        const int used = (past[s] + fresh[s] + c->page - 1) / c->page;
        const int *mine = table + static_cast<int64_t>(s) * stride;
        for (int i = 0; i < fresh[s]; ++i, ++t) {
            const int pos = past[s] + i;
            h[plan->at_slot + t] = mine[pos / c->page] * c->page + pos % c->page;
            h[plan->at_pos + t] = pos;
        }
        if (fresh[s] == 0) continue;  // nobody asks for its keys
        plan->table_at[s] = at;
        memcpy(h + plan->at_table + at, mine, sizeof(int) * used);
        at += used;
    }
    for (int i = 0; i < lists.n_items; ++i) lists.items[i].table = plan->table_at[lists.items[i].table];
    for (int i = 0; i < lists.n_wide; ++i) lists.wide[i].table = plan->table_at[lists.wide[i].table];
    h[0] = t;
    h[1] = lists.n_items;
    h[2] = lists.n_merges;
    h[3] = lists.n_wide;
    h[4] = lists.n_many;
    // One kernel that reads the host's memory: with a copy command for each piece the call took 10 us longer.
    const Segments segments = {{0, plan->at_wide, plan->at_merges, plan->at_slot, plan->at_pos, plan->at_table},
                               {plan->at_items + 8 * static_cast<size_t>(lists.n_items), 8 * static_cast<size_t>(lists.n_wide),
                                8 * static_cast<size_t>(lists.n_merges), static_cast<size_t>(t), static_cast<size_t>(t),
                                static_cast<size_t>(at)}};
    const size_t most = *std::max_element(segments.count, segments.count + kSegments);
    send_plan_kernel<<<dim3(static_cast<unsigned>(std::min<size_t>((most + 255) / 256, 512)), kSegments), dim3(256), 0, stream>>>(
        segments, h, plan->dev);
    hipCheck(hipGetLastError());
    hipCheck(hipEventRecord(plan->copied[plan->turn], stream));
    plan->n_tokens = t;
    plan->n_items = lists.n_items;
    plan->n_wide = lists.n_wide;
    plan->n_many = lists.n_many;
    plan->n_few = lists.n_merges - lists.n_many;
    plan->merge_rows = lists.merge_rows;
    plan->is_set = true;
}

// ---- append ----

namespace {

struct AppendParams {
    const float *qkv, *rotary;
    float *q_out;
    void *k, *v;
    const int *head, *slot, *pos;  // head[0]: the step's tokens
    int rows, H, KV, D, page_shift, rot;
    bool interleaved;
};

typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));

template <int W>
struct Vec {
    float e[W];
};

template <int W>
__device__ __forceinline__ Vec<W> load_vec(const float *p) {
    Vec<W> r;
    if constexpr (W == 4) {
        const f32x4_t x = *reinterpret_cast<const f32x4_t *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) r.e[i] = x[i];
    } else {
        r.e[0] = *p;
    }
    return r;
}

template <int W>
__device__ __forceinline__ void store_vec(float *p, const Vec<W> &x) {
    if constexpr (W == 4)
        *reinterpret_cast<f32x4_t *>(p) = f32x4_t{x.e[0], x.e[1], x.e[2], x.e[3]};
    else
        *p = x.e[0];
}

// Rounded to nearest even: the one rounding that bf16 pages bring.
template <int W>
__device__ __forceinline__ void store_vec(__bf16 *p, const Vec<W> &x) {
    if constexpr (W == 4) {
        bf16x4_t y;
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = static_cast<__bf16>(x.e[i]);
        *reinterpret_cast<bf16x4_t *>(p) = y;
    } else {
        *p = static_cast<__bf16>(x.e[0]);
    }
}

// One thread per W consecutive values of a head of a token.  A pass over the data and nothing else: each value is
// read once (a rotated one's partner comes from the same cache lines) and written once, so HBM bounds it for
// prompts and the launch for single tokens.  Without rotation the queries stay where they are.  MI355X: 5740 tokens of
// prompts, 32 and 8 heads of 128 into bf16 pages (262 MB) 51 us, 5.1 TB/s (a copy of that size reaches 5.1); 8 single
// tokens 3.4 us.
template <typename T, int W>
__global__ __launch_bounds__(256) void append_kernel(const AppendParams a) {
    const int per_head = a.D / W;
    const int first = a.rotary != nullptr ? 0 : a.H;  // first head to move
    const int heads = a.H + 2 * a.KV - first;
    const int i = blockIdx.y * 256 + threadIdx.x;
    const int t = blockIdx.x;
    if (t >= a.head[0] || i >= heads * per_head) return;
    const int head = first + i / per_head, d = (i % per_head) * W;
    const float *src = a.qkv + static_cast<int64_t>(t) * (a.H + 2 * a.KV) * a.D + static_cast<int64_t>(head) * a.D + d;
    Vec<W> x = load_vec<W>(src);
    if (a.rotary != nullptr && head < a.H + a.KV && d < a.rot) {
        const int half = a.rot / 2;
        const float *cs = a.rotary + static_cast<int64_t>(a.pos[t]) * a.rot;
        if (!a.interleaved) {
            const bool low = d < half;
            const int p = low ? d : d - half;
            const Vec<W> y = load_vec<W>(src + (low ? half : -half)), c = load_vec<W>(cs + p), s = load_vec<W>(cs + half + p);
#pragma unroll
            for (int e = 0; e < W; ++e) x.e[e] = fmaf(x.e[e], c.e[e], low ? -(y.e[e] * s.e[e]) : y.e[e] * s.e[e]);
        } else if constexpr (W == 4) {
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float c = cs[(d + e) / 2], s = cs[half + (d + e) / 2], one = x.e[e], two = x.e[e + 1];
                x.e[e] = fmaf(one, c, -(two * s));
                x.e[e + 1] = fmaf(two, c, one * s);
            }
        } else {
            const bool low = (d & 1) == 0;
            const float y = src[low ? 1 : -1], c = cs[d / 2], s = cs[half + d / 2];
            x.e[0] = fmaf(x.e[0], c, low ? -(y * s) : y * s);
        }
    }
    if (head < a.H) {
        store_vec<W>(a.q_out + (static_cast<int64_t>(t) * a.H + head) * a.D + d, x);
        return;
    }
    const int kv = head - a.H;
    const bool is_k = kv < a.KV;
    const int slot = a.slot[t];
    const int64_t page = slot >> a.page_shift, in = slot & ((1 << a.page_shift) - 1);
    T *dst = static_cast<T *>(is_k ? a.k : a.v) +
             (((page * a.KV + (is_k ? kv : kv - a.KV)) << a.page_shift) + in) * a.D + d;
    store_vec<W>(dst, x);
}

int log2_of(int page) { return __builtin_ctz(static_cast<unsigned>(page)); }

// The checks that both entry points share.
void check_step(const gptc_paged_plan_t *plan, int layer, const char *fn) {
    CHECK_ERROR(plan == NULL, "%s(): argument `plan` is NULL.", fn);
    CHECK_ERROR(layer < 0 || layer >= plan->cache->n_layers, "Expected 0 <= layer < %d, but got %d.",
                plan->cache->n_layers, layer);
}

}  // namespace

extern "C" tensor_t *gptc_rotary_table(const int rows, const int rot, const double theta) {
    CHECK_ERROR(rows < 1 || rot < 2 || rot % 2 != 0, "Expected rows >= 1 and an even rot >= 2, but got %d, %d.", rows, rot);
    CHECK_ERROR(!(theta > 0.0), "Expected theta > 0, but got %g.", theta);
    CHECK_ERROR(static_cast<int64_t>(rows) * rot > INT32_MAX, "A table of %d x %d values is too large.", rows, rot);
    int shp[2] = {rows, rot};
    tensor_t *t = create_tensor(shp, 2, CPU);
    for (int p = 0; p < rows; ++p)
        for (int i = 0; i < rot / 2; ++i) {
            const double a = p * pow(theta, -2.0 * i / rot);
            t->t[static_cast<int64_t>(p) * rot + i] = static_cast<float>(cos(a));
            t->t[static_cast<int64_t>(p) * rot + rot / 2 + i] = static_cast<float>(sin(a));
        }
    t->to(t, CUDA);
    return t;
}

extern "C" void gptc_paged_append_cuda(gptc_paged_plan_t *plan, const int layer, const tensor_t *qkv,
                                       const tensor_t *rotary, const int interleaved, tensor_t *q_out) {
    check_step(plan, layer, __func__);
    const gptc_paged_cache_t *c = plan->cache;
    const int H = plan->n_heads, KV = c->n_kv_heads, D = c->head_dim;
    check_gpu(qkv, "qkv");
    CHECK_ERROR(last_dim(qkv) != (H + 2 * KV) * D, "Expected qkv rows of (%d + 2 * %d) * %d values, but got %d.", H, KV,
                D, last_dim(qkv));
    const int rows = leading_rows(qkv);
    CHECK_ERROR((rotary == NULL) != (q_out == NULL), "Expected rotary and q_out together, or neither.");
    int rot = 0;
    if (rotary != NULL) {
        check_gpu(rotary, "rotary");
        check_gpu(q_out, "q_out");
        rot = last_dim(rotary);
        CHECK_ERROR(rotary->ndims != 2 || rot < 2 || rot % 2 != 0 || rot > D,
                    "Expected a (positions, rot) table with an even rot <= %d.", D);
        CHECK_ERROR(rotary->shape[0] < plan->max_len, "The rotary table has %d rows: the plan's sequences reach %d.",
                    rotary->shape[0], plan->max_len);
        CHECK_ERROR(last_dim(q_out) != H * D || leading_rows(q_out) != rows, "Expected q_out to be (%d, %d).", rows, H * D);
        CHECK_ERROR(overlap(q_out, qkv) || overlap(q_out, rotary), "q_out may not overlap qkv or the rotary table.");
    }
    CHECK_ERROR(!plan->is_set, "The plan has not been set.");
    CHECK_ERROR(rows < plan->n_tokens, "The step has %d new tokens, but qkv has %d rows.", plan->n_tokens, rows);
    hipStream_t s = gptc_stream_checked();
    AppendParams a{};
    a.qkv = qkv->t;
    a.rotary = rotary != NULL ? rotary->t : nullptr;
    a.q_out = q_out != NULL ? q_out->t : nullptr;
    a.k = c->k[layer];
    a.v = c->v[layer];
    a.head = plan->dev;
    a.slot = plan->dev + plan->at_slot;
    a.pos = plan->dev + plan->at_pos;
    a.rows = rows;
    a.H = H;
    a.KV = KV;
    a.D = D;
    a.page_shift = log2_of(c->page);
    a.rot = rot;
    a.interleaved = interleaved != 0;
    // A captured launch covers what the plan can hold; the kernel reads what it does hold.
    int tokens = plan->n_tokens;
    if (gptc_stream_capturing()) tokens = plan->max_tokens < rows ? plan->max_tokens : rows;
    if (tokens == 0) return;
    // Groups of four values where they are whole, aligned, and rotated as a group.
    const bool vec = D % 4 == 0 && aligned16(a.qkv) && aligned16(a.q_out) && aligned16(a.rotary) &&
                     (rot == 0 || (a.interleaved ? rot % 4 == 0 : rot % 8 == 0));
    const int work = ((rotary != NULL ? H : 0) + 2 * KV) * (vec ? D / 4 : D);
    const dim3 grid(tokens, (work + 255) / 256);
    if (c->dtype == GPTC_F32) {
        if (vec) append_kernel<float, 4><<<grid, dim3(256), 0, s>>>(a);
        else append_kernel<float, 1><<<grid, dim3(256), 0, s>>>(a);
    } else {
        if (vec) append_kernel<__bf16, 4><<<grid, dim3(256), 0, s>>>(a);
        else append_kernel<__bf16, 1><<<grid, dim3(256), 0, s>>>(a);
    }
    hipCheck(hipGetLastError());
}

extern "C" void gptc_paged_attention_cuda(gptc_paged_plan_t *plan, const int layer, const tensor_t *q,
                                          tensor_t *output) {
    check_step(plan, layer, __func__);
    const gptc_paged_cache_t *c = plan->cache;
    const int H = plan->n_heads, KV = c->n_kv_heads, D = c->head_dim;
    check_gpu(q, "q");
    check_gpu(output, "output");
    const int width = last_dim(q), rows = leading_rows(q);
    CHECK_ERROR(width != H * D && width != (H + 2 * KV) * D, "Expected q rows of %d or %d values, but got %d.", H * D,
                (H + 2 * KV) * D, width);
    CHECK_ERROR(last_dim(output) != H * D || leading_rows(output) != rows, "Expected output to be (%d, %d).", rows, H * D);
    CHECK_ERROR(overlap(q, output), "output may not overlap q.");
    CHECK_ERROR(!plan->is_set, "The plan has not been set.");
    CHECK_ERROR(rows < plan->n_tokens, "The step has %d new tokens, but q has %d rows.", plan->n_tokens, rows);
    hipStream_t s = gptc_stream_checked();
    const bool capturing = gptc_stream_capturing();
    PagedAttnParams a{};
    a.q = q->t;
    a.out = output->t;
    a.k = c->k[layer];
    a.v = c->v[layer];
    a.head = plan->dev;
    a.items = reinterpret_cast<const PagedItem *>(plan->dev + plan->at_items);
    a.wide = reinterpret_cast<const PagedItem *>(plan->dev + plan->at_wide);
    a.merges = reinterpret_cast<const PagedMerge *>(plan->dev + plan->at_merges);
    a.table = plan->dev + plan->at_table;
    a.part_o = plan->part_o;
    a.part_ml = plan->part_ml;
    a.q_stride = width;
    a.rows = rows;
    a.H = H;
    a.KV = KV;
    a.group = plan->group;
    a.D = D;
    a.page_shift = log2_of(c->page);
    a.scale_log2 = static_cast<float>(1.4426950408889634 / sqrt(static_cast<double>(D)));
    a.n_items = capturing ? plan->item_cap : plan->n_items;
    a.n_wide = capturing ? plan->wide_cap : plan->n_wide;
    a.merge_rows = plan->merge_rows;
    a.merge_groups = (plan->n_many * plan->merge_rows + plan->n_few) * KV;
    if (capturing) {
        a.merge_rows = kPagedRows;
        a.merge_groups = std::min(KV * plan->merge_cap, 1024);
    }
    a.bf16 = c->dtype == GPTC_BF16;
    a.vec = D % (a.bf16 ? 8 : 4) == 0 && aligned16(a.q) && aligned16(a.out);
    if (a.n_items + a.n_wide == 0 || rows == 0) return;
    launch_paged_attention(a, s);
}
