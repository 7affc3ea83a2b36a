// Embedding lookup with scaling and positions, and its gradient by sorted
// tokens.  No counterpart in gpt.c, whose GPT2 looks both tables up apart and
// adds them sequence by sequence (src/transformer.c:69-111), and whose gradient
// walks the rows in turn (kernels/src/cpu/Embedding.c:27-47):
//   out[i] = s W[id[i]] (+ P[i mod T]);
//   dW[v] (+)= s sum of g[i] over id[i] = v;   dP[t] (+)= sum of g over i mod T = t.
//
// The gradient sorts the rows by (id, row) and adds each id's rows in that
// order.  A wave takes a fixed number of sorted places and 256 columns; an id
// whose rows go on into the next places leaves a partial sum, and a second
// kernel adds these in the order of their places.  So sums depend on the ids
// alone (no float atomics), and a token that fills the batch is shared by all
// waves.
#include <algorithm>
#include "gpu_kernels.h"
#include "ops_common.hpp"

namespace gptc {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

// An id held in a float, truncated; -1 for what is not in [0, V).
__device__ __forceinline__ int id_of(float f, int V) {
    if (!(f > -1.0f && f < 2147483648.0f)) return -1;
    const int i = static_cast<int>(f);
    return i < V ? i : -1;
}

template <typename T>
__device__ __forceinline__ T splat(float x);
template <>
__device__ __forceinline__ float splat<float>(float x) {
    return x;
}
template <>
__device__ __forceinline__ f32x4_t splat<f32x4_t>(float x) {
    return f32x4_t{x, x, x, x};
}
__device__ __forceinline__ float fma_of(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ f32x4_t fma_of(float a, f32x4_t b, f32x4_t c) {
    return f32x4_t{fmaf(a, b[0], c[0]), fmaf(a, b[1], c[1]), fmaf(a, b[2], c[2]), fmaf(a, b[3], c[3])};
}

// A wave a row; cols: columns in units of T.
template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_kernel(const T *__restrict__ W, const T *__restrict__ P,
                                                         const float *__restrict__ ids, float scale,
                                                         T *__restrict__ out, int rows, int seq, int cols, int V) {
    const int lane = threadIdx.x & (kWave - 1);
    const int row = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (row >= rows) return;
    const int id = id_of(ids[row], V);
    T *o = out + static_cast<int64_t>(row) * cols;
    if (id < 0) {
        for (int j = lane; j < cols; j += kWave) o[j] = splat<T>(NAN);
        return;
    }
    const T *w = W + static_cast<int64_t>(id) * cols;
    if (P != nullptr) {
        const T *p = P + static_cast<int64_t>(row % seq) * cols;
        for (int j = lane; j < cols; j += kWave) o[j] = fma_of(scale, w[j], p[j]);
    } else {
        for (int j = lane; j < cols; j += kWave) o[j] = scale * w[j];
    }
}

// ---- sorting ----
// The sort's launches are short and mostly wait; where dW is to be overwritten, further workgroups of
// the same launches clear it meanwhile (8192 rows of 768 on 50257: 25 us beside the ranking's 13).
struct Clear {
    f32x4_t *at;  // n of them from here on, by the workgroups after the first `blocks` of a launch
    int64_t n;
    int blocks;
};

__device__ __forceinline__ void clear_part(const Clear &c) {
    const int64_t stride = static_cast<int64_t>(gridDim.x - c.blocks) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - c.blocks) * blockDim.x + threadIdx.x; i < c.n; i += stride)
        c.at[i] = splat<f32x4_t>(0.0f);
}

// Workgroups for a part: eight waves a CU.
int clear_blocks(const Clear &c, int threads) {
    return static_cast<int>(std::min<int64_t>((c.n + threads - 1) / threads, 256 * 512 / threads));
}

// order[r] = (key, row) of the r-th row by (key, row); key: the id, V for rows
// without one.

// Up to kRankRows rows: a row's place is the number of rows before it, counted
// by comparing it with all of them, in one launch.
constexpr int kRankRows = 12288;
constexpr int kRankThreads = 512;
constexpr int kRankPer = 32;  // rows a workgroup
constexpr int kRankSlices = kRankThreads / kRankPer;

__global__ __launch_bounds__(kRankThreads) void rank_kernel(const float *__restrict__ ids, int n, int V,
                                                           int2 *__restrict__ order, Clear clear) {
    if (static_cast<int>(blockIdx.x) >= clear.blocks) {
        clear_part(clear);
        return;
    }
    extern __shared__ uint32_t keys[];  // all rows, padded to slices of whole 16 bytes with keys past all others
    __shared__ int count[kRankPer];
    const int per = ((n + kRankSlices - 1) / kRankSlices + 3) & ~3;  // rows a slice
    for (int j0 = threadIdx.x; j0 < per * kRankSlices; j0 += 8 * kRankThreads) {
        float id[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) id[k] = ids[min(j0 + k * kRankThreads, n - 1)];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const int j = j0 + k * kRankThreads;
            if (j >= per * kRankSlices) break;
            const int key = id_of(id[k], V);
            keys[j] = j >= n ? 0xffffffffu : key < 0 ? static_cast<uint32_t>(V) : static_cast<uint32_t>(key);
        }
    }
    if (threadIdx.x < kRankPer) count[threadIdx.x] = 0;
    __syncthreads();
    const int i0 = blockIdx.x * kRankPer, i = i0 + static_cast<int>(threadIdx.x % kRankPer);
    const int first = (threadIdx.x / kRankPer) * per;
    if (i < n) {
        const uint32_t key = keys[i];
        int before = 0;
        // Rows of this key count up to row i.  Before the workgroup's rows all of them do, behind them none.
        const int upto = max(first, min(first + per, i0 & ~3)), from = max(first, min(first + per, i0 + kRankPer));
#pragma unroll 4
        for (int j = first; j < upto; j += 4) {
            const uint4 k = *reinterpret_cast<const uint4 *>(keys + j);
            before += (k.x <= key) + (k.y <= key) + (k.z <= key) + (k.w <= key);
        }
        for (int j = upto; j < from; ++j) before += keys[j] < key + (j < i);
#pragma unroll 4
        for (int j = from; j < first + per; j += 4) {
            const uint4 k = *reinterpret_cast<const uint4 *>(keys + j);
            before += (k.x < key) + (k.y < key) + (k.z < key) + (k.w < key);
        }
        atomicAdd(&count[threadIdx.x % kRankPer], before);  // whole numbers: in any order the same
    }
    __syncthreads();
    if (threadIdx.x < kRankPer && i < n) order[count[threadIdx.x]] = make_int2(static_cast<int>(keys[i]), i);
}

// More rows: passes over the key's digits of eight bits from the lowest, each
// keeping the order of equal digits: count the digits of every block, sum the
// counts up, move every row to its place.
constexpr int kDigits = 256;
constexpr int kSortThreads = 256;
constexpr int kSortItems = 16;  // 64 rows at a time of a wave
constexpr int kSortBlock = kSortThreads * kSortItems;

struct SortArgs {
    const float *ids;  // the first pass reads the ids, the others `in`
    const int2 *in;
    int2 *out;
    int *hist;  // digit-major: (kDigits, blocks)
    int n, V, shift, blocks;
    Clear clear;
};

__device__ __forceinline__ int2 sort_item(const SortArgs &a, int i) {
    if (a.ids == nullptr) return a.in[i];
    const int id = id_of(a.ids[i], a.V);
    return make_int2(id < 0 ? a.V : id, i);
}

__global__ __launch_bounds__(kSortThreads) void digit_count_kernel(const SortArgs a) {
    if (static_cast<int>(blockIdx.x) >= a.blocks) {
        clear_part(a.clear);
        return;
    }
    __shared__ int count[kDigits];
    count[threadIdx.x] = 0;
    __syncthreads();
    int key[kSortItems];
#pragma unroll
    for (int t = 0; t < kSortItems; ++t)
        key[t] = sort_item(a, min(blockIdx.x * kSortBlock + t * kSortThreads + static_cast<int>(threadIdx.x), a.n - 1)).x;
#pragma unroll
    for (int t = 0; t < kSortItems; ++t)
        if (static_cast<int>(blockIdx.x * kSortBlock + t * kSortThreads + threadIdx.x) < a.n)
            atomicAdd(&count[(key[t] >> a.shift) & (kDigits - 1)], 1);
    __syncthreads();
    a.hist[threadIdx.x * a.blocks + blockIdx.x] = count[threadIdx.x];
}

// hist := its running sums, the entry itself left out; one workgroup.
constexpr int kScanThreads = 1024;
__global__ __launch_bounds__(kScanThreads) void digit_scan_kernel(int *hist, int n, Clear clear) {
    if (blockIdx.x > 0) {
        clear_part(clear);
        return;
    }
    __shared__ int part[kScanThreads];
    const int per = (n + kScanThreads - 1) / kScanThreads;
    const int lo = min(n, static_cast<int>(threadIdx.x) * per), hi = min(n, lo + per);
    int sum = 0;
#pragma unroll 8
    for (int i = lo; i < hi; ++i) sum += hist[i];
    part[threadIdx.x] = sum;
    __syncthreads();
    for (int off = 1; off < kScanThreads; off <<= 1) {
        const int add = static_cast<int>(threadIdx.x) >= off ? part[threadIdx.x - off] : 0;
        __syncthreads();
        part[threadIdx.x] += add;
        __syncthreads();
    }
    int at = part[threadIdx.x] - sum;
    for (int i = lo; i < hi; ++i) {
        const int v = hist[i];
        hist[i] = at;
        at += v;
    }
}

__global__ __launch_bounds__(kSortThreads) void digit_move_kernel(const SortArgs a) {
    if (static_cast<int>(blockIdx.x) >= a.blocks) {
        clear_part(a.clear);
        return;
    }
    constexpr int kW = kSortThreads / kWave;
    __shared__ int at[kW][kDigits];  // where a wave's next row of a digit goes
    const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave;
#pragma unroll
    for (int k = 0; k < kW; ++k) at[k][threadIdx.x] = 0;
    __syncthreads();
    // Wave w takes the w-th quarter of the block, 64 rows at a time.
    const int first = blockIdx.x * kSortBlock + w * (kSortItems * kWave) + lane;
    int2 item[kSortItems];
#pragma unroll
    for (int t = 0; t < kSortItems; ++t) {
        const int i = first + t * kWave;
        item[t] = i < a.n ? sort_item(a, i) : make_int2(0, -1);
    }
#pragma unroll
    for (int t = 0; t < kSortItems; ++t)
        if (item[t].y >= 0) atomicAdd(&at[w][(item[t].x >> a.shift) & (kDigits - 1)], 1);
    __syncthreads();
    {
        int next = a.hist[threadIdx.x * a.blocks + blockIdx.x];
#pragma unroll
        for (int k = 0; k < kW; ++k) {
            const int c = at[k][threadIdx.x];
            at[k][threadIdx.x] = next;
            next += c;
        }
    }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < kSortItems; ++t) {
        const bool live = item[t].y >= 0;
        const int digit = (item[t].x >> a.shift) & (kDigits - 1);
        uint64_t same = __ballot(live);  // the lanes of this digit
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint64_t set = __ballot((digit >> b) & 1);
            same &= (digit >> b) & 1 ? set : ~set;
        }
        if (live) {
            const int before = __popcll(same & ((1ull << lane) - 1));
            const int place = at[w][digit] + before;
            a.out[place] = item[t];
            wave_lds_order();
            if (before == __popcll(same) - 1) at[w][digit] = place + 1;
        }
        wave_lds_order();
    }
}

// ---- the sums ----

struct GatherArgs {
    const float *g;
    const int2 *order;
    float *dW;
    float *part;  // (chunks, 2, columns): a chunk's share of the run that goes on behind it, and of the one it ends
    float scale;
    int n, V, C, chunk, blocks;  // blocks: of columns
    bool add;
    float *dP;  // or null
    int seqs, seq, positions;
};

// dP[t] (+)= the sequences' rows t, in their order; rows past the sequences' length: 0.  By the workgroups
// after the first `before` of a launch.
template <typename T>
__device__ __forceinline__ void position_sums(const GatherArgs &a, int before) {
    const int cols = a.C / (sizeof(T) / sizeof(float));
    const int64_t n = static_cast<int64_t>(a.seq) * cols, total = static_cast<int64_t>(a.positions) * cols;
    const int64_t stride = static_cast<int64_t>(gridDim.x - before) * kThreads;
    const T *g = reinterpret_cast<const T *>(a.g);
    T *dP = reinterpret_cast<T *>(a.dP);
    for (int64_t i = static_cast<int64_t>(blockIdx.x - before) * kThreads + threadIdx.x; i < total; i += stride) {
        T sum = splat<T>(0.0f);
        if (i < n) {
            int b = 0;
            for (; b + 8 <= a.seqs; b += 8) {
                T v[8];
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = g[(b + k) * n + i];
#pragma unroll
                for (int k = 0; k < 8; ++k) sum += v[k];
            }
            for (; b < a.seqs; ++b) sum += g[b * n + i];
        } else if (a.add) {
            return;
        }
        dP[i] = a.add ? dP[i] + sum : sum;
    }
}

// One wave: `chunk` sorted places x 64 columns in units of T.
template <typename T>
__global__ __launch_bounds__(kThreads) void gather_kernel(const GatherArgs a, int items) {
    constexpr int kAhead = 8;  // rows whose loads are on their way together
    const int gather_blocks = (items + kWaves - 1) / kWaves;
    if (static_cast<int>(blockIdx.x) >= gather_blocks) {
        position_sums<T>(a, gather_blocks);
        return;
    }
    const int lane = threadIdx.x & (kWave - 1);
    const int item = blockIdx.x * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    if (item >= items) return;
    const int chunk = item / a.blocks, col = (item - chunk * a.blocks) * kWave + lane;
    const int cols = a.C / (sizeof(T) / sizeof(float));
    const int p0 = chunk * a.chunk, left = min(a.chunk, a.n - p0);
    const int2 mine = lane < left ? a.order[p0 + lane] : make_int2(a.V, 0);
    const int after = lane < left && p0 + lane + 1 < a.n ? a.order[p0 + lane + 1].x : a.V;
    const int before = p0 > 0 ? a.order[p0 - 1].x : -1;
    const int live = __popcll(__ballot(mine.x < a.V));  // rows without an id are the last ones
    if (live == 0) return;
    const uint64_t ends = __ballot(mine.x != after);
    bool open = __builtin_amdgcn_readlane(mine.x, 0) == before;  // the first run began in an earlier chunk
    const bool on = col < cols;
    const T *g = reinterpret_cast<const T *>(a.g);
    T *dW = reinterpret_cast<T *>(a.dW);
    T *part = reinterpret_cast<T *>(a.part) + (static_cast<int64_t>(chunk) * 2) * cols;
    T sum = splat<T>(0.0f);
    for (int i0 = 0; i0 < live; i0 += kAhead) {
        T v[kAhead], old[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = min(i0 + k, live - 1);
            const int64_t row = __builtin_amdgcn_readlane(mine.y, i);
            v[k] = on ? g[row * cols + col] : splat<T>(0.0f);
        }
        if (a.add)
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                old[k] = splat<T>(0.0f);
                if (i0 + k < live && ((ends >> (i0 + k)) & 1)) {
                    const int64_t id = __builtin_amdgcn_readlane(mine.x, i0 + k);
                    if (on) old[k] = dW[id * cols + col];
                }
            }
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            const int i = i0 + k;
            if (i >= live) break;
            sum += v[k];
            if ((ends >> i) & 1) {
                const int64_t id = __builtin_amdgcn_readlane(mine.x, i);
                if (on) {
                    if (open)
                        part[cols + col] = sum;
                    else
                        dW[id * cols + col] = a.add ? fma_of(a.scale, sum, old[k]) : a.scale * sum;
                }
                open = false;
                sum = splat<T>(0.0f);
            }
        }
    }
    if (((ends >> (live - 1)) & 1) == 0 && on) part[col] = sum;
}

// The runs of several chunks: workgroup (chunk, column block) takes the one that
// ends in its chunk and began earlier, if there is one.  Wave w adds the w-th
// quarter of its chunks, then the quarters are added in order.
template <typename T>
__global__ __launch_bounds__(kThreads) void join_kernel(const GatherArgs a) {
    __shared__ T red[kWaves][kWave];
    const int chunk = blockIdx.x + 1, p0 = chunk * a.chunk;
    const int key = a.order[p0].x;
    if (key >= a.V || a.order[p0 - 1].x != key) return;
    const int last = min(p0 + a.chunk, a.n) - 1;
    // Goes on behind this chunk: a later workgroup's.
    if (a.order[last].x == key && last + 1 < a.n && a.order[last + 1].x == key) return;
    const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    int first = chunk - 1;  // the run's first chunk: back from here while chunks start with this key, 64 at a time
    for (;;) {
        const int c = first - lane;
        const bool same = c > 0 && a.order[c * static_cast<int64_t>(a.chunk)].x == key &&
                          a.order[c * static_cast<int64_t>(a.chunk) - 1].x == key;
        const uint64_t others = __ballot(!same);
        if (others != 0) {
            first -= __builtin_ctzll(others);
            break;
        }
        first -= kWave;
    }
    const int count = chunk - first, per = (count + kWaves - 1) / kWaves;
    const int cols = a.C / (sizeof(T) / sizeof(float)), col = blockIdx.y * kWave + lane;
    const bool on = col < cols;
    const T *part = reinterpret_cast<const T *>(a.part);
    T sum = splat<T>(0.0f);
    if (on) {
        const int end = first + min(count, (w + 1) * per);
        int c = first + w * per;
        for (; c + 8 <= end; c += 8) {
            T v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = part[static_cast<int64_t>(c + k) * 2 * cols + col];
#pragma unroll
            for (int k = 0; k < 8; ++k) sum += v[k];
        }
        for (; c < end; ++c) sum += part[static_cast<int64_t>(c) * 2 * cols + col];
    }
    red[w][lane] = sum;
    __syncthreads();
    if (w != 0 || !on) return;
#pragma unroll
    for (int k = 1; k < kWaves; ++k) sum += red[k][lane];
    sum += part[(static_cast<int64_t>(chunk) * 2 + 1) * cols + col];
    T *at = reinterpret_cast<T *>(a.dW) + static_cast<int64_t>(key) * cols + col;
    *at = a.add ? fma_of(a.scale, sum, *at) : a.scale * sum;
}

__global__ __launch_bounds__(kThreads) void clear_kernel(float *p, int64_t n) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n; i += stride)
        p[i] = 0.0f;
}

// The rows sorted by (id, row); `clear`, if it has any, is zeroed on the way.
void launch_sort(const float *ids, int n, int V, int2 *order, Clear clear, hipStream_t s) {
    if (n <= kRankRows) {
        const int per = ((n + kRankSlices - 1) / kRankSlices + 3) & ~3;
        clear.blocks = (n + kRankPer - 1) / kRankPer;
        rank_kernel<<<dim3(clear.blocks + clear_blocks(clear, kRankThreads)), dim3(kRankThreads),
                      static_cast<size_t>(per) * kRankSlices * sizeof(uint32_t), s>>>(ids, n, V, order, clear);
        hipCheck(hipGetLastError());
        return;
    }
    int passes = 1;  // over the digits of V, the largest key
    while (passes < 4 && (V >> (8 * passes)) != 0) ++passes;
    const int blocks = (n + kSortBlock - 1) / kSortBlock;
    int2 *other = static_cast<int2 *>(alloc_cuda(sizeof(int2) * static_cast<size_t>(n)));
    int *hist = static_cast<int *>(alloc_cuda(sizeof(int) * kDigits * static_cast<size_t>(blocks)));
    const int64_t share = (clear.n + 3 * passes - 1) / (3 * passes);  // an equal part with every launch
    int64_t left = clear.n;
    auto part = [&](int before) {
        const Clear c{clear.at + (clear.n - left), std::min(left, share), before};
        left -= c.n;
        return c;
    };
    SortArgs a{ids, nullptr, passes & 1 ? order : other, hist, n, V, 0, blocks, {}};
    for (int p = 0; p < passes; ++p) {
        a.clear = part(blocks);
        digit_count_kernel<<<dim3(blocks + clear_blocks(a.clear, kSortThreads)), dim3(kSortThreads), 0, s>>>(a);
        hipCheck(hipGetLastError());
        const Clear c = part(1);
        digit_scan_kernel<<<dim3(1 + clear_blocks(c, kScanThreads)), dim3(kScanThreads), 0, s>>>(hist, kDigits * blocks, c);
        hipCheck(hipGetLastError());
        a.clear = part(blocks);
        digit_move_kernel<<<dim3(blocks + clear_blocks(a.clear, kSortThreads)), dim3(kSortThreads), 0, s>>>(a);
        hipCheck(hipGetLastError());
        a.ids = nullptr;
        a.in = a.out;
        a.out = a.out == order ? other : order;
        a.shift += 8;
    }
    free_cuda(hist);
    free_cuda(other);
}

template <typename T>
void launch_gather(const float *ids, GatherArgs a, hipStream_t s) {
    constexpr int kW = sizeof(T) / sizeof(float);
    const int cols = a.C / kW;
    a.blocks = (cols + kWave - 1) / kWave;
    // A wave each for 32 places, fewer where that leaves less than eight waves a CU.
    a.chunk = 32;
    while (a.chunk > 8 && static_cast<int64_t>(a.n) * a.blocks < 2048ll * a.chunk) a.chunk /= 2;
    const int chunks = (a.n + a.chunk - 1) / a.chunk;
    const int64_t items = static_cast<int64_t>(chunks) * a.blocks;
    CHECK_ERROR(items > INT32_MAX / 2, "Too many rows and columns for one call: %d x %d.", a.n, a.C);
    int2 *order = static_cast<int2 *>(alloc_cuda(sizeof(int2) * static_cast<size_t>(a.n)));
    a.part = static_cast<float *>(alloc_cuda(sizeof(float) * 2 * static_cast<size_t>(chunks) * a.C));
    a.order = order;
    Clear clear{nullptr, 0, 0};
    if (!a.add) {
        const int64_t n = static_cast<int64_t>(a.V) * a.C;
        if (aligned16(a.dW)) clear = {reinterpret_cast<f32x4_t *>(a.dW), n / 4, 0};
        const int64_t rest = n - 4 * clear.n;
        if (rest > 0) {
            clear_kernel<<<dim3(blocks_for(rest, kThreads)), dim3(kThreads), 0, s>>>(a.dW + 4 * clear.n, rest);
            hipCheck(hipGetLastError());
        }
    }
    launch_sort(ids, a.n, a.V, order, clear, s);
    const int gather_blocks = static_cast<int>((items + kWaves - 1) / kWaves);
    const int extra = a.dP != nullptr ? blocks_for(static_cast<int64_t>(a.positions) * cols, kThreads) : 0;
    gather_kernel<T><<<dim3(gather_blocks + extra), dim3(kThreads), 0, s>>>(a, static_cast<int>(items));
    hipCheck(hipGetLastError());
    if (chunks > 1) {
        join_kernel<T><<<dim3(chunks - 1, a.blocks), dim3(kThreads), 0, s>>>(a);
        hipCheck(hipGetLastError());
    }
    free_cuda(a.part);
    free_cuda(order);
}

// Checks shared by both directions; returns the number of ids.
int check_tables(const tensor_t *W, const char *name, const tensor_t *pos, const char *pos_name, const tensor_t *ids,
                 const tensor_t *rows, const char *rows_name) {
    check_gpu(W, name);
    check_gpu(ids, "ids");
    check_gpu(rows, rows_name);
    CHECK_ERROR(W->ndims != 2, "Expected %s to be (num_embeddings, embedding_dim), but got %d dims.", name, W->ndims);
    const int V = W->shape[0], C = W->shape[1], n = ids->length;
    CHECK_ERROR(V < 1 || C < 1, "Expected %s to have rows and columns, but got %d x %d.", name, V, C);
    CHECK_ERROR(n < 0 || static_cast<int64_t>(n) * C != rows->length,
                "Expected %s to hold %d x %d elements, but it holds %d.", rows_name, n, C, rows->length);
    if (pos != NULL) {
        check_gpu(pos, pos_name);
        CHECK_ERROR(pos->ndims != 2 || pos->shape[1] != C, "Expected %s to be (positions, %d).", pos_name, C);
        CHECK_ERROR(n > 0 && (ids->ndims < 1 || last_dim(ids) > pos->shape[0]),
                    "Expected at least %d rows of %s, but got %d.", last_dim(ids), pos_name, pos->shape[0]);
    }
    return n;
}

}  // namespace

}  // namespace gptc

using namespace gptc;

extern "C" void gptc_embedding_forward_scaled_cuda(const tensor_t *W, const tensor_t *pos, const tensor_t *ids,
                                                   const float scale, tensor_t *output) {
    const int n = check_tables(W, "W", pos, "pos", ids, output, "output");
    CHECK_ERROR(overlap(output, W) || overlap(output, ids) || (pos != NULL && overlap(output, pos)),
                "output may not overlap another tensor of the call.");
    if (n == 0) return;
    const int V = W->shape[0], C = W->shape[1], seq = pos != NULL ? last_dim(ids) : 1;
    const dim3 grid((n + kWaves - 1) / kWaves);
    hipStream_t s = gptc_stream_checked();
    if (C % 4 == 0 && aligned16(W->t) && aligned16(output->t) && (pos == NULL || aligned16(pos->t)))
        lookup_kernel<f32x4_t><<<grid, dim3(kThreads), 0, s>>>(
            reinterpret_cast<const f32x4_t *>(W->t), reinterpret_cast<const f32x4_t *>(pos != NULL ? pos->t : nullptr),
            ids->t, scale, reinterpret_cast<f32x4_t *>(output->t), n, seq, C / 4, V);
    else
        lookup_kernel<float><<<grid, dim3(kThreads), 0, s>>>(W->t, pos != NULL ? pos->t : nullptr, ids->t, scale,
                                                             output->t, n, seq, C, V);
    hipCheck(hipGetLastError());
}

extern "C" void gptc_embedding_backward_sorted_cuda(const tensor_t *global_grad, const tensor_t *ids,
                                                    const float scale, tensor_t *dW, tensor_t *dpos,
                                                    const int accumulate) {
    const int n = check_tables(dW, "dW", dpos, "dpos", ids, global_grad, "global_grad");
    CHECK_ERROR(overlap(dW, global_grad) || overlap(dW, ids) ||
                    (dpos != NULL && (overlap(dpos, global_grad) || overlap(dpos, ids) || overlap(dpos, dW))),
                "dW and dpos may not overlap another tensor of the call.");
    CHECK_ERROR(gptc_stream_capturing(), "gptc_embedding_backward_sorted_cuda takes scratch: not under graph capture.");
    hipStream_t s = gptc_stream_checked();
    const int V = dW->shape[0], C = dW->shape[1];
    if (n == 0) {
        if (accumulate) return;
        clear_kernel<<<dim3(blocks_for(dW->length, kThreads)), dim3(kThreads), 0, s>>>(dW->t, dW->length);
        hipCheck(hipGetLastError());
        if (dpos != NULL && dpos->length > 0) {
            clear_kernel<<<dim3(blocks_for(dpos->length, kThreads)), dim3(kThreads), 0, s>>>(dpos->t,
                                                                                                  dpos->length);
            hipCheck(hipGetLastError());
        }
        return;
    }
    const int seq = last_dim(ids);
    const GatherArgs a{global_grad->t, nullptr, dW->t, nullptr, scale, n, V, C, 0, 0, accumulate != 0,
                       dpos != NULL ? dpos->t : nullptr, n / seq, seq, dpos != NULL ? dpos->shape[0] : 0};
    if (C % 4 == 0 && aligned16(a.g) && aligned16(a.dW) && aligned16(a.dP))
        launch_gather<f32x4_t>(ids->t, a, s);
    else
        launch_gather<float>(ids->t, a, s);
}
