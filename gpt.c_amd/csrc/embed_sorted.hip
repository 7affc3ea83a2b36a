// Embedding lookup with scaling and positions, and its gradient by sorted
// tokens.  No counterpart in gpt.c, whose GPT2 looks both tables up apart and
// adds them sequence by sequence (src/transformer.c:69-111), and whose gradient
// walks the rows in turn (kernels/src/cpu/Embedding.c:27-47):
//   out[i] = s W[id[i]] (+ P[i mod T]);
//   dW[v] (+)= s sum of g[i] over id[i] = v;   dP[t] (+)= sum of g over i mod T = t.
//
// The gradient adds each id's rows in their order.  Up to 1024 rows find the
// others of their id by comparing; more are sorted by (id, row).  There a wave
// takes a fixed number of sorted places and 256 columns; an id whose rows go on
// into the next places leaves a partial sum, and a second kernel adds these in
// the order of their places.  So sums depend on the ids alone (no float atomics),
// and a token that fills the batch is shared by all waves.
#include <algorithm>
#include "gpu_kernels.h"
#include "ops_common.hpp"

namespace gptc {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxGroups = 1 << 24;  // a launch's threads are counted in 32 bits

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

// A wave a row; cols: columns in units of T.  8 x 1024 rows of 768 and their positions: 8.0 us, 53 MB that partly stay
// in the caches; 8 rows: 3.7, the launch.
template <typename T>
__global__ __launch_bounds__(kThreads) void lookup_kernel(const T *__restrict__ W, const T *__restrict__ P,
                                                         const float *__restrict__ ids, float scale,
                                                         T *__restrict__ out, int rows, int before, int seq, int cols,
                                                         int V) {
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
        const T *p = P + static_cast<int64_t>((static_cast<uint32_t>(before) + row) % seq) * cols;
        for (int j = lane; j < cols; j += kWave) o[j] = fma_of(scale, w[j], p[j]);
    } else {
        for (int j = lane; j < cols; j += kWave) o[j] = scale * w[j];
    }
}

// ---- sorting ----
// The sort's launches are short and mostly wait; where dW is to be overwritten, further workgroups of
// the same launches clear it meanwhile (8192 rows of 768 on 50257: 23 us for the ranking alone).  What is written of dW is
// marked as not to be read again soon, here and in the sums: the caches keep the rows that are read twice (the call 53 us
// without the marks, 40 with them; 65536 rows of 1600: 224, 208).
struct Clear {
    f32x4_t *at;  // n of them from here on, by the workgroups after the first `blocks` of a launch
    int64_t n;
    int blocks;
    const uint32_t *hit;  // or null; else n counts rows of `units`, of which those that are hit stay
    int units;
};

__device__ __forceinline__ void clear_part(const Clear &c) {
    if (c.hit != nullptr) {
        // A wave a row, 64 rows' flags at a time.
        const int lane = threadIdx.x & (kWave - 1), per = blockDim.x / kWave;
        const int64_t waves = static_cast<int64_t>(gridDim.x - c.blocks) * per;
        const int64_t first = static_cast<int64_t>(blockIdx.x - c.blocks) * per +
                              __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
        for (int64_t r0 = first; r0 < c.n; r0 += kWave * waves) {
            const int64_t mine = r0 + lane * waves;
            uint64_t left = __ballot(mine < c.n && c.hit[min(mine, c.n - 1)] == 0);
            for (; left != 0; left &= left - 1) {
                f32x4_t *row = c.at + (r0 + __builtin_ctzll(left) * waves) * c.units;
                for (int j = lane; j < c.units; j += kWave) __builtin_nontemporal_store(splat<f32x4_t>(0.0f), row + j);
            }
        }
        return;
    }
    const int64_t stride = static_cast<int64_t>(gridDim.x - c.blocks) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x - c.blocks) * blockDim.x + threadIdx.x; i < c.n; i += stride)
        __builtin_nontemporal_store(splat<f32x4_t>(0.0f), c.at + i);
}

// Workgroups for a part, up to `waves` waves in all (65536 rows of 1600: 208 us with 2048, 220 with 512).
constexpr int kClearWaves = 2048;
int clear_blocks(const Clear &c, int threads, int waves = kClearWaves) {
    const int64_t units = c.hit != nullptr ? c.n * kWave : c.n;
    return static_cast<int>(std::min<int64_t>((units + threads - 1) / threads, waves * kWave / threads));
}

// order[r] = (key, row) of the r-th row by (key, row); key: the id, V for rows
// without one.

// Up to kRankRows rows: a row's place is the number of rows before it, counted
// by comparing it with all of them, in one launch.
constexpr int kRankRows = 12288;
constexpr int kRankThreads = 512;
constexpr int kRankPer = 32;  // rows a workgroup
constexpr int kRankSlices = kRankThreads / kRankPer;
// Enough to clear while the others rank; more only fill the queues that the ids have to pass.  The call in us with 384, 448,
// 512, 576, 1024 and 2048 waves:
//   1100 rows of 768 on 50257: 37 33 32 35 33 34;  8192: 47 44 41 43 44 53;  12288: 56 56 57 58 61 72
//   1100 rows of 1600 on 50257: 66 59 61 69 63 63;  12288: 97 91 88 95 95 95
//   8192 rows of 512 on 130000: 63 58 56 61 60 60;  of 100 on 50257: 30 30 30 30 30 31;  of 768 on 5003: 38 in all
constexpr int kRankClearWaves = 512;

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
// Rows a thread: few rows in many workgroups of short chains (65536 rows of 1600 on 50257: the sort 52 us with 4,
// 72 with 16), until the counts of all workgroups cost their one summing workgroup more.
constexpr int kSortFew = 4, kSortMany = 16, kSortFewRows = 1 << 17;

struct SortArgs {
    const float *ids;  // the first pass reads the ids, the others `in`
    const int2 *in;
    int2 *out;
    int *hist;  // digit-major: (kDigits, blocks)
    int n, V, shift, blocks;
    uint32_t *hit;  // or null: set where an id occurs, by the first count
    Clear clear;
};

__device__ __forceinline__ int2 sort_item(const SortArgs &a, int i) {
    if (a.ids == nullptr) return a.in[i];
    const int id = id_of(a.ids[i], a.V);
    return make_int2(id < 0 ? a.V : id, i);
}

template <int kItems>
__global__ __launch_bounds__(kSortThreads) void digit_count_kernel(const SortArgs a) {
    if (static_cast<int>(blockIdx.x) >= a.blocks) {
        clear_part(a.clear);
        return;
    }
    __shared__ int count[kDigits];
    count[threadIdx.x] = 0;
    __syncthreads();
    const int first = blockIdx.x * (kSortThreads * kItems) + threadIdx.x;
    int key[kItems];
#pragma unroll
    for (int t = 0; t < kItems; ++t)
        key[t] = sort_item(a, min(first + t * kSortThreads, a.n - 1)).x;
#pragma unroll
    for (int t = 0; t < kItems; ++t)
        if (first + t * kSortThreads < a.n) {
            atomicAdd(&count[(key[t] >> a.shift) & (kDigits - 1)], 1);
            if (a.hit != nullptr && key[t] < a.V) a.hit[key[t]] = 1;  // all that write here write the same
        }
    __syncthreads();
    a.hist[threadIdx.x * a.blocks + blockIdx.x] = count[threadIdx.x];
}

// hist (n entries, n a multiple of 4) := its running sums, the entry itself left out; one workgroup,
// 16384 entries at a time in one exchange between its waves.
constexpr int kScanThreads = 1024;
constexpr int kScanParts = 4;
__global__ __launch_bounds__(kScanThreads) void digit_scan_kernel(int *hist, int n, Clear clear) {
    if (blockIdx.x > 0) {
        clear_part(clear);
        return;
    }
    constexpr int kW = kScanThreads / kWave;
    __shared__ int total[kScanParts * kW];
    const int lane = threadIdx.x & (kWave - 1), w = threadIdx.x / kWave, units = n / 4;
    int4 *at = reinterpret_cast<int4 *>(hist);
    int before = 0;
    for (int u0 = 0; u0 < units; u0 += kScanParts * kScanThreads) {
        int4 v[kScanParts];
        int up[kScanParts];  // this lane's entries and those of the lanes before it
#pragma unroll
        for (int k = 0; k < kScanParts; ++k) {
            const int u = u0 + k * kScanThreads + static_cast<int>(threadIdx.x);
            v[k] = u < units ? at[u] : make_int4(0, 0, 0, 0);
        }
#pragma unroll
        for (int k = 0; k < kScanParts; ++k) {
            up[k] = v[k].x + v[k].y + v[k].z + v[k].w;
#pragma unroll
            for (int off = 1; off < kWave; off <<= 1) {
                const int other = __shfl_up(up[k], off, kWave);
                up[k] += lane >= off ? other : 0;
            }
            if (lane == kWave - 1) total[k * kW + w] = up[k];
        }
        __syncthreads();
        // Every wave sums up all waves' totals for itself.
        static_assert(kScanParts * kW == kWave, "a total a lane");
        const int own = total[lane];
        int sum = own;
#pragma unroll
        for (int off = 1; off < kWave; off <<= 1) {
            const int other = __shfl_up(sum, off, kWave);
            sum += lane >= off ? other : 0;
        }
#pragma unroll
        for (int k = 0; k < kScanParts; ++k) {
            const int u = u0 + k * kScanThreads + static_cast<int>(threadIdx.x);
            int4 out;
            out.x = before + __shfl(sum - own, k * kW + w, kWave) + up[k] - (v[k].x + v[k].y + v[k].z + v[k].w);
            out.y = out.x + v[k].x;
            out.z = out.y + v[k].y;
            out.w = out.z + v[k].z;
            if (u < units) at[u] = out;
        }
        before += __shfl(sum, kWave - 1, kWave);
        __syncthreads();
    }
}

template <int kItems>
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
    const int first = blockIdx.x * (kSortThreads * kItems) + w * (kItems * kWave) + lane;
    int2 item[kItems];
#pragma unroll
    for (int t = 0; t < kItems; ++t) {
        const int i = first + t * kWave;
        item[t] = i < a.n ? sort_item(a, i) : make_int2(0, -1);
    }
#pragma unroll
    for (int t = 0; t < kItems; ++t)
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
    for (int t = 0; t < kItems; ++t) {
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

// dP[t] (+)= the sequences' rows t, in a fixed order; rows past the sequences' length: 0.
template <typename T>
__device__ __forceinline__ void position_sum(const GatherArgs &a, int t, int col) {
    const int cols = a.C / (sizeof(T) / sizeof(float));
    if (col >= cols || (a.add && t >= a.seq)) return;
    const int64_t n = static_cast<int64_t>(a.seq) * cols, i = static_cast<int64_t>(t) * cols + col;
    const T *g = reinterpret_cast<const T *>(a.g) + i;
    T *dP = reinterpret_cast<T *>(a.dP) + i;
    T sum = splat<T>(0.0f);
    if (t < a.seq) {
        int b = 0;
        for (; b + 8 <= a.seqs; b += 8) {
            T v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = g[(b + k) * n];
            // Eight by themselves, in pairs: one chain of 64 sequences was off by twice as much.
            sum += ((v[0] + v[1]) + (v[2] + v[3])) + ((v[4] + v[5]) + (v[6] + v[7]));
        }
        for (; b < a.seqs; ++b) sum += g[b * n];
    }
    *dP = a.add ? *dP + sum : sum;
}

// One wave: `chunk` sorted places x 64 columns in units of T, or such columns of a position.  Workgroups go
// through one block of columns after the other, so that the rows are still near when they are read for the
// second time (64 x 1024 rows of 1600, with the positions: 139 us; one chunk after the other 50 more).
template <typename T>
__global__ __launch_bounds__(kThreads) void gather_kernel(const GatherArgs a, int chunks) {
    constexpr int kAhead = 8;  // rows whose loads are on their way together
    const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int position_blocks = a.dP != nullptr ? (a.positions + kWaves - 1) / kWaves : 0;
    const int per = position_blocks + (chunks + kWaves - 1) / kWaves;
    const int block = blockIdx.x / per, at = blockIdx.x - block * per, col = block * kWave + lane;
    if (at < position_blocks) {
        if (at * kWaves + w < a.positions) position_sum<T>(a, at * kWaves + w, col);
        return;
    }
    const int chunk = (at - position_blocks) * kWaves + w;
    if (chunk >= chunks) return;
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
                        __builtin_nontemporal_store(a.add ? fma_of(a.scale, sum, old[k]) : a.scale * sum,
                                                    dW + id * cols + col);
                }
                open = false;
                sum = splat<T>(0.0f);
            }
        }
    }
    if (((ends >> (live - 1)) & 1) == 0 && on) part[col] = sum;
}

// The runs of several chunks: workgroup (chunk, column block) takes the one that ends in its chunk and began earlier, if
// there is one.  Wave w adds the w-th quarter of its chunks, then the quarters are added in order.  6 us at 8192 rows, 15
// at 65536 of 1600: a launch of short workgroups.
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

// ---- few rows: no sort ----

// Up to kFewRows rows, in one launch: a workgroup a row and 64 columns in units of T compares the row's id with all
// others, and if it is the first of its id adds their rows, a quarter of them a wave.  The first a.clears workgroups
// clear the rows that no id names.  3 x 333 rows of 100 on 5003: 5.6 us, sorted 13.2; 1000 of 768 on 50257: 26.2, sorted
// 29.6; of 1600: 56, sorted 63.  With room for more ids it is behind: 2048 rows of 768 on 50257 50.5, sorted 30.9.
constexpr int kFewRows = 1024;
constexpr int kFewItems = kFewRows / kThreads;  // ids a thread
constexpr int kClearRows = 1 << 16;             // whose ids are marked at a time

// `count` rows of C floats from `base` on to zero, but for those whose bit in `named` (LDS) is set, by `groups` workgroups
// together: 16 bytes at a time, whatever rows they belong to, so that what is written at a time is one stretch.
template <typename T>
__device__ __forceinline__ void clear_unnamed(float *base, int C, int count, const uint32_t *named, int groups) {
    auto stays = [&](int row) { return ((named[row / 32] >> (row % 32)) & 1) != 0; };
    auto clear = [](float *to) {
        __builtin_nontemporal_store(splat<f32x4_t>(0.0f), reinterpret_cast<f32x4_t *>(to));
    };
    const int total = count * C, step = 4 * kThreads * groups, rows = step / C, rest = step - rows * C;
    const int first = blockIdx.x * kThreads + threadIdx.x;
    int before = 0;  // the first whole 16 bytes
    if constexpr (sizeof(T) == sizeof(float)) {
        before = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(base) & 15)) / 4 & 3);
        if (first < min(before, total) && !stays(first / C)) base[first] = 0.0f;
    }
    int64_t at = before + 4ll * first;
    int row = static_cast<int>(at / C), in = static_cast<int>(at - static_cast<int64_t>(row) * C);
    for (; at < total; at += step) {
        if constexpr (sizeof(T) == sizeof(f32x4_t)) {
            if (!stays(row)) clear(base + at);
        } else {
            const bool one = in + 3 < C;  // of one row, else of two or more
            if (!stays(row) && (one || (C >= 4 && at + 3 < total && !stays(row + 1)))) {
                clear(base + at);
            } else if (!one) {
                int r = row, i = in;
                for (int e = 0; e < 4; ++e, ++i) {
                    if (i >= C) {
                        i = 0;
                        ++r;
                    }
                    if (at + e < total && !stays(r)) base[at + e] = 0.0f;
                }
            }
        }
        row += rows;
        in += rest;
        if (in >= C) {
            in -= C;
            ++row;
        }
    }
}

struct FewArgs {
    GatherArgs a;
    const float *ids;
    int clears, position_blocks;  // workgroups: the first ones, and the next ones of each block of columns
};

template <typename T>
__global__ __launch_bounds__(kThreads) void gather_few_kernel(const FewArgs f) {
    const GatherArgs &a = f.a;
    const int lane = threadIdx.x & (kWave - 1), w = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int cols = a.C / (sizeof(T) / sizeof(float));
    T *dW = reinterpret_cast<T *>(a.dW);
    // Wave w has rows w * 256 .. , 64 at a time.
    int key[kFewItems];
#pragma unroll
    for (int k = 0; k < kFewItems; ++k) {
        const int i = (w * kFewItems + k) * kWave + lane;
        key[k] = i < a.n ? id_of(f.ids[i], a.V) : -1;
    }
    if (static_cast<int>(blockIdx.x) < f.clears) {
        __shared__ uint32_t named[kClearRows / 32];
        for (int first = 0; first < a.V; first += kClearRows) {
            const int count = min(kClearRows, a.V - first);
            __syncthreads();
            for (int i = threadIdx.x; i < (count + 31) / 32; i += kThreads) named[i] = 0;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < kFewItems; ++k) {
                const int v = key[k] - first;
                if (key[k] >= 0 && v >= 0 && v < count) atomicOr(&named[v / 32], 1u << (v % 32));
            }
            __syncthreads();
            clear_unnamed<T>(a.dW + static_cast<int64_t>(first) * a.C, a.C, count, named, f.clears);
        }
        return;
    }
    __shared__ T red[kWaves][kWave];
    __shared__ int later;  // a row before this one has its id
    const int per = f.position_blocks + a.n, i = static_cast<int>(blockIdx.x) - f.clears;
    const int block = i / per, at = i - block * per, col = block * kWave + lane;
    if (at < f.position_blocks) {
        if (at * kWaves + w < a.positions) position_sum<T>(a, at * kWaves + w, col);
        return;
    }
    const int row = at - f.position_blocks, id = id_of(f.ids[row], a.V);
    if (id < 0) return;
    if (threadIdx.x == 0) later = 0;
    __syncthreads();
    uint64_t same[kFewItems];
    bool before = false;
#pragma unroll
    for (int k = 0; k < kFewItems; ++k) {
        const int i0 = (w * kFewItems + k) * kWave;
        same[k] = __ballot(key[k] == id);
        before = before || (row > i0 && (same[k] & (~0ull >> max(0, i0 + kWave - row))) != 0);
    }
    if (before && lane == 0) later = 1;
    __syncthreads();
    if (later) return;
    const bool on = col < cols;
    const T *g = reinterpret_cast<const T *>(a.g);
    T sum = splat<T>(0.0f);
#pragma unroll 1
    for (int k = 0; k < kFewItems; ++k) {
        constexpr int kAhead = 16;  // rows whose loads are on their way together
        uint64_t left = same[0];
#pragma unroll
        for (int q = 0; q + 1 < kFewItems; ++q) same[q] = same[q + 1];
        const int64_t i0 = (w * kFewItems + k) * kWave;
        while (left != 0) {
            T v[kAhead];
#pragma unroll
            for (int e = 0; e < kAhead; ++e) {
                v[e] = splat<T>(0.0f);
                if (left != 0) {
                    if (on) v[e] = g[(i0 + __builtin_ctzll(left)) * cols + col];
                    left &= left - 1;
                }
            }
#pragma unroll
            for (int e = 0; e < kAhead; ++e) sum += v[e];
        }
    }
    red[w][lane] = sum;
    __syncthreads();
    if (w != 0 || !on) return;
#pragma unroll
    for (int k = 1; k < kWaves; ++k) sum += red[k][lane];
    T *to = dW + static_cast<int64_t>(id) * cols + col;
    *to = a.add ? fma_of(a.scale, sum, *to) : a.scale * sum;
}

__global__ __launch_bounds__(kThreads) void clear_kernel(float *p, int64_t n) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * kThreads;
    for (int64_t i = blockIdx.x * static_cast<int64_t>(kThreads) + threadIdx.x; i < n; i += stride)
        p[i] = 0.0f;
}

// Rows times units that are worth flags: 34 MB are 7 us of writing at the rate of a copy, the flags' launch 4.6.
constexpr int64_t kHitUnits = 1 << 21;

// The rows sorted by (id, row); `clear`, if it has any, is zeroed on the way.
void launch_sort(const float *ids, int n, int V, int2 *order, Clear clear, hipStream_t s) {
    if (n <= kRankRows) {
        const int per = ((n + kRankSlices - 1) / kRankSlices + 3) & ~3;
        clear.blocks = (n + kRankPer - 1) / kRankPer;
        rank_kernel<<<dim3(clear.blocks + clear_blocks(clear, kRankThreads, kRankClearWaves)), dim3(kRankThreads),
                      static_cast<size_t>(per) * kRankSlices * sizeof(uint32_t), s>>>(ids, n, V, order, clear);
        hipCheck(hipGetLastError());
        return;
    }
    int passes = 1;  // over the digits of V, the largest key
    while (passes < 4 && (V >> (8 * passes)) != 0) ++passes;
    const bool few = n <= kSortFewRows;
    const int per = kSortThreads * (few ? kSortFew : kSortMany), blocks = (n + per - 1) / per;
    auto count_kernel = few ? digit_count_kernel<kSortFew> : digit_count_kernel<kSortMany>;
    auto move_kernel = few ? digit_move_kernel<kSortFew> : digit_move_kernel<kSortMany>;
    int2 *other = static_cast<int2 *>(alloc_cuda(sizeof(int2) * static_cast<size_t>(n)));
    int *hist = static_cast<int *>(alloc_cuda(sizeof(int) * kDigits * static_cast<size_t>(blocks)));
    // Rows of ids that occur are not cleared, where this spares more than the flags cost.
    uint32_t *hit = nullptr;
    if (clear.units > 0 && static_cast<int64_t>(std::min(n, V)) * clear.units >= kHitUnits) {
        hit = static_cast<uint32_t *>(alloc_cuda(sizeof(uint32_t) * static_cast<size_t>(V)));
        clear_kernel<<<dim3(blocks_for(V, kThreads)), dim3(kThreads), 0, s>>>(reinterpret_cast<float *>(hit), V);
        hipCheck(hipGetLastError());
    }
    // An equal part with every launch, but for the one that sets the flags.
    const int64_t unit = hit != nullptr ? clear.units : 1, count = clear.n / unit;
    const int shares = 3 * passes - (hit != nullptr);
    int64_t done = 0;
    auto part = [&](int before) {
        const int64_t n = std::min(count - done, (count + shares - 1) / shares);
        const Clear c{clear.at + done * unit, n, before, hit != nullptr ? hit + done : nullptr, clear.units};
        done += n;
        return c;
    };
    SortArgs a{ids, nullptr, passes & 1 ? order : other, hist, n, V, 0, blocks, hit, {}};
    for (int p = 0; p < passes; ++p) {
        a.clear = p == 0 && hit != nullptr ? Clear{} : part(blocks);
        count_kernel<<<dim3(blocks + clear_blocks(a.clear, kSortThreads)), dim3(kSortThreads), 0, s>>>(a);
        hipCheck(hipGetLastError());
        const Clear c = part(1);
        digit_scan_kernel<<<dim3(1 + clear_blocks(c, kScanThreads)), dim3(kScanThreads), 0, s>>>(hist, kDigits * blocks, c);
        hipCheck(hipGetLastError());
        a.clear = part(blocks);
        move_kernel<<<dim3(blocks + clear_blocks(a.clear, kSortThreads)), dim3(kSortThreads), 0, s>>>(a);
        hipCheck(hipGetLastError());
        a.ids = nullptr;
        a.hit = nullptr;
        a.in = a.out;
        a.out = a.out == order ? other : order;
        a.shift += 8;
    }
    if (hit != nullptr) free_cuda(hit);
    free_cuda(hist);
    free_cuda(other);
}

template <typename T>
void launch_gather(const float *ids, GatherArgs a, hipStream_t s) {
    constexpr int kW = sizeof(T) / sizeof(float);
    const int cols = a.C / kW;
    a.blocks = (cols + kWave - 1) / kWave;
    if (a.n <= kFewRows) {
        // Clearing: a workgroup a CU (26 rows of 1600 on 50257: 56 us; 272 workgroups 70, 512 61, as many as 16 KB each 58;
        // 1000 rows 56, 70, 64, 65), a few more where rows share 16 bytes (64 rows of 1601: 51 us with 320, 58 with 256, 64
        // with 384).
        const int64_t bytes = static_cast<int64_t>(a.V) * a.C * sizeof(float);
        FewArgs f{a, ids, 0, a.dP != nullptr ? (a.positions + kWaves - 1) / kWaves : 0};
        if (!a.add) f.clears = static_cast<int>(std::min<int64_t>(kW == 4 ? 256 : 320, (bytes + 16383) / 16384));
        const int64_t grid = static_cast<int64_t>(f.position_blocks + a.n) * a.blocks + f.clears;
        CHECK_ERROR(grid >= kMaxGroups, "Too many positions for one call: %d x %d.", a.positions, a.C);
        gather_few_kernel<T><<<dim3(static_cast<unsigned>(grid)), dim3(kThreads), 0, s>>>(f);
        hipCheck(hipGetLastError());
        return;
    }
    // A wave each for 32 places, fewer where that leaves less than eight waves a CU.
    a.chunk = 32;
    while (a.chunk > 8 && static_cast<int64_t>(a.n) * a.blocks < 2048ll * a.chunk) a.chunk /= 2;
    const int chunks = static_cast<int>((static_cast<int64_t>(a.n) + a.chunk - 1) / a.chunk);
    const int position_blocks = a.dP != nullptr ? (a.positions + kWaves - 1) / kWaves : 0;
    const int per = position_blocks + (chunks + kWaves - 1) / kWaves;
    CHECK_ERROR(static_cast<int64_t>(std::max(per, chunks)) * a.blocks >= kMaxGroups,
                "Too many rows or positions for one call: %d, %d x %d.", a.n, a.positions, a.C);
    int2 *order = static_cast<int2 *>(alloc_cuda(sizeof(int2) * static_cast<size_t>(a.n)));
    a.part = static_cast<float *>(alloc_cuda(sizeof(float) * 2 * static_cast<size_t>(chunks) * a.C));
    a.order = order;
    Clear clear{};
    if (!a.add) {
        const int64_t n = static_cast<int64_t>(a.V) * a.C;
        if (aligned16(a.dW)) clear = {reinterpret_cast<f32x4_t *>(a.dW), n / 4, 0, nullptr, a.C % 4 == 0 ? a.C / 4 : 0};
        const int64_t rest = n - 4 * clear.n;
        if (rest > 0) {
            clear_kernel<<<dim3(blocks_for(rest, kThreads)), dim3(kThreads), 0, s>>>(a.dW + 4 * clear.n, rest);
            hipCheck(hipGetLastError());
        }
    }
    launch_sort(ids, a.n, a.V, order, clear, s);
    gather_kernel<T><<<dim3(per * a.blocks), dim3(kThreads), 0, s>>>(a, chunks);
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
    const float *P = pos != NULL ? pos->t : nullptr;
    hipStream_t s = gptc_stream_checked();
    const bool vec = C % 4 == 0 && aligned16(W->t) && aligned16(output->t) && aligned16(P);
    // A wave a row, and as many launches as that takes (of more than 2^26 rows).
    constexpr int kMost = (kMaxGroups - 1) * kWaves;
    for (int64_t r = 0; r < n; r += kMost) {
        const int rows = static_cast<int>(std::min<int64_t>(n - r, kMost)), before = static_cast<int>(r % seq);
        const dim3 grid((rows + kWaves - 1) / kWaves);
        float *out = output->t + r * C;
        if (vec)
            lookup_kernel<f32x4_t><<<grid, dim3(kThreads), 0, s>>>(
                reinterpret_cast<const f32x4_t *>(W->t), reinterpret_cast<const f32x4_t *>(P), ids->t + r, scale,
                reinterpret_cast<f32x4_t *>(out), rows, before, seq, C / 4, V);
        else
            lookup_kernel<float><<<grid, dim3(kThreads), 0, s>>>(W->t, P, ids->t + r, scale, out, rows, before, seq, C, V);
        hipCheck(hipGetLastError());
    }
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
