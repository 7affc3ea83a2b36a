// Drawing tokens from rows of logits (gptc_sample_cuda): temperature, top-k, top-p and min-p, then a draw from a
// given random number.  gpt.c's infer_gpt.c draws on the host from the softmax of one row (sample_mult); it has
// no filters.
//
// The filters each keep a head of one order, logits descending and equal ones by index, so their result is a
// bound: the last (logit, index) kept.  With M the row's maximum and weights w_i = exp((l_i - M) / T), top-k keeps
// the first k; top-p, of those, the shortest head whose weight reaches top_p of theirs; min-p the weights that are
// at least min_p.  The token is then the first, in the order of the vocabulary, at which the kept weights' sum
// passes u times their total.
//
// Sums decide which token comes out, so they are exact: weights are whole numbers, w 2^shift rounded from 64-bit
// floats, and every sum of them is a 64-bit integer, the same in any order (atomics too).  shift leaves room for a
// whole vocabulary (46 bits at 50257 tokens: a weight is off by at most 2^-47 of the largest).
//
// A workgroup of 1024 threads takes a row and passes over its logits, which stay in cache between the passes.
// Nothing is sorted:
//   maximum the first pass; greedy rows end there.
//   top-k   the k-th largest of the threads' own maxima is a lower bound of the k-th logit, and few tokens lie
//           above it: a second pass gathers them, they are ranked by counting, and the rest of the work is theirs.
//   else    a bound is found in histograms: over 8192 steps of (M - l) / T first, then over the bits of the logits
//           in the one step where the bound lies, until it holds at most 1024 tokens, which are ranked, or equal
//           logits only, whose order is that of the vocabulary.  The kept tokens are gathered where they are few, and
//           the draw finds the stretch of the vocabulary where the sum is passed, and the token in it.
// The weights bind it, eleven 64-bit operations each, and then the adds to the histogram.  Logits held in registers
// between the passes (49152 of a row at 512 threads) spilled more and came out 1.1 to 1.3 times as slow; as it is the
// kernel fills the 128 registers that 1024 threads leave each, and spills 11 (44 bytes a lane) outside its inner loops.
//
// MI355X, rows of 50257 logits: greedy 6 us, top-k 40 15 us, min-p 14 us, no filter 23 us, top-p 37 to 50 us, for one row
// as for 64.  256 rows of 131072 (134 MB): greedy 26 us (5.2 TB/s), top-k 54 us, top-p 97 to 142 us (three to four
// passes of 23 us or more).
#include <hip/hip_runtime.h>
#include <cstdint>
#include "gpu_kernels.h"
#include "ops_common.hpp"

namespace gptc {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kChunk = 8;            // logits of a thread that are worked on together, and that are on their way
constexpr int kBins = 8192;          // of a histogram; tokens that can be gathered
constexpr int kList = kThreads;      // tokens that can be ranked
constexpr int kTable = 32;           // entries of 8 bytes: one for every two LDS banks, so lanes never collide

struct SampleParams {
    const float *logits, *params, *u;
    float *ids, *prob;
    int V, param_rows, shift;
};

struct Token {
    float l;
    int i;
};

struct Lds {
    union {
        u64 mass[kBins];
        Token kept[kBins];
    };
    Token list[kList];
    u64 list_w[kList];
    u64 ahead[kList];
    double table[kTable];  // 2^(-j / 32)
    u64 wave_sum[kWaves];
    float wave_max[kWaves];
    uint32_t key_lo, key_hi;
    int n, found;
    u64 before;
    Token bound;
};

// Order-preserving bits of a float that is no NaN (-0 counts as 0), and back.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l + 0.0f);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __uint_as_float(k ^ (k >> 31 ? 0x80000000u : 0xffffffffu));
}

template <int kCtrl, int kRows>
__device__ __forceinline__ u64 dpp64(u64 v) {  // 0 where the control has no lane to read, or the row is not written
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(v), kCtrl, kRows, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(v >> 32), kCtrl, kRows, 0xf, false);
    return static_cast<u64>(hi) << 32 | lo;
}

// Inclusive sums over the lanes: within rows of 16 (shifts by 1, 2, 4 and 8), then the last lane of a row added to
// the next row, and that of the lower half to the upper.
__device__ __forceinline__ u64 wave_scan64(u64 v) {
    v += dpp64<0x111, 0xf>(v);
    v += dpp64<0x112, 0xf>(v);
    v += dpp64<0x114, 0xf>(v);
    v += dpp64<0x118, 0xf>(v);
    v += dpp64<0x142, 0xa>(v);
    return v + dpp64<0x143, 0xc>(v);
}

__device__ __forceinline__ int wave_scan32(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    return v + __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
}

__device__ __forceinline__ u64 lane_of(u64 v, int lane) {
    const uint32_t lo = __builtin_amdgcn_readlane(static_cast<int>(v), lane);
    const uint32_t hi = __builtin_amdgcn_readlane(static_cast<int>(v >> 32), lane);
    return static_cast<u64>(hi) << 32 | lo;
}

__device__ __forceinline__ u64 wave_sum64(u64 v) { return lane_of(wave_scan64(v), kWave - 1); }

// The sum over the workgroup (every thread gets it), and with `upto` the inclusive sums by thread.
__device__ __forceinline__ u64 block_sum64(Lds &s, u64 v, u64 *upto = nullptr) {
    const int w = threadIdx.x / kWave;
    u64 in = upto != nullptr ? wave_scan64(v) : wave_sum64(v);
    __syncthreads();
    if ((threadIdx.x & (kWave - 1)) == kWave - 1) s.wave_sum[w] = in;
    __syncthreads();
    u64 total = 0;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        const u64 x = s.wave_sum[i];
        if (upto != nullptr && i < w) in += x;
        total += x;
    }
    if (upto != nullptr) *upto = in;
    return total;
}

struct Row {
    const float *logits;
    int V;
    int from, to;  // the wave's stretch of the vocabulary
    float M;
    double per_entry;  // the weight is 2^(-(M - l) per_entry / kTable)
    int shift;
    float per_step;  // the histogram's steps by logit: monotone, whatever their rounding
    Token bound;
    u64 min_w;                  // the least weight that min-p keeps,
    float min_from, min_upto;   // and where it lies: before `from` every token is kept, from `upto` on none

    // NaN counts as -inf, and +inf as the largest number.
    static __device__ __forceinline__ float plain(float l) { return fminf(fmaxf(l, -INFINITY), 3.402823466e38f); }

    // What follows has no branches: the chains of a chunk's logits run side by side.
    __device__ __forceinline__ bool kept(float l, int i) const { return static_cast<int>(l > bound.l) | (static_cast<int>(l == bound.l) & static_cast<int>(i <= bound.i)); }

    // Where the logit lies in the histogram: kBins and more where the weight is nothing, 0 where the difference is 0
    // and the scale infinite (a vanishing temperature).
    __device__ __forceinline__ float step(float l) const { return fmaxf((M - l) * per_step, 0.0f); }

    // Where step(l) < kBins.  The exponent in steps of 1/32: a table's entry, and five terms of the exponential series
    // for the rest (at most ln 2 / 64: the next is below 2^-48 of the weight).  Whole numbers come out of additions of
    // 2^52, or 1.5 times that.  A table of 2048 entries with two terms took 1.4 times as long: its reads collide.
    __device__ __forceinline__ u64 weight(const Lds &s, float l) const {
        static_assert(kTable == 1 << 5, "the shift below");
        constexpr double kWhole = 6755399441055744.0, kLn = 0.6931471805599453 / kTable;
        const double t = (static_cast<double>(M) - static_cast<double>(l)) * per_entry;
        const double n = t + kWhole, x = (n - kWhole) - t;
        const int e = static_cast<int>(__double_as_longlong(n));
        double p = fma(x, kLn * kLn * kLn * kLn * kLn / 120, kLn * kLn * kLn * kLn / 24);
        p = fma(x, p, kLn * kLn * kLn / 6);
        p = fma(x, p, kLn * kLn / 2);
        p = fma(x, p, kLn);
        p = fma(x, p, 1.0) * s.table[e & (kTable - 1)];
        const double scale = __hiloint2double((1023 + shift - (e >> 5)) << 20, 0);
        return static_cast<u64>(__double_as_longlong(fma(p, scale, 4503599627370496.0))) & ((1ull << 52) - 1);
    }

    // Tokens i0 + lane + 64 e; -inf from `end` on.
    __device__ __forceinline__ void load(float (&l)[kChunk], int i0, int lane, int end) const {
        if (i0 + kChunk * kWave <= end) {
            const float *at = logits + i0 + lane;
#pragma unroll
            for (int e = 0; e < kChunk; ++e) l[e] = at[e * kWave];
#pragma unroll
            for (int e = 0; e < kChunk; ++e) l[e] = plain(l[e]);
            return;
        }
#pragma unroll
        for (int e = 0; e < kChunk; ++e) l[e] = logits[min(i0 + lane + e * kWave, V - 1)];
#pragma unroll
        for (int e = 0; e < kChunk; ++e) l[e] = i0 + lane + e * kWave < end ? plain(l[e]) : -INFINITY;
    }
};

// A wave's share of n tokens: contiguous, in whole turns of its lanes.
__device__ __forceinline__ int stretch(int n) { return (n + kThreads - 1) / kThreads * kWave; }

// f(l, i) over tokens from .. to of a wave in chunks: l[e] is the logit of token i + 64 e, -inf from `to` on.  The next
// chunk is on its way while this one is worked on.
template <typename F>
__device__ __forceinline__ void each(const Row &r, int from, int to, F f) {
    const int lane = threadIdx.x & (kWave - 1);
    float l[kChunk], next[kChunk];
    if (from < to) r.load(l, from, lane, to);
#pragma unroll 1
    for (int i = from; i < to; i += kChunk * kWave) {
        r.load(next, i + kChunk * kWave, lane, to);
        f(l, i + lane);
#pragma unroll
        for (int e = 0; e < kChunk; ++e) l[e] = next[e];
    }
}

// Gathers the tokens for which want(l); returns how many there are, of which the first `room` were written.  Their
// order is that of the waves' turns, so nothing may depend on it.  A token that the bound leaves out by its index
// alone is written as one of no weight.
template <typename F>
__device__ __forceinline__ int gather(const Row &r, Lds &s, Token *to, int room, F want) {
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    each(r, r.from, r.to, [&](const float (&l)[kChunk], int i) {
        uint32_t mask = 0;
#pragma unroll
        for (int e = 0; e < kChunk; ++e) mask |= want(l[e]) ? 1u << e : 0u;
        const int count = __popc(mask), upto = wave_scan32(count), all = __builtin_amdgcn_readlane(upto, kWave - 1);
        if (all == 0) return;
        int at = 0;
        // One for the wave: its lanes' would queue (top-k 3000 of 50257 tokens: 38 us with an add a lane, 31 us so).
        if ((threadIdx.x & (kWave - 1)) == 0) at = atomicAdd(&s.n, all);
        at = __builtin_amdgcn_readfirstlane(at) + upto - count;
        while (mask != 0) {
            if (at < room) to[at].i = i + (__ffs(mask) - 1) * kWave;
            ++at;
            mask &= mask - 1;
        }
    });
    __syncthreads();
    const int n = s.n;
    for (int j = threadIdx.x; j < min(n, room); j += kThreads) {
        const int i = to[j].i;
        const float l = Row::plain(r.logits[i]);
        to[j].l = r.kept(l, i) ? l : -INFINITY;
    }
    __syncthreads();
    return n;
}

// The same where few tokens are wanted: one comparison of wave masks for eight logits, most of which end there.
template <typename F>
__device__ __forceinline__ int gather_few(const Row &r, Lds &s, Token *to, int room, F want) {
    const u64 below = (1ull << (threadIdx.x & (kWave - 1))) - 1;
    __syncthreads();
    if (threadIdx.x == 0) s.n = 0;
    __syncthreads();
    each(r, r.from, r.to, [&](const float (&l)[kChunk], int i) {
        u64 who[kChunk], any = 0;
#pragma unroll
        for (int e = 0; e < kChunk; ++e) {
            who[e] = __ballot(want(l[e]));
            any |= who[e];
        }
        if (any == 0) return;
#pragma unroll
        for (int e = 0; e < kChunk; ++e) {
            if (who[e] == 0) continue;
            int at = 0;
            if (below == 0) at = atomicAdd(&s.n, __popcll(who[e]));
            at = __builtin_amdgcn_readfirstlane(at) + __popcll(who[e] & below);
            const int j = i + e * kWave;
            if ((who[e] & (below + 1)) != 0 && at < room) to[at] = Token{r.kept(l[e], j) ? l[e] : -INFINITY, j};
        }
    });
    __syncthreads();
    return s.n;
}

// ahead[i] = the sum over j < n of value(j) where before(j, i), for i < n <= kList: the pairs are shared out over
// all threads.
template <typename B, typename F>
__device__ __forceinline__ void sum_ahead(Lds &s, int n, B before, F value) {
    const int tid = threadIdx.x, parts = kThreads / n, i = tid % n, q = tid / n;
    __syncthreads();
    s.ahead[tid] = 0;
    __syncthreads();
    if (q < parts) {
        const int from = n * q / parts, to = n * (q + 1) / parts;
        u64 sum = 0;
        for (int j = from; j < to; ++j)
            if (before(j, i)) sum += value(j);
        if (sum != 0) atomicAdd(&s.ahead[i], sum);
    }
    __syncthreads();
}

__device__ __forceinline__ bool ahead_of(const Token &a, const Token &b) { return a.l > b.l || (a.l == b.l && a.i < b.i); }

// Finds in the histogram the step where `target` (counted in what it holds) is reached: its number, and what lies
// before it in `before`; -1 when the whole histogram holds less.  Each wave has a stretch of the steps.
__device__ int locate(Lds &s, u64 target, u64 &before) {
    constexpr int kPer = kBins / kThreads, kStretch = kPer * kWave;
    const int w = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    u64 sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) sum += s.mass[w * kStretch + e * kWave + lane];
    block_sum64(s, sum);
    u64 at = 0;
    int q = 0;
    while (q < kWaves && at + s.wave_sum[q] < target) at += s.wave_sum[q++];
    if (q == kWaves) return -1;
    if (w == q) {
        u64 v[kPer];
        sum = 0;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            v[e] = s.mass[w * kStretch + lane * kPer + e];
            sum += v[e];
        }
        at += wave_scan64(sum) - sum;
#pragma unroll
        for (int e = 0; e < kPer; ++e) {
            if (at < target && target <= at + v[e]) {
                s.found = w * kStretch + lane * kPer + e;
                s.before = at;
            }
            at += v[e];
        }
    }
    __syncthreads();
    before = s.before;
    return s.found;
}

__device__ __forceinline__ void clear(Lds &s) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kBins / kThreads; ++i) s.mass[i * kThreads + threadIdx.x] = 0;
    __syncthreads();
}

// The first token, in the order of the vocabulary, at which the sum of weigh(l, i) passes target(total); its
// weight, and the total.  Stretches first, then stretches of the one it lies in, then its tokens.  Where the total is
// known (not 0), the stretches are summed from the nearer end only as far as they have to.
template <typename W, typename T>
__device__ __forceinline__ int pick(const Row &r, Lds &s, W weigh, T target, u64 &weight, u64 &total) {
    const int w = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    auto sum_of = [&](int from, int to) {
        u64 sum = 0;
        each(r, from, to, [&](const float (&l)[kChunk], int i) {
#pragma unroll
            for (int e = 0; e < kChunk; ++e) sum += weigh(l[e], i + e * kWave);
        });
        return sum;
    };
    int lo, hi;
    u64 left;
    if (total != 0) {
        // Whole chunks of every thread: part of one takes as long.
        constexpr int kTurn = kChunk * kThreads;
        left = target(total);
        const bool back = left > total / 2;
        if (back) left = total - 1 - left;
        const int step = (r.V / 16 / kTurn + 1) * kTurn;
        lo = back ? max(r.V - step, 0) : 0;
        hi = back ? r.V : min(step, r.V);
#pragma unroll 1
        while (true) {
            const int len = stretch(hi - lo), a = min(lo + w * len, hi);
            const u64 sum = block_sum64(s, sum_of(a, min(a + len, hi)));
            if (left < sum || (back ? lo == 0 : hi == r.V)) {
                if (back) left = sum - 1 - min(left, sum - 1);
                break;
            }
            left -= sum;
            if (back) {
                hi = lo;
                lo = max(hi - step, 0);
            } else {
                lo = hi;
                hi = min(lo + step, r.V);
            }
        }
    } else {
        const u64 sum = wave_sum64(sum_of(r.from, r.to));
        __syncthreads();
        if (lane == 0) s.wave_sum[w] = sum;
        __syncthreads();
        for (int i = 0; i < kWaves; ++i) total += s.wave_sum[i];
        left = target(total);
        int q = 0;
        while (q < kWaves - 1 && left >= s.wave_sum[q]) left -= s.wave_sum[q++];
        const int len = stretch(r.V);
        lo = min(q * len, r.V);
        hi = min(lo + len, r.V);
    }
    while (hi - lo > kChunk * kWave) {
        const int len = stretch(hi - lo), a = min(lo + w * len, hi);
        const u64 sum = wave_sum64(sum_of(a, min(a + len, hi)));
        __syncthreads();
        if (lane == 0) s.wave_sum[w] = sum;
        __syncthreads();
        int q = 0;
        while (q < kWaves - 1 && left >= s.wave_sum[q]) left -= s.wave_sum[q++];
        lo = min(lo + q * len, hi);
        hi = min(lo + len, hi);
    }
    // Every wave does the last part, so that all end with the token.
    float l[kChunk];
    r.load(l, lo, lane, hi);
#pragma unroll
    for (int e = 0; e < kChunk; ++e) {
        const u64 mine = weigh(l[e], lo + e * kWave + lane), over_all = wave_scan64(mine);
        const u64 over = __ballot(over_all > left);
        if (over != 0) {
            const int at = __ffsll(over) - 1;
            weight = lane_of(mine, at);
            return lo + e * kWave + at;
        }
        left -= lane_of(over_all, kWave - 1);
    }
    weight = 0;
    return max(hi - 1, 0);  // not reached while target < total
}

// The weight that a head with `share` of the total has to reach.
__device__ __forceinline__ u64 head_of(double share, u64 total) {
    const double want = ceil(share * static_cast<double>(total));
    return want < 1.0 ? 1 : min(static_cast<u64>(want), total);
}

// Moves the row's bound to the last token of the shortest head of the order (of the tokens kept so far) that holds
// `target` tokens, or `share` of their weight.
//
// Returns how many tokens were gathered into s.kept on the way, all that are kept among them, or kBins + 1; and
// what is kept after min-p, in what the target counts, in `kept_sum` (0: not known).
__device__ __forceinline__ int bound_at(Row &r, Lds &s, bool mass, u64 target, double share, u64 &kept_sum) {
    const int tid = threadIdx.x;
    clear(s);
    const bool all = r.bound.l == -INFINITY;
    each(r, r.from, r.to, [&](const float (&l)[kChunk], int i) {
        u64 w[kChunk];
        if (mass) {
#pragma unroll
            for (int e = 0; e < kChunk; ++e) w[e] = r.weight(s, l[e]);
        } else {
#pragma unroll
            for (int e = 0; e < kChunk; ++e) w[e] = 1;
        }
#pragma unroll
        for (int e = 0; e < kChunk; ++e) {
            const float at = r.step(l[e]);
            if (at < kBins && (all || r.kept(l[e], i + e * kWave))) atomicAdd(&s.mass[static_cast<int>(at)], w[e]);
        }
    });
    __syncthreads();
    if (mass) {
        u64 sum = 0;
#pragma unroll
        for (int i = 0; i < kBins / kThreads; ++i) sum += s.mass[i * kThreads + tid];
        target = head_of(share, block_sum64(s, sum));
    }
    u64 before;
    int b = locate(s, target, before);
    kept_sum = 0;
    if (b < 0) return kBins + 1;  // fewer tokens than that have any weight
    target -= before;
    u64 ahead = before;
    if (mass && r.min_upto <= static_cast<float>(b)) return kBins + 1;  // min-p keeps less: the bound is its own
    // The tokens up to that step, and in it.
    const float from = static_cast<float>(b), upto = static_cast<float>(b + 1);
    // Gathered where they are few, going by the first ones of each wave.
    u64 some = 0;
    const int first_to = min(r.from + kChunk * kWave, r.to);
    each(r, r.from, first_to, [&](const float (&l)[kChunk], int) {
#pragma unroll
        for (int e = 0; e < kChunk; ++e) some += r.step(l[e]) < upto;
    });
    const bool few = static_cast<double>(block_sum64(s, some)) * r.V < static_cast<double>(kBins) * min(r.V, kChunk * kThreads);
    const int kept = few ? gather(r, s, s.kept, kBins, [&](float l) { return (r.step(l) < upto) & (l >= r.bound.l); }) : kBins + 1;
    if (tid == 0) s.n = 0;
    __syncthreads();
    if (kept <= kBins)
        for (int j = tid; j < kept; j += kThreads) {
            const Token t = s.kept[j];
            if (!(r.step(t.l) >= from)) continue;
            const int m = atomicAdd(&s.n, 1);
            if (m < kList) s.list[m] = t;
        }
    __syncthreads();
    int n = kept <= kBins ? s.n : gather(r, s, s.list, kList, [&](float l) {
        const float at = r.step(l);
        return (at >= from) & (at < upto) & (l >= r.bound.l);
    });
    bool first = true;  // and s.kept still holds the tokens
    uint32_t lo = 0, hi = 0;
    auto in_group = [&](float l, int i) {
        const uint32_t k = key_of(l);
        return r.kept(l, i) && (first ? static_cast<int>(r.step(l)) == b : k >= lo && k <= hi);
    };
    while (n > kList) {
        // The logits that the step holds; then its steps of them.
        __syncthreads();
        if (tid == 0) {
            s.key_lo = 0xffffffffu;
            s.key_hi = 0;
        }
        __syncthreads();
        uint32_t k0 = 0xffffffffu, k1 = 0;
        each(r, r.from, r.to, [&](const float (&l)[kChunk], int i) {
#pragma unroll
            for (int e = 0; e < kChunk; ++e) {
                if (!in_group(l[e], i + e * kWave)) continue;
                k0 = min(k0, key_of(l[e]));
                k1 = max(k1, key_of(l[e]));
            }
        });
        atomicMin(&s.key_lo, k0);
        atomicMax(&s.key_hi, k1);
        __syncthreads();
        lo = s.key_lo;
        hi = s.key_hi;
        first = false;
        if (lo == hi) {
            const float l = of_key(lo);
            if (mass) {
                const u64 w = r.weight(s, l);
                target = (target + w - 1) / w;
            }
            u64 weight, total = 0;
            const int i = pick(r, s, [&](float x, int j) { return static_cast<u64>(in_group(x, j)); },
                               [&](u64) { return target - 1; }, weight, total);
            r.bound = Token{l, i};
            return kBins + 1;  // the list made room for the histogram
        }
        const int bits = 32 - __clz(hi - lo), down = bits > 13 ? bits - 13 : 0;
        static_assert(kBins == 1 << 13, "steps of the logits' bits");
        clear(s);
        each(r, r.from, r.to, [&](const float (&l)[kChunk], int i) {
#pragma unroll
            for (int e = 0; e < kChunk; ++e) {
                if (!in_group(l[e], i + e * kWave)) continue;
                atomicAdd(&s.mass[(hi - key_of(l[e])) >> down], mass ? r.weight(s, l[e]) : 1ull);
            }
        });
        __syncthreads();
        b = locate(s, target, before);
        target -= before;
        ahead += before;
        hi -= static_cast<uint32_t>(b) << down;
        const uint32_t width = (1u << down) - 1;
        lo = hi - lo > width ? hi - width : lo;
        const float least = of_key(lo), most = of_key(hi);
        n = gather(r, s, s.list, kList, [&](float l) { return (l >= least) & (l <= most) & (l >= r.bound.l); });
    }
    if (tid < n) s.list_w[tid] = !mass ? 1 : r.step(s.list[tid].l) < kBins ? r.weight(s, s.list[tid].l) : 0;
    sum_ahead(s, n, [&](int j, int i) { return ahead_of(s.list[j], s.list[i]); },
              [&](int j) { return s.list_w[j]; });
    if (tid < n && s.ahead[tid] < target && target <= s.ahead[tid] + s.list_w[tid]) {
        s.bound = s.list[tid];
        s.before = s.ahead[tid] + s.list_w[tid];
    }
    __syncthreads();
    r.bound = s.bound;
    if (r.min_from >= upto) kept_sum = ahead + s.before;
    return first ? kept : kBins + 1;
}

// The sum that the drawn token passes.
__device__ __forceinline__ u64 draw_at(float u, u64 total) {
    const double t = u > 0.0f ? static_cast<double>(u) * static_cast<double>(total) : 0.0;
    return t < static_cast<double>(total) ? min(static_cast<u64>(t), total - 1) : total - 1;
}

__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams a) {
    __shared__ Lds s;
    const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid / kWave), lane = tid & (kWave - 1);
    const int row = blockIdx.x;
    Row r;
    r.logits = a.logits + static_cast<int64_t>(row) * a.V;
    r.V = a.V;
    r.from = min(w * stretch(a.V), a.V);
    r.to = min(r.from + stretch(a.V), a.V);
    const float *p = a.params + (a.param_rows > 1 ? 4 * row : 0);
    const float temperature = p[0], top_k = p[1], top_p = p[2], min_p = p[3], u = a.u[row];

    if (tid < kTable) s.table[tid] = exp2(-tid / static_cast<double>(kTable));

    auto block_max = [&](float x) {
        x = wave_max(x);
        __syncthreads();
        if (lane == 0) s.wave_max[w] = x;
        __syncthreads();
        x = s.wave_max[0];
#pragma unroll
        for (int i = 1; i < kWaves; ++i) x = fmaxf(x, s.wave_max[i]);
        return x;
    };
    auto answer = [&](int id, double prob) {
        a.ids[row] = static_cast<float>(id);
        if (a.prob != nullptr) a.prob[row] = static_cast<float>(prob);
    };
    if (!(temperature > 0.0f)) {
        Token top{-INFINITY, -1};
        each(r, r.from, r.to, [&](const float (&l)[kChunk], int i) {
#pragma unroll
            for (int e = 0; e < kChunk; ++e)
                if (l[e] > top.l) top = Token{l[e], i + e * kWave};
        });
        const float best = block_max(top.l);
        // The first place, as a float (V <= 2^24); -1 where there is none.
        const float first = block_max(top.l == best ? -static_cast<float>(top.i) : -INFINITY);
        if (tid == 0) answer(static_cast<int>(-first), best == -INFINITY ? 0.0 : 1.0);
        return;
    }
    float own_max = -INFINITY;
    each(r, r.from, r.to, [&](const float (&l)[kChunk], int) {
#pragma unroll
        for (int e = 0; e < kChunk; ++e) own_max = fmaxf(own_max, l[e]);
    });
    const float best = block_max(own_max);
    if (best == -INFINITY) {
        if (tid == 0) answer(-1, 0.0);
        return;
    }
    const double inv_t = 1.0 / static_cast<double>(fminf(temperature, 1e30f));
    r.M = best;
    r.shift = a.shift;
    r.per_entry = inv_t * (kTable * 1.4426950408889634);
    const double z_most = (a.shift + 2) * 0.6931471805599453 * 1.001;  // (M - l) / T from which on a weight is nothing
    r.per_step = static_cast<float>(inv_t * (kBins / z_most));
    r.bound = Token{-INFINITY, -1};
    const double one = static_cast<double>(1ull << a.shift);
    r.min_w = 1;
    r.min_from = r.min_upto = kBins;
    if (min_p > 0.0f) {  // (M - l) / T <= -log(min_p), with room for the roundings of both sides
        r.min_w = static_cast<u64>(ceil(fmin(static_cast<double>(min_p), 1.0) * one));
        const double z = fmax(-log(static_cast<double>(min_p)), 0.0), steps = kBins / z_most;
        r.min_from = static_cast<float>(fmin((z * 0.999 - 1e-3) * steps, kBins));
        r.min_upto = static_cast<float>(fmin((z * 1.001 + 1e-3) * steps, kBins));
    }
    const bool by_k = top_k >= 1.0f && top_k < static_cast<float>(a.V), by_p = top_p < 1.0f;
    const double share = fmax(static_cast<double>(top_p), 0.0);

    if (by_k) {
        const u64 k = static_cast<u64>(top_k);
        int n = kList + 1;
        if (k <= kList) {
            clear(s);
            const float own = r.step(own_max);
            if (own < kBins) atomicAdd(&s.mass[static_cast<int>(own)], 1ull);
            __syncthreads();
            u64 before;
            const int last = locate(s, k, before);
            if (last >= 0) {
                // The smallest of the maxima that were counted.
                const float bound = -block_max(own < static_cast<float>(last + 1) ? -own_max : -INFINITY);
                n = gather_few(r, s, s.list, kList, [&](float l) { return l >= bound; });
            }
        }
        if (n <= kList) {
            // All that counts is in the list: rank it, cut it, draw from it.
            auto before = [&](int j, int i) { return ahead_of(s.list[j], s.list[i]); };
            sum_ahead(s, n, before, [](int) { return 1ull; });
            Token mine{};
            int rank = kList;
            if (tid < n) {
                mine = s.list[tid];
                rank = static_cast<int>(s.ahead[tid]);
            }
            __syncthreads();
            if (rank < static_cast<int>(k)) s.list[rank] = mine;
            __syncthreads();
            n = static_cast<int>(k);
            u64 weight = 0, upto;
            if (tid < n) {
                mine = s.list[tid];
                weight = r.step(mine.l) < kBins ? r.weight(s, mine.l) : 0;
            }
            const u64 all = block_sum64(s, weight, &upto);
            if (by_p && upto - weight >= head_of(share, all)) weight = 0;
            if (weight < r.min_w) weight = 0;
            const u64 total = block_sum64(s, weight);
            if (tid < n) s.list_w[tid] = weight;
            sum_ahead(s, n, [&](int j, int i) { return s.list[j].i < s.list[i].i; }, [&](int j) { return s.list_w[j]; });
            const u64 at = draw_at(u, total);
            if (tid < n && weight != 0 && s.ahead[tid] <= at && at < s.ahead[tid] + weight)
                answer(mine.i, static_cast<double>(weight) / static_cast<double>(total));
            return;
        }
    }
    int n = kBins + 1;
    u64 kept_sum = 0;
#pragma unroll 1
    for (int mass = by_k ? 0 : 1; mass < (by_p ? 2 : 1); ++mass)
        n = bound_at(r, s, mass != 0, mass != 0 ? 0 : static_cast<u64>(top_k), share, kept_sum);
    if (!by_p) kept_sum = 0;  // it counts tokens

    auto weigh = [&](float l, int i) -> u64 {
        const u64 x = r.weight(s, l);
        const int in = static_cast<int>(r.kept(l, i)) & static_cast<int>(r.step(l) < kBins) & static_cast<int>(x >= r.min_w);
        return in ? x : 0;
    };
    if (by_k || by_p || min_p > 0.0f) {
        // The kept tokens, where they are few: not yet gathered, and not found to be many.
        if (n > kBins && r.bound.l == -INFINITY)
            n = gather(r, s, s.kept, kBins, [&](float l) { return (l >= r.bound.l) & (r.step(l) < r.min_upto); });
        if (n <= kBins) {
            const int per = (a.V + kList - 1) / kList;
            s.ahead[tid] = 0;
            __syncthreads();
            for (int j = tid; j < n; j += kThreads) {
                const Token t = s.kept[j];
                atomicAdd(&s.ahead[t.i / per], weigh(t.l, t.i));
            }
            __syncthreads();
            const u64 weight = s.ahead[tid];
            u64 upto;
            const u64 total = block_sum64(s, weight, &upto), at = draw_at(u, total);
            if (upto - weight <= at && at < upto) {
                s.found = tid;
                s.before = upto - weight;
            }
            if (tid == 0) s.n = 0;
            __syncthreads();
            const int found = s.found;
            const u64 left = at - s.before;
            for (int j = tid; j < n; j += kThreads) {
                const Token t = s.kept[j];
                if (t.i / per != found) continue;
                const u64 x = weigh(t.l, t.i);
                if (x == 0) continue;
                const int m = atomicAdd(&s.n, 1);
                if (m < kList) {
                    s.list[m] = t;
                    s.list_w[m] = x;
                }
            }
            __syncthreads();
            const int m = s.n;
            if (m <= kList) {
                sum_ahead(s, m, [&](int j, int i) { return s.list[j].i < s.list[i].i; }, [&](int j) { return s.list_w[j]; });
                if (tid < m && s.ahead[tid] <= left && left < s.ahead[tid] + s.list_w[tid])
                    answer(s.list[tid].i, static_cast<double>(s.list_w[tid]) / static_cast<double>(total));
                return;
            }
        }
    }
    auto target = [&](u64 sum) { return draw_at(u, sum); };
    u64 weight, total = kept_sum;
    int id;
    if (by_k || by_p || min_p > 0.0f)
        id = pick(r, s, weigh, target, weight, total);
    else
        id = pick(r, s, [&](float l, int) {
            const u64 x = r.weight(s, l);
            return r.step(l) < kBins ? x : 0;
        }, target, weight, total);
    if (tid == 0) answer(id, static_cast<double>(weight) / static_cast<double>(total));
}

}  // namespace
}  // namespace gptc

using namespace gptc;

extern "C" void gptc_sample_cuda(const tensor_t *logits, const tensor_t *params, const tensor_t *u, tensor_t *ids,
                                 tensor_t *prob) {
    check_gpu(logits, "logits");
    check_gpu(params, "params");
    check_gpu(u, "u");
    check_gpu(ids, "ids");
    const int V = last_dim(logits), rows = leading_rows(logits);
    CHECK_ERROR(logits->length > 0 && V > (1 << 24), "Vocabularies of up to 2^24 tokens are supported, but got %d.", V);
    CHECK_ERROR(rows >= (1 << 22), "Fewer than 2^22 rows are supported, but got %d.", rows);  // 2^32 threads
    CHECK_ERROR(params->length != 4 && params->length != 4 * static_cast<int64_t>(rows),
                "Expected 4 parameters, or 4 for each of %d rows, but got %d.", rows, params->length);
    CHECK_ERROR(u->length != rows, "Expected %d random numbers, but got %d.", rows, u->length);
    CHECK_ERROR(ids->length != rows, "Expected %d ids, but got %d.", rows, ids->length);
    if (prob != NULL) {
        check_gpu(prob, "prob");
        CHECK_ERROR(prob->length != rows, "Expected %d probabilities, but got %d.", rows, prob->length);
    }
    if (logits->length == 0 || rows == 0) return;
    // Rows are answered while others are still read.
    for (const tensor_t *out : {static_cast<const tensor_t *>(ids), static_cast<const tensor_t *>(prob)})
        CHECK_ERROR(out != NULL && (overlap(out, logits) || overlap(out, params) || overlap(out, u)),
                    "ids and prob may not overlap logits, params or u.");
    CHECK_ERROR(prob != NULL && overlap(ids, prob), "ids and prob may not overlap.");
    SampleParams a;
    a.logits = logits->t;
    a.params = params->t;
    a.u = u->t;
    a.ids = ids->t;
    a.prob = prob != NULL ? prob->t : nullptr;
    a.V = V;
    a.param_rows = params->length / 4;
    // V weights of up to 2^shift have to fit 62 bits, and one of them the 52 of a 64-bit float's fraction.
    int bits = 0;
    while ((1 << bits) < V) ++bits;
    a.shift = 62 - bits < 46 ? 62 - bits : 46;
    sample_kernel<<<dim3(rows), dim3(kThreads), 0, gptc_stream_checked()>>>(a);
    hipCheck(hipGetLastError());
}
