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
// Nothing is sorted.  A bound is found in histograms: over 2048 steps of (M - l) / T first, then over the bits of
// the logits in the one step where the bound lies, until it holds at most 1024 tokens, which are ranked by
// counting, or equal logits only, whose order is that of the vocabulary.
#include <hip/hip_runtime.h>
#include <cstdint>
#include "gpu_kernels.h"
#include "ops_common.hpp"

namespace gptc {
namespace {

typedef unsigned long long u64;

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / kWave;
constexpr int kBins = 2048;
constexpr int kList = 1024;  // tokens that are ranked by counting: one for each thread

struct SampleParams {
    const float *logits, *params, *u;
    float *ids, *prob;
    int V, param_rows, shift;
};

// Order-preserving bits of a float that is no NaN.
__device__ __forceinline__ uint32_t key_of(float l) {
    const uint32_t b = __float_as_uint(l);
    return b ^ (b >> 31 ? 0xffffffffu : 0x80000000u);
}

struct Lds {
    unsigned count[kBins];
    u64 mass[kBins];
    float list_l[kList];
    int list_i[kList];
    u64 list_w[kList];
    u64 wave_sum[kWaves];
    float wave_max[kWaves];
    int wave_idx[kWaves];
    uint32_t key_lo, key_hi;
    int n, found;
    float bound_l;
    int bound_i;
    u64 before;
};

__device__ __forceinline__ u64 wave_sum64(u64 v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v += __shfl_xor(v, off, kWave);
    return v;
}

// Inclusive sums over the lanes.
__device__ __forceinline__ u64 wave_scan64(u64 v) {
    const int lane = threadIdx.x & (kWave - 1);
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const u64 o = __shfl_up(v, off, kWave);
        if (lane >= off) v += o;
    }
    return v;
}

struct Row {
    const float *logits;
    int V;
    float M, inv_t_f;     // inv_t_f, limit_f: the histograms' steps, monotone in the logit whatever their rounding
    double inv_t, limit;  // limit: where a weight rounds to nothing
    float limit_f, bin_scale;
    double one;  // 2^shift
    float bound_l;
    int bound_i;
    u64 min_w;

    __device__ __forceinline__ float at(int i) const { return fmaxf(logits[i], -INFINITY) + 0.0f; }  // NaN: -inf; -0: 0

    __device__ __forceinline__ bool kept(float l, int i) const { return l > bound_l || (l == bound_l && i <= bound_i); }

    __device__ __forceinline__ u64 weight(float l) const {
        if (l == M) return static_cast<u64>(one);
        const double z = (static_cast<double>(M) - static_cast<double>(l)) * inv_t;
        if (!(z < limit)) return 0;
        // Rounded to a whole number by the addition.
        const double r = fma(exp(-z), one, 4503599627370496.0);
        return static_cast<u64>(__double_as_longlong(r)) & ((1ull << 52) - 1);
    }

    // The histogram's step, or -1 where the weight is nothing.
    __device__ __forceinline__ int bin(float l) const {
        const float z = l == M ? 0.0f : (M - l) * inv_t_f;
        return z < limit_f ? min(static_cast<int>(z * bin_scale), kBins - 1) : -1;
    }
};

// Tokens lo + lane, lo + lane + 64, ... below hi: f(logit, index), eight loads in flight.
template <typename F>
__device__ __forceinline__ void each(const Row &r, int lo, int hi, F f) {
    constexpr int kAhead = 8;
    for (int i0 = lo + (threadIdx.x & (kWave - 1)); i0 < hi; i0 += kAhead * kWave) {
        float l[kAhead];
#pragma unroll
        for (int e = 0; e < kAhead; ++e) l[e] = i0 + e * kWave < hi ? r.at(i0 + e * kWave) : -INFINITY;
#pragma unroll
        for (int e = 0; e < kAhead; ++e)
            if (i0 + e * kWave < hi) f(l[e], i0 + e * kWave);
    }
}

// Every token of the row: each wave takes a contiguous stretch.
__device__ __forceinline__ int stretch(int n) { return (n + kWaves * kWave - 1) / (kWaves * kWave) * kWave; }

template <typename F>
__device__ __forceinline__ void all(const Row &r, F f) {
    const int w = threadIdx.x / kWave, len = stretch(r.V);
    each(r, min(w * len, r.V), min(w * len + len, r.V), f);
}

// The first token, in the order of the vocabulary, at which the sum of weigh(l, i) passes target(total); its
// weight, and the total.  Stretches first, then stretches of the one it lies in, then its tokens.
template <typename W, typename T>
__device__ int pick(const Row &r, Lds &s, W weigh, T target, u64 &weight, u64 &total) {
    const int w = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
    int lo = 0, hi = r.V;
    u64 left = 0;
    for (int level = 0; level < 2; ++level) {
        const int len = stretch(hi - lo);
        const int a = min(lo + w * len, hi), b = min(lo + w * len + len, hi);
        u64 sum = 0;
        each(r, a, b, [&](float l, int i) { sum += weigh(l, i); });
        sum = wave_sum64(sum);
        __syncthreads();
        if (lane == 0) s.wave_sum[w] = sum;
        __syncthreads();
        if (level == 0) {
            total = 0;
            for (int i = 0; i < kWaves; ++i) total += s.wave_sum[i];
            left = target(total);
        }
        int q = 0;
        while (q < kWaves - 1 && left >= s.wave_sum[q]) left -= s.wave_sum[q++];
        const int from = min(lo + q * len, hi);
        hi = min(from + len, hi);
        lo = from;
    }
    // Every wave does the last part, so that all end with the token.
    int last = lo;
    weight = 0;
    for (int i0 = lo; i0 < hi; i0 += kWave) {
        const int i = i0 + lane;
        const u64 mine = i < hi ? weigh(r.at(i), i) : 0;
        const u64 upto = wave_scan64(mine);
        const u64 over = __ballot(upto > left);
        if (over != 0) {
            const int at = __ffsll(over) - 1;
            weight = __shfl(mine, at, kWave);
            return i0 + at;
        }
        left -= __shfl(upto, kWave - 1, kWave);
        last = min(i0 + kWave, hi) - 1;
    }
    return last;  // not reached while target < total
}

// Finds in the histogram the step where `target` (counted in tokens, or in weight) is reached: its number, and what
// lies before it in before; -1 when the whole histogram holds less.
__device__ int locate(Lds &s, bool by_mass, u64 target, u64 &before) {
    constexpr int kPer = kBins / kThreads;
    const int tid = threadIdx.x, w = tid / kWave, lane = tid & (kWave - 1);
    u64 v[kPer], sum = 0;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        v[e] = by_mass ? s.mass[tid * kPer + e] : s.count[tid * kPer + e];
        sum += v[e];
    }
    const u64 upto = wave_scan64(sum);
    if (lane == kWave - 1) s.wave_sum[w] = upto;
    if (tid == 0) s.found = -1;
    __syncthreads();
    u64 at = upto - sum;
    for (int i = 0; i < w; ++i) at += s.wave_sum[i];
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
        if (at < target && target <= at + v[e]) {
            s.found = tid * kPer + e;
            s.before = at;
        }
        at += v[e];
    }
    __syncthreads();
    const int found = s.found;
    before = s.before;
    return found;
}

__device__ __forceinline__ void clear(Lds &s) {
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
        s.count[i] = 0;
        s.mass[i] = 0;
    }
    __syncthreads();
}

// Moves the row's bound to the last token of the shortest head of the order (of the tokens kept so far) that holds
// `target` tokens, or share of their weight.
template <bool MASS>
__device__ void bound_at(Row &r, Lds &s, u64 target, double share) {
    const int tid = threadIdx.x;
    clear(s);
    all(r, [&](float l, int i) {
        const int b = r.bin(l);
        if (b < 0 || !r.kept(l, i)) return;
        atomicAdd(&s.count[b], 1u);
        if constexpr (MASS) atomicAdd(&s.mass[b], r.weight(l));
    });
    __syncthreads();
    if constexpr (MASS) {
        u64 sum = 0;
        for (int i = tid; i < kBins; i += kThreads) sum += s.mass[i];
        sum = wave_sum64(sum);
        if ((tid & (kWave - 1)) == 0) s.wave_sum[tid / kWave] = sum;
        __syncthreads();
        sum = 0;
        for (int i = 0; i < kWaves; ++i) sum += s.wave_sum[i];
        const double want = ceil(share * static_cast<double>(sum));
        target = want < 1.0 ? 1 : static_cast<u64>(want);
        if (target > sum) target = sum;
        __syncthreads();
    }
    u64 before;
    int b = locate(s, MASS, target, before);
    if (b < 0) return;  // fewer tokens than that have any weight
    target -= before;
    int n = s.count[b];
    bool first = true;
    uint32_t lo = 0, hi = 0;
    auto in_group = [&](float l, int i) {
        if (!r.kept(l, i)) return false;
        if (first) return r.bin(l) == b;
        const uint32_t k = key_of(l);
        return k >= lo && k <= hi;
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
        all(r, [&](float l, int i) {
            if (!in_group(l, i)) return;
            k0 = min(k0, key_of(l));
            k1 = max(k1, key_of(l));
        });
        atomicMin(&s.key_lo, k0);
        atomicMax(&s.key_hi, k1);
        __syncthreads();
        lo = s.key_lo;
        hi = s.key_hi;
        first = false;
        if (lo == hi) {
            const float l = __uint_as_float(lo ^ (lo >> 31 ? 0x80000000u : 0xffffffffu));
            if constexpr (MASS) {
                const u64 w = r.weight(l);
                target = (target + w - 1) / w;
            }
            u64 weight, total;
            const int i = pick(r, s, [&](float x, int j) { return static_cast<u64>(in_group(x, j)); },
                               [&](u64) { return target - 1; }, weight, total);
            r.bound_l = l;
            r.bound_i = i;
            return;
        }
        const int bits = 32 - __clz(hi - lo), down = bits > 11 ? bits - 11 : 0;
        clear(s);
        all(r, [&](float l, int i) {
            if (!in_group(l, i)) return;
            const int at = static_cast<int>((hi - key_of(l)) >> down);
            atomicAdd(&s.count[at], 1u);
            if constexpr (MASS) atomicAdd(&s.mass[at], r.weight(l));
        });
        __syncthreads();
        b = locate(s, MASS, target, before);
        target -= before;
        n = s.count[b];
        hi -= static_cast<uint32_t>(b) << down;
        const uint32_t width = (1u << down) - 1;
        lo = hi - lo > width ? hi - width : lo;
    }
    __syncthreads();
    if (tid == 0) s.n = 0;
    __syncthreads();
    all(r, [&](float l, int i) {
        if (!in_group(l, i)) return;
        const int at = atomicAdd(&s.n, 1);
        s.list_l[at] = l;
        s.list_i[at] = i;
        if constexpr (MASS) s.list_w[at] = r.weight(l);
    });
    __syncthreads();
    if (tid < n) {
        const float l = s.list_l[tid];
        const int i = s.list_i[tid];
        u64 ahead = 0;
        for (int j = 0; j < n; ++j)
            if (s.list_l[j] > l || (s.list_l[j] == l && s.list_i[j] < i)) ahead += MASS ? s.list_w[j] : 1;
        if (ahead < target && target <= ahead + (MASS ? s.list_w[tid] : 1)) {
            s.bound_l = l;
            s.bound_i = i;
        }
    }
    __syncthreads();
    r.bound_l = s.bound_l;
    r.bound_i = s.bound_i;
}

__global__ __launch_bounds__(kThreads) void sample_kernel(const SampleParams a) {
    __shared__ Lds s;
    const int tid = threadIdx.x, w = tid / kWave, lane = tid & (kWave - 1);
    const int row = blockIdx.x;
    Row r;
    r.logits = a.logits + static_cast<int64_t>(row) * a.V;
    r.V = a.V;
    const float *p = a.params + (a.param_rows > 1 ? 4 * row : 0);
    float temperature = p[0];
    const float top_k = p[1], top_p = p[2], min_p = p[3], u = a.u[row];

    // The maximum and its first place.
    float best = -INFINITY;
    int where = a.V;
    all(r, [&](float l, int i) {
        if (l > best) {
            best = l;
            where = i;
        }
    });
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) {
        const float l = __shfl_xor(best, off, kWave);
        const int i = __shfl_xor(where, off, kWave);
        if (l > best || (l == best && i < where)) {
            best = l;
            where = i;
        }
    }
    if (lane == 0) {
        s.wave_max[w] = best;
        s.wave_idx[w] = where;
    }
    __syncthreads();
    best = s.wave_max[0];
    where = s.wave_idx[0];
    for (int i = 1; i < kWaves; ++i)  // stretches rise: an equal one later is further back
        if (s.wave_max[i] > best) {
            best = s.wave_max[i];
            where = s.wave_idx[i];
        }
    if (best == -INFINITY || !(temperature > 0.0f)) {
        if (tid == 0) {
            const bool none = best == -INFINITY;
            a.ids[row] = none ? -1.0f : static_cast<float>(where);
            if (a.prob != nullptr) a.prob[row] = none ? 0.0f : 1.0f;
        }
        return;
    }
    r.M = best;
    temperature = fminf(temperature, 1e30f);
    r.inv_t = 1.0 / static_cast<double>(temperature);
    r.limit = (a.shift + 2) * 0.6931471805599453;
    r.limit_f = static_cast<float>(r.limit) * 1.001f;
    r.inv_t_f = static_cast<float>(r.inv_t);
    r.bin_scale = kBins / r.limit_f;
    r.one = static_cast<double>(1ull << a.shift);
    r.bound_l = -INFINITY;
    r.bound_i = a.V;
    r.min_w = min_p > 0.0f ? static_cast<u64>(ceil(fmin(static_cast<double>(min_p), 1.0) * r.one)) : 1;

    if (top_k >= 1.0f && top_k < static_cast<float>(a.V)) bound_at<false>(r, s, static_cast<u64>(top_k), 0.0);
    if (top_p < 1.0f) bound_at<true>(r, s, 0, fmax(static_cast<double>(top_p), 0.0));

    u64 weight, total;
    const int id = pick(r, s,
                        [&](float l, int i) -> u64 {
                            if (!r.kept(l, i) || r.bin(l) < 0) return 0;
                            const u64 x = r.weight(l);
                            return x >= r.min_w ? x : 0;
                        },
                        [&](u64 sum) {
                            const double t = u > 0.0f ? static_cast<double>(u) * static_cast<double>(sum) : 0.0;
                            return t < static_cast<double>(sum) ? min(static_cast<u64>(t), sum - 1) : sum - 1;
                        },
                        weight, total);
    if (tid == 0) {
        a.ids[row] = static_cast<float>(id);
        if (a.prob != nullptr) a.prob[row] = static_cast<float>(static_cast<double>(weight) / static_cast<double>(total));
    }
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
    CHECK_ERROR(params->length != 4 && params->length != 4 * static_cast<int64_t>(rows),
                "Expected 4 parameters, or 4 for each of %d rows, but got %d.", rows, params->length);
    CHECK_ERROR(u->length != rows, "Expected %d random numbers, but got %d.", rows, u->length);
    CHECK_ERROR(ids->length != rows, "Expected %d ids, but got %d.", rows, ids->length);
    if (prob != NULL) {
        check_gpu(prob, "prob");
        CHECK_ERROR(prob->length != rows, "Expected %d probabilities, but got %d.", rows, prob->length);
    }
    if (logits->length == 0 || rows == 0) return;
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
