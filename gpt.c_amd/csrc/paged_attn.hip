// Attention of a step's new tokens over keys and values in pages (include/paged.h).
//
// For query row (token i of its sequence, head h): with the sequence's keys and values j <= past + i,
//   t_j = (q . k_j) log2(e)/sqrt(D),  y = sum_j 2^(t_j - m) v_j / sum_j 2^(t_j - m),  m = max_j t_j,
// in one pass over the keys with a running m, sum and weighted sum, rescaled when m grows.  The query heads
// that share a kv head and the new tokens of a sequence are all rows of one product, 16 at a time, so a page is
// read once for a whole group, and single tokens and prompts run the same way.
//
// A workgroup takes an item of the plan: up to 16 rows and a range of keys, which its four waves take in turns
// of 16 (fp32 pages) or 32 (bf16) keys.  A wave's keys and values go from memory straight into the registers
// that the matrix instructions read: nothing is shared between waves, so LDS would only add a trip.  All
// products are transposed so that a lane holds one query (lane % 16):
//   S^T (keys x rows) = K Q^T.  K is the A operand: lane (m, g) = (lane % 16, lane / 16) holds values of key m.
//     The reduction may be taken in any order, so the lane reads 16 consecutive bytes of its key per load.
//   The result leaves lane (n, g) with t of row n and keys 4g .. 4g+3: m and the sums of a row are the lane's
//     own up to the four lanes n + 16 g, and p is, register for register, the B operand of the next product.
//   O^T (D x rows) += V^T P^T.  V^T is the A operand with row m of tile c standing for value m DP/16 + c, so
//     that lane m reads consecutive bytes of each value row (for bf16, where an operand register holds two
//     keys, 16-bit halves of two rows are swapped into place).
//
// fp32 pages are multiplied by v_mfma_f32_16x16x4_f32.  bf16 pages by v_mfma_f32_16x16x32_bf16 with the query
// and the weights as exact sums of three bf16 values (24 bits): three products at a sixteenth of the cost of an
// fp32 one each.  One or two rows over fp32 pages go without either (Dots).
//
// HBM bounds many or long contexts, each page being read once; round trips bound few and short ones.  MI355X: 64 tokens
// over up to 4000 keys, 12 heads of 64, fp32 (889 MB) 158 us, 5.6 TB/s; 16 over up to 30000, 32 heads on 8 of 128, bf16
// (836 MB) 154 us, 5.4 TB/s; one token over 300 keys 5.6 us.
#include <type_traits>
#include "hip_check.hpp"
#include "paged_attn_common.hpp"

namespace gptc {

namespace {

constexpr int kWaves = 4;

// A wave's operands: the query rows, and the keys and values of one turn.
template <typename T, int DP, Rows R>
struct Tile;

template <int DP, Rows R>
struct Tile<float, DP, R> {
    static constexpr int kGroups = 1;  // of 16 keys
    struct Q {
        uint32_t w[DP / 16][4];  // d = 16c + 4g + e
    };
    uint32_t k[DP / 16][4], v[4][DP / 64][4];  // v[i][h][c]: key 4g + i, d = 64h + 4m + c

    static __device__ __forceinline__ void load_q(Q &q, const float *row, int g, int D) {
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            if (row != nullptr) {
                load_words<float, 4, R, true>(q.w[c], row, 16 * c + 4 * g, D);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) q.w[c][e] = 0;
            }
        }
    }
    // kp, vp: row 0 of each group of 16 keys.
    __device__ __forceinline__ void load(const float *const (&kp)[1], const float *const (&vp)[1], int m, int g, int D) {
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) load_words<float, 4, R, false>(k[c], kp[0] + m * D, 16 * c + 4 * g, D);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < DP / 64; ++h)
                load_words<float, 4, R, false>(v[i][h], vp[0] + (4 * g + i) * D, 64 * h + 4 * m, D);
    }
    __device__ __forceinline__ void clear_values(int g, int left) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (4 * g + i >= left)
#pragma unroll
                for (int h = 0; h < DP / 64; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) v[i][h][c] = 0;
    }
    // Takes out what is not finite; whether there was any.
    __device__ __forceinline__ bool take_out() {
        bool any = false;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < DP / 64; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const uint32_t w = finite_part<float>(v[i][h][c]);
                    any |= w != v[i][h][c];
                    v[i][h][c] = w;
                }
        return any;
    }
    __device__ __forceinline__ void scores(const Q &q, f32x4 (&s)[1]) const {
        s[0] = zero4();
#pragma unroll
        for (int c = 0; c < DP / 16; ++c)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                s[0] = mfma16(__builtin_bit_cast(float, k[c][e]), __builtin_bit_cast(float, q.w[c][e]), s[0]);
    }
    __device__ __forceinline__ void values(const f32x4 (&p)[1], f32x4 (&o)[DP / 16]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < DP / 64; ++h)
#pragma unroll
                for (int c = 0; c < 4; ++c)
                    o[4 * h + c] = mfma16(__builtin_bit_cast(float, v[i][h][c]), p[0][i], o[4 * h + c]);
    }
    // o[4 (j / 4) + c][r], c < 4, are d .. d+3 of this row.
    static __device__ __forceinline__ int dim(int j, int g, int r) { return 16 * j + 16 * g + 4 * r; }
};

template <int DP, Rows R>
struct Tile<__bf16, DP, R> {
    static constexpr int kGroups = 2;
    static constexpr int kWords = DP / 32;  // of a value row per lane
    struct Q {
        uint32_t w[3][DP / 32][4];  // d = 32c + 8g + 2e, + 1
    };
    uint32_t k[2][DP / 32][4], v[8][kWords];  // v[j]: key 4g + j of the first group, or 4g + j - 4 of the second

    static __device__ __forceinline__ void load_q(Q &q, const float *row, int g, int D) {
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            uint32_t x[2][4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (row != nullptr) {
                    load_words<float, 4, R, true>(x[h], row, 32 * c + 8 * g + 4 * h, D);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[h][e] = 0;
                }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t p[3];
                split3(__builtin_bit_cast(float, x[e / 2][2 * (e % 2)]), __builtin_bit_cast(float, x[e / 2][2 * (e % 2) + 1]), p);
#pragma unroll
                for (int i = 0; i < 3; ++i) q.w[i][c][e] = p[i];
            }
        }
    }
    __device__ __forceinline__ void load(const __bf16 *const (&kp)[2], const __bf16 *const (&vp)[2], int m, int g, int D) {
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) load_words<__bf16, 4, R, false>(k[t][c], kp[t] + m * D, 32 * c + 8 * g, D);
#pragma unroll
        for (int j = 0; j < 8; ++j)
            load_words<__bf16, kWords, R, false>(v[j], vp[j / 4] + (4 * g + j % 4) * D, 2 * kWords * m, D);
    }
    __device__ __forceinline__ void clear_values(int g, int left) {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (16 * (j / 4) + 4 * g + j % 4 >= left)
#pragma unroll
                for (int c = 0; c < kWords; ++c) v[j][c] = 0;
    }
    __device__ __forceinline__ bool take_out() {
        bool any = false;
#pragma unroll
        for (int j = 0; j < 8; ++j)
#pragma unroll
            for (int c = 0; c < kWords; ++c) {
                const uint32_t w = finite_part<__bf16>(v[j][c]);
                any |= w != v[j][c];
                v[j][c] = w;
            }
        return any;
    }
    __device__ __forceinline__ void scores(const Q &q, f32x4 (&s)[2]) const {
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            s[t] = zero4();
#pragma unroll
            for (int i = 2; i >= 0; --i)  // the smallest parts first
#pragma unroll
                for (int c = 0; c < DP / 32; ++c) s[t] = mfma_bf16(k[t][c], q.w[i][c], s[t]);
        }
    }
    __device__ __forceinline__ void values(const f32x4 (&p)[2], f32x4 (&o)[DP / 16]) const {
        uint32_t w[3][4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t x[3];
            split3(p[e / 2][2 * (e % 2)], p[e / 2][2 * (e % 2) + 1], x);
#pragma unroll
            for (int i = 0; i < 3; ++i) w[i][e] = x[i];
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) {
            uint32_t a[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                a[e] = __builtin_amdgcn_perm(v[2 * e + 1][c / 2], v[2 * e][c / 2], c % 2 ? 0x07060302u : 0x05040100u);
#pragma unroll
            for (int i = 2; i >= 0; --i) o[c] = mfma_bf16(a, w[i], o[c]);
        }
    }
    static __device__ __forceinline__ int dim(int j, int g, int r) { return DP / 4 * g + DP / 16 * r + j; }
};

// One or two query rows over fp32 pages: a wave's products as multiplications and additions, sixteen lanes to a key.  Keys
// come in the layout of the values (lane (m, g) holds values 64h + 4m + c of key 4g + i), so that after the sums over m
// every lane has the weights that its values need.  The running maximum and sum are those of the lane's own g; they are
// joined after the last key.
// The matrix instruction takes 16 rows for the price of one: 12 heads of 64, one token over 300 keys 8.1 us by it, 5.6 us
// so; 8 heads of 128, 8 over 400 keys 18.7 and 9.8 us.  Four rows take as long or longer (32 heads on 8 of 128, 8 over
// 3500 keys: 43 us by the matrix instruction, 46 us so).
template <int DP, Rows R, int NR>
struct Dots {
    static constexpr int kH = DP / 64;
    uint32_t q[NR][kH][4];
    float m[NR], l[NR];
    f32x4 o[NR][kH];

    __device__ __forceinline__ void init(const float *const (&rows)[NR], int lane, int D) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int h = 0; h < kH; ++h) {
                o[r][h] = zero4();
                load_words<float, 4, R, true>(q[r][h], rows[r], 64 * h + 4 * (lane & 15), D);
            }
        }
    }
    static __device__ __forceinline__ void load(Tile<float, DP, R> &x, const float *kp, const float *vp, int m, int g, int D) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < kH; ++h) load_words<float, 4, R, false>(x.k[i * kH + h], kp + (4 * g + i) * D, 64 * h + 4 * m, D);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int h = 0; h < kH; ++h) load_words<float, 4, R, false>(x.v[i][h], vp + (4 * g + i) * D, 64 * h + 4 * m, D);
    }
    // key: of the lane's first; hides: some of the keys are past an end.
    __device__ __forceinline__ void step(const Tile<float, DP, R> &x, int key, const int (&end)[NR], bool hides, float scale_log2) {
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float s[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                s[i] = 0.0f;
#pragma unroll
                for (int h = 0; h < kH; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c)
                        s[i] = fmaf(__builtin_bit_cast(float, x.k[i * kH + h][c]), __builtin_bit_cast(float, q[r][h][c]), s[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[i] = row16_sum(s[i]) * scale_log2;
            if (hides) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (key + i >= end[r]) s[i] = -INFINITY;
            }
            const float mx = fmaxf(fmaxf(m[r], fmaxf(s[0], s[1])), fmaxf(s[2], s[3]));
            const float base = mx == -INFINITY ? 0.0f : mx;
            const float f = fast_exp2(m[r] - base);
            l[r] *= f;
#pragma unroll
            for (int h = 0; h < kH; ++h) o[r][h] *= f;
            m[r] = mx;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = fast_exp2(s[i] - base);
                l[r] += p;
#pragma unroll
                for (int h = 0; h < kH; ++h)
#pragma unroll
                    for (int c = 0; c < 4; ++c) o[r][h][c] = fmaf(p, __builtin_bit_cast(float, x.v[i][h][c]), o[r][h][c]);
            }
        }
    }
    // The wave's state of row r in all its lanes.
    __device__ __forceinline__ void join(int r) {
        const float big = max4_rows(m[r]);
        const float f = m[r] == -INFINITY ? l[r] : fast_exp2(m[r] - big);  // 0; NaN where a key's score was
        m[r] = big;
        l[r] = sum4_rows(l[r] * f);
#pragma unroll
        for (int h = 0; h < kH; ++h)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[r][h][c] = sum4_rows(o[r][h][c] * f);
    }
};

// Up to heads of 64 two workgroups share a CU, which the plan counts on: without the bound the kernel for bf16 rows that are
// no whole vectors took 260 registers and ran alone (12 heads of 60, 64 contexts of 2000: 163 us, with it 149 us).
template <typename T, int DP, Rows R>
__global__ __launch_bounds__(64 * kWaves, DP <= 64 ? 2 : 1) void paged_attn_kernel(const PagedAttnParams a) {
    using Step = Tile<T, DP, R>;
    constexpr int kKeys = 16 * Step::kGroups;
    static_assert(kPagedWideTarget <= kPagedTarget, "kMaxParts");
    static_assert(kKeys * kWaves == paged_unit(sizeof(T) == 2 ? GPTC_BF16 : GPTC_F32), "the plan's rounds");
    constexpr int kRow = DP + 4;  // floats of an LDS row: the four lanes of a row fall on other banks than its neighbours
    __shared__ __attribute__((aligned(16))) float o_s[kWaves][kPagedRows][kRow];
    __shared__ float m_s[kWaves][kPagedRows], l_s[kWaves][kPagedRows];
    __shared__ bool again_s[kWaves];

    const int item = blockIdx.x / a.KV, kv = blockIdx.x - item * a.KV;
    if (item >= a.head[1]) return;
    const PagedItem it = a.items[item];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int total = it.past + it.rows / a.group;  // the sequence's tokens: slots past them hold anything

    const int first_end = it.past + it.row0 / a.group + 1;  // the end of the first row's keys, which is the first
    // Row i of the item: its end, and its query, or NULL for rows that are not there.
    auto end_of = [&](int i) { return it.past + (it.row0 + i) / a.group + 1; };
    auto query_of = [&](int i) {
        const int row = it.row0 + i, token = row / a.group;
        const bool live = row < it.rows && it.tok0 + token < a.rows;
        return live ? a.q + static_cast<int64_t>(it.tok0 + token) * a.q_stride + (kv * a.group + row - token * a.group) * a.D
                    : nullptr;
    };

    const T *kpool = static_cast<const T *>(a.k), *vpool = static_cast<const T *>(a.v);
    const int *table = a.table + it.table;
    const int mask = (1 << a.page_shift) - 1;
    const int steps = (it.key1 - it.key0 - w * kKeys + kWaves * kKeys - 1) / (kWaves * kKeys);  // <= 0: none
    int pages[Step::kGroups];  // lane i: the pages of the wave's step i, i + 64, ...
    auto rows_of = [&](int i, const T *(&kp)[Step::kGroups], const T *(&vp)[Step::kGroups]) {
        if ((i & 63) == 0) {
#pragma unroll
            for (int t = 0; t < Step::kGroups; ++t) {
                const int key = it.key0 + (w + kWaves * (i + lane)) * kKeys + 16 * t;
                pages[t] = table[min(key, total - 1) >> a.page_shift];
            }
        }
        const int key = it.key0 + (w + kWaves * i) * kKeys;
#pragma unroll
        for (int t = 0; t < Step::kGroups; ++t) {
            const int64_t page = __builtin_amdgcn_readlane(pages[t], i & 63);
            const int64_t at = (((page * a.KV + kv) << a.page_shift) + ((key + 16 * t) & mask)) * a.D;
            kp[t] = kpool + at;
            vp[t] = vpool + at;
        }
    };
    bool again = false;  // see rows_by_key

    // All rows, on the matrix units.
    auto products = [&] {
        typename Step::Q q;
        Step::load_q(q, query_of(n), g, a.D);
        const int end = end_of(n);
        float m = -INFINITY, l = 0.0f;
        f32x4 o[DP / 16];
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) o[c] = zero4();
        auto step = [&](Step &x, int i) {
            const int key = it.key0 + (w + kWaves * i) * kKeys;
            if (key + kKeys > total) x.clear_values(g, total - key);
            if (key + kKeys > first_end) again |= x.take_out();
            f32x4 s[Step::kGroups];
            x.scores(q, s);
#pragma unroll
            for (int t = 0; t < Step::kGroups; ++t) settled(s[t]);
#pragma unroll
            for (int t = 0; t < Step::kGroups; ++t) s[t] *= a.scale_log2;
            if (key + kKeys > first_end) {
#pragma unroll
                for (int t = 0; t < Step::kGroups; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key + 16 * t + 4 * g + r >= end) s[t][r] = -INFINITY;
            }
            float mx = m;
#pragma unroll
            for (int t = 0; t < Step::kGroups; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[t][r]);
            mx = max4_rows(mx);
            const float base = mx == -INFINITY ? 0.0f : mx;  // no key of this row yet
            if (__any(mx > m)) {
                const float f = fast_exp2(m - base);
                l *= f;
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) o[c] *= f;
                m = mx;
            }
#pragma unroll
            for (int t = 0; t < Step::kGroups; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    s[t][r] = fast_exp2(s[t][r] - base);
                    l += s[t][r];
                }
            x.values(s, o);
        };
        // Two steps in turn: the loads of one are in flight while the other is multiplied.  Four, as below, were slower
        // here (16 heads of 128 on bf16 pages: 8 to 20 %), the matrix instructions of a step covering its loads.
        auto load_step = [&](Step &x, int i) {
            const T *kp[Step::kGroups], *vp[Step::kGroups];
            rows_of(i, kp, vp);
            x.load(kp, vp, n, g, a.D);
        };
        Step x, y;
        if (steps > 0) load_step(x, 0);
        for (int i = 0; i < steps; i += 2) {
            if (i + 1 < steps) load_step(y, i + 1);
            step(x, i);
            if (i + 1 >= steps) break;
            if (i + 2 < steps) load_step(x, i + 2);
            step(y, i + 1);
        }

        drain();
        l = sum4_rows(l);
        if (g == 0) {
            m_s[w][n] = m;
            l_s[w][n] = l;
        }
#pragma unroll
        for (int j = 0; j < DP / 16; j += 4)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                *reinterpret_cast<f32x4 *>(&o_s[w][n][Step::dim(j, g, r)]) = f32x4{o[j][r], o[j + 1][r], o[j + 2][r], o[j + 3][r]};
    };
    // One or two, fp32 pages.
    auto dots = [&](auto count) {
        constexpr int NR = decltype(count)::value, kAhead = 4;  // steps on their way: the work of one is short
        Dots<DP, R, NR> dots;
        const float *src[NR];
        int end[NR];
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            src[r] = query_of(r);
            if (src[r] == nullptr) src[r] = a.q;  // its result is not stored
            end[r] = end_of(r);
        }
        dots.init(src, lane, a.D);
        Step x[kAhead];
        auto load_step = [&](Step &x, int i) {
            const T *kp[Step::kGroups], *vp[Step::kGroups];
            rows_of(i, kp, vp);
            dots.load(x, kp[0], vp[0], n, g, a.D);
        };
#pragma unroll
        for (int i = 0; i < kAhead; ++i)
            if (i < steps) load_step(x[i], i);
        for (int i0 = 0; i0 < steps; i0 += kAhead) {
#pragma unroll
            for (int j = 0; j < kAhead; ++j) {
                const int i = i0 + j;
                if (i >= steps) break;
                const int key = it.key0 + (w + kWaves * i) * kKeys;
                if (key + kKeys > total) x[j].clear_values(g, total - key);
                const bool hides = key + kKeys > first_end;
                if (hides) again |= x[j].take_out();
                dots.step(x[j], key + 4 * g, end, hides, a.scale_log2);
                if (i + kAhead < steps) load_step(x[j], i + kAhead);
            }
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            dots.join(r);
            if (g != 0) continue;
            m_s[w][r] = dots.m[r];
            l_s[w][r] = dots.l[r];
#pragma unroll
            for (int h = 0; h < DP / 64; ++h) *reinterpret_cast<f32x4 *>(&o_s[w][r][64 * h + 4 * n]) = dots.o[r][h];
        }
    };
    const int n_rows = it.rows - it.row0;
    if constexpr (sizeof(T) == 4) {
        if (n_rows == 1)
            dots(std::integral_constant<int, 1>());
        else if (n_rows == 2)
            dots(std::integral_constant<int, 2>());
        else
            products();
    } else {
        products();
    }

    // The waves' states joined: sums of o 2^(m_w - M).
    again = __any(again);
    if (lane == 0) again_s[w] = again;
    __syncthreads();
    if (again_s[0] | again_s[1] | again_s[2] | again_s[3]) {
        constexpr int kEach = kPagedRows / kWaves;
        rows_by_key<T>(a, it, kv, it.row0 + kEach * w, kEach,
                       (static_cast<int64_t>(it.part) * a.KV + kv) * kPagedRows + kEach * w);
        return;
    }
    constexpr int kPerRow = 4 * kWaves;  // threads
    const int r = tid / kPerRow, place = tid % kPerRow;
    float big = m_s[0][r];
#pragma unroll
    for (int i = 1; i < kWaves; ++i) big = fmaxf(big, m_s[i][r]);
    float f[kWaves], sum = 0.0f;
#pragma unroll
    for (int i = 0; i < kWaves; ++i) {
        f[i] = m_s[i][r] == -INFINITY ? l_s[i][r] : fast_exp2(m_s[i][r] - big);  // 0; NaN where a key's score was
        sum = fmaf(l_s[i][r], f[i], sum);
    }
    const int out_row = it.row0 + r, out_token = it.tok0 + out_row / a.group;
    if (out_row >= it.rows || out_token >= a.rows) return;
    float *dst;
    float scale = 1.0f;
    if (it.part < 0) {
        dst = a.out + (static_cast<int64_t>(out_token) * a.H + kv * a.group + out_row % a.group) * a.D;
        scale = 1.0f / sum;
    } else {
        const int64_t slot = (static_cast<int64_t>(it.part) * a.KV + kv) * kPagedRows + r;
        dst = a.part_o + slot * a.D;
        if (place == 0) *reinterpret_cast<f32x2 *>(a.part_ml + 2 * slot) = f32x2{big, sum};
    }
    for (int d = 4 * place; d < a.D; d += 4 * kPerRow) {
        f32x4 y4 = zero4();
#pragma unroll
        for (int i = 0; i < kWaves; ++i) y4 += f[i] * *reinterpret_cast<const f32x4 *>(&o_s[i][r][d]);
        store4<R != kAny>(dst, d, a.D, y4 * scale);
    }
}

// The parts of rows whose keys were cut are joined by one launch, in two ways (paged_many).  Few parts: 16 rows a
// workgroup, 16 threads a row.
template <bool VEC>
__device__ __forceinline__ void merge_few(const PagedAttnParams &a, const PagedMerge &mg, int kv) {
    const int r = threadIdx.x >> 4, row = mg.row0 + r;
    const int token = mg.tok0 + row / a.group;
    if (row >= mg.rows || token >= a.rows) return;
    const int64_t first = (static_cast<int64_t>(mg.part0) * a.KV + kv) * kPagedRows + r;
    const int64_t next = static_cast<int64_t>(mg.step) * a.KV * kPagedRows;
    float big = -INFINITY;
#pragma unroll 4
    for (int p = 0; p < mg.n; ++p) big = fmaxf(big, a.part_ml[2 * (first + p * next)]);
    float *dst = a.out + (static_cast<int64_t>(token) * a.H + kv * a.group + row % a.group) * a.D;
    for (int d = 4 * (threadIdx.x & 15); d < a.D; d += 64) {
        f32x4 y = zero4();
        float sum = 0.0f;
#pragma unroll 4
        for (int p = 0; p < mg.n; ++p) {
            const f32x2 ml = *reinterpret_cast<const f32x2 *>(a.part_ml + 2 * (first + p * next));
            const float f = ml[0] == -INFINITY ? ml[1] : fast_exp2(ml[0] - big);
            sum = fmaf(ml[1], f, sum);
            y += f * load4<VEC>(a.part_o + (first + p * next) * a.D, d, a.D);
        }
        store4<VEC>(dst, d, a.D, y / sum);
    }
}

// Many parts: a workgroup takes one row.  Its threads weigh a part each, then sum the parts in groups of threads that
// hold four values each, and the groups' sums are added in order.
constexpr int kMergeThreads = 256;
constexpr int kMaxParts = kPagedTarget + 1;  // a tile is cut into at most target / kv heads + 1 items

template <bool VEC>
__device__ __forceinline__ void merge_many(const PagedAttnParams &a, const PagedMerge &mg, int kv, int r) {
    __shared__ float f_s[kMaxParts];
    __shared__ float red[2][kMergeThreads / 64];
    __shared__ __attribute__((aligned(16))) float y_s[kMergeThreads][4];
    const int row = mg.row0 + r, token = mg.tok0 + row / a.group;
    if (row >= mg.rows || token >= a.rows) return;
    const int64_t first = (static_cast<int64_t>(mg.part0) * a.KV + kv) * kPagedRows + r;
    const int64_t next = static_cast<int64_t>(mg.step) * a.KV * kPagedRows;
    const int tid = threadIdx.x, w = tid >> 6;
    __syncthreads();  // the workgroup's row before has been read
    float big = -INFINITY;
    for (int p = tid; p < mg.n; p += kMergeThreads) big = fmaxf(big, a.part_ml[2 * (first + p * next)]);
    big = wave_max(big);
    if ((tid & 63) == 0) red[0][w] = big;
    __syncthreads();
    big = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
    float sum = 0.0f;
    for (int p = tid; p < mg.n; p += kMergeThreads) {
        const f32x2 ml = *reinterpret_cast<const f32x2 *>(a.part_ml + 2 * (first + p * next));
        const float f = ml[0] == -INFINITY ? ml[1] : fast_exp2(ml[0] - big);
        f_s[p] = f;
        sum = fmaf(ml[1], f, sum);
    }
    sum = wave_sum(sum);
    if ((tid & 63) == 0) red[1][w] = sum;
    __syncthreads();
    sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
    const int lanes = a.D <= 64 ? 16 : 32, groups = kMergeThreads / lanes;  // 4 values a thread
    const int q = tid / lanes, d = tid % lanes * 4;
    f32x4 y = zero4();
    if (d < a.D) {
#pragma unroll 4
        for (int p = q; p < mg.n; p += groups) y += f_s[p] * load4<VEC>(a.part_o + (first + p * next) * a.D, d, a.D);
    }
    *reinterpret_cast<f32x4 *>(y_s[tid]) = y;
    __syncthreads();
    if (q > 0 || d >= a.D) return;
    for (int k = 1; k < groups; ++k) y += *reinterpret_cast<const f32x4 *>(y_s[k * lanes + tid]);
    store4<VEC>(a.out + (static_cast<int64_t>(token) * a.H + kv * a.group + row % a.group) * a.D, d, a.D, y / sum);
}

// Many parts of few rows go faster by the second (4 contexts of 1900, 32 heads on 8 of 128, bf16, 5 to 8 parts of 4 rows:
// 15.3 us with the attention by few, 12.9 by many; of 14 parts 17 and 5 us for the join alone); up to four parts take the
// same.  Full tiles of 16 rows by the first: a prompt of 1024 (up to 4 parts) 5 us by few and 14 by many, a chunk of 200 on
// 3000 keys (13 parts) 9 and 17 us.
//
// A workgroup takes what lies `gridDim.x` apart: a captured launch has no more of them than run at once, whatever the
// plan can hold.
template <bool VEC>
__global__ __launch_bounds__(kMergeThreads) void paged_merge_kernel(const PagedAttnParams a) {
    const int n_many = a.head[4], many = n_many * a.KV * a.merge_rows, all = many + (a.head[2] - n_many) * a.KV;
    for (int at = blockIdx.x; at < all; at += gridDim.x) {
        if (at < many) {
            const int i = at / (a.KV * a.merge_rows), left = at - i * a.KV * a.merge_rows, kv = left / a.merge_rows;
            merge_many<VEC>(a, a.merges[i], kv, left - kv * a.merge_rows);
        } else {
            const int few = at - many, i = few / a.KV;
            merge_few<VEC>(a, a.merges[n_many + i], few - i * a.KV);
        }
    }
}

template <typename T, int DP>
void launch(const PagedAttnParams &p, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(p.n_items) * p.KV);
    if (p.vec && p.D == DP)
        paged_attn_kernel<T, DP, kFull><<<grid, dim3(64 * kWaves), 0, s>>>(p);
    else if (p.vec)
        paged_attn_kernel<T, DP, kVec><<<grid, dim3(64 * kWaves), 0, s>>>(p);
    else
        paged_attn_kernel<T, DP, kAny><<<grid, dim3(64 * kWaves), 0, s>>>(p);
    hipCheck(hipGetLastError());
}

}  // namespace

void launch_paged_attention(const PagedAttnParams &p, hipStream_t s) {
    if (p.n_wide > 0) launch_paged_wide(p, s);
    if (p.n_items > 0) {
        if (p.bf16) {
            if (p.D <= 64) launch<__bf16, 64>(p, s);
            else launch<__bf16, 128>(p, s);
        } else {
            if (p.D <= 64) launch<float, 64>(p, s);
            else launch<float, 128>(p, s);
        }
    }
    const unsigned n = p.merge_groups;
    if (n == 0) return;
    if (p.vec) paged_merge_kernel<true><<<dim3(n), dim3(kMergeThreads), 0, s>>>(p);
    else paged_merge_kernel<false><<<dim3(n), dim3(kMergeThreads), 0, s>>>(p);
    hipCheck(hipGetLastError());
}

}  // namespace gptc
