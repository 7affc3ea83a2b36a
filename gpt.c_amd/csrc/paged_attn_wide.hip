// The attention of csrc/paged_attn.hip for many query rows of one sequence (prompts and their chunks).
//
// There every 16 rows read all their keys from memory again, which binds it once a sequence brings more than a few
// tiles of rows.  Here a workgroup takes 64 rows (bf16 pages) or 128 (fp32), 16 or 32 for each of its waves,
// and the waves share each tile of keys and values through LDS: while a tile is multiplied the next one is on its way
// to registers, and it is written to the other of two LDS buffers, so a tile costs one barrier (kBuffers).
//
// All products run on v_mfma_f32_16x16x32_bf16 with operands that are exact sums of bf16 values ("parts"): queries
// and weights have three, bf16 pages one and fp32 pages three.  Products of parts below 2^-24 of the whole are left
// out, which leaves three for bf16 pages and six for fp32 pages, at a sixteenth of the cost of an fp32 product each.
// Parts of keys and values are formed once per tile, as it goes to LDS.
//   K tile: [part][key][D], rows padded by 16 bytes: the 16 rows that lanes read together start on other banks.
//   V tile: [part][d][keys], transposed on the way by swapping 16-bit halves in registers, the keys of 32 in the
//     order in which the scores' product leaves them with the lanes: place 8 g + j holds key 16 (j / 4) + 4 g + j % 4,
//     so a lane reads its eight keys as 16 bytes.
//
// The matrix cores bound long chunks: 2048 tokens on 8192 bf16 keys, 32 heads on 8 of 128, take 900 us, 344 TFLOP/s or
// 1031 in bf16 products (MI355X; a library product of 8192 reaches 1254).  A prompt of 1024, 12 heads of 64, fp32, has one
// workgroup a CU, whose waves do their loads, splits, products and exponentials in step: 21 us and 5 to join, where the
// products alone would take 8.
#include <mutex>
#include "hip_check.hpp"
#include "paged_attn_common.hpp"

namespace gptc {

namespace {

template <typename T>
constexpr int kType = sizeof(T) == 4 ? GPTC_F32 : GPTC_BF16;
template <typename T, int DP>
struct Shape {
    static constexpr int kParts = sizeof(T) == 4 ? 3 : 1;
    static constexpr int kKeys = paged_wide_keys(kType<T>, DP);
    static constexpr int kKRow = DP + 8;      // bf16 values of an LDS row
    static constexpr int kVRow = kKeys + 8;
    static constexpr int kKPart = kKeys * kKRow, kVPart = DP * kVRow;
    static constexpr int kBuffer = kParts * (kKPart + kVPart);
    // Two of fp32 pages with heads past 64 would take 114 KB and leave a CU to one workgroup: one is 1.04 times as fast
    // there at a second barrier, and 1.07 to 1.15 times once two workgroups share the CU.
    static constexpr int kBuffers = sizeof(T) == 4 && DP > 64 ? 1 : 2;
};

// Two floats as three bf16 values each, packed in pairs.
__device__ __forceinline__ void parts_of(uint32_t x0, uint32_t x1, uint32_t (&p)[3]) {
    split3(__builtin_bit_cast(float, x0), __builtin_bit_cast(float, x1), p);
}

// G: groups of 16 rows that a wave takes.  Two read each operand from LDS once for both.
template <typename T, int DP, Rows R, int G, int THREADS>
__global__ __launch_bounds__(THREADS, 2) void paged_wide_kernel(const PagedAttnParams a) {
    using S = Shape<T, DP>;
    constexpr int kThreads = THREADS, kKeys = S::kKeys, kParts = S::kParts, kTiles = kKeys / 16;
    extern __shared__ __attribute__((aligned(16))) uint16_t lds[];
    __shared__ int again_s;  // see rows_by_key

    const int item = blockIdx.x / a.KV, kv = blockIdx.x - item * a.KV;
    if (item >= a.head[3]) return;
    const PagedItem it = a.wide[item];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int total = it.past + it.rows / a.group;

    // The lane's query rows, one of each of the wave's groups, and the end of their keys.
    const int row0 = it.row0 + 16 * G * w;  // the wave's first row, whose keys end first
    const int first_end = it.past + row0 / a.group + 1;
    // Nothing of a tile that starts here or later is for this wave.
    const int wave_end = row0 < it.rows ? min(it.past + min(row0 + 16 * G - 1, it.rows - 1) / a.group + 1, it.key1) : 0;
    int row[G], token[G], end[G];
    bool live[G];
    uint32_t q[G][3][DP / 32][4];  // [group][part][c][e]: d = 32c + 8g + 2e, + 1
#pragma unroll
    for (int u = 0; u < G; ++u) {
        row[u] = row0 + 16 * u + n;
        token[u] = row[u] / a.group;
        live[u] = row[u] < it.rows && it.tok0 + token[u] < a.rows;
        end[u] = it.past + token[u] + 1;
        const float *src = a.q;  // a captured launch may hold items of tokens that its tensors have no rows for
        if (live[u])
            src += static_cast<int64_t>(it.tok0 + token[u]) * a.q_stride + (kv * a.group + row[u] - token[u] * a.group) * a.D;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
            uint32_t x[2][4];
            load_words<float, 4, R, true>(x[0], src, 32 * c + 8 * g, a.D);
            load_words<float, 4, R, true>(x[1], src, 32 * c + 8 * g + 4, a.D);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t p[3];
                split3(live[u] ? __builtin_bit_cast(float, x[e / 2][2 * (e % 2)]) : 0.0f,
                       live[u] ? __builtin_bit_cast(float, x[e / 2][2 * (e % 2) + 1]) : 0.0f, p);
#pragma unroll
                for (int i = 0; i < 3; ++i) q[u][i][c][e] = p[i];
            }
        }
    }

    // What this thread brings of a tile.  Keys: kKLoads pieces of 16 bytes, piece i being row i / per row.  Values:
    // kVDims neighbouring values of the eight keys of a place 8g.
    constexpr int kPiece = 16 / sizeof(T), kPieces = DP / kPiece;
    // Where that does not come out even, some threads bring nothing: their loads are clamped into the tile.
    constexpr int kKAll = kKeys * kPieces, kKLoads = (kKAll + kThreads - 1) / kThreads;
    constexpr int kVAll = kKeys / 8 * DP, kVDims = kVAll > 2 * kThreads ? 4 : kVAll > kThreads || sizeof(T) == 2 ? 2 : 1;
    constexpr int kVWords = kVDims * sizeof(T) / 4;
    static_assert(kVAll <= kVDims * kThreads && DP % kVDims == 0, "the values of a tile are brought at once");
    const bool brings_v = kVAll == kVDims * kThreads || tid < kVAll / kVDims;
    const int v_place = min(tid / (DP / kVDims), kKeys / 8 - 1), v_dim = tid % (DP / kVDims) * kVDims;
    const int v_key = v_place / 4 * 32 + v_place % 4 * 4;  // and the 3 after it, and 16 further
    const T *kpool = static_cast<const T *>(a.k), *vpool = static_cast<const T *>(a.v);
    const int *table = a.table + it.table;
    const int mask = (1 << a.page_shift) - 1;
    int k_page[kKLoads], v_page[2];
    auto load_pages = [&](int key) {
#pragma unroll
        for (int i = 0; i < kKLoads; ++i) k_page[i] = table[min(key + min(tid + i * kThreads, kKAll - 1) / kPieces, total - 1) >> a.page_shift];
#pragma unroll
        for (int h = 0; h < 2; ++h) v_page[h] = table[min(key + v_key + 16 * h, total - 1) >> a.page_shift];
    };
    uint32_t kr[kKLoads][4], vr[8][kVWords];
    auto load_tile = [&](int key) {
#pragma unroll
        for (int i = 0; i < kKLoads; ++i) {
            const int p = min(tid + i * kThreads, kKAll - 1), r = p / kPieces;
            const int64_t at = ((static_cast<int64_t>(k_page[i]) * a.KV + kv) << a.page_shift) + ((key + r) & mask);
            load_words<T, 4, R, false>(kr[i], kpool + at * a.D, p % kPieces * kPiece, a.D);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int r = v_key + 16 * (j / 4) + j % 4;
            const int64_t at = ((static_cast<int64_t>(v_page[j / 4]) * a.KV + kv) << a.page_shift) + ((key + r) & mask);
            load_words<T, kVWords, R, false>(vr[j], vpool + at * a.D, v_dim, a.D);
        }
    };
    const int item_end = it.past + it.row0 / a.group + 1;  // of the item's first row
    auto store_tile = [&](uint16_t *buf, int key) {
        uint16_t *kb = buf, *vb = buf + kParts * S::kKPart;
#pragma unroll
        for (int i = 0; i < kKLoads; ++i) {
            const int p = tid + i * kThreads;
            if (kKAll % kThreads != 0 && p >= kKAll) break;
            uint16_t *dst = kb + p / kPieces * S::kKRow + p % kPieces * kPiece;
            if constexpr (kParts == 1) {
                *reinterpret_cast<u32x4 *>(dst) = u32x4{kr[i][0], kr[i][1], kr[i][2], kr[i][3]};
            } else {
                uint32_t p0[3], p1[3];
                parts_of(kr[i][0], kr[i][1], p0);
                parts_of(kr[i][2], kr[i][3], p1);
#pragma unroll
                for (int t = 0; t < 3; ++t) *reinterpret_cast<u32x2 *>(dst + t * S::kKPart) = u32x2{p0[t], p1[t]};
            }
        }
        if (!brings_v) return;
        // Slots past the sequence's end hold anything: their weights are 0, and 0 times NaN is not.
        if (key + kKeys > total) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (key + v_key + 16 * (j / 4) + j % 4 >= total)
#pragma unroll
                    for (int i = 0; i < kVWords; ++i) vr[j][i] = 0;
        }
        if (key + kKeys > item_end) {
            bool any = false;
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int i = 0; i < kVWords; ++i) {
                    const uint32_t x = finite_part<T, true>(vr[j][i]);
                    any |= x != vr[j][i];
                    vr[j][i] = x;
                }
            if (any) again_s = 1;
        }
#pragma unroll
        for (int i = 0; i < kVDims; ++i) {
            uint16_t *dst = vb + (v_dim + i) * S::kVRow + 8 * v_place;
            if constexpr (kParts == 1) {
                u32x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    x[e] = __builtin_amdgcn_perm(vr[2 * e + 1][i / 2], vr[2 * e][i / 2], i % 2 ? 0x07060302u : 0x05040100u);
                *reinterpret_cast<u32x4 *>(dst) = x;
            } else {
                u32x4 x[3];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t p[3];
                    parts_of(vr[2 * e][i], vr[2 * e + 1][i], p);
#pragma unroll
                    for (int t = 0; t < 3; ++t) x[t][e] = p[t];
                }
#pragma unroll
                for (int t = 0; t < 3; ++t) *reinterpret_cast<u32x4 *>(dst + t * S::kVPart) = x[t];
            }
        }
    };

    float m[G], l[G];
    f32x4 o[G][DP / 16];
#pragma unroll
    for (int u = 0; u < G; ++u) {
        m[u] = -INFINITY;
        l[u] = 0.0f;
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) o[u][c] = zero4();
    }
    auto read4 = [](uint32_t (&x)[4], const uint16_t *p) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    };
    auto multiply = [&](const uint16_t *buf, int key) {
        const uint16_t *kb = buf + n * S::kKRow + 8 * g, *vb = buf + kParts * S::kKPart + n * S::kVRow + 8 * g;
        f32x4 s[G][kTiles];
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
#pragma unroll
            for (int u = 0; u < G; ++u) s[u][t] = zero4();
#pragma unroll
            for (int c = 0; c < DP / 32; ++c) {
#pragma unroll
                for (int j = kParts - 1; j >= 0; --j) {
                    uint32_t k[4];
                    read4(k, kb + j * S::kKPart + 16 * t * S::kKRow + 32 * c);
#pragma unroll
                    for (int i = 2 - j; i >= 0; --i)
#pragma unroll
                        for (int u = 0; u < G; ++u) s[u][t] = mfma_bf16(k, q[u][i][c], s[u][t]);
                }
            }
        }
        float base[G];
#pragma unroll
        for (int u = 0; u < G; ++u) {
#pragma unroll
            for (int t = 0; t < kTiles; ++t) settled(s[u][t]);
#pragma unroll
            for (int t = 0; t < kTiles; ++t) s[u][t] *= a.scale_log2;
            if (key + kKeys > first_end) {
#pragma unroll
                for (int t = 0; t < kTiles; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (key + 16 * t + 4 * g + r >= end[u]) s[u][t][r] = -INFINITY;
            }
            float mx = m[u];
#pragma unroll
            for (int t = 0; t < kTiles; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = fmaxf(mx, s[u][t][r]);
            mx = max4_rows(mx);
            base[u] = mx == -INFINITY ? 0.0f : mx;
            if (__any(mx > m[u])) {
                const float f = fast_exp2(m[u] - base[u]);
                l[u] *= f;
#pragma unroll
                for (int c = 0; c < DP / 16; ++c) o[u][c] *= f;
                m[u] = mx;
            }
        }
#pragma unroll
        for (int b = 0; b < kTiles / 2; ++b) {
            uint32_t p[G][3][4];
#pragma unroll
            for (int u = 0; u < G; ++u)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int t = 2 * b + e / 2, r = 2 * (e % 2);
                    const float p0 = fast_exp2(s[u][t][r] - base[u]), p1 = fast_exp2(s[u][t][r + 1] - base[u]);
                    l[u] += p0 + p1;
                    uint32_t x[3];
                    split3(p0, p1, x);
#pragma unroll
                    for (int i = 0; i < 3; ++i) p[u][i][e] = x[i];
                }
#pragma unroll
            for (int c = 0; c < DP / 16; ++c)
#pragma unroll
                for (int j = kParts - 1; j >= 0; --j) {
                    uint32_t v[4];
                    read4(v, vb + j * S::kVPart + 16 * c * S::kVRow + 32 * b);
#pragma unroll
                    for (int i = 2 - j; i >= 0; --i)
#pragma unroll
                        for (int u = 0; u < G; ++u) o[u][c] = mfma_bf16(v, p[u][i], o[u][c]);
                }
        }
    };

    load_pages(it.key0);
    load_tile(it.key0);
    load_pages(it.key0 + kKeys);
    if (tid == 0) again_s = 0;
    __syncthreads();
    int turn = 0;
    for (int key = it.key0; key < it.key1; key += kKeys, turn ^= 1) {
        uint16_t *buf = lds + (S::kBuffers == 2 ? turn * S::kBuffer : 0);
        if (S::kBuffers == 1) __syncthreads();
        store_tile(buf, key);
        __syncthreads();
        if (key + kKeys < it.key1) {
            load_tile(key + kKeys);
            load_pages(key + 2 * kKeys);
        }
        if (key < wave_end) multiply(buf, key);
    }
    drain();
    if (again_s != 0) {  // set before the last tile's barrier at the latest
        for (int u = 0; u < G; ++u)
            rows_by_key<T>(a, it, kv, row0 + 16 * u, 16, (static_cast<int64_t>(it.part + G * w + u) * a.KV + kv) * kPagedRows);
        return;
    }
#pragma unroll
    for (int u = 0; u < G; ++u) {
        const float sum = sum4_rows(l[u]);
        if (!live[u]) continue;
        float *dst;
        float scale = 1.0f;
        if (it.part < 0) {
            dst = a.out + (static_cast<int64_t>(it.tok0 + token[u]) * a.H + kv * a.group + row[u] - token[u] * a.group) * a.D;
            scale = 1.0f / sum;
        } else {
            const int64_t slot = (static_cast<int64_t>(it.part + G * w + u) * a.KV + kv) * kPagedRows + n;
            dst = a.part_o + slot * a.D;
            if (g == 0) *reinterpret_cast<f32x2 *>(a.part_ml + 2 * slot) = f32x2{m[u], sum};
        }
#pragma unroll
        for (int c = 0; c < DP / 16; ++c) store4<R != kAny>(dst, 16 * c + 4 * g, a.D, o[u][c] * scale);
    }
}

template <typename T, int DP, Rows R, int G>
void launch(const PagedAttnParams &p, hipStream_t s) {
    constexpr size_t kBytes = Shape<T, DP>::kBuffers * sizeof(uint16_t) * Shape<T, DP>::kBuffer;
    constexpr int kThreads = paged_wide_rows(kType<T>) / (16 * G) * 64;
    const auto kernel = paged_wide_kernel<T, DP, R, G, kThreads>;
    if constexpr (kBytes > 65536) {
        static std::once_flag once;
        std::call_once(once, [&] {
            hipCheck(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize,
                                         kBytes));
        });
    }
    kernel<<<dim3(static_cast<unsigned>(p.n_wide) * p.KV), dim3(kThreads), kBytes, s>>>(p);
    hipCheck(hipGetLastError());
}

template <typename T, int DP, int G>
void launch(const PagedAttnParams &p, hipStream_t s) {
    if (p.vec && p.D == DP)
        launch<T, DP, kFull, G>(p, s);
    else if (p.vec)
        launch<T, DP, kVec, G>(p, s);
    else
        launch<T, DP, kAny, G>(p, s);
}

}  // namespace

void launch_paged_wide(const PagedAttnParams &p, hipStream_t s) {
    // Groups of 16 rows to a wave, fp32 pages.  With two a workgroup has half the waves, and two of them fit a CU: worth
    // it from one and a half per CU on.  12 heads of 64, a prompt of 4096: 239 us with one group and 219 with two; of
    // 1024 (240 workgroups): 24 and 29 us.  Heads of 128, 64 tokens each of 8 sequences over 2000: 82 and 76 us; a
    // prompt of 1024 with 12 heads: 42 and 52 us.  Both give the same sums.  With two, heads past 96 spill 8 registers a
    // lane (21 where rows are no whole vectors), which these figures include.
    const bool two = static_cast<int64_t>(p.n_wide) * p.KV >= 384;
    // Tiles of 64, 96 and 128 values of a head: what pads a head is multiplied too.  Heads of 80 as 128, fp32 and bf16
    // pages: a prompt of 4096 with 12 heads 383 and 217 us, as 96 294 and 191 us.
    if (p.bf16) {
        if (p.D <= 64) launch<__bf16, 64, 1>(p, s);
        else if (p.D <= 96) launch<__bf16, 96, 1>(p, s);
        else launch<__bf16, 128, 1>(p, s);
    } else if (p.D <= 64) {
        if (two) launch<float, 64, 2>(p, s);
        else launch<float, 64, 1>(p, s);
    } else if (p.D <= 96) {
        if (two) launch<float, 96, 2>(p, s);
        else launch<float, 96, 1>(p, s);
    } else {
        if (two) launch<float, 128, 2>(p, s);
        else launch<float, 128, 1>(p, s);
    }
}

}  // namespace gptc
