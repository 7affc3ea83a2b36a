// Products of operands laid out as two fp16 parts (gemm_halves.hpp), fp32 results.
//
// A float times a power of two is the sum of two fp16 values to 2^-24 of it (11 +
// 11 bits and the low part's sign), as close as fp32 itself.  Of the four products
// of two such sums three are formed, low high, high low and high high; the fourth
// is at most 2^-24 of the product.  A product of fp16 values is exact in fp32, so
// three v_mfma_f32_32x32x16_f16 do what takes six bf16 instructions from three-part
// sums (gemm_split.hip), whose parts need no common scale.
//
// Sums.  As there: the matrix core drops bits below its accumulator towards minus
// infinity, so 64 terms at a time are summed in a fresh accumulator, smallest products
// first, and taken into the tile by a rounded fp32 add; every other 64 are formed
// negated and subtracted, which cancels what shift is left.
//
// What bounds them: the matrix cores' power.  8192 rows of 768 against 50257 tokens,
// 1.9e12 fp16 operations for each of the three products, take 1.73 to 1.9 ms for the
// logits and 1.7 to 1.9 for a gradient, from box to box: 1000 to 1130 TFLOP/s beside the
// library's fp16 product of 8192^3 on such values, 1145 (1594 on zeros, as the clock
// falls with what toggles).  Tiles of 256 x 256 were no quicker.
//
// A workgroup forms 128 x 128 outputs, its four waves 64 x 64 each.  The operands lie
// in memory as the instruction takes them, so a step's 32 KB go to LDS by 32 loads
// of 1 KB that pass no register, and every LDS access is 1 KB in a row.  Two buffers:
// a step's fragments are read to registers at once, and the loads of the step after
// next go out into the same buffer as soon as all waves have read it.
#include <algorithm>
#include "gpu_kernels.h"
#include "head_loss.hpp"
#include "ops_common.hpp"

namespace gptc {

namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ hf32x16 mfma(hu32x4 a, hu32x4 b, hf32x16 c) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// ---- operands ----

// A wave a row, which is read once: its first kRowsKeep * 256 terms stay in registers (the others are read again for their
// parts).  A workgroup's eight rows fill lines of 128 bytes.  8192 rows of 768 in three pieces: 24 us.
constexpr int kRowsWaves = 8;
constexpr int kRowsKeep = 4;
__global__ __launch_bounds__(64 * kRowsWaves) void halves_rows_kernel(const float *__restrict__ x,
                                                                     const float *__restrict__ weights, int rows,
                                                                     int terms, bool vec, HalvesRows t) {
    const int lane = threadIdx.x & 63;
    const int row = blockIdx.x * kRowsWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    for (int i = blockIdx.x * (64 * kRowsWaves) + threadIdx.x; i < t.zeros; i += gridDim.x * (64 * kRowsWaves)) t.zero[i] = 0;
    const bool live = row < rows && (weights == nullptr || weights[row] != 0.0f);
    const float *p = x + static_cast<int64_t>(row) * terms;
    auto four = [&](int k) {
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (vec) {
            if (live && k < terms) v = *reinterpret_cast<const f32x4_t *>(p + k);
        } else if (live) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = k + e < terms ? p[k + e] : 0.0f;
        }
        return v;
    };
    f32x4_t own[kRowsKeep];
    float top = 0.0f;
    auto larger = [&](f32x4_t v) {
        top = fmaxf(fmaxf(top, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
    };
#pragma unroll
    for (int i = 0; i < kRowsKeep; ++i) own[i] = four(256 * i + 4 * lane);
#pragma unroll 4
    for (int k = 256 * kRowsKeep + 4 * lane; k < terms; k += 256) larger(four(k));
#pragma unroll
    for (int i = 0; i < kRowsKeep; ++i) larger(own[i]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    const int up = halves_shift(top);
    if (lane == 0) t.shift[row] = up;
    uint2 *out = reinterpret_cast<uint2 *>(t.data + static_cast<int64_t>(row >> 5) * t.term_blocks * 128 + (row & 31));
    auto put = [&](int k, f32x4_t v) {
        if (k >= 16 * t.term_blocks) return;
        const uint32_t flip = t.in_lines && halves_negated(k) ? 0x80008000u : 0;
        uint2 high, low;
        halves_split(__builtin_amdgcn_ldexpf(v[0], up), __builtin_amdgcn_ldexpf(v[1], up), high.x, low.x);
        halves_split(__builtin_amdgcn_ldexpf(v[2], up), __builtin_amdgcn_ldexpf(v[3], up), high.y, low.y);
        // Block, lanes' half and place in 16 bytes of term k = 32 j + 16 a + 8 b + 4 c.
        const int j = k >> 5, a = (k >> 4) & 1, b = (k >> 3) & 1, c = (k >> 2) & 1;
        const int kb = 2 * j + (t.in_lines ? b : a), hf = t.in_lines ? a : c, half = t.in_lines ? c : b;
        uint2 *at = out + 2 * (kb * 128 + 32 * hf) + half;
        at[0] = make_uint2(high.x ^ flip, high.y ^ flip);
        at[2 * 64] = make_uint2(low.x ^ flip, low.y ^ flip);
    };
#pragma unroll
    for (int i = 0; i < kRowsKeep; ++i) put(256 * i + 4 * lane, own[i]);
    for (int k = 256 * kRowsKeep + 4 * lane; k < 16 * t.term_blocks; k += 256) put(k, four(k));
}

constexpr int kTableThreads = 512;

// 64 rows by one shift, in one pass: a workgroup's values stay in registers until the largest is known, its lines are read
// whole and written whole, through LDS.  PIECES of 32 terms stay, up to 24 with two workgroups a CU (768 x 50257: 69 us,
// 4.5 TB/s; a pass for the largest value and one for the parts 88), else 52 with one (1600 x 50257: 166 us; with 24, and
// the others read again, 206); MORE: there are more, which are read again.
template <int PIECES, bool MORE>
__global__ __launch_bounds__(kTableThreads) __attribute__((amdgpu_waves_per_eu(PIECES > 24 ? 2 : 4))) void halves_table_kernel(
    const float *__restrict__ x, Halves h, bool vec) {
    __shared__ hu32x4 lds[2][8 * 128];  // of each block of 32 rows, 128 terms
    __shared__ float red[kTableThreads / 64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, kbs = h.term_blocks(), pieces = kbs / 2;
    // Piece i of a wave: rows 8 w .. + 7, terms 32 i .. + 31.
    const int in = w * 8 + (lane >> 3), row = blockIdx.x * 64 + in;
    const float *p = x + static_cast<int64_t>(row) * h.terms;
    auto four = [&](int i) {
        const int k = 32 * i + 4 * (lane & 7);
        f32x4_t v = {0.0f, 0.0f, 0.0f, 0.0f};
        if (vec) {
            if (row < h.rows && k < h.terms) v = *reinterpret_cast<const f32x4_t *>(p + k);
        } else if (row < h.rows) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = k + e < h.terms ? p[k + e] : 0.0f;
        }
        return v;
    };
    float top = 0.0f;
    auto larger = [&](f32x4_t v) {
        top = fmaxf(fmaxf(top, fmaxf(fabsf(v[0]), fabsf(v[1]))), fmaxf(fabsf(v[2]), fabsf(v[3])));
    };
    f32x4_t own[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) own[i] = four(i);
    if (MORE)
#pragma unroll 4
        for (int i = PIECES; i < pieces; ++i) larger(four(i));
#pragma unroll
    for (int i = 0; i < PIECES; ++i) larger(own[i]);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off, 64));
    if (lane == 0) red[w] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kTableThreads / 64; ++i) top = fmaxf(top, red[i]);
    const int up = min(halves_shift(top), 126);
    if ((lane & 7) == 0) h.shift[row] = up;
    uint2 *to = reinterpret_cast<uint2 *>(lds[in >> 5]);
#pragma unroll 1
    for (int p0 = 0; p0 < pieces; p0 += 4) {
        f32x4_t v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = !MORE || p0 < PIECES ? own[i] : four(p0 + i);
#pragma unroll
        for (int i = 0; i + 4 < PIECES; ++i) own[i] = own[i + 4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int c = 8 * i + (lane & 7), q = c & 3;  // four terms of block c / 4
            const uint32_t flip = halves_negated((2 * p0 + (c >> 2)) * 16) ? 0x80008000u : 0;
            uint2 high, low;
            halves_split(__builtin_amdgcn_ldexpf(v[i][0], up), __builtin_amdgcn_ldexpf(v[i][1], up), high.x, low.x);
            halves_split(__builtin_amdgcn_ldexpf(v[i][2], up), __builtin_amdgcn_ldexpf(v[i][3], up), high.y, low.y);
            const int at = (c >> 2) * 256 + ((q & 1) * 32 + (in & 31)) * 2 + (q >> 1);
            to[at] = make_uint2(high.x ^ flip, high.y ^ flip);
            to[at + 128] = make_uint2(low.x ^ flip, low.y ^ flip);
        }
        __syncthreads();
        const int chunks = min(8, kbs - 2 * p0) * 128;
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            hu32x4 *out = h.data + (static_cast<int64_t>(blockIdx.x * 2 + b) * kbs + 2 * p0) * 128;
#pragma unroll
            for (int i = 0; i < 8 * 128; i += kTableThreads)
                if (i + static_cast<int>(threadIdx.x) < chunks) out[i + threadIdx.x] = lds[b][i + threadIdx.x];
        }
        __syncthreads();
    }
}

// The factor of term k of an operand that is read across its rows.
__device__ __forceinline__ float term_factor(const float *weights, float divisor, int k) {
    return weights != nullptr ? weights[k] / divisor : 1.0f / divisor;
}

constexpr int kLargestTerms = 64;  // terms a workgroup

// largest[c] = bits of the largest magnitude of column c so far (whole numbers: in any order the same).
// A workgroup: 64 columns in units of T, its waves take the terms in turns.
template <typename T>
__global__ __launch_bounds__(kThreads) void column_largest_kernel(const float *__restrict__ x, int ld,
                                                                 const float *__restrict__ weights, float divisor,
                                                                 int terms, int cols, uint32_t *largest) {
    constexpr int kW = sizeof(T) / sizeof(float);
    __shared__ uint32_t red[64 * kW];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = (blockIdx.y * 64 + lane) * kW;
    for (int i = threadIdx.x; i < 64 * kW; i += kThreads) red[i] = 0;
    __syncthreads();
    if (c < cols) {
        float m[kW];
#pragma unroll
        for (int e = 0; e < kW; ++e) m[e] = 0.0f;
        const int k1 = min(terms, static_cast<int>(blockIdx.x + 1) * kLargestTerms);
#pragma unroll 8
        for (int k = blockIdx.x * kLargestTerms + w; k < k1; k += 4) {
            const T v = *reinterpret_cast<const T *>(x + static_cast<int64_t>(k) * ld + c);
            const float f = term_factor(weights, divisor, k);
#pragma unroll
            for (int e = 0; e < kW; ++e)
                if (f != 0.0f) m[e] = fmaxf(m[e], fabsf(f * reinterpret_cast<const float *>(&v)[e]));
        }
#pragma unroll
        for (int e = 0; e < kW; ++e) atomicMax(&red[lane * kW + e], __float_as_uint(m[e]));
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 64 * kW; i += kThreads) {
        const int at = blockIdx.y * 64 * kW + i;
        if (at < cols && red[i] != 0) atomicMax(largest + at, red[i]);
    }
}

// A workgroup: 32 columns, kColumnTerms terms; with `largest` null these are all terms.
__global__ __launch_bounds__(kThreads) void halves_columns_kernel(const float *__restrict__ x, int ld,
                                                                 const float *__restrict__ weights, float divisor,
                                                                 Halves h, bool negate,
                                                                 const uint32_t *__restrict__ largest) {
    const int lane = threadIdx.x & 63, hf = lane >> 5, w = threadIdx.x >> 6;
    const int rb = blockIdx.x, c = rb * 32 + (lane & 31), kbs = h.term_blocks();
    const int first = blockIdx.y * (kColumnTerms / 16) + w * (kColumnTerms / 64);
    float v[kColumnTerms / 64][8];
#pragma unroll
    for (int i = 0; i < kColumnTerms / 64; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int k = (first + i) * 16 + 4 * hf + (e & 3) + 8 * (e >> 2), at = min(k, h.terms - 1);
            const float f = term_factor(weights, divisor, at);
            const float y = x[static_cast<int64_t>(at) * ld + min(c, h.rows - 1)];
            v[i][e] = f != 0.0f && k < h.terms && c < h.rows ? f * y : 0.0f;
        }
    float top = largest != nullptr && c < h.rows ? __uint_as_float(largest[c]) : 0.0f;
    if (largest == nullptr) {
        __shared__ float red[kThreads / 64][32];
#pragma unroll
        for (int i = 0; i < kColumnTerms / 64; ++i)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[i][e]));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        if (hf == 0) red[w][lane] = top;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kThreads / 64; ++i) top = fmaxf(top, red[i][lane & 31]);
    }
    const int up = halves_shift(top);
    if (blockIdx.y == 0 && w == 0 && hf == 0) h.shift[c] = up;
    hu32x4 *out = h.data + (static_cast<int64_t>(rb) * kbs * 2) * 64 + lane;
#pragma unroll
    for (int i = 0; i < kColumnTerms / 64; ++i) {
        const int kb = first + i;
        if (kb >= kbs) return;
        const uint32_t flip = negate && halves_negated(kb * 16) ? 0x80008000u : 0;
        hu32x4 high, low;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint32_t hi, lo;
            halves_split(__builtin_amdgcn_ldexpf(v[i][2 * e], up), __builtin_amdgcn_ldexpf(v[i][2 * e + 1], up), hi, lo);
            high[e] = hi ^ flip;
            low[e] = lo ^ flip;
        }
        out[(kb * 2) * 64] = high;
        out[(kb * 2 + 1) * 64] = low;
    }
}

// ---- the product's loop ----

struct Tile {
    const hu32x4 *A, *B;
    const int *shift_a, *shift_b;  // of the rows; shift_a for logits alone
    int all_a;                     // where shift_a is null
    int tiles_m, tiles_n, kbs, stages, slice;  // stages of 32 terms in all, and of a slice
    int kbs_across;  // blocks of 16 of what are rows here of the operand that is read across
};

// The tile and slice of this workgroup (grid: tiles by slices, or slices of few tiles one after the other).  Workgroup i
// runs on XCD i % 8: 8 contiguous ranges of a slice's tiles, or of all slices' where those are few (so that a slice's
// operands go to one L2 or two), one per XCD.  In a range, columns of G row tiles, so that the tiles that run together
// share rows and columns.  Few columns come one after the other (G = 1): the workgroups of a row start one by one as
// others end, and what lies between them has to stay in the L2.
__device__ __forceinline__ void tile_of(const Tile &t, int &tm, int &tn, int &slice) {
    const int tiles = t.tiles_m * t.tiles_n, n = gridDim.x;
    int i = blockIdx.x;
    const int x = i & 7, q = n >> 3, r = n & 7;
    i = (i >> 3) + x * q + min(x, r);
    slice = blockIdx.y;
    if (n > tiles) {
        slice = i / tiles;
        i -= slice * tiles;
    }
    const int G = t.tiles_n <= 8 ? 1 : 8, per = G * t.tiles_n;
    const int g = i / per, first = g * G, h = min(G, t.tiles_m - first);
    const int in = i - g * per;
    tm = first + in % h;
    tn = in / h;
}

// The workgroup's shapes: waves WM x WN, each forming 32 NI x 64 outputs.
template <int WM_, int WN_, int NI_>
struct Shape {
    static constexpr int WM = WM_, WN = WN_, NI = NI_;
    static constexpr int kWaves = WM * WN, kThreads = 64 * kWaves;
    static constexpr int BM = WM * NI * 32, BN = WN * 64;
    static constexpr int kBlocks = (BM + BN) / 32;             // blocks of 32 rows of either operand, 4 KB a step each
    static constexpr int kLoads = kBlocks / kWaves;            // of a wave
    static constexpr int kStage = kBlocks * 4096;              // bytes
};

// Loads of 4 KB from `base` on to LDS at `to` and behind, lane l's 16 bytes of a kilobyte from `first` there, of the last
// two from `last`.  They write no register but m0, which nothing else of these kernels uses (it cannot be named as written:
// the compiler keeps it to itself); the compiler does not count them, so its own waits wait for more than they need.
__device__ __forceinline__ void load_block(const hu32x4 *base, uint32_t to, uint32_t first, uint32_t last) {
    asm volatile(
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %2\n\t"
        "global_load_lds_dwordx4 %0, %2 offset:1024\n\t"
        "global_load_lds_dwordx4 %1, %2 offset:2048\n\t"
        "global_load_lds_dwordx4 %1, %2 offset:%4"
        :
        : "v"(first), "v"(last), "s"(base), "s"(to), "n"(3 << 10)
        : "memory");
}

// Four fp16 values, 16 lanes transposed: lane j receives value j % 4 of lanes j / 4 + {0, 4, 8, 12} of its 16.
__device__ __forceinline__ uint2 read_across(uint32_t at) {
    typedef short s16x4 __attribute__((ext_vector_type(4)));
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
        reinterpret_cast<__attribute__((address_space(3))) s16x4 *>(static_cast<uintptr_t>(at))));
}

// acc = the wave's outputs of tile (tm, tn) over steps [s0, s1), without the shifts.
// The operand that is read `Across` comes as the first one of another product, its rows as terms and its terms as
// rows: four consecutive terms of a row are 8 bytes in LDS, which a transposing read gives to four lanes.  There 16-byte
// chunk c of a kilobyte lies at c ^ 4 (c / 32), and ^ 8 in every other block of 16 terms, so that no two of a read's
// lanes meet in a bank.  The sign of every other 64 terms is a sign of the outputs' rows or columns here, and the other
// operand holds that of the reduction.
enum class Across { kNone, kA, kB };

template <class S, Across ACROSS>
__device__ __forceinline__ void tile_product(const Tile &t, int tm, int tn, int s0, int s1, hu32x4 *lds,
                                             hf32x16 (&acc)[S::NI][2]) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    constexpr int kA = S::BM / 32, kB = S::BN / 32;
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
        (__attribute__((address_space(3))) void *)lds));
    const uint32_t lane16 = lane * 16, hf = lane >> 5;
    constexpr int kAt = ACROSS == Across::kA ? 0 : ACROSS == Across::kB ? 1 : -1;  // which of a wave's blocks it is
    static_assert(kAt < 0 || (kA == S::kWaves && S::kLoads == 2), "a wave loads one block of A, then one of B");
    // Wave w loads blocks w, w + kWaves .. of A's and B's rows.
    const hu32x4 *from[S::kLoads];
    int64_t step[S::kLoads];
#pragma unroll
    for (int i = 0; i < S::kLoads; ++i) {
        const int block = w + i * S::kWaves;
        const int kbs = i == kAt ? 2 : t.kbs;
        const hu32x4 *p = block < kA ? t.A + static_cast<int64_t>(tm * kA + block) * kbs * 128
                                     : t.B + static_cast<int64_t>(tn * kB + block - kA) * kbs * 128;
        step[i] = i == kAt ? static_cast<int64_t>(t.kbs_across) * 128 : 256;
        from[i] = p + s0 * step[i];
    }
    const uint32_t lane_first = lane16 ^ (64 * hf), lane_last = lane_first ^ 128;
    // Past the last step the last one is loaded again, into a buffer that nobody reads any more: the
    // loop needs no branch then, and its waits are the same in every step.
    int next = s0;
    auto load_stage = [&](uint32_t off) {
#pragma unroll
        for (int i = 0; i < S::kLoads; ++i)
            load_block(from[i], base + off + (w + i * S::kWaves) * 4096, i == kAt ? lane_first : lane16,
                       i == kAt ? lane_last : lane16);
        if (++next < s1) {
#pragma unroll
            for (int i = 0; i < S::kLoads; ++i) from[i] += step[i];
        }
    };
#pragma unroll
    for (int i = 0; i < S::NI; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;
    load_stage(0);
    load_stage(S::kStage);
    const hu32x4 *at_a = lds + (w / S::WN) * S::NI * 256 + lane;
    const hu32x4 *at_b = lds + (kA + (w % S::WN) * 2) * 256 + lane;
    // Lane l reads, of terms (rows of the block) 4 (l / 32) + l / 4 % 4 and 8 behind, rows (terms) 16 (l / 16 % 2) +
    // 4 (l % 4) and the next three.
    const uint32_t in16 = lane & 15, half16 = (lane >> 4) & 1;
    const uint32_t block_across = ACROSS == Across::kA ? (w / S::WN) * S::NI : kA + (w % S::WN) * 2;
    const uint32_t across = block_across * 4096 + half16 * 2048 + (in16 & 1) * 512 + half16 * 128 +
                            (hf ^ (in16 & 1)) * 64 + (in16 >> 2) * 16 + ((in16 >> 1) & 1) * 8;
    const uint32_t across_first = base + across, across_last = base + (across ^ 128);
    auto fragment_across = [&](int half, int i) {
        const uint32_t at = half * S::kStage + (i >> 2) * 4096 + ((i >> 1) & 1) * 256 + (i & 1) * 1024;
        const uint2 one = read_across(across_first + at), two = read_across(across_last + at);
        return hu32x4{one.x, one.y, two.x, two.y};
    };
    // A wave's 64 rows and 64 columns are of one sign each.
    static_assert(S::NI == 2 && S::BM % 128 == 0 && S::BN % 128 == 0, "");
    const bool minus = ACROSS == Across::kA ? ((w / S::WN) & 1) != 0 : ACROSS == Across::kB ? ((w % S::WN) & 1) != 0 : false;
    float sign = ((s0 & 2) != 0) != minus ? -1.0f : 1.0f;
    int shifts = 0;  // of B read across: lane l holds that of the 64 terms after 64 l others
    // There A's scale goes too: sums that kept it would pass the largest float with values of B 2^15 below it.
    if (ACROSS == Across::kB) sign = __builtin_amdgcn_ldexpf(sign, -t.all_a);
    for (int s = s0; s < s1; s += 2) {
        float times = sign;
        if constexpr (ACROSS == Across::kB) {
            if (((s - s0) & 127) == 0) shifts = t.shift_b[32 * min(s + 2 * lane, t.stages - 1)];
            times = __builtin_amdgcn_ldexpf(sign, -__builtin_amdgcn_readlane(shifts, ((s - s0) & 127) >> 1));
        }
        hf32x16 p[S::NI][2];
#pragma unroll
        for (int i = 0; i < S::NI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) p[i][j][r] = 0.0f;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int off = half * (S::kStage / 16);
            // This wave's loads of the step have landed (those of the next are on their way), then all waves'.
            static_assert(S::kLoads == 2, "4 kLoads loads a step");
            asm volatile("s_waitcnt vmcnt(8)\n\ts_barrier" ::: "memory");
            hu32x4 fb[2][2][2], fa[S::NI][2][2];  // blocks of 32 rows, of 16 terms, parts
#pragma unroll
            for (int i = 0; i < 8; ++i)
                fb[i >> 2][(i >> 1) & 1][i & 1] = ACROSS == Across::kB ? fragment_across(half, i) : at_b[off + i * 64];
#pragma unroll
            for (int i = 0; i < 4 * S::NI; ++i)
                fa[i >> 2][(i >> 1) & 1][i & 1] = ACROSS == Across::kA ? fragment_across(half, i) : at_a[off + i * 64];
            // All waves have read this buffer: the step after next goes there.
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
            load_stage(half * S::kStage);
            constexpr int kProd[3][2] = {{1, 0}, {0, 1}, {0, 0}};
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < S::NI; ++i)
#pragma unroll
                        for (int j = 0; j < 2; ++j)
                            p[i][j] = mfma(fa[i][k][kProd[q][0]], fb[j][k][kProd[q][1]], p[i][j]);
        }
#pragma unroll
        for (int i = 0; i < S::NI; ++i)
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) acc[i][j][r] = fmaf(times, p[i][j][r], acc[i][j][r]);
        sign = -sign;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
}

template <class S>
__global__ __launch_bounds__(S::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void logits_kernel(
    const Tile t, const LogitsArgs l) {
    __shared__ hu32x4 lds[2 * S::kStage / 16];
    int tm, tn, slice;
    tile_of(t, tm, tn, slice);
    hf32x16 acc[S::NI][2];
    tile_product<S, Across::kNone>(t, tm, tn, 0, t.stages, lds, acc);
    const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int token0 = tm * S::BM + (w / S::WN) * (S::NI * 32), row0 = tn * S::BN + (w % S::WN) * 64;
    // In a loop, as its code is fetched by every workgroup.
#pragma unroll 1
    for (int j = 0; j < 2; ++j) {
        const int up = t.shift_b[row0 + 32 * j + l32];
        hf32x16 x[S::NI];
#pragma unroll
        for (int i = 0; i < S::NI; ++i) {
            x[i] = acc[i][0];
            acc[i][0] = acc[i][1];
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int4 back = *reinterpret_cast<const int4 *>(t.shift_a + token0 + 32 * i + 8 * q + 4 * hf);
                const int shift[4] = {back.x, back.y, back.z, back.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) x[i][4 * q + e] = __builtin_amdgcn_ldexpf(x[i][4 * q + e], -up - shift[e]);
            }
        }
        const float2 stat = put_logits<S::NI, true>(l, x, token0, (row0 >> 5) + j);
        if (hf == 0) l.stats[static_cast<int64_t>(token0 / (S::NI * 32)) * l.row_stride + row0 + 32 * j + l32] = stat;
    }
}

struct ProductArgs {
    HalvesProduct p;
    int M, N;
    float *part;  // the slices' sums, (M, N) each, or null
};

__device__ __forceinline__ float times_row_factor(const HalvesProduct &p, int row, float v) {
    const float f = p.row_factor != nullptr ? p.row_factor[row] : 1.0f;
    return f != 0.0f ? v * (f / p.divisor) : 0.0f;
}

template <class S, Across ACROSS>
__global__ __launch_bounds__(S::kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void product_kernel(
    const Tile t, const ProductArgs a) {
    __shared__ hu32x4 lds[2 * S::kStage / 16];
    int tm, tn, slice;
    tile_of(t, tm, tn, slice);
    hf32x16 acc[S::NI][2];
    const int s0 = slice * t.slice;
    tile_product<S, ACROSS>(t, tm, tn, s0, min(t.stages, s0 + t.slice), lds, acc);
    const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int m0 = tm * S::BM + (w / S::WN) * (S::NI * 32), n0 = tn * S::BN + (w % S::WN) * 64;
    // One block of 32 x 32 after the other, in a loop: its code is fetched by every workgroup.
#pragma unroll 1
    for (int block = 0; block < 2 * S::NI; ++block) {
        hf32x16 v = acc[0][0];
#pragma unroll
        for (int i = 0; i < S::NI; ++i) {
            acc[i][0] = acc[i][1];
            if (i + 1 < S::NI) acc[i][1] = acc[i + 1][0];
        }
        const int n = n0 + 32 * (block & 1) + l32, first = m0 + 32 * (block >> 1), m = first + 4 * hf;
        if (first >= a.M) break;
        const int up = ACROSS == Across::kB ? 0 : -t.all_a - t.shift_b[min(n, a.N - 1)];
#pragma unroll
        for (int r = 0; r < 16; ++r) v[r] = __builtin_amdgcn_ldexpf(v[r], up);
        // The block's rows of C or of the slice's part; what lies past the last row or column is neither read nor written.
        const int ld = a.part != nullptr ? a.N : a.p.ldc;
        float *C = a.part != nullptr ? a.part + static_cast<int64_t>(slice) * a.M * a.N : a.p.C;
        const int bytes = 4 * min(32, a.M - first) * ld;
        const __amdgpu_buffer_rsrc_t rows =
            __builtin_amdgcn_make_buffer_rsrc(C + static_cast<int64_t>(first) * ld, 0, bytes, 0x00020000);
        const uint32_t mine = n < a.N ? 4 * (static_cast<uint32_t>(4 * hf) * ld + n) : 0x80000000u;
        auto row_at = [&](int r) { return min(4 * (8 * (r >> 2) + (r & 3)) * ld, bytes); };
        if (a.part == nullptr) {
            if (a.p.row_factor != nullptr || a.p.divisor != 1.0f) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    v[r] = times_row_factor(a.p, min(m + 8 * (r >> 2) + (r & 3), a.M - 1), v[r]);
            }
            if (a.p.add) {
                float old[16];
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    old[r] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rows, mine, row_at(r), 0));
#pragma unroll
                for (int r = 0; r < 16; ++r) v[r] = old[r] + v[r];
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[r]), rows, mine, row_at(r),
                                                  ACROSS == Across::kA ? kStreamed : 0);
    }
}

// C = the slices' sums, times the row's factor (+ C).  Many slices go to eight threads, every eighth slice to one, whose
// sums are added in their order (2 rows of 45, 393 slices: 4 us, by one thread 16; 100 rows of 768, 85 slices: 6.2, 7.4).
constexpr int kJoinGroups = 8, kJoinMany = 32;
template <int GROUPS>
__global__ __launch_bounds__(kThreads) void join_slices_kernel(const float *__restrict__ part, int M, int N, int slices,
                                                              const HalvesProduct p) {
    constexpr int kOwn = kThreads / GROUPS;  // results of a workgroup
    const int64_t n = static_cast<int64_t>(M) * N, stride = static_cast<int64_t>(gridDim.x) * kOwn;
    const int group = threadIdx.x / kOwn, mine = threadIdx.x % kOwn;
    for (int64_t i0 = blockIdx.x * static_cast<int64_t>(kOwn); i0 < n; i0 += stride) {
        const int64_t i = i0 + mine;
        float v = 0.0f;
        if (i < n) {
            if (GROUPS == 1) v = part[i];
#pragma unroll 8
            for (int s = GROUPS == 1 ? 1 : group; s < slices; s += GROUPS) v += part[s * n + i];
        }
        if (GROUPS > 1) {
            __shared__ float sums[GROUPS][kOwn];
            __syncthreads();
            sums[group][mine] = v;
            __syncthreads();
            if (group > 0) continue;
#pragma unroll
            for (int g = 1; g < GROUPS; ++g) v += sums[g][mine];
        }
        if (i >= n) continue;
        const int m = static_cast<int>(i / N);
        float *c = p.C + static_cast<int64_t>(m) * p.ldc + (i - static_cast<int64_t>(m) * N);
        v = times_row_factor(p, m, v);
        *c = p.add ? *c + v : v;
    }
}

template <class S>
Tile tile_args(const Halves &A, const Halves &B) {
    CHECK_ERROR(A.terms != B.terms || B.rows >= 1 << 22 || B.shift == nullptr,
                "Operands of %d and %d terms, %d columns, or one shift for all of them.", A.terms, B.terms, B.rows);
    const int stages = A.term_blocks() / 2;
    return {A.data, B.data, A.shift, B.shift, A.shift_all, (A.rows + S::BM - 1) / S::BM,
            (B.rows + S::BN - 1) / S::BN, A.term_blocks(), stages, stages, 0};
}

using Small = Shape<2, 2, 2>;  // 128 x 128

template <class S>
void run_logits(const Halves &A, const Halves &B, LogitsArgs l, hipStream_t s) {
    Tile t = tile_args<S>(A, B);
    t.tiles_m = A.row_blocks() * 32 / S::BM;  // the padding too: its parts are joined
    t.tiles_n = B.row_blocks() * 32 / S::BN;
    logits_kernel<S><<<dim3(t.tiles_m * t.tiles_n), dim3(S::kThreads), 0, s>>>(t, l);
    hipCheck(hipGetLastError());
}

// Slices of the reduction so that the last round of workgroups (kSlots at once) is full.  In steps of
// 32 terms: a workgroup's start and end cost about 8, a slice's sums go out and come back.
template <class S, Across ACROSS>
void run_product(const Halves &A, const Halves &B, int kbs_across, const HalvesProduct &p, hipStream_t s) {
    constexpr int kSlots = 256 * (8 / S::kWaves);
    CHECK_ERROR(A.shift != nullptr, "A first operand with a shift a row.");
    Tile t = tile_args<S>(A, B);
    t.kbs_across = kbs_across;
    const int tiles = t.tiles_m * t.tiles_n;
    int best = 1;
    double best_cost = 1e30;
    for (int n = 1; n <= 32 && n <= t.stages; ++n) {
        const int mine = (t.stages + n - 1) / n;
        const int rounds = (tiles * n + kSlots - 1) / kSlots;
        const double cost = rounds * (mine + 8.0) + (n > 1 ? 8.0 + n * 0.02 * tiles * (S::BM / 128) : 0.0);
        if (cost < best_cost) {
            best_cost = cost;
            best = n;
        }
    }
    t.slice = ((t.stages + best - 1) / best + 1) & ~1;
    const int slices = (t.stages + t.slice - 1) / t.slice;
    ProductArgs a{p, A.rows, B.rows, nullptr};
    if (slices > 1) a.part = static_cast<float *>(alloc_cuda(sizeof(float) * static_cast<size_t>(A.rows) * B.rows * slices));
    // dx with its slices one after the other / side by side: 1024 rows of 768 (48 tiles) 252 / 265 us, 3328 rows (156
    // tiles) 638 / 643, 2000 rows of 1600 (208 tiles) 975 / 943.
    const bool in_turn = tiles <= 3 * kSlots / 8;
    product_kernel<S, ACROSS><<<in_turn ? dim3(tiles * slices) : dim3(tiles, slices), dim3(S::kThreads), 0, s>>>(t, a);
    hipCheck(hipGetLastError());
    if (slices == 1) return;
    launch_join_slices(a.part, A.rows, B.rows, slices, p, s);
    free_cuda(a.part);
}

}  // namespace

void launch_join_slices(const float *part, int M, int N, int slices, const HalvesProduct &p, hipStream_t s) {
    const int64_t n = static_cast<int64_t>(M) * N;
    if (slices >= kJoinMany)
        join_slices_kernel<kJoinGroups><<<dim3(blocks_for(n, kThreads / kJoinGroups)), dim3(kThreads), 0, s>>>(part, M, N,
                                                                                                              slices, p);
    else
        join_slices_kernel<1><<<dim3(blocks_for(n, kThreads)), dim3(kThreads), 0, s>>>(part, M, N, slices, p);
    hipCheck(hipGetLastError());
}

void launch_rows(const float *x, const float *weights, int rows, int terms, const HalvesRows &t, hipStream_t s) {
    halves_rows_kernel<<<dim3(t.row_blocks * 32 / kRowsWaves), dim3(64 * kRowsWaves), 0, s>>>(
        x, weights, rows, terms, terms % 4 == 0 && aligned16(x), t);
    hipCheck(hipGetLastError());
}

void launch_halves_rows(const float *x, const float *weights, const Halves &h, uint32_t *zero, int zeros,
                        hipStream_t s) {
    launch_rows(x, weights, h.rows, h.terms, {h.data, h.shift, h.row_blocks(), h.term_blocks(), false, zero, zeros}, s);
}

void launch_halves_table(const float *x, const Halves &h, hipStream_t s) {
    auto kernel = h.terms <= 32 * 24   ? halves_table_kernel<24, false>
                  : h.terms <= 32 * 52 ? halves_table_kernel<52, false>
                                       : halves_table_kernel<52, true>;
    kernel<<<dim3(h.row_blocks() / 2), dim3(kTableThreads), 0, s>>>(x, h, h.terms % 4 == 0 && aligned16(x));
    hipCheck(hipGetLastError());
}

void launch_column_largest(const float *x, int ld, const float *weights, float divisor, int terms, int cols,
                           uint32_t *largest, hipStream_t s) {
    const int chunks = (terms + kLargestTerms - 1) / kLargestTerms;
    if (ld % 4 == 0 && cols % 4 == 0 && aligned16(x))
        column_largest_kernel<f32x4_t><<<dim3(chunks, (cols + 255) / 256), dim3(kThreads), 0, s>>>(
            x, ld, weights, divisor, terms, cols, largest);
    else
        column_largest_kernel<float><<<dim3(chunks, (cols + 63) / 64), dim3(kThreads), 0, s>>>(x, ld, weights, divisor,
                                                                                              terms, cols, largest);
    hipCheck(hipGetLastError());
}

void launch_halves_columns(const float *x, int ld, const float *weights, float divisor, const Halves &h,
                           bool negate, const uint32_t *largest, hipStream_t s) {
    const int chunks = (h.term_blocks() * 16 + kColumnTerms - 1) / kColumnTerms;
    halves_columns_kernel<<<dim3(h.row_blocks(), chunks), dim3(kThreads), 0, s>>>(x, ld, weights, divisor, h, negate, largest);
    hipCheck(hipGetLastError());
}

int launch_logits(const Halves &A, const Halves &B, const LogitsArgs &l, hipStream_t s) {
    run_logits<Small>(A, B, l, s);
    return 64;
}

void launch_halves_product(const Halves &A, const Halves &B, const HalvesProduct &p, hipStream_t s) {
    run_product<Small, Across::kNone>(A, B, 0, p, s);
}

// Of the operand that is read across only its size counts from here on, as it is in this product.
void launch_product_across_a(const Halves &A, const Halves &B, const HalvesProduct &p, hipStream_t s) {
    CHECK_ERROR(A.rows != B.terms, "Operands of %d and %d terms.", A.rows, B.terms);
    run_product<Small, Across::kA>({A.data, A.shift, A.shift_all, A.terms, A.rows}, B, A.term_blocks(), p, s);
}

void launch_product_across_b(const Halves &A, const Halves &B, const HalvesProduct &p, hipStream_t s) {
    CHECK_ERROR(A.terms != B.rows, "Operands of %d and %d terms.", A.terms, B.rows);
    run_product<Small, Across::kB>(A, {B.data, B.shift, 0, B.terms, B.rows}, B.term_blocks(), p, s);
}

}  // namespace gptc
