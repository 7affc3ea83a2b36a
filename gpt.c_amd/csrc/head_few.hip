// Few rows against a whole vocabulary: the logits x W^T, and the gradient d W.
//
// Reading W is the time there (154 MB for GPT-2 small's, 29 us at the rate of a large
// copy), so W is read as it comes and each of its floats split once for up to 128
// rows.  The parts are those of gemm_halves.hpp, two fp16 values by a common scale; W's
// is the largest value of a row (logits) or column (d W) within a step of 32 terms,
// whose products are summed apart and come into the sum times that scale.  The other
// operand is small; its parts are formed once, in the order of the fragments.
//
// 768 features, 50257 tokens: 16 rows' logits 28 us (5.5 TB/s), where W comes from HBM 35
// to 37; 100 rows' 53 to 58, d W 44 to 47.  With three bf16 parts, which need no scale but
// six products instead of three, those took 70 and 60.
#include <algorithm>
#include "gpu_kernels.h"
#include "head_loss.hpp"

namespace gptc {

namespace {

constexpr int kThreads = 256;
constexpr int kFewWaves = 4;
__device__ __forceinline__ hf32x16 mfma_f16(hu32x4 a, hu32x4 b, hf32x16 c) {
    typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// The larger one of lanes l and l ^ 32.
__device__ __forceinline__ float across_halves(float x) {
    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(both[0]), __uint_as_float(both[1]));
}

// A kilobyte to LDS at `to` by loads that write no register but m0, which nothing else of these kernels uses (the compiler
// does not count them, so that its own waits wait for more than they need).
__device__ __forceinline__ void load_kilobyte(const hu32x4 *from, uint32_t lane_at, uint32_t to) {
    asm volatile(
        "s_mov_b32 m0, %2\n\t"
        "s_nop 0\n\t"
        "global_load_lds_dwordx4 %0, %1"
        :
        : "v"(lane_at), "s"(from), "s"(to)
        : "memory");
}
__device__ __forceinline__ void load_kilobyte(__amdgpu_buffer_rsrc_t from, uint32_t lane_at, uint32_t at, uint32_t to) {
    asm volatile(
        "s_mov_b32 m0, %3\n\t"
        "s_nop 0\n\t"
        "buffer_load_dwordx4 %0, %1, %2 offen lds"
        :
        : "v"(lane_at), "s"(from), "s"(at), "s"(to)
        : "memory");
}

// W from row `first` on; what lies past it reads as zero.  Offsets that are the same for all lanes are kept
// within `bytes`, as the range check is against what they leave of it.
struct RowsOfW {
    __amdgpu_buffer_rsrc_t rsrc;
    uint32_t bytes;
    __device__ __forceinline__ RowsOfW(const float *W, int V, int C, int first) {
        const int64_t skip = static_cast<int64_t>(min(first, V)) * C, left = 4 * (static_cast<int64_t>(V) * C - skip);
        bytes = static_cast<uint32_t>(min(left, static_cast<int64_t>(0xfffffffc)));
        rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float *>(W + skip), 0, static_cast<int>(bytes), 0x00020000);
    }
};

struct FewArgs {
    const float *W;
    int V, C;
    FewRows small;  // x or d
    LogitsArgs l;
    int rows, slice, columns;  // of the gradient: blocks of 16 tokens a workgroup, workgroups side by side
    float *part;
};

// 128 tokens (logits) or 128 columns (the gradient, DX) by 32 NB rows a workgroup, 32 by up to 64 a wave.  Both
// operands go to LDS, kDepth - 1 steps of 32 terms ahead: the waves share the small one, and W's rows come in
// whole lines (a lane a row, as the fragments want them, costs a cycle of the address path for every lane: the
// logits of 16 rows of 768 on 50257 tokens took 39 us so and take 28).  Up to four waves a SIMD, which hide
// each other's chain of loads, largest value, split and products.
constexpr int kSmallShift = kHalvesTop + 1;  // the small operand is held below 2^15: d by this shift, x by its rows'
template <int NB>
struct FewShape {
    static constexpr int kBlocks = NB < 2 ? NB : 2;                      // of 32 rows a wave
    static constexpr int kWaves = 4 * NB / kBlocks;
    static constexpr int kSmall = NB * 256, kStage = kSmall + 4 * 256;  // 16-byte chunks
    static constexpr int kDepth = NB == 1 ? 4 : NB == 2 ? 3 : 2;         // two workgroups a CU in 160 KB
    static constexpr int kLoadsSmall = NB * 4 / kWaves, kLoadsW = 16 / kWaves;  // kilobytes of a wave
};

template <int NB, bool DX>
__global__ __launch_bounds__(64 * FewShape<NB>::kWaves)
    __attribute__((amdgpu_waves_per_eu(FewShape<NB>::kWaves / 2))) void few_kernel(const FewArgs a) {
    using S = FewShape<NB>;
    __shared__ hu32x4 lds[S::kDepth * S::kStage];
    const int lane = threadIdx.x & 63, hf = lane >> 5, l32 = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), mine = w & 3;
    const int kbs = a.small.term_blocks(), rb = blockIdx.y * NB;
    int first = 0, count = kbs;  // blocks of 16 terms
    int at128 = blockIdx.x;      // which 128 tokens or columns
    if (DX) {
        // A slice's workgroups, which read the same rows of W and the same of d, go to one XCD (workgroup i runs on
        // XCD i % 8).
        const int turn = blockIdx.x >> 3;
        first = (turn / a.columns * 8 + static_cast<int>(blockIdx.x & 7)) * a.slice;
        if (first >= kbs) return;
        count = min(a.slice, kbs - first);
        at128 = turn % a.columns;
    }
    const int steps = count / 2;
    const RowsOfW rows(a.W, a.V, a.C, DX ? first * 16 : at128 * 128);
    const uint32_t base = static_cast<uint32_t>(reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) void *)lds));
    const hu32x4 *small = a.small.data + (static_cast<int64_t>(rb) * kbs + first) * 128;

    // Kilobyte q of W's 16 of a step.  Logits: eight rows' 128 bytes, whose 16-byte chunk c lies at c ^ (row / 2 % 8).
    // Gradient: two rows' 512 bytes, whose columns change places with the next 32 in every other four rows.  So a
    // row or a column a lane, the fragments' reads meet no bank twice.
    uint32_t lane_at[S::kLoadsW];
#pragma unroll
    for (int i = 0; i < S::kLoadsW; ++i) {
        const int q = w * S::kLoadsW + i;
        lane_at[i] = DX ? 4 * (static_cast<uint32_t>(hf) * a.C + 4 * (l32 ^ (8 * ((q >> 1) & 1))))
                        : 4 * (static_cast<uint32_t>(lane >> 3) * a.C + 4 * ((lane & 7) ^ (4 * (q & 1) + (lane >> 4))));
    }
    auto load_stage = [&](int step, int buffer) {
        const uint32_t to = base + buffer * (S::kStage * 16);
#pragma unroll
        for (int i = 0; i < S::kLoadsSmall; ++i) {
            const int c = w + i * S::kWaves;  // a kilobyte of block c / 4
            load_kilobyte(small + (static_cast<int64_t>(c / 4) * kbs + 2 * step) * 128 + (c % 4) * 64, lane * 16,
                          to + c * 1024);
        }
#pragma unroll
        for (int i = 0; i < S::kLoadsW; ++i) {
            const uint32_t q = w * S::kLoadsW + i;
            const uint32_t at = DX ? 4 * ((32 * step + 2 * q) * a.C + 128 * at128) : 4 * (8 * q * a.C + 32 * step);
            load_kilobyte(rows.rsrc, lane_at[i], min(at, rows.bytes), to + S::kSmall * 16 + q * 1024);
        }
    };
    hf32x16 acc[S::kBlocks];
#pragma unroll
    for (int i = 0; i < S::kBlocks; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][r] = 0.0f;
#pragma unroll
    for (int d = 0; d + 1 < S::kDepth; ++d) load_stage(min(d, steps - 1), d);
    int buffer = 0, free_buffer = S::kDepth - 1;
    for (int step = 0; step < steps; ++step) {
        // This step's loads have landed, all waves', and the buffer of the step before has been read.
        constexpr int kLoads = S::kLoadsSmall + S::kLoadsW;
        constexpr int kAhead = (S::kDepth - 2) * kLoads;
        static_assert(kAhead == 0 || kAhead == 6 || kAhead == 10, "the waits");
        if constexpr (kAhead == 0)
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else if constexpr (kAhead == 6)
            asm volatile("s_waitcnt vmcnt(6) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        else
            asm volatile("s_waitcnt vmcnt(10) lgkmcnt(0)\n\ts_barrier" ::: "memory");
        load_stage(min(step + S::kDepth - 1, steps - 1), free_buffer);
        const hu32x4 *at = lds + buffer * S::kStage;
        float v[2][8];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (DX) {
                const float *p = reinterpret_cast<const float *>(at + S::kSmall) + 4 * hf * 128 + (mine ^ hf) * 32 + l32;
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k][e] = p[(16 * k + (e & 3) + 8 * (e >> 2)) * 128];
            } else {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const hu32x4 c = at[S::kSmall + mine * 256 + l32 * 8 + ((4 * hf + 2 * k + e) ^ (l32 >> 1 & 7))];
#pragma unroll
                    for (int i = 0; i < 4; ++i) v[k][4 * e + i] = __uint_as_float(c[i]);
                }
            }
        }
        // Past a row's last feature lie the next row's, which its scale may not see.
        if (!DX && 32 * (step + 1) > a.C) {
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (32 * step + 16 * hf + 8 * k + e >= a.C) v[k][e] = 0.0f;
        }
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = fmaxf(top, fabsf(v[k][e]));
        top = across_halves(top);
        const int up = min(halves_shift(top), 126);
        hf32x16 t[S::kBlocks];
#pragma unroll
        for (int i = 0; i < S::kBlocks; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) t[i][r] = 0.0f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            hu32x4 f[2], g[S::kBlocks][2];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t hi, lo;
                halves_split(__builtin_amdgcn_ldexpf(v[k][2 * e], up), __builtin_amdgcn_ldexpf(v[k][2 * e + 1], up), hi, lo);
                f[0][e] = hi;
                f[1][e] = lo;
            }
#pragma unroll
            for (int i = 0; i < S::kBlocks; ++i)
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    g[i][q] = at[((w >> 2) * S::kBlocks + i) * 256 + k * 128 + q * 64 + lane];
            constexpr int kParts[3][2] = {{1, 0}, {0, 1}, {0, 0}};  // smallest products first
#pragma unroll
            for (int q = 0; q < 3; ++q)
#pragma unroll
                for (int i = 0; i < S::kBlocks; ++i) t[i] = mfma_f16(g[i][kParts[q][0]], f[kParts[q][1]], t[i]);
        }
        // 64 terms of a sign.  Both scales go: with the small operand's, values of W 2^15 below the largest float would take
        // the sums past it.
        const float down = __builtin_amdgcn_ldexpf(step & 2 ? -1.0f : 1.0f, -up - kSmallShift);
#pragma unroll
        for (int i = 0; i < S::kBlocks; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[i][r] = fmaf(down, t[i][r], acc[i][r]);
        free_buffer = buffer;
        buffer = buffer + 1 == S::kDepth ? 0 : buffer + 1;
    }
    asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");  // from here on `lds` is free
    const int block = rb + (w >> 2) * S::kBlocks;
    // A lane holds a token (or column) and 16 rows.  The logits are put with a row a lane, and change over in LDS.
    constexpr int kStride = 36;  // words of a row
    float2 *stats = reinterpret_cast<float2 *>(lds);  // (blocks of 32 rows, the four waves' tokens, rows)
    float *across = reinterpret_cast<float *>(stats + NB * 128) + w * (32 * kStride);
    static_assert(DX || NB * 1024 + S::kWaves * 32 * kStride * 4 <= S::kDepth * S::kStage * 16, "room");
    // In a loop over the blocks, whose sums move up: code that runs once a wave is paid by its fetch.
#pragma unroll 1
    for (int i = 0; i < S::kBlocks; ++i) {
        hf32x16 v[1] = {acc[0]};
        if (S::kBlocks == 2) acc[0] = acc[S::kBlocks - 1];
        if (!DX) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int4 back = *reinterpret_cast<const int4 *>(a.small.shift + (block + i) * 32 + 8 * q + 4 * hf);
                const int shift[4] = {back.x, back.y, back.z, back.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    across[(8 * q + 4 * hf + e) * kStride + l32] =
                        __builtin_amdgcn_ldexpf(v[0][4 * q + e], kSmallShift - shift[e]);
            }
            wave_lds_order();
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const f32x4_t x = *reinterpret_cast<const f32x4_t *>(across + l32 * kStride + 8 * q + 4 * hf);
#pragma unroll
                for (int e = 0; e < 4; ++e) v[0][4 * q + e] = x[e];
            }
            wave_lds_order();
            const float2 stat = put_logits<1, false>(a.l, v, at128 * 128 + mine * 32, block + i);
            if (hf == 0) stats[((w >> 2) * S::kBlocks + i) * 128 + mine * 32 + l32] = stat;
            continue;
        }
        // Rows past the last one and columns past the last one are not written.
        const int bytes = 4 * a.rows * a.C, c = at128 * 128 + mine * 32 + l32;
        const __amdgpu_buffer_rsrc_t out = __builtin_amdgcn_make_buffer_rsrc(
            a.part + static_cast<int64_t>(first / a.slice) * a.rows * a.C, 0, bytes, 0x00020000);
        const uint32_t lane_out = c < a.C ? 4 * (static_cast<uint32_t>((block + i) * 32 + 4 * hf) * a.C + c) : 0x80000000u;
#pragma unroll
        for (int r = 0; r < 16; ++r)
            __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v[0][r]), out, lane_out,
                                                  min(4 * (8 * (r >> 2) + (r & 3)) * a.C, bytes), 0);
    }
    if (DX) return;
    __syncthreads();
    if (threadIdx.x >= 32 * NB) return;
    const float2 *p = stats + (threadIdx.x >> 5) * 128 + l32;
    float m = p[0].x, s = 0.0f;
#pragma unroll
    for (int k = 1; k < 4; ++k) m = fmaxf(m, p[32 * k].x);
    constexpr float kLog2e = 1.4426950408889634f;
    const float ref = m == -INFINITY ? 0.0f : m;  // no logit but minus infinity or NaN, which stays in the sum
#pragma unroll
    for (int k = 0; k < 4; ++k) s += p[32 * k].y * __builtin_amdgcn_exp2f((p[32 * k].x - ref) * kLog2e);
    a.l.stats[static_cast<int64_t>(at128) * a.l.row_stride + rb * 32 + threadIdx.x] = make_float2(m, s);
}

template <bool DX>
void run_few(const FewArgs &a, int n, int across, hipStream_t s) {
    auto kernel = n == 1 ? few_kernel<1, DX> : n == 2 ? few_kernel<2, DX> : few_kernel<4, DX>;
    const int waves = n == 1 ? FewShape<1>::kWaves : n == 2 ? FewShape<2>::kWaves : FewShape<4>::kWaves;
    kernel<<<dim3(across, a.small.row_blocks / n), dim3(64 * waves), 0, s>>>(a);
    hipCheck(hipGetLastError());
}

// dW = d^T x for up to 16 KB terms (rows): writing dW is the time (100 rows of 768 on 50257: 40 us for 154 MB out and
// 26 in; 7 more without the order by XCD, 8 more without the stores' hint).  Both operands come as two fp16 parts
// (Halves).  A workgroup keeps its 128 columns of x in LDS and its waves stream blocks of 32 tokens.
template <int KB>
__global__ __launch_bounds__(kThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void few_dw_kernel(
    const Halves dt, const Halves xt, const HalvesProduct p, int columns) {
    __shared__ hu32x4 lds[4 * KB * 128];
    const int lane = threadIdx.x & 63, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // The workgroups that read the same blocks of d^T and write the same rows go to one XCD (workgroup i runs on XCD i % 8).
    const int turn = blockIdx.x >> 3, column = turn % columns, group = turn / columns * 8 + static_cast<int>(blockIdx.x & 7);
    const hu32x4 *from = xt.data + static_cast<int64_t>(column) * (4 * KB * 128);
    {
        constexpr int kPer = 4 * KB * 128 / kThreads;
        hu32x4 v[kPer];
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = from[threadIdx.x + i * kThreads];
#pragma unroll
        for (int i = 0; i < kPer; ++i) lds[threadIdx.x + i * kThreads] = v[i];
    }
    const int blocks = (dt.rows + 31) / 32, stride = static_cast<int>(gridDim.x) / columns * kFewWaves;
    int m = group * kFewWaves + w;
    hu32x4 a[KB][2];
    auto load = [&](int block) {
        const hu32x4 *at = dt.data + static_cast<int64_t>(min(block, blocks - 1)) * (KB * 128) + lane;
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int q = 0; q < 2; ++q) a[k][q] = at[(2 * k + q) * 64];
    };
    load(m);
    __syncthreads();
    for (; m < blocks; m += stride) {
        hu32x4 now[KB][2];
#pragma unroll
        for (int k = 0; k < KB; ++k)
#pragma unroll
            for (int q = 0; q < 2; ++q) now[k][q] = a[k][q];
        load(m + stride);
#pragma unroll 1
        for (int j = 0; j < 4; ++j) {
            // A block's rows of C; what lies past the last row or column is neither read nor written.
            const int bytes = 4 * min(32, dt.rows - m * 32) * p.ldc;
            const __amdgpu_buffer_rsrc_t C = __builtin_amdgcn_make_buffer_rsrc(
                p.C + static_cast<int64_t>(m) * 32 * p.ldc, 0, bytes, 0x00020000);
            auto row_at = [&](int r) { return min(4 * (8 * (r >> 2) + (r & 3)) * p.ldc, bytes); };
            const int c = column * 128 + 32 * j + (lane & 31);
            const int up = -dt.shift_all - xt.shift[c];
            const uint32_t mine = c < xt.rows ? 4 * (static_cast<uint32_t>(4 * hf) * p.ldc + c) : 0x80000000u;
            float old[16];
            if (p.add)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    old[r] = __uint_as_float(
                        __builtin_amdgcn_raw_buffer_load_b32(C, mine, row_at(r), 0));
            // Steps of 64 terms, every other one negated in d^T.
            hf32x16 t[KB / 4];
            constexpr int kParts[3][2] = {{1, 0}, {0, 1}, {0, 0}};
#pragma unroll
            for (int i = 0; i < KB / 4; ++i) {
                hu32x4 b[4][2];
#pragma unroll
                for (int k = 0; k < 4; ++k)
#pragma unroll
                    for (int q = 0; q < 2; ++q) b[k][q] = lds[(j * KB + 4 * i + k) * 128 + q * 64 + lane];
#pragma unroll
                for (int r = 0; r < 16; ++r) t[i][r] = 0.0f;
#pragma unroll
                for (int q = 0; q < 3; ++q)
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        t[i] = mfma_f16(now[4 * i + k][kParts[q][0]], b[k][kParts[q][1]], t[i]);
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                float v = t[0][r];
                if (KB == 8) v -= t[KB / 4 - 1][r];
                v = __builtin_amdgcn_ldexpf(v, up);
                if (p.add) v = old[r] + v;
                __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(v), C, mine, row_at(r), kStreamed);
            }
        }
    }
}

}  // namespace

// Waves of one block of rows take one, two or four.
int few_row_blocks(int rows) {
    const int blocks = (rows + 31) / 32;
    return blocks <= 2 ? blocks : (blocks + 3) / 4 * 4;
}

void launch_few_rows(const float *x, const float *weights, int rows, const FewRows &t, uint32_t *zero, int zeros,
                     hipStream_t s) {
    launch_rows(x, weights, rows, t.terms, {t.data, t.shift, t.row_blocks, t.term_blocks(), true, zero, zeros}, s);
}

int launch_few_logits(const float *W, int V, int C, const FewRows &x, const LogitsArgs &l, hipStream_t s) {
    const int across = l.token_blocks / 4;
    int n = std::min(x.row_blocks, 4);
    // Rather W again than CUs without work: 450 rows of 1820 on 2029 tokens 77 us in 64 workgroups, 57 in 128, 49 in 256;
    // 64 of 768 on 20000 33 in 157, 40 in 314; 200 of 768 on 5003 40 in 80, 32 in 160, 34 in 320.
    while (n > 1 && across * (x.row_blocks / n) < 144) n /= 2;
    run_few<false>({W, V, C, x, l, 0, 0, 0, nullptr}, n, across, s);
    return 128;
}

void launch_few_dx(const FewRows &d, const float *W, int V, int C, int rows, const HalvesProduct &p, hipStream_t s) {
    CHECK_ERROR(static_cast<int64_t>(rows) * C >= 1 << 29, "few_dx: %d x %d results.", rows, C);
    const int groups = d.row_blocks <= 2 ? 1 : d.row_blocks / 4, columns = (C + 127) / 128, kbs = d.term_blocks();
    // About two workgroups a CU, at least 128 terms each; a slice's offsets stay within 32 bits.
    const int least = static_cast<int>(static_cast<int64_t>(V) * C / (1 << 28)) + 1;
    int slices = std::max(least, 512 / (columns * groups));
    slices = std::min(slices, kbs / 8);
    const int slice = ((kbs + slices - 1) / slices + 7) / 8 * 8;  // whole steps, whose signs alternate
    slices = (kbs + slice - 1) / slice;
    float *part = static_cast<float *>(alloc_cuda(sizeof(float) * static_cast<size_t>(rows) * C * slices));
    CHECK_ERROR(d.shift != nullptr || d.shift_all != kSmallShift, "few_dx: shares times 2^%d.", d.shift_all);
    run_few<true>({W, V, C, d, {}, rows, slice, columns, part}, std::min(d.row_blocks, 4),
                  columns * ((slices + 7) / 8 * 8), s);
    launch_join_slices(part, rows, C, slices, p, s);
    free_cuda(part);
}

void launch_few_dw(const Halves &dt, const Halves &xt, const HalvesProduct &p, hipStream_t s) {
    CHECK_ERROR(dt.terms != xt.terms || dt.terms > kFewDwTerms || p.ldc >= 1 << 22, "few_dw: %d and %d terms, rows of %d.",
                dt.terms, xt.terms, p.ldc);
    const int columns = (xt.rows + 127) / 128, blocks = (dt.rows + 31) / 32;
    // Two workgroups a CU, the same number for each XCD.
    const int groups = std::max(1, std::min((blocks + 8 * kFewWaves - 1) / (8 * kFewWaves), 64 / columns)) * 8;
    auto kernel = dt.term_blocks() == 4 ? few_dw_kernel<4> : few_dw_kernel<8>;
    kernel<<<dim3(columns * groups), dim3(kThreads), 0, s>>>(dt, xt, p, columns);
    hipCheck(hipGetLastError());
}

}  // namespace gptc
