// Products of block-scaled 8-bit matrices (tsne_operators.h has the format): c = a b^T.
//
// The 8-bit matrix instructions take the scales themselves, so that a product of blocks is one instruction for 16 x 16
// results and nothing is rescaled.  They add products in groups of eight and drop, in each, what lies more than 2^-13 below
// the largest (the groups' sums are added in 32 bits).  What that comes to, of a result: 1.5e-5 for normally distributed
// factors, a hundredth of a bfloat16's half unit (2^-9) and not of a half's (2^-11) or a float's; at most 7 * 2^-13 of the
// sum of its groups' largest products, which is more than any half unit where those cancel.  So results in halves and floats
// are summed from exact products (kExact), and bfloat16 where the caller asks for it: values times scales are bf16 numbers,
// and the bf16 instructions lose nothing, at half the rate.
//
// What a product is bound by changes with its size, and so does its form (cut_of).  us (TFLOP/s) into bfloat16 by the 8-bit
// instructions and into floats, exactly; alone the instructions reach 3890 TFLOP/s on normally distributed values, a library's
// 8-bit product with one scale a matrix 2650 at the second size:
//   256 x 256 tiles       8192 x 8192 x 512      54 (1280)   96 (716)   storing: 134 MB of bfloat16 are 28 us at a copy's rate
//                         8192 x 8192 x 4096    220 (2500)  435 (1265)  the clock, which falls with what is multiplied, and
//                                                                       64 KB of factors a block through each unit's load path
//   128 x 128, two teams  4096 x 1024 x 8192     38 (1835)   68 (1014)  the same, for half the products a byte
//   64 x 64, four teams   512 x 2048 x 4096      12 (710)    16 (551)   a block's way from memory through LDS, 1.2 us a step
//   64 x 64               1203 x 1111 x 784       6 (335)     9 (225)   the first loads' latency (7 on factors just written)
//   16 rows               1 x 8192 x 8192        15          17         reading b, 4.4 TB/s (a copy runs at 4.8)
#include "../../include/tsnecuda/tsne_operators.h"
#include "lds_load.h"
#include "operators.h"

#include <algorithm>
#include <type_traits>

namespace tsnehip {

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// 32 of the 128 values of a row's block, as one lane of a 16 x 16 x 128 product holds them.
struct Fragment {
    u32x4 lo, hi;
};

// acc (16 x 16) += a (16 x 128) b (16 x 128)^T with the lanes' row scales (in the low byte).
__device__ __forceinline__ f32x4 multiply(const Fragment &a, const Fragment &b, unsigned int sa, unsigned int sb,
                                          f32x4 acc) {
    i32x8 x, y;
    for (int i = 0; i < 4; ++i) {
        x[i] = (int)a.lo[i], x[4 + i] = (int)a.hi[i];
        y[i] = (int)b.lo[i], y[4 + i] = (int)b.hi[i];
    }
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, acc, 0, 0, 0, (int)sa, 0, (int)sb);
}

// 2^(byte - 127) of a byte that plain_scales() lets through.
__device__ __forceinline__ float scale_value(unsigned int byte) { return __uint_as_float(byte << 23); }
// Values times scales from 2^-111 to 2^119 are bf16 numbers: nothing below the range's end, and 448 * 2^119 within it.
__device__ __forceinline__ bool plain_scales(unsigned int least, unsigned int most) { return least >= 16 && most <= 246; }

// Eight values times a scale, as bf16 numbers: exactly.
__device__ __forceinline__ bf16x8 widen(unsigned int w0, unsigned int w1, float scale) {
    const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, false),
                 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w0, scale, true),
                 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, false),
                 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w1, scale, true);
    return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// A lane's 32 values, as the four 16 x 16 x 32 products of a block take them.
__device__ __forceinline__ void widen(const Fragment &f, float scale, bf16x8 *out) {
    out[0] = widen(f.lo[0], f.lo[1], scale), out[1] = widen(f.lo[2], f.lo[3], scale);
    out[2] = widen(f.hi[0], f.hi[1], scale), out[3] = widen(f.hi[2], f.hi[3], scale);
}

// A block's products, exact, before their scales.
__device__ __forceinline__ f32x4 multiply_exactly(const Fragment &a, const Fragment &b) {
    bf16x8 wa[4], wb[4];
    widen(a, 1.0f, wa);
    widen(b, 1.0f, wb);
    f32x4 block = {};
#pragma unroll
    for (int q = 0; q < 4; ++q) block = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa[q], wb[q], block, 0, 0, 0);
    return block;
}
// acc += block times its rows' and its column's scales, whatever they are.  A lane's four results are of rows 4 (lane / 16)
// and on of a, whose scales those lanes have, and of the row of b whose scale it has itself.
__device__ __forceinline__ void add_scaled(f32x4 &acc, f32x4 block, unsigned int ea, unsigned int eb) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const unsigned int of_row = __shfl((int)(ea & 255), (int)(threadIdx.x % kWave) / 16 * 4 + q, kWave), of_column = eb & 255;
        const float v = ldexpf(block[q], (int)of_row + (int)of_column - 254);
        acc[q] += of_row == 255 || of_column == 255 ? __builtin_nanf("") : v;
    }
}

typedef u32x2 u32x2_unaligned __attribute__((aligned(2)));
__device__ __forceinline__ unsigned int pack_bf16(float a, float b) {
    return (unsigned int)__builtin_bit_cast(unsigned short, (__bf16)a) | (unsigned int)__builtin_bit_cast(unsigned short, (__bf16)b) << 16;
}
__device__ __forceinline__ void store4(float *to, f32x4 v) {
    const float w[4] = {v[0], v[1], v[2], v[3]};
    store_vec(to, w);
}
__device__ __forceinline__ void store4(__bf16 *to, f32x4 v) {
    *reinterpret_cast<u32x2_unaligned *>(to) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
}

// A workgroup's tile: kWM x kWN waves of kFM x kFN fragments of 16 x 16 results, and how many blocks of it LDS holds.  With
// several teams of such waves each takes its share of the blocks in turn, and their sums are added in LDS.
template <int kWMs, int kWNs, int kFMs, int kFNs, int kHeld, int kTeamsOf = 1>
struct TileShape {
    static constexpr int kWM = kWMs, kWN = kWNs, kFM = kFMs, kFN = kFNs, kStages = kHeld, kTeams = kTeamsOf;
    static constexpr int kWaves = kWM * kWN, kThreads = kWave * kWaves * kTeams;
    static constexpr int kRows = 16 * kFM * kWM, kCols = 16 * kFN * kWN;
    static constexpr int kData = (kRows + kCols) * kBlock;           // a block of both factors
    static constexpr int kScales = (kRows + kCols) * 4;              // ... and the four bytes of scales that hold its own
    static constexpr int kTeamLds = kStages * (kData + kScales), kLds = kTeams * kTeamLds;
    // A wave's loads of a block: eight rows of data an instruction, and one instruction of 64 rows' scales.
    static constexpr int kLoadsA = kRows / 8 / kWaves, kLoadsB = kCols / 8 / kWaves, kLoads = kLoadsA + kLoadsB + 1;
    static_assert((kRows + kCols) / 64 <= kWaves && kLds <= 160 * 1024 && (kTeams - 1) * kRows * kCols * 4 <= kLds);
};

// Where a row's 16 bytes `chunk` of a block lie in its 128 bytes of LDS: eight rows that are read together, and 16 as well,
// take every bank alike.
__device__ __forceinline__ int place_of(int row, int chunk) { return chunk ^ (row & 7) ^ ((row >> 3) & 1); }

struct Product {
    const uint8_t *a, *a_scales, *b, *b_scales;
    int64_t m, n, k;
    void *c;
    int64_t c_stride;
    int exact;
    float *partial;  // room for the partial results
};

// All of the wave's reads of LDS are here.
__device__ __forceinline__ void wait_for_lds() {
    __builtin_amdgcn_s_waitcnt(0xc07f);  // lgkmcnt(0)
    asm volatile("" ::: "memory");
}
// A barrier that nothing is moved across, and that waits for nothing else.
__device__ __forceinline__ void phase_end() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");
}

// Workgroups go to the XCDs in turn: each takes a run of tiles, in bands of four tile rows, so that what it reads at a time is
// a few panels of both factors.
__device__ __forceinline__ void tile_origin(unsigned int which, unsigned int row_tiles, unsigned int column_tiles, int rows,
                                            int cols, int64_t &r0, int64_t &c0) {
    const unsigned int tiles = row_tiles * column_tiles, xcd = which % 8, share = tiles / 8, extra = tiles % 8;
    const unsigned int tile = xcd * share + min(xcd, extra) + which / 8;
    const unsigned int band = tile / (4 * column_tiles), in_band = tile % (4 * column_tiles);
    const unsigned int band_rows = min(4u, row_tiles - 4 * band);
    r0 = (int64_t)(4 * band + in_band % band_rows) * rows;
    c0 = (int64_t)(in_band / band_rows) * cols;
}

// blockIdx.y: one of the parts of the sum, of `part` blocks, whose results go to c + that many times c_part.
template <typename T, bool kExact, class Shape>
__global__ __launch_bounds__(Shape::kThreads, 2) void tiled_product_kernel(
    const uint8_t *__restrict__ a, const uint8_t *__restrict__ a_scales, const uint8_t *__restrict__ b,
    const uint8_t *__restrict__ b_scales, int64_t m, int64_t n, int blocks, int part, int64_t data_stride,
    int64_t scale_stride, T *__restrict__ c, int64_t c_stride, int64_t c_part, unsigned int row_tiles,
    unsigned int column_tiles) {
    extern __shared__ unsigned char all_lds[];
    constexpr int kRows = Shape::kRows, kCols = Shape::kCols, kWaves = Shape::kWaves, kStages = Shape::kStages, kTeams = Shape::kTeams;
    constexpr bool kEach = kStages > 2 || kTeams > 1;
    constexpr int kWN = Shape::kWN, kFM = Shape::kFM, kFN = Shape::kFN;
    int64_t r0, c0;
    tile_origin(blockIdx.x, row_tiles, column_tiles, kRows, kCols, r0, c0);
    const int lane = threadIdx.x % kWave, any_wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int team = kTeams > 1 ? any_wave / kWaves : 0, wave = kTeams > 1 ? any_wave % kWaves : any_wave;
    unsigned char *const lds = all_lds + team * Shape::kTeamLds;
    const unsigned int base = __builtin_amdgcn_readfirstlane((unsigned int)(size_t)(LdsByte *)lds);
    // The team's blocks: first, first + kTeams, ... before end.
    const int part_first = blockIdx.y * part, end = min(part_first + part, blocks), first = part_first + team;

    // Loading: a wave's instruction brings eight rows' blocks.  (Rows behind the last are the last once more.)
    unsigned int from_a[Shape::kLoadsA], from_b[Shape::kLoadsB];
#pragma unroll
    for (int i = 0; i < Shape::kLoadsA; ++i) {
        const int row = (i * kWaves + wave) * 8 + lane / 8;
        from_a[i] = (unsigned int)(min((int64_t)row, m - 1 - r0) * data_stride) + 16 * place_of(row, lane % 8);
    }
#pragma unroll
    for (int i = 0; i < Shape::kLoadsB; ++i) {
        const int row = (i * kWaves + wave) * 8 + lane / 8;
        from_b[i] = (unsigned int)(min((int64_t)row, n - 1 - c0) * data_stride) + 16 * place_of(row, lane % 8);
    }
    const int scale_rows = wave % ((kRows + kCols) / 64) * 64;
    const bool scales_of_a = scale_rows < kRows;
    const int scale_row = (scales_of_a ? scale_rows : scale_rows - kRows) + lane;
    const unsigned int from_s = (unsigned int)(min((int64_t)scale_row, scales_of_a ? m - 1 - r0 : n - 1 - c0) * scale_stride);
    const uint8_t *pa = a + r0 * data_stride, *pb = b + c0 * data_stride;
    const uint8_t *ps = scales_of_a ? a_scales + r0 * scale_stride : b_scales + c0 * scale_stride;
    auto load_block = [&](int k, int stage) {
        const unsigned int to = base + stage * Shape::kData;
#pragma unroll
        for (int i = 0; i < Shape::kLoadsA; ++i)
            load_to_lds(pa + (int64_t)k * kBlock, from_a[i], to + (i * kWaves + wave) * 1024);
#pragma unroll
        for (int i = 0; i < Shape::kLoadsB; ++i)
            load_to_lds(pb + (int64_t)k * kBlock, from_b[i], to + kRows * kBlock + (i * kWaves + wave) * 1024);
        // (Four blocks' scales at once; where several blocks are in flight, or a team leaves some out, each brings them.)
        if (kEach || k == first || k % 4 == 0)
            load_word_to_lds(ps + (k & ~3), from_s,
                             base + kStages * Shape::kData + (kEach ? stage : k / 4 & 1) * Shape::kScales + scale_rows * 4);
    };

    // Reading: the wave's fragments.
    const int wm = wave / kWN, wn = wave % kWN, group = lane / 16, lr = lane % 16;
    auto fragment = [&](const unsigned char *from, int row) {
        Fragment f;
        f.lo = *reinterpret_cast<const u32x4 *>(from + row * kBlock + 16 * place_of(row, 2 * group));
        f.hi = *reinterpret_cast<const u32x4 *>(from + row * kBlock + 16 * place_of(row, 2 * group + 1));
        return f;
    };
    f32x4 acc[kFM][kFN] = {};
    unsigned int ea[kFM], eb[kFN];
    auto read_scales = [&](int k, int stage) __attribute__((always_inline)) {
        if (kEach || k == first || k % 4 == 0) {
            const unsigned int *scales = reinterpret_cast<const unsigned int *>(
                lds + kStages * Shape::kData + (kEach ? stage : k / 4 & 1) * Shape::kScales);
            const int shift = 8 * (k & 3);
#pragma unroll
            for (int i = 0; i < kFM; ++i) ea[i] = scales[(wm * kFM + i) * 16 + lr] >> shift;
#pragma unroll
            for (int j = 0; j < kFN; ++j) eb[j] = scales[kRows + (wn * kFN + j) * 16 + lr] >> shift;
        } else {
#pragma unroll
            for (int i = 0; i < kFM; ++i) ea[i] >>= 8;
#pragma unroll
            for (int j = 0; j < kFN; ++j) eb[j] >>= 8;
        }
    };
    auto scales_are_plain = [&]() __attribute__((always_inline)) {
        unsigned int least = 255, most = 0;
#pragma unroll
        for (int i = 0; i < kFM; ++i) least = min(least, ea[i] & 255), most = max(most, ea[i] & 255);
#pragma unroll
        for (int j = 0; j < kFN; ++j) least = min(least, eb[j] & 255), most = max(most, eb[j] & 255);
        return (bool)__all(plain_scales(least, most));
    };
    // Exact products of a block at la and lb, whatever its scales are.  (Seldom run: it may be slow, but not take registers.)
    auto multiply_any = [&](const unsigned char *la, const unsigned char *lb) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < kFM; ++i)
#pragma unroll
            for (int j = 0; j < kFN; ++j) {
                add_scaled(acc[i][j], multiply_exactly(fragment(la, (wm * kFM + i) * 16 + lr),
                                                       fragment(lb, (wn * kFN + j) * 16 + lr)), ea[i], eb[j]);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    // The products of a block; read_a(i) and read_b(j) give the fragments, which are in LDS at la and lb.
    auto multiply_block = [&](const unsigned char *la, const unsigned char *lb, auto read_a, auto read_b) __attribute__((always_inline)) {
        if constexpr (!kExact) {
            Fragment fb[kFN];
#pragma unroll
            for (int j = 0; j < kFN; ++j) fb[j] = read_b(j);
            // (b's fragments first: a lane then holds four neighbouring columns of one row of the result)
#pragma unroll
            for (int i = 0; i < kFM; ++i) {
                const Fragment fa = read_a(i);
#pragma unroll
                for (int j = 0; j < kFN; ++j) acc[i][j] = multiply(fb[j], fa, eb[j], ea[i], acc[i][j]);
            }
            return;
        }
        if (__builtin_expect(scales_are_plain(), 1)) {
            bf16x8 wb[kFN][4];
#pragma unroll
            for (int j = 0; j < kFN; ++j) widen(read_b(j), scale_value(eb[j] & 255), wb[j]);
#pragma unroll
            for (int i = 0; i < kFM; ++i) {
                bf16x8 wa[4];
                widen(read_a(i), scale_value(ea[i] & 255), wa);
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int j = 0; j < kFN; ++j)
                        acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa[q], wb[j][q], acc[i][j], 0, 0, 0);
            }
        } else {
            multiply_any(la, lb);
        }
    };
    if constexpr (kTeams == 2) {
        // Two waves share a SIMD, one of each team, and the teams take turns: while the one multiplies the other loads (which
        // holds up whoever does), reads and, for exact products, widens b's fragments; a's are widened between products.
        Fragment fa[kFM], fb[kFN];
        bf16x8 wb[kExact ? kFN : 1][4];
        int stage = 0;
        if (first < end) load_block(first, 0);
        wait_for_loads();
        phase_end();
        if (team == 1) phase_end();
        for (int step = part_first; step < end; step += kTeams) {
            const int k = step + team;
            if (k + kTeams < end) load_block(k + kTeams, stage ^ 1);
            const unsigned char *la = lds + stage * Shape::kData, *lb = la + kRows * kBlock;
            bool plain = true;
            if (k < end) {
                read_scales(k, stage);
#pragma unroll
                for (int j = 0; j < kFN; ++j) fb[j] = fragment(lb, (wn * kFN + j) * 16 + lr);
                if constexpr (!kExact) {
#pragma unroll
                    for (int i = 0; i < kFM; ++i) fa[i] = fragment(la, (wm * kFM + i) * 16 + lr);
                } else {
                    fa[0] = fragment(la, wm * kFM * 16 + lr);
                    plain = scales_are_plain();
#pragma unroll
                    for (int j = 0; j < kFN; ++j) widen(fb[j], scale_value(eb[j] & 255), wb[j]);
                }
            }
            wait_for_lds();
            phase_end();
            if (k < end) {
                __builtin_amdgcn_s_setprio(1);
                if constexpr (!kExact) {
                    multiply_block(la, lb, [&](int i) { return fa[i]; }, [&](int j) { return fb[j]; });
                } else if (__builtin_expect(plain, 1)) {
                    bf16x8 wa[2][4];
                    widen(fa[0], scale_value(ea[0] & 255), wa[0]);
#pragma unroll
                    for (int i = 0; i < kFM; ++i) {
                        if (i + 1 < kFM) fa[i + 1] = fragment(la, (wm * kFM + i + 1) * 16 + lr);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
#pragma unroll
                            for (int j = 0; j < kFN; ++j)
                                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa[i % 2][q], wb[j][q], acc[i][j], 0, 0, 0);
                        if (i + 1 < kFM) widen(fa[i + 1], scale_value(ea[i + 1] & 255), wa[(i + 1) % 2]);
#pragma unroll
                        for (int t = 0; t < kFN * 4; ++t) {  // a product, a conversion, ...
                            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                            __builtin_amdgcn_sched_group_barrier(0x002, 1, 0);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                } else {
                    multiply_any(la, lb);
                }
                __builtin_amdgcn_s_setprio(0);
            }
            wait_for_loads();
            phase_end();
            stage ^= 1;
        }
        if (team == 0) phase_end();
    } else {
        // Blocks in flight: all that LDS holds but the one that is multiplied.
        auto all_blocks = [&](auto multiply_one) __attribute__((always_inline)) {
#pragma unroll
            for (int i = 0; i < kStages - 1; ++i)
                if (first + i * kTeams < end) load_block(first + i * kTeams, i);
            int stage = 0;
            for (int step = part_first; step < end; step += kTeams) {
                const int k = step + team;
                // This block is here, and everybody is done with the one before, whose place the next load takes.
                if (k + (kStages - 2) * kTeams < end) wait_for_loads<(kStages - 2) * Shape::kLoads>();
                else wait_for_loads<0>();
                __syncthreads();
                if (k + (kStages - 1) * kTeams < end) load_block(k + (kStages - 1) * kTeams, stage == 0 ? kStages - 1 : stage - 1);
                if (kTeams > 1 && k >= end) continue;  // (the last step, for some teams)
                const unsigned char *la = lds + stage * Shape::kData, *lb = la + kRows * kBlock;
                read_scales(k, stage);
                stage = stage + 1 == kStages ? 0 : stage + 1;
                multiply_one(la, lb);
            }
        };
        if constexpr (kExact && kFM * kFN > 16) {
            // So many results leave no registers for a choice in every block: each wave looks at all its scales first, and
            // as the ways that follow have barriers, all waves take the same.
            unsigned int least = 255, most = 0;
            for (int row = lane; row < 16 * (kFM + kFN); row += kWave) {
                const bool of_a = row < 16 * kFM;
                const int64_t r = of_a ? min(r0 + wm * 16 * kFM + row, m - 1) : min(c0 + wn * 16 * kFN + row - 16 * kFM, n - 1);
                const unsigned int *words = reinterpret_cast<const unsigned int *>((of_a ? a_scales : b_scales) + r * scale_stride);
                for (int i = part_first / 4; i * 4 < end; ++i) {
                    const unsigned int four = words[i];
#pragma unroll
                    for (int q = 0; q < 4; ++q) least = min(least, four >> 8 * q & 255), most = max(most, four >> 8 * q & 255);
                }
            }
            if (__syncthreads_and(plain_scales(least, most))) {
                all_blocks([&](const unsigned char *la, const unsigned char *lb) __attribute__((always_inline)) {
                    bf16x8 wb[kFN][4];
#pragma unroll
                    for (int j = 0; j < kFN; ++j) widen(fragment(lb, (wn * kFN + j) * 16 + lr), scale_value(eb[j] & 255), wb[j]);
#pragma unroll
                    for (int i = 0; i < kFM; ++i) {
                        bf16x8 wa[4];
                        widen(fragment(la, (wm * kFM + i) * 16 + lr), scale_value(ea[i] & 255), wa);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
#pragma unroll
                            for (int j = 0; j < kFN; ++j)
                                acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wa[q], wb[j][q], acc[i][j], 0, 0, 0);
                    }
                });
            } else {
                all_blocks(multiply_any);
            }
        } else {
            all_blocks([&](const unsigned char *la, const unsigned char *lb) __attribute__((always_inline)) {
                multiply_block(la, lb, [&](int i) { return fragment(la, (wm * kFM + i) * 16 + lr); },
                               [&](int j) { return fragment(lb, (wn * kFN + j) * 16 + lr); });
            });
        }
    }
    c += blockIdx.y * c_part;
    if constexpr (kTeams > 1) {
        // The other teams' sums, in the layout of the lanes, and in the teams' order.
        constexpr int kEachTeam = kFM * kFN * kWave * kWaves;
        f32x4 *const sums = reinterpret_cast<f32x4 *>(all_lds) + wave * kFM * kFN * kWave + lane;
        __syncthreads();
        if (team > 0) {
#pragma unroll
            for (int i = 0; i < kFM * kFN; ++i) sums[(team - 1) * kEachTeam + i * kWave] = acc[i / kFN][i % kFN];
        }
        __syncthreads();
        if (team > 0) return;
#pragma unroll
        for (int t = 0; t < kTeams - 1; ++t)
#pragma unroll
            for (int i = 0; i < kFM * kFN; ++i) acc[i / kFN][i % kFN] += sums[t * kEachTeam + i * kWave];
    }
#pragma unroll
    for (int i = 0; i < kFM; ++i)
#pragma unroll
        for (int j = 0; j < kFN; ++j) {
            if constexpr (!kExact) {
                const int64_t r = r0 + (wm * kFM + i) * 16 + lr, col = c0 + (wn * kFN + j) * 16 + 4 * group;
                if (r >= m) continue;
                T *to = c + r * c_stride + col;
                if (col + 4 <= n) {
                    store4(to, acc[i][j]);
                } else {
                    for (int q = 0; q < 4; ++q)
                        if (col + q < n) to[q] = (T)acc[i][j][q];
                }
            } else {
                const int64_t col = c0 + (wn * kFN + j) * 16 + lr;
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const int64_t r = r0 + (wm * kFM + i) * 16 + 4 * group + q;
                    if (r < m && col < n) c[r * c_stride + col] = (T)acc[i][j][q];
                }
            }
        }
}

// Large results in bfloat16: tiles of 256 x 256, eight waves of 128 x 64.  Two waves share a SIMD, one of each half of the
// tile's rows, and they take turns: while the one multiplies (a phase of matrix instructions and nothing else) the other reads
// its fragments of a block, and the first half's waves load.  Phase 2 k: the first half reads block k, the second multiplies
// block k - 1; phase 2 k + 1: the first multiplies block k, the second reads it.
// LDS holds two blocks.  What is loaded when follows from who reads it last: the first half's rows of a are free after phase
// 2 k and have three phases to be filled again (by the second half's waves, in phase 2 k + 1), the second half's rows are free
// after phase 2 k + 1 and have three as well, b's have two.  (A wave's loads arrive in order, so the later needed are issued
// after the others and left outstanding.)
// There are at least 256 rows and columns: the last tiles begin earlier instead of ending late, and what two tiles share they
// compute alike.
// A workgroup goes from tile to tile, and the blocks of all its tiles are one stream: the next tile's first blocks are on
// their way while this one's results are stored, and nobody waits for the stores before the loads behind them.
constexpr int kLargeSide = 256;
typedef TileShape<2, 4, 8, 4, 2> LargeShape;

// 16 bytes a lane.  (As an instruction that the compiler does not count, merge or move: the waits for loads count it.  Its
// data may not be written in the cycle after it, which the compiler sees to for instructions it knows only.)
__device__ __forceinline__ void store_sixteen(const void *to, unsigned int offset, u32x4 v) {
    const void *at;
    asm volatile("s_mov_b64 %0, %1\n\tglobal_store_dwordx4 %2, %3, %0\n\ts_nop 0" : "=&s"(at) : "s"(to), "v"(offset), "v"(v) : "memory");
}

__global__ __launch_bounds__(LargeShape::kThreads) void large_product_kernel(
    const uint8_t *__restrict__ a, const uint8_t *__restrict__ a_scales, const uint8_t *__restrict__ b,
    const uint8_t *__restrict__ b_scales, int64_t m, int64_t n, int blocks, int64_t data_stride, int64_t scale_stride,
    __bf16 *c, int64_t c_stride, unsigned int row_tiles, unsigned int column_tiles) {
    using Shape = LargeShape;
    extern __shared__ unsigned char lds[];
    constexpr int kFM = Shape::kFM, kFN = Shape::kFN, kLoadsB = 8, kLoadsA = 4, kLoadsS = 2, kStores = kFM * kFN / 2;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int half = wave / 4, w = wave % 4, group = lane / 16, lr = lane % 16;
    const unsigned int base = __builtin_amdgcn_readfirstlane((unsigned int)(size_t)(LdsByte *)lds);
    const unsigned int tiles = row_tiles * column_tiles;

    // Where in the stream a load, or a product, is: the tile's first row and column, and the block.
    struct Place {
        unsigned int tile;
        int k;
        int64_t r0, c0;
    };
    auto find = [&](Place &p) {
        tile_origin(p.tile, row_tiles, column_tiles, kLargeSide, kLargeSide, p.r0, p.c0);
        p.r0 = min(p.r0, m - kLargeSide);
        p.c0 = min(p.c0, n - kLargeSide);
    };
    auto next = [&](Place &p) {
        if (++p.k < blocks) return;
        p.k = 0;
        p.tile += gridDim.x;
        if (p.tile < tiles) find(p);
    };

    // A load brings eight rows, 8 * (4 i + w) and on: place_of() goes by the row's last three bits and by w's last.
    const unsigned int from = (unsigned int)(lane / 8 * data_stride) + 16 * place_of(8 * w + lane / 8, lane % 8);
    const unsigned int from_scales = (unsigned int)(lane * scale_stride);
    const int64_t turn = 32 * data_stride;
    const unsigned int to_a = base + w * 1024, to_b = to_a + kLargeSide * kBlock;
    auto load_a = [&](const Place &at, int slot, int rows) {  // rows: 0 or 128, the half
        const uint8_t *p = a + (at.r0 + rows + 8 * w) * data_stride + (int64_t)at.k * kBlock;
        const unsigned int to = to_a + slot * Shape::kData + rows * kBlock;
#pragma unroll
        for (int i = 0; i < kLoadsA; ++i) load_to_lds(p + i * turn, from, to + i * 4096);
    };
    auto load_b = [&](const Place &at, int slot) {
        const uint8_t *p = b + (at.c0 + 8 * w) * data_stride + (int64_t)at.k * kBlock;
        const unsigned int to = to_b + slot * Shape::kData;
#pragma unroll
        for (int i = 0; i < kLoadsB; ++i) load_to_lds(p + i * turn, from, to + i * 4096);
    };
    // (Four blocks' scales, with every one of them, so that there are always as many loads.)
    auto load_scales = [&](const Place &at, int slot) {
        const unsigned int to = base + 2 * Shape::kData + slot * Shape::kScales + w * 256;
        load_word_to_lds(a_scales + (at.r0 + 64 * w) * scale_stride + (at.k & ~3), from_scales, to);
        load_word_to_lds(b_scales + (at.c0 + 64 * w) * scale_stride + (at.k & ~3), from_scales, to + kLargeSide * 4);
    };

    Fragment fa[kFM], fb[kFN];
    unsigned int ea[kFM], eb[kFN];
    f32x4 acc[kFM][kFN] = {};
    auto fragment = [&](const unsigned char *at, int row) {
        Fragment f;
        f.lo = *reinterpret_cast<const u32x4 *>(at + row * kBlock + 16 * place_of(row, 2 * group));
        f.hi = *reinterpret_cast<const u32x4 *>(at + row * kBlock + 16 * place_of(row, 2 * group + 1));
        return f;
    };
    auto read = [&](int k, int slot) {
        const unsigned char *la = lds + slot * Shape::kData, *lb = la + kLargeSide * kBlock;
        if (k % 4 == 0) {
            const unsigned int *scales = reinterpret_cast<const unsigned int *>(lds + 2 * Shape::kData + slot * Shape::kScales);
#pragma unroll
            for (int i = 0; i < kFM; ++i) ea[i] = scales[(half * kFM + i) * 16 + lr];
#pragma unroll
            for (int j = 0; j < kFN; ++j) eb[j] = scales[kLargeSide + (w * kFN + j) * 16 + lr];
        } else {
#pragma unroll
            for (int i = 0; i < kFM; ++i) ea[i] >>= 8;
#pragma unroll
            for (int j = 0; j < kFN; ++j) eb[j] >>= 8;
        }
#pragma unroll
        for (int j = 0; j < kFN; ++j) fb[j] = fragment(lb, (w * kFN + j) * 16 + lr);
#pragma unroll
        for (int i = 0; i < kFM; ++i) fa[i] = fragment(la, (half * kFM + i) * 16 + lr);
        wait_for_lds();
    };

    Place now = {blockIdx.x, 0, 0, 0};
    find(now);
    const int steps = blocks * (int)((tiles - blockIdx.x + gridDim.x - 1) / gridDim.x);
    Place ahead = now;  // the next to be loaded: by the first half's waves one block ahead, by the second's two
    if (half == 0) {
        load_scales(ahead, 0);
        load_b(ahead, 0);
        load_a(ahead, 0, 128);
        next(ahead);
        wait_for_loads();
    } else {
        load_a(ahead, 0, 0);
        next(ahead);
        if (steps > 1) {
            load_a(ahead, 1, 0);
            next(ahead);
            wait_for_loads<kLoadsA>();
        } else {
            wait_for_loads();
        }
    }
    phase_end();
    if (half == 1) phase_end();
    bool stored = false;  // whether the stores of a tile stand between the loads that are waited for and those behind them
    for (int s = 0; s < steps; ++s) {
        const int slot = s & 1;
        if (half == 0) {
            if (s + 1 < steps) {
                load_scales(ahead, slot ^ 1);
                load_b(ahead, slot ^ 1);
                load_a(ahead, slot ^ 1, 128);
                next(ahead);
            }
        } else if (s + 2 < steps) {
            load_a(ahead, slot, 0);
            next(ahead);
        }
        read(now.k, slot);
        if (half == 0) {  // the second half's rows of this block
            if (s + 1 == steps) wait_for_loads();
            else if (stored) wait_for_loads<kStores + kLoadsS + kLoadsB + kLoadsA>();
            else wait_for_loads<kLoadsS + kLoadsB + kLoadsA>();
        } else {          // the first half's rows of the next
            if (s + 2 >= steps) wait_for_loads();
            else if (stored) wait_for_loads<kStores + kLoadsA>();
            else wait_for_loads<kLoadsA>();
        }
        phase_end();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int i = 0; i < kFM; ++i)
#pragma unroll
            for (int j = 0; j < kFN; ++j) acc[i][j] = multiply(fb[j], fa[i], eb[j], ea[i], acc[i][j]);
        __builtin_amdgcn_s_setprio(0);
        if (half == 0) {  // the next block's b
            if (s + 1 < steps) wait_for_loads<kLoadsA>();
        }
        stored = now.k + 1 == blocks;
        if (stored) {
            // A lane has four columns of two neighbouring fragments; the groups of 16 lanes exchange them so that it has
            // eight of one, and 64 bytes of a row are stored at once: the first two groups the first eight columns of either
            // fragment, the others the last.
            const unsigned int to = (unsigned int)(lr * c_stride + group % 2 * 16 + group / 2 * 8) * 2;
#pragma unroll
            for (int i = 0; i < kFM; ++i)
#pragma unroll
                for (int j = 0; j < kFN; j += 2) {
                    const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(
                        pack_bf16(acc[i][j][0], acc[i][j][1]), pack_bf16(acc[i][j + 1][0], acc[i][j + 1][1]), false, false));
                    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane16_swap(
                        pack_bf16(acc[i][j][2], acc[i][j][3]), pack_bf16(acc[i][j + 1][2], acc[i][j + 1][3]), false, false));
                    store_sixteen(c + (now.r0 + (half * kFM + i) * 16) * c_stride + now.c0 + (w * kFN + j) * 16, to,
                                  u32x4{x[0], y[0], x[1], y[1]});
                    acc[i][j] = f32x4{};
                    acc[i][j + 1] = f32x4{};
                }
        }
        next(now);
        phase_end();
    }
    if (half == 0) phase_end();
}

// At most 16 rows of a: what there is to do is reading b once.  A workgroup takes 16 of b's rows, its waves every eighth
// block of them each, and the waves' sums are added in their order.  Nothing of b goes through LDS, since nothing of it is
// used twice; all loads of up to 32 blocks are under way before the first product.  With kQuantize a is still to be
// quantised: every workgroup does so for itself, into LDS, while b's first blocks are on their way.
constexpr int kFewRows = 16, kFewWaves = 8, kFewHeld = 4;
// Bytes of a that every workgroup quantises for itself rather than a kernel of its own once (16 x 1024 into 1024 columns 5.0 us
// within, 5.2 apart; 4 x 4096 into 4096 7.7 and 8.2; beyond it 8 x 4096 10.4 and 8.6, 16 x 2048 7.9 and 6.4).
constexpr int64_t kFewQuantized = 16384;

template <typename T, bool kExact, bool kQuantize>
__global__ __launch_bounds__(kFewWaves *kWave) void few_rows_kernel(
    const void *__restrict__ a, const uint8_t *__restrict__ a_scales, int64_t x_stride, const uint8_t *__restrict__ b,
    const uint8_t *__restrict__ b_scales, int m, int64_t n, int64_t k, int blocks, int64_t data_stride,
    int64_t scale_stride, T *__restrict__ c, int64_t c_stride) {
    extern __shared__ unsigned char lds[];  // kQuantize: a's rows, data_stride apart, and their scales, scale_stride apart
    __shared__ float sums[kFewWaves][16 * 16];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, group = lane / 16, lr = lane % 16;
    const int64_t c0 = (int64_t)blockIdx.x * 16, row_b = min(c0 + lr, n - 1);
    const int row_a = min(lr, m - 1);
    const uint8_t *pb = b + row_b * data_stride + 32 * group, *psb = b_scales + row_b * scale_stride;
    const uint8_t *pa = (const uint8_t *)a + (int64_t)row_a * data_stride + 32 * group,
                  *psa = a_scales + (int64_t)row_a * scale_stride;
    Fragment fb[kFewHeld];
    unsigned int eb[kFewHeld];
    auto load = [&](int i, int at) {
        if (at < blocks) {
            fb[i].lo = *reinterpret_cast<const u32x4 *>(pb + (int64_t)at * kBlock);
            fb[i].hi = *reinterpret_cast<const u32x4 *>(pb + (int64_t)at * kBlock + 16);
            eb[i] = psb[at];
        }
    };
#pragma unroll
    for (int i = 0; i < kFewHeld; ++i) load(i, wave + kFewWaves * i);
    if constexpr (kQuantize) {
        // Eight values a thread, 16 threads a block.
        const int units = m * blocks;
        for (int u = threadIdx.x / 16; u < units; u += kFewWaves * kWave / 16) {
            const int r = u / blocks, at = u % blocks;
            const int64_t col = (int64_t)at * kBlock + threadIdx.x % 16 * 8;
            float v[8], peak = 0.0f;
            load_eight((const T *)a + r * x_stride, col, k, v);
#pragma unroll
            for (int j = 0; j < 8; ++j) peak = fmaxf(peak, scale_magnitude(v[j]));
            const int e = scale_exponent(max_of_sixteen(peak));
            const float inv = inverse_scale(e);
            const u32x2 q = {pack4(v[0], v[1], v[2], v[3], inv), pack4(v[4], v[5], v[6], v[7], inv)};
            const int half = threadIdx.x % 16;
            *reinterpret_cast<u32x2 *>(lds + r * data_stride + at * kBlock + 16 * place_of(r, half / 2) + half % 2 * 8) = q;
            if (half == 0) lds[m * data_stride + r * scale_stride + at] = (uint8_t)(e + 127);
        }
        __syncthreads();
    }
    f32x4 acc = {};
    for (int at = wave; at < blocks; at += kFewWaves * kFewHeld) {
#pragma unroll
        for (int i = 0; i < kFewHeld; ++i) {
            const int here = at + kFewWaves * i;
            if (here < blocks) {
                Fragment fa;
                unsigned int ea;
                if constexpr (kQuantize) {
                    const unsigned char *la = lds + row_a * data_stride + here * kBlock;
                    fa.lo = *reinterpret_cast<const u32x4 *>(la + 16 * place_of(row_a, 2 * group));
                    fa.hi = *reinterpret_cast<const u32x4 *>(la + 16 * place_of(row_a, 2 * group + 1));
                    ea = lds[m * data_stride + row_a * scale_stride + here];
                } else {
                    fa.lo = *reinterpret_cast<const u32x4 *>(pa + (int64_t)here * kBlock);
                    fa.hi = *reinterpret_cast<const u32x4 *>(pa + (int64_t)here * kBlock + 16);
                    ea = psa[here];
                }
                if constexpr (!kExact) {
                    acc = multiply(fa, fb[i], ea, eb[i], acc);
                } else {
                    add_scaled(acc, multiply_exactly(fa, fb[i]), ea, eb[i]);
                }
            }
            load(i, here + kFewWaves * kFewHeld);
        }
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) sums[wave][(4 * group + q) * 16 + lr] = acc[q];
    __syncthreads();
    const int r = threadIdx.x / 16, col = threadIdx.x % 16;
    if (r < m && c0 + col < n) {
        float v = sums[0][threadIdx.x];
#pragma unroll
        for (int w = 1; w < kFewWaves; ++w) v += sums[w][threadIdx.x];
        c[r * c_stride + c0 + col] = (T)v;
    }
}

// The parts' sums, in their order.
template <typename T>
__global__ __launch_bounds__(256) void join_parts_kernel(const float *__restrict__ partial, int parts, int64_t m, int64_t n,
                                                         T *__restrict__ c, int64_t c_stride) {
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4, size = m * n;
    if (i >= size) return;
    float v[4] = {};
    if (i + 4 <= size) {
        for (int p = 0; p < parts; ++p) {
            const Vec<float> w = load_vec(partial + p * size + i);
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] += w[q];
        }
    } else {
        for (int p = 0; p < parts; ++p)
            for (int q = 0; i + q < size; ++q) v[q] += partial[p * size + i + q];
    }
    for (int q = 0; q < 4 && i + q < size; ++q) c[(i + q) / n * c_stride + (i + q) % n] = (T)v[q];
}

constexpr int64_t kComputeUnits = 256;  // (a multiple of the eight XCDs)

// How a product is cut.  The larger a tile the fewer times the factors are read; the smaller the more units have one.  us into
// bfloat16 / floats, the side that is taken first:
// - up to 16 rows of at most so many bytes, as every workgroup reads them all: 16 columns a workgroup, no LDS
//   (16 x 4096 x 4096 7.7, in tiles 8.9; beyond it 16 x 8192 x 8192 in tiles 17.5, this way 24.0);
constexpr int64_t kFewData = 65536;
// - 256 x 256 where as many rounds of them on all units take no longer than the rounds of 128 x 128: one is 3 of those,
//   3.5 exactly (196 tiles, 3584 x 3584 x 2048: 33.8 / 59.3 and 38.2 / 67.5; 121 tiles, 2816 x 2816 x 2048: by 128
//   23.0 / 39.4, by 256 31.7 / 57.4), but for short exact sums (4096 x 4096 x 256 floats: 19.5 by 128, 22.5 by 256);
constexpr int64_t kShortExact = 4;
// - 128 x 128 where every second unit has one, by two teams where there is no second tile a unit and the sum is long enough to
//   pay for joining them (256 tiles, 2000 x 2000 x 8192: 39 / 71 by two, 50 / 93 by one; 2000 x 2000 x 512: 8.2 / 11.9 by one,
//   9.1 / 12.6 by two);
constexpr int64_t kTeamBlocks = 8;
// - else 64 x 64.  Too few of them for all units: the sum in parts, which a kernel joins, if it is long (200 x 200 x 4096
//   9.3 / 10.4 in four, 12 / 15 whole; 200 x 200 x 2048 7.3 / 9.8 whole, 8.2 / 8.9 in four).  Enough of them: parts of
//   128 x 128 tiles if those are long (1203 x 1111 x 8192 28 / 44 in two parts, by 64 x 64 39 / 54; 1203 x 1111 x 2048
//   11 / 17 by 64 x 64, 19 / 24 in parts).  At most one to a unit: four teams (512 x 2048 x 4096 12.5 / 16.2, one team
//   13.3 / 23.0).
constexpr int64_t kPartBlocks = 24, kLongPart = 16;
// At most 64 rows or columns leave half of each larger tile empty.
constexpr int64_t kThin = 64;

constexpr int64_t kManyColumns = (int64_t)1 << 26;  // (32 threads each, of fewer than 2^32)
bool few_rows(int64_t m, int64_t n, int64_t k) {
    return m <= kFewRows && n <= kManyColumns && m * block_data_stride(k) <= kFewData;
}

// Tiles of `side`, of so many teams, and the sum in `parts`.
struct Cut {
    int side, parts, teams;
};
Cut cut_of(int64_t m, int64_t n, int64_t k, bool exact) {
    if (few_rows(m, n, k)) return {16, 1, 1};
    const int64_t blocks = (k + kBlock - 1) / kBlock;
    auto tiles = [&](int64_t side) { return ((m + side - 1) / side) * ((n + side - 1) / side); };
    auto rounds = [&](int64_t side) { return (tiles(side) + kComputeUnits - 1) / kComputeUnits; };
    auto parts_of = [&](int64_t parts) {  // none of them empty
        const int64_t part = (blocks + parts - 1) / parts;
        return (int)((blocks + part - 1) / part);
    };
    const bool thin = std::min(m, n) <= kThin;
    if (!thin && std::min(m, n) >= 256 && k > 0 && !(exact && blocks <= kShortExact) && (exact ? 7 : 6) * rounds(256) <= 2 * rounds(128))
        return {256, 1, 1};
    if (!thin && tiles(128) >= kComputeUnits / 2)
        return {128, 1, tiles(128) <= kComputeUnits && blocks > kTeamBlocks ? 2 : 1};
    if (tiles(64) * 2 <= kComputeUnits) {
        if (blocks >= kPartBlocks) return {64, parts_of(std::min(kComputeUnits / tiles(64), blocks / 8)), 4};
    } else if (!thin && blocks >= kLongPart * (kComputeUnits / tiles(128))) {
        return {128, parts_of(kComputeUnits / tiles(128)), 2};
    }
    return {64, 1, tiles(64) <= kComputeUnits && blocks >= 8 ? 4 : 1};
}

template <typename T, bool kExact, class Shape>
int launch_tiled(const Product &p, int parts, T *c, int64_t c_stride, hipStream_t s) {
    const int64_t row_tiles = (p.m + Shape::kRows - 1) / Shape::kRows, column_tiles = (p.n + Shape::kCols - 1) / Shape::kCols;
    TSNE_OPERATOR_REQUIRE(row_tiles <= 0xffffffff / Shape::kThreads / column_tiles, "matmul_blocks: a result of %lld x %lld is more "
                          "than one launch holds", (long long)p.m, (long long)p.n);  // (fewer than 2^32 threads)
    const int blocks = (int)((p.k + kBlock - 1) / kBlock);
    const auto kernel = tiled_product_kernel<T, kExact, Shape>;
    TSNE_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, Shape::kLds));
    kernel<<<dim3((unsigned int)(row_tiles * column_tiles), parts), Shape::kThreads, Shape::kLds, s>>>(
        p.a, p.a_scales, p.b, p.b_scales, p.m, p.n, blocks, parts > 1 ? (blocks + parts - 1) / parts : blocks,
        block_data_stride(p.k), block_scale_stride(p.k), c, c_stride, p.m * p.n, (unsigned int)row_tiles,
        (unsigned int)column_tiles);
    TSNE_LAUNCHED(s);
    return 0;
}

constexpr int64_t kLargeStride = (int64_t)1 << 26;  // (16 rows of results are within 32 bits)
int launch_large(const Product &p, hipStream_t s) {
    const int64_t row_tiles = (p.m + kLargeSide - 1) / kLargeSide, column_tiles = (p.n + kLargeSide - 1) / kLargeSide;
    TSNE_OPERATOR_REQUIRE(row_tiles <= 0x7fffffff / column_tiles, "matmul_blocks: a result of %lld x %lld is more than "
                          "one launch holds", (long long)p.m, (long long)p.n);
    TSNE_TRY(hipFuncSetAttribute(reinterpret_cast<const void *>(large_product_kernel),
                                 hipFuncAttributeMaxDynamicSharedMemorySize, LargeShape::kLds));
    large_product_kernel<<<(unsigned int)std::min<int64_t>(row_tiles * column_tiles, kComputeUnits), LargeShape::kThreads, LargeShape::kLds, s>>>(
        p.a, p.a_scales, p.b, p.b_scales, p.m, p.n, (int)((p.k + kBlock - 1) / kBlock), block_data_stride(p.k),
        block_scale_stride(p.k), (__bf16 *)p.c, p.c_stride, (unsigned int)row_tiles, (unsigned int)column_tiles);
    TSNE_LAUNCHED(s);
    return 0;
}

// x: a is still to be quantised, from rows of T, x_stride apart.
template <typename T, bool kExact, bool kQuantize>
int launch_few_rows(const Product &p, const void *x, int64_t x_stride, hipStream_t s) {
    const int64_t groups = (p.n + 15) / 16;
    const size_t lds = kQuantize ? (size_t)(p.m * (block_data_stride(p.k) + block_scale_stride(p.k))) : 0;
    few_rows_kernel<T, kExact, kQuantize><<<(unsigned int)groups, kFewWaves * kWave, lds, s>>>(
        kQuantize ? x : p.a, p.a_scales, x_stride, p.b, p.b_scales, (int)p.m, p.n, p.k, (int)((p.k + kBlock - 1) / kBlock),
        block_data_stride(p.k), block_scale_stride(p.k), (T *)p.c, p.c_stride);
    TSNE_LAUNCHED(s);
    return 0;
}

template <typename T, bool kExact>
int launch_as(const Product &p, hipStream_t s) {
    const Cut cut = cut_of(p.m, p.n, p.k, kExact);
    if (cut.side == 16) return launch_few_rows<T, kExact, false>(p, nullptr, 0, s);
    if (cut.parts > 1) {
        if (cut.side == 128 ? launch_tiled<float, kExact, TileShape<2, 2, 4, 4, 2, 2>>(p, cut.parts, p.partial, p.n, s)
                            : launch_tiled<float, kExact, TileShape<2, 2, 2, 2, 2, 4>>(p, cut.parts, p.partial, p.n, s))
            return 1;
        join_parts_kernel<T><<<div_up(p.m * p.n, 1024), 256, 0, s>>>(p.partial, cut.parts, p.m, p.n, (T *)p.c, p.c_stride);
        TSNE_LAUNCHED(s);
        return 0;
    }
    if (cut.side == 256) {
        if constexpr (kExact) return launch_tiled<T, kExact, TileShape<2, 4, 8, 4, 2>>(p, 1, (T *)p.c, p.c_stride, s);
        else if (p.c_stride < kLargeStride) return launch_large(p, s);
        else return launch_tiled<T, kExact, TileShape<2, 2, 4, 4, 2>>(p, 1, (T *)p.c, p.c_stride, s);
    }
    if (cut.side == 128 && cut.teams == 2) return launch_tiled<T, kExact, TileShape<2, 2, 4, 4, 2, 2>>(p, 1, (T *)p.c, p.c_stride, s);
    if (cut.side == 128) return launch_tiled<T, kExact, TileShape<2, 2, 4, 4, 2>>(p, 1, (T *)p.c, p.c_stride, s);
    if (cut.teams == 4) return launch_tiled<T, kExact, TileShape<2, 2, 2, 2, 2, 4>>(p, 1, (T *)p.c, p.c_stride, s);
    return launch_tiled<T, kExact, TileShape<2, 2, 2, 2, 4>>(p, 1, (T *)p.c, p.c_stride, s);
}

int launch_product(const Product &p, int type, hipStream_t s) {
    if (type == kTypeF32) return launch_as<float, true>(p, s);
    if (type == kTypeF16) return launch_as<_Float16, true>(p, s);
    return p.exact ? launch_as<__bf16, true>(p, s) : launch_as<__bf16, false>(p, s);
}

constexpr int64_t kMostSummed = (int64_t)1 << 24;  // (a tile's rows are within 32 bits of its first)
int check_type(const char *who, int type) {
    TSNE_OPERATOR_REQUIRE(type >= 0 && type <= 2, "%s: unknown type %d (0 = float, 1 = half, 2 = bfloat16)", who, type);
    return 0;
}

int check_product(const char *who, int64_t m, int64_t n, int64_t k, int64_t c_stride) {
    TSNE_OPERATOR_REQUIRE(m >= 0 && n >= 0 && k >= 0 && k <= kMostSummed, "%s: a product of %lld x %lld x %lld (at most %lld are summed)", who,
                          (long long)m, (long long)n, (long long)k, (long long)kMostSummed);
    TSNE_OPERATOR_REQUIRE(c_stride >= n, "%s: rows of %lld values are only %lld apart", who, (long long)n,
                          (long long)c_stride);
    return 0;
}

}  // namespace
}  // namespace tsnehip

using namespace tsnehip;

extern "C" int64_t tsne_hip_matmul_blocks_workspace(int64_t m, int64_t n, int64_t k, int type, int exact) {
    if (m <= 0 || n <= 0 || k <= 0) return 0;
    const int parts = cut_of(m, n, k, exact || type == kTypeF32 || type == kTypeF16).parts;
    return parts > 1 ? parts * m * n * 4 : 0;
}

extern "C" int tsne_hip_matmul_blocks(const uint8_t *a, const uint8_t *a_scales, const uint8_t *b,
                                      const uint8_t *b_scales, int64_t m, int64_t n, int64_t k, void *c, int type,
                                      int64_t c_stride, int exact, void *workspace, int64_t workspace_bytes,
                                      void *stream) {
    if (check_product("matmul_blocks", m, n, k, c_stride) || check_type("matmul_blocks", type)) return 1;
    TSNE_OPERATOR_REQUIRE(exact == 0 || exact == 1, "matmul_blocks: exact must be 0 or 1 (got %d)", exact);
    if (m == 0 || n == 0) return 0;
    TSNE_OPERATOR_REQUIRE(c && (k == 0 || (a && a_scales && b && b_scales)), "matmul_blocks: null argument");
    TSNE_OPERATOR_REQUIRE((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) % 16 == 0,
                          "matmul_blocks: data must be aligned to 16 bytes");
    TSNE_OPERATOR_REQUIRE((reinterpret_cast<uintptr_t>(a_scales) | reinterpret_cast<uintptr_t>(b_scales)) % 16 == 0,
                          "matmul_blocks: scales must be aligned to 16 bytes");
    if (check_workspace("matmul_blocks", workspace, workspace_bytes, tsne_hip_matmul_blocks_workspace(m, n, k, type, exact)))
        return 1;
    return launch_product({a, a_scales, b, b_scales, m, n, k, c, c_stride, exact, (float *)workspace}, type,
                          (hipStream_t)stream);
}

namespace {
// Whether linear_blocks quantises its input in the product's kernel.
bool quantized_within(int64_t m, int64_t n, int64_t k) { return few_rows(m, n, k) && m * block_data_stride(k) <= kFewQuantized; }
int64_t round_up_16(int64_t n) { return (n + 15) / 16 * 16; }
}  // namespace

extern "C" int64_t tsne_hip_linear_blocks_workspace(int64_t m, int64_t n, int64_t k, int type) {
    if (m <= 0 || n <= 0 || k <= 0 || quantized_within(m, n, k)) return 0;
    return m * block_data_stride(k) + round_up_16(m * block_scale_stride(k)) +
           tsne_hip_matmul_blocks_workspace(m, n, k, type, 0);
}

extern "C" int tsne_hip_linear_blocks(const void *x, int type, int64_t m, int64_t k, int64_t x_stride, const uint8_t *w,
                                      const uint8_t *w_scales, int64_t n, void *c, int64_t c_stride, void *workspace,
                                      int64_t workspace_bytes, void *stream) {
    if (check_product("linear_blocks", m, n, k, c_stride) || check_type("linear_blocks", type)) return 1;
    TSNE_OPERATOR_REQUIRE(x_stride >= k, "linear_blocks: rows of %lld values are only %lld apart", (long long)k,
                          (long long)x_stride);
    if (m == 0 || n == 0) return 0;
    TSNE_OPERATOR_REQUIRE(c && (k == 0 || (x && w && w_scales)), "linear_blocks: null argument");
    TSNE_OPERATOR_REQUIRE((reinterpret_cast<uintptr_t>(w) | reinterpret_cast<uintptr_t>(w_scales)) % 16 == 0,
                          "linear_blocks: w and its scales must be aligned to 16 bytes");
    if (check_workspace("linear_blocks", workspace, workspace_bytes, tsne_hip_linear_blocks_workspace(m, n, k, type))) return 1;
    const hipStream_t s = (hipStream_t)stream;
    if (k > 0 && quantized_within(m, n, k)) {
        const Product p = {nullptr, nullptr, w, w_scales, m, n, k, c, c_stride, 0, nullptr};
        if (type == kTypeF32) return launch_few_rows<float, true, true>(p, x, x_stride, s);
        if (type == kTypeF16) return launch_few_rows<_Float16, true, true>(p, x, x_stride, s);
        return launch_few_rows<__bf16, false, true>(p, x, x_stride, s);
    }
    uint8_t *data = (uint8_t *)workspace, *scales = data + m * block_data_stride(k);
    if (k > 0 && launch_quantize(x, type, m, k, x_stride, 0, data, scales, nullptr, nullptr, s)) return 1;
    float *partial = (float *)(scales + round_up_16(m * block_scale_stride(k)));
    return launch_product({data, scales, w, w_scales, m, n, k, c, c_stride, 0, partial}, type, s);
}
