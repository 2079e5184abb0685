// A teacher's top list, and distillation from one (tsne_operators.h has the formulas).
//
// Both are bound by reading the logits, and distillation by writing as much as a gradient.  A workgroup holds a row in its
// registers, as it came (16-bit values two to a register), so that it is read once however often it is gone over: maximum, sum
// of exponentials, and candidates or gradient.  The shorter the row the fewer threads, so that a compute unit has several rows
// at different stages, one loading while another computes or stores.  Few long rows, and rows beyond registers, are cut into
// stretches whose results a second kernel joins.  us, and GB/s of what has to be moved (a copy's rate is 4785):
//                            loss and gradient, rest   loss alone    top list
//   4096 x 60000 bf16, k 90      217.8  4513           131.7  3732   131.5  3737   (reading alone: a large sum runs at 4012)
//   2048 x 32003 bf16, k 45       67.3  3896            31.1  4214    36.6  3584
//   4096 x 2000  bf16, k 45       13.4  2440             7.4  2211    15.4  1063   (the list's own work)
//    600 x 1200  bf16, k 90        8.1                   5.4          13.2         (latency: loads, barriers, one list)
//      7 x 131071 bf16, k 90      11.0                   8.1          15.2         (and a second launch's)
//   1000 x 131072 f32, k 90      291.8  3593           105.3  4979                 (no rest; beyond registers, so that both kernels of
//                                                                                  a gradient read the logits: 5390 of three transfers)
#include <algorithm>
#include <type_traits>

#include "../../include/tsnecuda/tsne_operators.h"
#include "operators.h"

namespace tsnehip {

namespace {

constexpr int kMostListed = 1024;
constexpr int64_t kMostDistilled = (int64_t)1 << 20;
constexpr float kLog2E = 1.4426950408889634f;

__device__ __forceinline__ float lowest() { return -__builtin_inff(); }

// (What all lanes hold alike: in a scalar register, of which there are enough.)
__device__ __forceinline__ float uniform(float v) { return lane_value(v, 0); }

__device__ __forceinline__ float exp2_of(float x) { return __builtin_amdgcn_exp2f(x); }  // (0 below 2^-126)

// (fmaxf adds a quieting move an operand.  A signalling NaN comes out as NaN here, a quiet one is passed over; the sums that
// follow catch both.)
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}

// Running maximum of some z and the sum of 2^((z - maximum) c) over them.
struct Stat {
    float m, s;
};
// What the maximum is taken as where it is none (then every term is 2^-inf = 0).
__device__ __forceinline__ float base_of(float m) { return m == lowest() ? 0.0f : m; }
__device__ __forceinline__ void add(Stat &a, float z, float c) {
    const float m = fmaxf(a.m, z);  // (a NaN is passed over here and caught by the sum)
    if (m > a.m) {
        a.s *= exp2f((a.m - m) * c);
        a.m = m;
    }
    a.s += exp2f((z - base_of(a.m)) * c);
}
__device__ __forceinline__ Stat join(Stat a, Stat b, float c) {
    const float m = fmaxf(a.m, b.m), base = base_of(m);
    return {m, a.s * exp2f((a.m - base) * c) + b.s * exp2f((b.m - base) * c)};
}
// 2^((z - base) c) of many z.  The difference first would be two instructions and an exponent; z c + shift, shift = -base c, is
// one, but off by shift's rounding, which grows with the row's distance from zero and which a softmax must not depend on (100
// equal columns of 1e6 would sum to 101.5, of -1e30 to infinity).  What the rounding has taken away is a number that a fused
// multiplication gives exactly, and as it is the same for all of a row's z, its power multiplies their sum, or whatever else
// they are multiplied by.  From 2^20 on (masks of the lowest values) the difference comes first, as everywhere else.
// (4096 x 60000 bfloat16 with gradient and rest, pass after pass: 210 us, and 223 with the difference first.)
struct Powers {
    float base, c, shift;
    bool fused;
    __device__ __forceinline__ Powers(float b, float by) : base(uniform(b)), c(uniform(by)), shift(uniform(-b * by)), fused(fabsf(shift) <= 1048576.0f) {}
    __device__ __forceinline__ float near(float z) const { return exp2_of(fmaf(z, c, shift)); }  // times more(), where fused
    __device__ __forceinline__ float far(float z) const { return exp2_of((z - base) * c); }
    __device__ __forceinline__ float more() const { return exp2_of(fmaf(-base, c, -shift)); }  // (2^(1/16) at most)
};

// Over all threads.  scratch: an entry a wave; a barrier has to lie between its last use and this.
template <int kThreads>
__device__ __forceinline__ float max_all(float v, float *scratch) {
    v = wave_max(v);
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) v = fmaxf(v, scratch[w]);
    return uniform(v);
}
template <int kThreads>
__device__ __forceinline__ float sum_all(float v, float *scratch) {
    v = wave_sum(v);
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = v;
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) v += scratch[w];
    return uniform(v);
}
template <int kThreads>
__device__ __forceinline__ Stat join_all(Stat v, float c, Stat *scratch) {
    const float m = wave_max(v.m), s = wave_sum(v.s * exp2f((v.m - base_of(m)) * c));
    if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = {m, s};
    __syncthreads();
    v = scratch[0];
#pragma unroll
    for (int w = 1; w < kThreads / kWave; ++w) v = join(v, scratch[w], c);
    return v;
}

// A stretch of a row in registers: kHeld times kVec values a thread, in turns of 16 bytes.  What lies behind its end is
// -infinity.
template <typename T, int kThreads, int kHeld>
struct Held {
    Vec<T> v[kHeld];
    static constexpr int kMost = kThreads * kHeld * kVec<T>;

    static __device__ __forceinline__ int place(int h) { return (h * kThreads + (int)threadIdx.x) * kVec<T>; }
    __device__ __forceinline__ void load(const T *z, int n) {
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
            const int i = place(h);
            if (i + kVec<T> <= n) {
                v[h] = load_vec(z + i);
            } else {
                float w[kVec<T>];
#pragma unroll
                for (int j = 0; j < kVec<T>; ++j) w[j] = i + j < n ? value_of(z[i + j]) : lowest();
                v[h].raw = pack_vec<T>(w);
            }
        }
    }
    // What is held is unpacked again in every pass: kept unpacked from one to the next it would take twice the registers.
    __device__ __forceinline__ void keep_packed() {
#pragma unroll
        for (int h = 0; h < kHeld; ++h) asm volatile("" : "+v"(v[h].raw));
    }
    __device__ __forceinline__ float max() {
        keep_packed();
        float m = lowest();
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
#pragma unroll
            for (int j = 0; j < kVec<T>; j += 2) m = max3(m, v[h][j], v[h][j + 1]);
        return m;
    }
    // Sum of 2^((z - base) c).
    __device__ __forceinline__ float sum(float base, float c) {
        keep_packed();
        float s[4] = {};
        const Powers power(base, c);
        if (power.fused) {
#pragma unroll
            for (int h = 0; h < kHeld; ++h)
#pragma unroll
                for (int j = 0; j < kVec<T>; ++j) s[j % 4] += power.near(v[h][j]);
        } else {  // (far from zero, or infinity)
#pragma unroll 1
            for (int h = 0; h < kHeld; ++h) {
                Vec<T> w = v[0];
#pragma unroll
                for (int i = 1; i < kHeld; ++i) w.raw = h == i ? v[i].raw : w.raw;
#pragma unroll
                for (int j = 0; j < kVec<T>; ++j) s[j % 4] += power.far(w[j]);
            }
        }
        const float all = (s[0] + s[1]) + (s[2] + s[3]);
        return power.fused ? all * power.more() : all;
    }
};

// ---- the top list -------------------------------------------------------------------------------------------------

// Order of a value: NaN above everything, -infinity 0x007fffff, 0 and -0 alike.
__device__ __forceinline__ unsigned int key_of(float v) { return v != v ? 0xffffffffu : float_to_ordered(v + 0.0f); }
constexpr unsigned int kKeyOfNothing = 0x007fffffu;
__device__ __forceinline__ float value_of_key(unsigned int key) {
    return key == 0xffffffffu ? __builtin_nanf("") : ordered_to_float(key);
}

typedef unsigned long long u64;

// An entry: a value's key above its column's complement, so that no two are equal and of equal values the lower column is
// the larger.
__device__ __forceinline__ u64 entry_of(float v, unsigned int column) { return (u64)key_of(v) << 32 | ~column; }

// The largest digit d such that at least `want` of the counted have d or more; want becomes which of those with d it is.
// Every wave finds it for itself.
__device__ __forceinline__ int find_digit(const unsigned int *counts, int &want) {
    const int lane = threadIdx.x % kWave;
    unsigned int mine[4], sum = 0;  // of digits 255 - 4 lane and the three below it
#pragma unroll
    for (int i = 0; i < 4; ++i) sum += mine[i] = counts[255 - 4 * lane - i];
    // Sums up to and with every lane: within 16 lanes, then over the groups of 16 before.
    unsigned int upto = sum;
    upto += __builtin_amdgcn_update_dpp(0u, upto, 0x111, 15, 15, true);
    upto += __builtin_amdgcn_update_dpp(0u, upto, 0x112, 15, 15, true);
    upto += __builtin_amdgcn_update_dpp(0u, upto, 0x114, 15, 15, true);
    upto += __builtin_amdgcn_update_dpp(0u, upto, 0x118, 15, 15, true);
    upto += __builtin_amdgcn_update_dpp(0u, upto, 0x142, 10, 15, true);
    upto += __builtin_amdgcn_update_dpp(0u, upto, 0x143, 12, 15, true);
    const u64 reached = __ballot(upto >= (unsigned int)want);
    const int who = __builtin_amdgcn_readfirstlane(reached ? __ffsll(reached) - 1 : kWave - 1);
    unsigned int left = want - (upto - sum);
    int digit = 255 - 4 * lane;
#pragma unroll
    for (int i = 0; i < 3; ++i)
        if (digit == 255 - 4 * lane - i && left > mine[i]) {
            left -= mine[i];
            --digit;
        }
    want = __builtin_amdgcn_readlane((int)left, who);
    return __builtin_amdgcn_readlane(digit, who);
}

// The k-th largest of n threads' maxima leaves about -n ln(1 - k / n) candidates, so that lists are a good deal shorter than
// the threads are many: 4096 x 2000, k = 48 16.0 us by a wave a row and 18.8 by 256 threads, k = 52 20.1 and 19.5; 2048 x 8000,
// k = 240 39 us by 256 threads and 89 by 1024.  (Rows of few threads are short, and many of them share a compute unit's LDS.)
constexpr int kWaveListed = 48, kGroupListed = 240;
template <int kThreads>
struct TopShared {
    // Candidates: more than are expected of the longest list that these threads are given.
    static constexpr int kMost = kThreads == kWave ? 512 : kThreads == 256 ? 1024 : 4096;
    unsigned int counts[256];
    u64 candidates[kMost];
    unsigned int count;
    float floats[16];
    float sums[16];
};

// The n candidates in descending order: where there are few each one's place is counted, else by a bitonic network.
template <int kThreads>
__device__ __forceinline__ void sort_candidates(TopShared<kThreads> &sh, int n) {
    const int t = threadIdx.x;
    if (n * 4 <= kThreads) {
        // Four threads a candidate count those above it.
        const int who = t / 4;
        u64 e = 0;
        int place = 0;
        if (who < n) {
            e = sh.candidates[who];
            for (int j = t % 4; j < n; j += 4) place += sh.candidates[j] > e;
        }
        place += exchanged<kByOne>(place);
        place += exchanged<kByTwo>(place);
        __syncthreads();
        if (who < n && t % 4 == 0) sh.candidates[place] = e;
        __syncthreads();
        return;
    }
    if (n <= 2 * kWave) {  // (threads too few for four each)
        u64 e[2] = {};
        int place[2] = {};
#pragma unroll
        for (int q = 0; q < 2; ++q)
            if (t + q * kThreads < n) e[q] = sh.candidates[t + q * kThreads];
        for (int j = 0; j < n; ++j) {
            const u64 other = sh.candidates[j];
#pragma unroll
            for (int q = 0; q < 2; ++q) place[q] += other > e[q];
        }
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 2; ++q)
            if (t + q * kThreads < n) sh.candidates[place[q]] = e[q];
        __syncthreads();
        return;
    }
    int size = 2;
    while (size < n) size *= 2;
    for (int i = n + t; i < size; i += kThreads) sh.candidates[i] = 0;
    for (int half = 1; half < size; half *= 2)
        for (int step = half; step > 0; step /= 2) {
            __syncthreads();
            for (int i = t; i < size / 2; i += kThreads) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const u64 x = sh.candidates[a], y = sh.candidates[b];
                if ((x < y) != ((a & (2 * half)) != 0)) {
                    sh.candidates[a] = y;
                    sh.candidates[b] = x;
                }
            }
        }
    __syncthreads();
}

// Entries of a row or of a stretch of it, from which the k largest are taken.  Few are larger than the k-th largest of the
// threads' own maxima, which is thus a threshold that leaves the k largest and little else: it is found to 16 bits of the key,
// eight at a time.  The counts of the first eight lie where candidates come later.
template <int kThreads>
__device__ __forceinline__ unsigned int *first_counts(TopShared<kThreads> &sh) {
    return reinterpret_cast<unsigned int *>(sh.candidates);
}
template <int kThreads>
__device__ __forceinline__ void clear_top(TopShared<kThreads> &sh) {
    for (int i = threadIdx.x; i < 256; i += kThreads) first_counts(sh)[i] = sh.counts[i] = 0;
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
}
// From the k-th largest of the threads' keys on, after clear_top(); k is at most kThreads.
template <int kThreads>
__device__ __forceinline__ unsigned int threshold_of(TopShared<kThreads> &sh, int k, unsigned int key) {
    int want = k;
    atomicAdd(&first_counts(sh)[key >> 24], 1u);
    __syncthreads();
    const unsigned int digit = (unsigned int)find_digit(first_counts(sh), want);
    if (key >> 24 == digit) atomicAdd(&sh.counts[key >> 16 & 255], 1u);
    __syncthreads();
    return digit << 24 | (unsigned int)find_digit(sh.counts, want) << 16;
}

// The k-th largest of some entries (0 where there are fewer), found eight bits at a time; each(visit) calls visit(entry) for
// all of this thread's share.
template <int kThreads, typename Each>
__device__ __forceinline__ u64 kth_entry(TopShared<kThreads> &sh, int k, Each each) {
    u64 found = 0;
    int want = k;
    for (int shift = 56; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += kThreads) sh.counts[i] = 0;
        __syncthreads();
        each([&](u64 e) {
            if (shift == 56 || e >> (shift + 8) == found) atomicAdd(&sh.counts[(e >> shift) & 255], 1u);
        });
        __syncthreads();
        const int d = find_digit(sh.counts, want);
        found = found << 8 | (unsigned int)d;
        if ((int)sh.counts[d] == want) return found << shift;  // all that share these digits are among the k
    }
    return found;
}

// The k largest and perhaps a few more, in any order; their number.  Where a threshold (of a key, see above) leaves more than
// there is room for (columns that are all alike, say) the k-th largest is found first, and so it is where it leaves many more
// than k: sorting costs by powers of two (300 x 3000, k = 600, which takes all 3000: 44 us, and 69 with all of them sorted;
// 4096 x 1000, k = 230 49 and 82; where it halves them only, 300 x 3000, k = 300, 34 and 30).
// each_from(least, visit) calls visit(value, column) for this thread's share of the entries, those below `least` left out or
// not; each(visit) for all of some share.
template <int kThreads, typename From, typename Each>
__device__ __forceinline__ int take_top(TopShared<kThreads> &sh, int k, unsigned int prefix, From each_from, Each each) {
    constexpr int kMost = TopShared<kThreads>::kMost, kEach = kMost / kThreads;
    const int t = threadIdx.x;
    const bool all = prefix <= kKeyOfNothing;  // (then nothing but -infinity is left out)
    const float least = all ? lowest() : value_of_key(prefix);
    each_from(least, [&](float v, unsigned int column) {
        if (!(v < least) && v != lowest()) {
            const unsigned int at = atomicAdd(&sh.count, 1u);
            if (at < kMost) sh.candidates[at] = entry_of(v, column);
        }
    });
    __syncthreads();
    const int n = (int)sh.count;
    if (__builtin_expect(n <= kMost, 1)) {
        const int room = k > 1 ? 1 << (32 - __clz(k - 1)) : 1;
        if (__builtin_expect(n <= 2 * kWave || n <= 2 * room, 1)) return n;
        u64 mine[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) mine[i] = t + i * kThreads < n ? sh.candidates[t + i * kThreads] : 0;
        const u64 found = kth_entry(sh, k, [&](auto visit) {
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                if (mine[i] != 0) visit(mine[i]);
        });
        __syncthreads();
        if (t == 0) sh.count = 0;
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (mine[i] != 0 && mine[i] >= found) sh.candidates[atomicAdd(&sh.count, 1u)] = mine[i];
        __syncthreads();
        return (int)sh.count;
    }
    const u64 found = kth_entry(sh, k, [&](auto visit) {
        each([&](float v, unsigned int column) { visit(entry_of(v, column)); });
    });
    __syncthreads();
    if (t == 0) sh.count = 0;
    __syncthreads();
    each([&](float v, unsigned int column) {
        const u64 e = entry_of(v, column);
        if (e >= found && v != lowest()) sh.candidates[atomicAdd(&sh.count, 1u)] = e;
    });
    __syncthreads();
    return (int)sh.count;
}

template <int kThreads>
__device__ __forceinline__ void write_top(const TopShared<kThreads> &sh, int n, int k, float *values, int *indices) {
    for (int i = threadIdx.x; i < k; i += kThreads) {
        const u64 e = i < n ? sh.candidates[i] : 0;
        values[i] = i < n ? value_of_key((unsigned int)(e >> 32)) : lowest();
        indices[i] = i < n ? (int)~(unsigned int)e : -1;
    }
}
__device__ __forceinline__ float lse_of(Stat a, float temperature) {
    return a.m == lowest() ? a.s + lowest() : a.m / temperature + logf(a.s);
}

// One workgroup a row or, with parts, a stretch of `part` columns of it, whose k largest (as entries, in no order; 0 for
// none) and statistics go to the workspace.
template <typename T, int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads, kHeld == 8 && kThreads > 256 ? 8 : 4) void top_logits_kernel(const T *__restrict__ logits, int64_t cols, int64_t row_stride,
                                                              int k, float temperature, int parts, int part,
                                                              float *__restrict__ values, int *__restrict__ indices,
                                                              float *__restrict__ lse, u64 *__restrict__ part_entries,
                                                              Stat *__restrict__ part_stats) {
    __shared__ TopShared<kThreads> sh;
    const int64_t row = blockIdx.x / parts;
    const int which = (int)(blockIdx.x % parts);
    const int64_t c0 = (int64_t)which * part;
    const int n = (int)min((int64_t)part, cols - c0);
    const float c = kLog2E / temperature;
    clear_top(sh);
    Held<T, kThreads, kHeld> held;
    held.load(logits + row * row_stride + c0, n);
    // threshold_of(), but that the barriers of the maximum and of the sum are its own too.
    const float my_max = held.max();
    const unsigned int key = key_of(my_max);
    int want = k;
    atomicAdd(&first_counts(sh)[key >> 24], 1u);
    Stat st = {max_all<kThreads>(my_max, sh.floats), 0.0f};
    const unsigned int digit = (unsigned int)find_digit(first_counts(sh), want);
    if (key >> 24 == digit) atomicAdd(&sh.counts[key >> 16 & 255], 1u);
    const float my_sum = held.sum(base_of(st.m), c);
    st.s = sum_all<kThreads>(my_sum, sh.sums);
    unsigned int prefix = digit << 24 | (unsigned int)find_digit(sh.counts, want) << 16;
    bool my_nan = false;
    if (st.s != st.s) {  // NaN, of which the maxima know nothing, or infinity
#pragma unroll
        for (int h = 0; h < kHeld; ++h)
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) my_nan |= held.v[h][j] != held.v[h][j];
        __syncthreads();
        clear_top(sh);
        prefix = threshold_of(sh, k, my_nan ? 0xffffffffu : key);
    }
    const int found = take_top<kThreads>(sh, k, prefix, [&](float least, auto visit) {
        held.keep_packed();
#pragma unroll
        for (int h = 0; h < kHeld; ++h) {
            float m = held.v[h][0];
#pragma unroll
            for (int j = 0; j < kVec<T>; j += 2) m = max3(m, held.v[h][j], held.v[h][j + 1]);
            if (my_nan || !(m < least)) {
#pragma unroll
                for (int j = 0; j < kVec<T>; ++j) visit(held.v[h][j], (unsigned int)(c0 + held.place(h) + j));
            }
        }
    }, [&](auto visit) {
        for (int i = threadIdx.x; i < n; i += kThreads) visit(value_of(logits[row * row_stride + c0 + i]), (unsigned int)(c0 + i));
    });
    if (parts == 1) {
        sort_candidates<kThreads>(sh, found);
        write_top<kThreads>(sh, found, k, values + row * k, indices + row * k);
        if (threadIdx.x == 0) lse[row] = lse_of(st, temperature);
        return;
    }
    // (Of more than k candidates only the k largest can be among the row's.)
    if (found > k) sort_candidates<kThreads>(sh, found);
    for (int i = threadIdx.x; i < k; i += kThreads) part_entries[(int64_t)blockIdx.x * k + i] = i < found ? sh.candidates[i] : 0;
    if (threadIdx.x == 0) part_stats[blockIdx.x] = st;
}

// The parts' entries of a row, and their statistics.
__global__ __launch_bounds__(1024) void join_top_kernel(const u64 *__restrict__ part_entries, const Stat *__restrict__ part_stats,
                                                        int parts, int k, float temperature, float *__restrict__ values,
                                                        int *__restrict__ indices, float *__restrict__ lse) {
    constexpr int kThreads = 1024;
    __shared__ TopShared<kThreads> sh;
    const int64_t row = blockIdx.x;
    const u64 *const e = part_entries + row * parts * k;
    const int n = parts * k;
    u64 mine = 0;
    for (int i = threadIdx.x; i < n; i += kThreads) mine = mine > e[i] ? mine : e[i];
    auto each = [&](auto visit) {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const u64 w = e[i];
            if (w != 0) visit(value_of_key((unsigned int)(w >> 32)), ~(unsigned int)w);
        }
    };
    clear_top(sh);
    const unsigned int key = max((unsigned int)(mine >> 32), kKeyOfNothing);
    const int found = take_top<kThreads>(sh, k, threshold_of(sh, k, key), [&](float, auto visit) { each(visit); }, each);
    sort_candidates<kThreads>(sh, found);
    write_top<kThreads>(sh, found, k, values + row * k, indices + row * k);
    if (threadIdx.x == 0) {
        Stat st = part_stats[row * parts];
        for (int p = 1; p < parts; ++p) st = join(st, part_stats[row * parts + p], kLog2E / temperature);
        lse[row] = lse_of(st, temperature);
    }
}

// ---- distillation -------------------------------------------------------------------------------------------------

struct Distill {
    int64_t cols, row_stride;
    const int *indices;
    const float *values;
    int k;
    const float *lse, *weights;
    float temperature;
    int rest;
    float *loss;
    int64_t grad_stride;
    int parts, part;      // stretches of a row, and their columns
    Stat *part_stats;     // rows x parts, of the columns that are not listed (of all without rest)
    float *listed_logits; // rows x k
    int *part_doubles;    // rows x parts: whether the list has one of the stretch's columns more than once
    int mark;             // whether that is asked for: with rest, or for a gradient
};

// The teacher's list of a row in LDS.
struct List {
    int *at;     // columns, -1 for none
    float *p;    // probabilities
    float *lp;   // ... and their logarithms
    float *z;    // the columns' logits
    float *own;  // everything that the list says of a column; the sign bit set where the column stands before in the list
};
__device__ __forceinline__ int list_room(int k) { return (k + 7) / 8 * 8; }
__device__ __forceinline__ List list_in(unsigned int *shared, int k) {
    const int room = list_room(k);
    float *const f = reinterpret_cast<float *>(shared) + room;
    return {reinterpret_cast<int *>(shared), f, f + room, f + 2 * room, f + 3 * room};
}
inline size_t list_bytes(int k) { return (size_t)(k + 7) / 8 * 8 * 5 * 4; }

// Reads the list and makes its probabilities; ends with a barrier.  scratch: an entry a wave.
template <int kThreads>
__device__ __forceinline__ void read_list(const Distill &d, int64_t row, const List &l, Stat *scratch) {
    const float c = kLog2E / d.temperature;
    Stat st = {lowest(), 0.0f};
    for (int j = threadIdx.x; j < list_room(d.k); j += kThreads) {
        const int i = j < d.k ? d.indices[row * d.k + j] : -1;
        const float said = j < d.k ? d.values[row * d.k + j] : lowest();
        const bool there = i >= 0 && i < d.cols;
        const float v = there ? said : lowest();
        l.at[j] = there ? i : -1;
        l.p[j] = v;
        if (!d.lse) add(st, v, c);
    }
    float base = 0.0f, offset;
    if (d.lse) {
        offset = d.lse[row];
    } else {
        st = join_all<kThreads>(st, c, scratch);
        base = base_of(st.m);
        offset = logf(st.s);
    }
    for (int j = threadIdx.x; j < list_room(d.k); j += kThreads) {
        const float lp = (l.p[j] - base) / d.temperature - offset;
        l.p[j] = l.p[j] == lowest() ? 0.0f : expf(lp);
        l.lp[j] = lp;
    }
    __syncthreads();
}
// What the list says of every column in it (eight threads an entry); ends with a barrier.
template <int kThreads>
__device__ __forceinline__ void join_doubles(const Distill &d, const List &l) {
    const int room = list_room(d.k);
    for (int j = threadIdx.x / 8; j < room; j += kThreads / 8) {
        const int mine = l.at[j];
        float sum = 0.0f;
        int before = 0;
        for (int i = threadIdx.x % 8 * 4; i < room; i += 32) {
            const int4 at = *reinterpret_cast<const int4 *>(l.at + i);
            if (at.x == mine || at.y == mine || at.z == mine || at.w == mine) {
                if (at.x == mine) sum += l.p[i], before |= i < j;
                if (at.y == mine) sum += l.p[i + 1], before |= i + 1 < j;
                if (at.z == mine) sum += l.p[i + 2], before |= i + 2 < j;
                if (at.w == mine) sum += l.p[i + 3], before |= i + 3 < j;
            }
        }
        sum += exchanged<kByOne>(sum);
        sum += exchanged<kByTwo>(sum);
        sum += exchanged<kMirrorEight>(sum);
        before |= exchanged<kByOne>(before);
        before |= exchanged<kByTwo>(before);
        before |= exchanged<kMirrorEight>(before);
        if (threadIdx.x % 8 == 0) l.own[j] = before ? -sum : sum;
    }
    __syncthreads();
}
__device__ __forceinline__ bool stands_before(float own) { return __float_as_uint(own) >> 31; }

// A row's loss, and what its gradient is made of.
struct Parts {
    float all_base, all_sum, total;  // q = 2^((z - all_base) c) / all_sum; total = sum p + p_r
    float out_base, factor;          // outside the list: scale * factor * 2^((z - out_base) c)
    float scale;
};
// out: the statistics of the columns outside the list (of all without rest).  scratch, sums: an entry a wave each.
template <int kThreads>
__device__ __forceinline__ Parts make_parts(const Distill &d, const List &l, Stat out, float w, float *loss, Stat *scratch,
                                            float *sums, float *more_sums) {
    const float c = kLog2E / d.temperature;
    Stat all = out;
    if (d.rest) {
        Stat in = {lowest(), 0.0f};
        for (int j = threadIdx.x; j < d.k; j += kThreads)
            if (l.at[j] >= 0 && !stands_before(l.own[j])) add(in, l.z[j], c);
        all = join(join_all<kThreads>(in, c, scratch), out, c);
    }
    const float base = base_of(all.m), ln_all = logf(all.s);
    auto ln_q = [&](float v) { return v == lowest() ? v : (v - base) / d.temperature - ln_all; };
    float part = 0.0f, mass = 0.0f;
    for (int j = threadIdx.x; j < d.k; j += kThreads) {
        const float p = l.p[j];
        if (p != 0.0f) part += p * (l.lp[j] - ln_q(l.z[j]));
        mass += p;
    }
    part = sum_all<kThreads>(part, sums);
    mass = sum_all<kThreads>(mass, more_sums);
    float pr = 0.0f;
    if (d.rest && out.s != 0.0f) {
        pr = fmaxf(0.0f, 1.0f - mass);
        if (pr > 0.0f) part += pr * (logf(pr) - (ln_q(out.m) + logf(out.s)));
    }
    if (loss && threadIdx.x == 0) *loss = w * (all.s != all.s ? all.s : part);  // (no number, also where no p asks for one)
    // Outside the list q total - p_r q / q_r, from those columns' own maximum, so that nothing overflows where they are far
    // below the list's.  (Where nothing is finite out there every term is 0; a sum that is no number goes everywhere.)
    Parts r = {base, all.s, mass + pr, base_of(out.m), all.s != all.s ? all.s : 0.0f, w / d.temperature};
    if (out.m > lowest() && all.s > 0.0f)
        r.factor = r.total * exp2f((r.out_base - base) * c) / all.s - (pr > 0.0f ? pr / out.s : 0.0f);
    return r;
}
__device__ __forceinline__ float listed_gradient(const Parts &r, float z, float own, float c) {
    const float q = r.all_sum > 0.0f ? exp2f((z - r.all_base) * c) / r.all_sum : r.all_sum;
    return r.scale * (q * r.total - fabsf(own));
}

// The columns of a stretch that are listed, a bit each, and whether any is listed twice; ends with a barrier.
template <int kThreads>
__device__ __forceinline__ bool mark_listed(const Distill &d, const List &l, unsigned int *bits, int *doubles, int c0, int n) {
    for (int i = threadIdx.x; i < (n + 31) / 32; i += kThreads) bits[i] = 0;
    if (threadIdx.x == 0) *doubles = 0;
    __syncthreads();
    for (int j = threadIdx.x; j < d.k; j += kThreads) {
        const int i = l.at[j] - c0;
        if (l.at[j] < 0 || i < 0 || i >= n) continue;
        const unsigned int bit = 1u << (i % 32);
        if (atomicOr(&bits[i / 32], bit) & bit) *doubles = 1;
    }
    __syncthreads();
    return *doubles != 0;
}
// ... are taken out of what is held.
template <typename T, int kThreads, int kHeld>
__device__ __forceinline__ void take_out(Held<T, kThreads, kHeld> &held, const unsigned int *bits, int n) {
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const int i = held.place(h);
        const unsigned int b = i < n ? bits[i / 32] >> (i % 32) & ((1u << kVec<T>) - 1) : 0;
        if (b != 0) {
            float w[kVec<T>];
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) w[j] = b >> j & 1 ? lowest() : held.v[h][j];
            held.v[h].raw = pack_vec<T>(w);
        }
    }
}

template <typename T, int kThreads, int kHeld>
__device__ __forceinline__ void write_gradient(Held<T, kThreads, kHeld> &held, const Parts &r, float c, T *g, int n) {
    held.keep_packed();
    const Powers power(r.out_base, c);
    const float factor = uniform(r.scale * r.factor * (power.fused ? power.more() : 1.0f));
#pragma unroll
    for (int h = 0; h < kHeld; ++h) {
        const int i = held.place(h);
        if (i >= n) break;
        float w[kVec<T>];
        if (power.fused) {
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) w[j] = factor * power.near(held.v[h][j]);
        } else {
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) w[j] = factor * power.far(held.v[h][j]);
        }
        if (i + kVec<T> <= n) {
            store_vec(g + i, w);
        } else {
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j)
                if (i + j < n) g[i + j] = (T)w[j];
        }
    }
}

struct DistillShared {
    Stat stats[16];
    float floats[16], sums[16], more_sums[16];
    int doubles;
};

// One workgroup a row, all of it in registers: it is read once.
template <typename T, int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads, kHeld == 8 && kThreads > 256 ? 8 : 4) void distill_kernel(const T *logits, T *grad, Distill d) {
    extern __shared__ unsigned int shared[];
    __shared__ DistillShared sh;
    const int64_t row = blockIdx.x;
    const T *z = logits + row * d.row_stride;
    T *g = grad ? grad + row * d.grad_stride : nullptr;
    const int n = (int)d.cols;
    const float w = d.weights ? d.weights[row] : 1.0f, c = kLog2E / d.temperature;
    if (w == 0.0f) {
        if (threadIdx.x == 0) d.loss[row] = 0.0f;
        if (g)
            for (int i = threadIdx.x; i < n; i += kThreads) g[i] = (T)0.0f;
        return;
    }
    const List l = list_in(shared, d.k);
    unsigned int *const bits = shared + 5 * list_room(d.k);
    Held<T, kThreads, kHeld> held;
    held.load(z, n);
    read_list<kThreads>(d, row, l, sh.stats);
    for (int j = threadIdx.x; j < d.k; j += kThreads) l.z[j] = l.at[j] >= 0 ? value_of(z[l.at[j]]) : 0.0f;
    if (g || d.rest) {
        if (mark_listed<kThreads>(d, l, bits, &sh.doubles, 0, n)) {
            join_doubles<kThreads>(d, l);
        } else {  // (each thread for the entries that it alone reads)
            for (int j = threadIdx.x; j < d.k; j += kThreads) l.own[j] = l.p[j];
        }
    }
    if (d.rest) take_out(held, bits, n);
    Stat out = {max_all<kThreads>(held.max(), sh.floats), 0.0f};
    out.s = sum_all<kThreads>(held.sum(base_of(out.m), c), sh.sums);
    __syncthreads();
    const Parts r = make_parts<kThreads>(d, l, out, w, d.loss + row, sh.stats, sh.sums, sh.more_sums);
    if (!g) return;
    write_gradient(held, r, c, g, n);
    __syncthreads();
    for (int j = threadIdx.x; j < d.k; j += kThreads)
        if (l.at[j] >= 0) g[l.at[j]] = (T)listed_gradient(r, l.z[j], l.own[j], c);
}

// Rows in stretches, a workgroup each: the statistics of every stretch, and the listed columns' logits (the gradient may go
// where the logits are) ...
template <typename T, int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads) void distill_stats_kernel(const T *__restrict__ logits, Distill d) {
    extern __shared__ unsigned int shared[];
    __shared__ DistillShared sh;
    const int64_t row = blockIdx.x / d.parts;
    const int which = (int)(blockIdx.x % d.parts), c0 = which * d.part, n = min(d.part, (int)d.cols - c0);
    const T *z = logits + row * d.row_stride;
    const float c = kLog2E / d.temperature;
    if (d.weights && d.weights[row] == 0.0f) return;
    // (Of the first stretch's threads; the columns first, so that what they lead to is not waited for at the end.)
    constexpr int kEach = kMostListed / kThreads;
    int at[kEach];
    float listed[kEach];
    if (which == 0) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int j = i * kThreads + (int)threadIdx.x;
            at[i] = j < d.k ? d.indices[row * d.k + j] : -1;
        }
    }
    Held<T, kThreads, kHeld> held;
    held.load(z + c0, n);
    if (which == 0) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) listed[i] = at[i] >= 0 && at[i] < d.cols ? value_of(z[at[i]]) : 0.0f;
    }
    if (d.mark) {
        const List l = list_in(shared, d.k);
        unsigned int *const bits = shared + list_room(d.k);
        for (int j = threadIdx.x; j < d.k; j += kThreads) {
            const int i = d.indices[row * d.k + j];
            l.at[j] = i >= 0 && i < d.cols ? i : -1;
        }
        const bool doubles = mark_listed<kThreads>(d, l, bits, &sh.doubles, c0, n);
        if (threadIdx.x == 0) d.part_doubles[blockIdx.x] = doubles;
        if (d.rest) take_out(held, bits, n);
    }
    Stat out = {max_all<kThreads>(held.max(), sh.floats), 0.0f};
    out.s = sum_all<kThreads>(held.sum(base_of(out.m), c), sh.sums);
    if (threadIdx.x == 0) d.part_stats[blockIdx.x] = out;
    if (which == 0) {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            const int j = i * kThreads + (int)threadIdx.x;
            if (j < d.k) d.listed_logits[row * d.k + j] = listed[i];
        }
    }
}
// ... and from all of a row's its loss, and a stretch's gradient.
template <typename T, int kThreads, int kHeld>
__global__ __launch_bounds__(kThreads) void distill_finish_kernel(const T *logits, T *grad, Distill d) {
    extern __shared__ unsigned int shared[];
    __shared__ DistillShared sh;
    const int parts = grad ? d.parts : 1;  // (the loss alone takes one workgroup)
    const int64_t row = blockIdx.x / parts;
    const int which = (int)(blockIdx.x % parts), c0 = which * d.part, n = min(d.part, (int)d.cols - c0);
    T *g = grad ? grad + row * d.grad_stride : nullptr;
    const float w = d.weights ? d.weights[row] : 1.0f, c = kLog2E / d.temperature;
    if (w == 0.0f) {
        if (which == 0 && threadIdx.x == 0) d.loss[row] = 0.0f;
        if (g)
            for (int i = threadIdx.x; i < n; i += kThreads) g[c0 + i] = (T)0.0f;
        return;
    }
    Held<T, kThreads, kHeld> held;
    if (g) held.load(logits + row * d.row_stride + c0, n);
    const List l = list_in(shared, d.k);
    read_list<kThreads>(d, row, l, sh.stats);
    for (int j = threadIdx.x; j < d.k; j += kThreads) l.z[j] = d.listed_logits[row * d.k + j];
    Stat out = {lowest(), 0.0f};
    int doubles = 0;
    for (int p = threadIdx.x; p < d.parts; p += kThreads) {
        out = join(out, d.part_stats[row * d.parts + p], c);
        if (d.mark) doubles |= d.part_doubles[row * d.parts + p];
    }
    // (Every pair of entries is looked at only where some column is listed twice.)
    if (__syncthreads_or(doubles)) {
        join_doubles<kThreads>(d, l);
    } else {  // (each thread for the entries that it alone reads)
        for (int j = threadIdx.x; j < d.k; j += kThreads) l.own[j] = l.p[j];
    }
    out = join_all<kThreads>(out, c, sh.stats);
    __syncthreads();
    const Parts r = make_parts<kThreads>(d, l, out, w, which == 0 ? d.loss + row : nullptr, sh.stats, sh.sums, sh.more_sums);
    if (!g) return;
    write_gradient(held, r, c, g + c0, n);
    __syncthreads();
    for (int j = threadIdx.x; j < d.k; j += kThreads)
        if (l.at[j] >= c0 && l.at[j] < c0 + n) g[l.at[j]] = (T)listed_gradient(r, l.z[j], l.own[j], c);
}

// How a row is held: by how many threads, 16 bytes how often each, in how many stretches of how many columns.
struct Holding {
    int threads, held, parts, part;
};
// Rows that one workgroup can hold are read once and need one launch; the fewer and the longer they are, the more compute
// units idle that way.  us, the side that is taken first:
// - distillation, up to 128 rows of more than 64 KB: stretches (60 x 131071 bfloat16 with gradient and rest 19.1, a workgroup a
//   row 31.7; 127 x 60000 18.1 and 18.6; more, 160 x 60000: a workgroup a row 19.4, stretches 20.7; shorter, 64 x 30000, the
//   loss: 6.3 and 7.8);
// - top lists, up to 32 rows of more than 65536 columns: stretches (7 x 131071 15.4, a workgroup a row 22.4; more rows,
//   64 x 131071: a workgroup a row 23.3, stretches 27.5; fewer columns, 16 x 60000 floats: 12.1 and 14.8), for lists that are
//   short to join (2 x 80000, k = 45: stretches 12.6, a workgroup a row 16.9; 1 x 70000, k = 240: 29.9 and 27.2);
// - many short rows: a wave each, which has no barriers to wait at.  Distillation from 512 rows on (4096 x 1000, loss 7.4,
//   by 256 threads 13.3; at 512 both take 5), top lists from 2048 on (2048 x 1000 9.1 and 10.5; 1024 rows: 7.7 by 256 threads,
//   8.3).
constexpr int kFewRows = 128, kFewTopRows = 32, kManyRows = 512, kManyTopRows = 2048, kStretch = 1024;
constexpr int64_t kLongRow = 65536;     // bytes, of a student's; columns, of a teacher's
constexpr int64_t kMostHeld = 16384;    // times 16 bytes
Holding holding_of(int64_t cols, int type, bool many, int least_threads, bool in_stretches, int stretch) {
    const int per = type == kTypeF32 ? 4 : 8;
    const int64_t vecs = (cols + per - 1) / per;
    if (vecs > kMostHeld || in_stretches) return {0, 0, (int)((vecs + stretch - 1) / stretch), stretch * per};
    if (many && least_threads <= kWave && vecs <= kWave * 8) return {kWave, vecs <= kWave * 4 ? 4 : 8, 1, (int)cols};
    const Holding all[] = {{256, 2, 1, (int)cols}, {256, 4, 1, (int)cols}, {256, 8, 1, (int)cols},
                           {512, 8, 1, (int)cols}, {1024, 8, 1, (int)cols}, {1024, 16, 1, (int)cols}};
    for (const Holding &h : all)
        if (h.threads >= least_threads && vecs <= (int64_t)h.threads * h.held) return h;
    return all[5];
}

// A stretch's list costs the more the more stretches there are: where rows are many, they are as long as two to a compute
// unit can be held (1000 x 131072 floats: 450 us with stretches of 4096, 120 with 32768).
int top_stretch(int64_t rows) { return rows <= kFewTopRows ? kStretch : 8 * kStretch; }

// (The threshold is the k-th largest of the threads' maxima: there are k of them at least, 1024 in stretches.)
static_assert(kWaveListed <= kWave && kGroupListed <= 256 && kMostListed <= 1024 && kMostListed <= kStretch);
int top_threads(int k) { return k <= kWaveListed ? kWave : k <= kGroupListed ? 256 : 1024; }

Holding top_holding(int64_t rows, int64_t cols, int type, int k) {
    return holding_of(cols, type, rows >= kManyTopRows, top_threads(k), rows <= kFewTopRows && cols > kLongRow && k <= kGroupListed, top_stretch(rows));
}
Holding distill_holding(int64_t rows, int64_t cols, int type) {
    const int64_t bytes = cols * (type == kTypeF32 ? 4 : 2);
    return holding_of(cols, type, rows >= kManyRows, kWave, rows <= kFewRows && bytes > kLongRow, kStretch);
}

// f(first row, number of rows) for as many rows at a time as a launch can take: its threads, 1024 a row or stretch at most, are
// fewer than 2^32.
template <typename F>
int by_rows(int64_t rows, const Holding &h, F f) {
    const int64_t most = std::max<int64_t>(1, ((int64_t)1 << 21) / h.parts);
    for (int64_t r = 0; r < rows; r += most)
        if (f(r, std::min(most, rows - r))) return 1;
    return 0;
}

// f(number of threads, how often each holds 16 bytes), as constants.
template <typename F>
int by_holding(const Holding &h, F f) {
    using std::integral_constant;
    if (h.threads == kWave) {
        if (h.held == 4) return f(integral_constant<int, kWave>(), integral_constant<int, 4>());
        return f(integral_constant<int, kWave>(), integral_constant<int, 8>());
    }
    if (h.threads == 256) {
        if (h.held == 2) return f(integral_constant<int, 256>(), integral_constant<int, 2>());
        if (h.held == 4) return f(integral_constant<int, 256>(), integral_constant<int, 4>());
        return f(integral_constant<int, 256>(), integral_constant<int, 8>());
    }
    if (h.threads == 512) return f(integral_constant<int, 512>(), integral_constant<int, 8>());
    if (h.held == 8) return f(integral_constant<int, 1024>(), integral_constant<int, 8>());
    return f(integral_constant<int, 1024>(), integral_constant<int, 16>());
}

// Whether a gradient has values where other logits are, so that what one workgroup reads another may have written.  (Rows of
// both that are equally far apart may lie between one another; otherwise the two have to be apart.)
bool overlap(const void *logits, int64_t row_stride, const void *grad, int64_t grad_stride, int64_t rows, int64_t cols, int type) {
    const int64_t size = (int64_t)type_size(type);
    const int64_t apart = (int64_t)(reinterpret_cast<uintptr_t>(grad) - reinterpret_cast<uintptr_t>(logits));  // (bytes)
    if (apart == 0) return false;
    auto extent = [&](int64_t stride) { return ((rows - 1) * stride + cols) * size; };
    if (apart >= extent(row_stride) || -apart >= extent(grad_stride)) return false;
    if (rows == 1 || row_stride != grad_stride) return true;
    const int64_t step = row_stride * size, within = (apart % step + step) % step;  // from a row of logits to the next gradient
    return within < cols * size || within > step - cols * size;
}

}  // namespace
}  // namespace tsnehip

using namespace tsnehip;

extern "C" int64_t tsne_hip_top_logits_workspace(int64_t rows, int64_t cols, int type, int k) {
    if (rows <= 0 || cols <= 0) return 0;
    const Holding h = top_holding(rows, cols, type, k);
    return h.parts > 1 ? rows * h.parts * ((int64_t)sizeof(Stat) + k * (int64_t)sizeof(u64)) : 0;
}

extern "C" int tsne_hip_top_logits(const void *logits, int type, int64_t rows, int64_t cols, int64_t row_stride, int k,
                                   float temperature, float *values, int *indices, float *lse, void *workspace,
                                   int64_t workspace_bytes, void *stream) {
    TSNE_OPERATOR_REQUIRE(rows >= 0 && rows <= 0x7fffffff && cols >= 1 && cols <= 0x7fffffff,
                          "top_logits: a matrix of %lld x %lld", (long long)rows, (long long)cols);
    TSNE_OPERATOR_REQUIRE(row_stride >= cols, "top_logits: rows of %lld values are only %lld apart", (long long)cols,
                          (long long)row_stride);
    TSNE_OPERATOR_REQUIRE(k >= 1 && k <= kMostListed && k <= cols, "top_logits: k must be in [1, min(%lld, %d)] (got %d)",
                          (long long)cols, kMostListed, k);
    if (check_temperature("top_logits", temperature)) return 1;
    if (rows == 0) return 0;
    TSNE_OPERATOR_REQUIRE(logits && values && indices && lse, "top_logits: null argument");
    if (check_workspace("top_logits", workspace, workspace_bytes, tsne_hip_top_logits_workspace(rows, cols, type, k))) return 1;
    const hipStream_t s = (hipStream_t)stream;
    const Holding h = top_holding(rows, cols, type, k);
    return by_type(type, "top_logits", [&](auto zero) {
        using T = decltype(zero);
        u64 *const entries = (u64 *)workspace;
        Stat *const stats = (Stat *)(entries + rows * h.parts * k);
        return by_rows(rows, h, [&](int64_t first, int64_t n) {
            const T *z = (const T *)logits + first * row_stride;
            float *const v = values + first * k, *const l = lse + first;
            int *const at = indices + first * k;
            if (h.parts > 1) {
                const auto kernel = top_stretch(rows) == kStretch ? top_logits_kernel<T, kStretch, 1> : top_logits_kernel<T, kStretch, 8>;
                kernel<<<(unsigned int)(n * h.parts), kStretch, 0, s>>>(z, cols, row_stride, k, temperature, h.parts, h.part, v, at, l,
                                                                       entries, stats);
                TSNE_LAUNCHED(s);
                join_top_kernel<<<(unsigned int)n, 1024, 0, s>>>(entries, stats, h.parts, k, temperature, v, at, l);
                TSNE_LAUNCHED(s);
                return 0;
            }
            return by_holding(h, [&](auto threads, auto held) {
                constexpr int kThreads = decltype(threads)::value, kHeld = decltype(held)::value;
                top_logits_kernel<T, kThreads, kHeld><<<(unsigned int)n, kThreads, 0, s>>>(z, cols, row_stride, k, temperature, 1, h.part,
                                                                                         v, at, l, nullptr, nullptr);
                TSNE_LAUNCHED(s);
                return 0;
            });
        });
    });
}

extern "C" int64_t tsne_hip_distill_workspace(int64_t rows, int64_t cols, int type, int k) {
    if (rows <= 0 || cols <= 0) return 0;
    const Holding h = distill_holding(rows, cols, type);
    return h.parts > 1 ? rows * (h.parts * (int64_t)(sizeof(Stat) + sizeof(int)) + k * (int64_t)sizeof(float)) : 0;
}

extern "C" int tsne_hip_distill(const void *logits, int type, int64_t rows, int64_t cols, int64_t row_stride,
                                const int *indices, const float *values, int k, const float *lse, const float *weights,
                                float temperature, int rest, float *loss, void *grad, int64_t grad_stride,
                                void *workspace, int64_t workspace_bytes, void *stream) {
    TSNE_OPERATOR_REQUIRE(rows >= 0 && rows <= 0x7fffffff && cols >= 1 && cols <= kMostDistilled,
                          "distill: a matrix of %lld x %lld (at most %lld columns)", (long long)rows, (long long)cols,
                          (long long)kMostDistilled);
    TSNE_OPERATOR_REQUIRE(row_stride >= cols && (!grad || grad_stride >= cols),
                          "distill: rows of %lld values are only %lld and %lld apart", (long long)cols,
                          (long long)row_stride, (long long)grad_stride);
    TSNE_OPERATOR_REQUIRE(k >= 1 && k <= kMostListed, "distill: k must be in [1, %d] (got %d)", kMostListed, k);
    if (check_temperature("distill", temperature)) return 1;
    TSNE_OPERATOR_REQUIRE(rest == 0 || rest == 1, "distill: rest must be 0 or 1 (got %d)", rest);
    TSNE_OPERATOR_REQUIRE(rest == 0 || lse, "distill: rest needs the teacher's lse");
    if (rows == 0) return 0;
    TSNE_OPERATOR_REQUIRE(logits && indices && values && loss, "distill: null argument");
    TSNE_OPERATOR_REQUIRE(grad != logits || grad_stride == row_stride,
                          "distill: a gradient in the logits' place has to have their stride");
    TSNE_OPERATOR_REQUIRE(!grad || !overlap(logits, row_stride, grad, grad_stride, rows, cols, type),
                          "distill: the gradient overlaps the logits, and is not in their place");
    if (check_workspace("distill", workspace, workspace_bytes, tsne_hip_distill_workspace(rows, cols, type, k))) return 1;
    const hipStream_t s = (hipStream_t)stream;
    const Holding h = distill_holding(rows, cols, type);
    Distill d = {cols, row_stride, indices, values, k, lse, weights, temperature, rest, loss, grad_stride, h.parts, h.part,
                 (Stat *)workspace, nullptr, nullptr, rest || grad};
    d.listed_logits = (float *)(d.part_stats + rows * h.parts);
    d.part_doubles = (int *)(d.listed_logits + rows * k);
    const size_t bits = rest || grad ? ((size_t)h.part + 31) / 32 * 4 : 0;
    return by_type(type, "distill", [&](auto zero) {
        using T = decltype(zero);
        return by_rows(rows, h, [&](int64_t first, int64_t n) {
            const T *z = (const T *)logits + first * row_stride;
            T *const g = grad ? (T *)grad + first * grad_stride : nullptr;
            d.indices = indices + first * k;
            d.values = values + first * k;
            d.lse = lse ? lse + first : nullptr;
            d.weights = weights ? weights + first : nullptr;
            d.loss = loss + first;
            if (h.parts > 1) {
                constexpr int kThreads = 256;
                distill_stats_kernel<T, kThreads, kStretch / kThreads><<<(unsigned int)(n * h.parts), kThreads, list_bytes(k) / 5 + bits, s>>>(z, d);
                TSNE_LAUNCHED(s);
                distill_finish_kernel<T, kThreads, kStretch / kThreads><<<(unsigned int)(n * (g ? h.parts : 1)), kThreads, list_bytes(k), s>>>(z, g, d);
                TSNE_LAUNCHED(s);
                return 0;
            }
            return by_holding(h, [&](auto threads, auto held) {
                constexpr int kThreads = decltype(threads)::value, kHeld = decltype(held)::value;
                distill_kernel<T, kThreads, kHeld><<<(unsigned int)n, kThreads, list_bytes(k) + bits, s>>>(z, g, d);
                TSNE_LAUNCHED(s);
                return 0;
            });
        });
    });
}
