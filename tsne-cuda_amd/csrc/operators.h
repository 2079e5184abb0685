// What the encoder operators (quantize.hip, block_product.hip, distill.hip) share.
#ifndef TSNE_HIP_OPERATORS_INTERNAL_H_
#define TSNE_HIP_OPERATORS_INTERNAL_H_

#include "common.h"

namespace tsnehip {

enum { kTypeF32 = 0, kTypeF16 = 1, kTypeBf16 = 2 };

inline size_t type_size(int type) { return type == kTypeF32 ? 4 : 2; }

constexpr int kBlock = 128;  // values that share a scale
// Bytes from one row to the next of a block-scaled matrix of `cols` columns, and of its scales.
inline int64_t block_data_stride(int64_t cols) { return (cols + kBlock - 1) / kBlock * kBlock; }
inline int64_t block_scale_stride(int64_t cols) { return (cols + 4 * kBlock - 1) / (4 * kBlock) * 4; }

#define TSNE_OPERATOR_REQUIRE(cond, ...) \
    do {                                 \
        if (!(cond)) {                   \
            set_error(__VA_ARGS__);      \
            return 1;                    \
        }                                \
    } while (0)

inline int check_workspace(const char *who, const void *workspace, int64_t bytes, int64_t needed) {
    TSNE_OPERATOR_REQUIRE(bytes >= needed && (workspace || needed == 0), "%s: the workspace has %lld bytes and not %lld", who,
                          (long long)bytes, (long long)needed);
    TSNE_OPERATOR_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "%s: the workspace must be aligned to 16 bytes", who);
    return 0;
}

// (Below 2^-126 its reciprocal is infinite, and a difference of nothing times that no number.)
inline int check_temperature(const char *who, float temperature) {
    TSNE_OPERATOR_REQUIRE(temperature >= 0x1p-126f && temperature < __builtin_inff(),
                          "%s: the temperature must be positive, 2^-126 at least (got %g)", who, (double)temperature);
    return 0;
}

int launch_quantize(const void *x, int type, int64_t rows, int64_t cols, int64_t row_stride, int square, uint8_t *data,
                    uint8_t *scales, uint8_t *data_t, uint8_t *scales_t, hipStream_t s);

#ifdef __HIPCC__
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
// (16 bytes at any address a value may have: the machine's loads and stores need no more)
typedef u32x4 u32x4_unaligned __attribute__((aligned(2)));

__device__ __forceinline__ float value_of(float v) { return v; }
__device__ __forceinline__ float value_of(_Float16 v) { return (float)v; }
__device__ __forceinline__ float value_of(__bf16 v) { return (float)v; }

// kVec<T> values are 16 bytes.
template <typename T>
constexpr int kVec = 16 / (int)sizeof(T);

template <typename T>
struct Vec {
    u32x4 raw;
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(raw[i]);
        const unsigned short h = (unsigned short)(raw[i / 2] >> (16 * (i & 1)));
        return value_of(__builtin_bit_cast(T, h));
    }
};
template <>
__device__ __forceinline__ float Vec<float>::operator[](int i) const {
    return __uint_as_float(raw[i]);
}
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T *p) {
    return Vec<T>{*reinterpret_cast<const u32x4_unaligned *>(p)};
}
template <typename T>
__device__ __forceinline__ u32x4 pack_vec(const float *v) {
    u32x4 raw;
    if constexpr (sizeof(T) == 4) {
        for (int i = 0; i < 4; ++i) raw[i] = __float_as_uint(v[i]);
    } else {
        for (int i = 0; i < 4; ++i)
            raw[i] = (unsigned int)__builtin_bit_cast(unsigned short, (T)v[2 * i]) |
                     (unsigned int)__builtin_bit_cast(unsigned short, (T)v[2 * i + 1]) << 16;
    }
    return raw;
}
template <typename T>
__device__ __forceinline__ void store_vec(T *p, const float *v) {
    *reinterpret_cast<u32x4_unaligned *>(p) = pack_vec<T>(v);
}

// Exchanges among 16 lanes in the vector unit (shuffles go through LDS, at ten times the latency), all lanes taking part:
// with the lane whose number differs in the last bit, in the last but one, and with the mirrored one of eight and of 16.
template <int kControl>
__device__ __forceinline__ int exchanged(int v) {
    return __builtin_amdgcn_mov_dpp(v, kControl, 15, 15, false);
}
template <int kControl>
__device__ __forceinline__ float exchanged(float v) {
    return __int_as_float(exchanged<kControl>(__float_as_int(v)));
}
__device__ __forceinline__ float lane_value(float v, int lane) {
    return __uint_as_float((unsigned int)__builtin_amdgcn_readlane((int)__float_as_uint(v), lane));
}
constexpr int kByOne = 0xb1, kByTwo = 0x4e, kMirrorEight = 0x141, kMirrorSixteen = 0x140;
// Over a wave, in a fixed order, for all lanes.
__device__ __forceinline__ float wave_sum(float v) {
    v += exchanged<kByOne>(v);
    v += exchanged<kByTwo>(v);
    v += exchanged<kMirrorEight>(v);
    v += exchanged<kMirrorSixteen>(v);
    return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ __forceinline__ float max_of_eight(float v) {
    v = fmaxf(v, exchanged<kByOne>(v));
    v = fmaxf(v, exchanged<kByTwo>(v));
    return fmaxf(v, exchanged<kMirrorEight>(v));
}
__device__ __forceinline__ float max_of_sixteen(float v) {
    v = max_of_eight(v);
    return fmaxf(v, exchanged<kMirrorSixteen>(v));
}
__device__ __forceinline__ float wave_max(float v) {
    v = max_of_sixteen(v);
    return fmaxf(fmaxf(lane_value(v, 0), lane_value(v, 16)), fmaxf(lane_value(v, 32), lane_value(v, 48)));
}

// Quantising a block of 128 values.
// Eight values of a row from column c on, zeros from column `cols` on.
template <typename T>
__device__ __forceinline__ void load_eight(const T *row, int64_t c, int64_t cols, float *v) {
    if (c + 8 <= cols) {
#pragma unroll
        for (int h = 0; h < 8 / kVec<T>; ++h) {
            const Vec<T> w = load_vec(row + c + h * kVec<T>);
#pragma unroll
            for (int j = 0; j < kVec<T>; ++j) v[h * kVec<T> + j] = w[j];
        }
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = c + j < cols ? value_of(row[c + j]) : 0.0f;
    }
}
// Magnitude that a block's scale goes by: nothing of NaN and infinities.
__device__ __forceinline__ float scale_magnitude(float v) {
    const float a = fabsf(v);
    return a < __builtin_inff() ? a : 0.0f;
}

// The least e >= -127 with a <= 448 * 2^e = 0.875 * 2^(e + 9); 0 for a = 0.
__device__ __forceinline__ int scale_exponent(float a) {
    if (a == 0.0f) return 0;
    int x;
    const float m = frexpf(a, &x);  // a = m 2^x, 0.5 <= m < 1
    const int e = x - 9 + (m > 0.875f ? 1 : 0);
    return e < -127 ? -127 : e;
}
// 2^-e: v * 2^-e is exact unless it underflows, and what underflows is 0 in eight bits.
__device__ __forceinline__ float inverse_scale(int e) { return __uint_as_float((unsigned int)(127 - e) << 23); }

__device__ __forceinline__ float or_nan(float v, float inv) {  // (448 is the conversion's largest)
    return fabsf(v) < __builtin_inff() ? v * inv : __builtin_nanf("");
}
__device__ __forceinline__ unsigned int pack4(float a, float b, float c, float d, float inv) {
    int r = __builtin_amdgcn_cvt_pk_fp8_f32(or_nan(a, inv), or_nan(b, inv), 0, false);
    return (unsigned int)__builtin_amdgcn_cvt_pk_fp8_f32(or_nan(c, inv), or_nan(d, inv), r, true);
}
#endif  // __HIPCC__

// Calls f with a value of the matrix's type.
template <typename F>
inline int by_type(int type, const char *who, F f) {
    switch (type) {
        case kTypeF32: return f(0.0f);
        case kTypeF16: return f((_Float16)0.0f);
        case kTypeBf16: return f((__bf16)0.0f);
    }
    set_error("%s: unknown type %d (0 = float, 1 = half, 2 = bfloat16)", who, type);
    return 1;
}

}  // namespace tsnehip

#endif  // TSNE_HIP_OPERATORS_INTERNAL_H_
