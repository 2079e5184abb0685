// 8-bit floating point with a power-of-two scale for each block of 128 values (tsne_operators.h has the format).
//
// Bound: memory, two bytes in and one or two out a value of bfloat16.  Rows alone need nobody else's values: 16 threads a
// block, nothing in LDS (by these and by the tiles below: 1203 x 784 floats 2.8 and 4.9 us, 8195 x 1024 bfloat16 6.0 and 7.7;
// large ones alike, 8192 x 8192 33.6, 6.0 TB/s, in part from the cache).  Where the transpose or squares are asked for, a
// workgroup takes 128 x 128 values, so that rows', columns' and square blocks are all whole in it and x is read once for
// everything.  A row's block is complete in the 16 threads that load it and is written at once; the values go to LDS as they
// came, where eight threads find a column's (a word's two columns at a time) with 16 rows each.  Both orientations of
// 8192 x 4096 bfloat16 27 us (5.0 TB/s; a copy runs at 4.8; 31 with the rows read from LDS again and a column at a time), of
// 4096 x 4096 floats 20.1 (5.0; by squares 22.9); of 8195 x 1024 11.5 to 12.4 (2.7 to 2.9), where the tiles are too few to cover one
// another's loads, way through LDS and stores.
#include "../../include/tsnecuda/tsne_operators.h"
#include "operators.h"

namespace tsnehip {

namespace {

constexpr int kThreads = 512;
constexpr int kTile = kBlock;
constexpr int kRowTurns = kTile * 16 / kThreads;

// A tile's row in LDS: 128 values and a pad that spreads a column's over the banks.
template <typename T>
constexpr int kPerWord = 4 / sizeof(T);
template <typename T>
constexpr int kRowWords = kTile / kPerWord<T> + 1;
template <typename T>
constexpr int kColumnTurns = kTile * 8 / kThreads / kPerWord<T>;

template <typename T>
__global__ __launch_bounds__(kThreads) void quantize_kernel(const T *__restrict__ x, int64_t rows, int64_t cols,
                                                            int64_t row_stride, int square, uint8_t *__restrict__ data,
                                                            uint8_t *__restrict__ scales, uint8_t *__restrict__ data_t,
                                                            uint8_t *__restrict__ scales_t, int64_t data_stride,
                                                            int64_t scale_stride, int64_t data_t_stride,
                                                            int64_t scale_t_stride, unsigned int column_tiles) {
    __shared__ unsigned int tile[kTile * kRowWords<T>];
    __shared__ float square_max[kThreads / kWave];
    const int64_t r0 = (int64_t)(blockIdx.x / column_tiles) * kTile, c0 = (int64_t)(blockIdx.x % column_tiles) * kTile;
    const int t = threadIdx.x;
    auto at = [&](int r, int c) -> float {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(tile[r * kRowWords<T> + c]);
        } else {
            const unsigned int w = tile[r * kRowWords<T> + c / 2];
            return value_of(__builtin_bit_cast(T, (unsigned short)(w >> (16 * (c & 1)))));
        }
    };
    // Values of this thread: columns 8 (t % 16) ... + 8 of rows t / 16, + kThreads / 16, ...  Their rows' blocks are complete
    // in 16 threads, and are written right away; squares' wait for the other threads'.
    const int c = t % 16 * 8;
    float peak = 0.0f;  // of everything this thread has loaded
    auto write_row = [&](int r, int e, const float *v) {
        const float inv = inverse_scale(e);
        *reinterpret_cast<u32x2 *>(data + (r0 + r) * data_stride + c0 + c) =
            u32x2{pack4(v[0], v[1], v[2], v[3], inv), pack4(v[4], v[5], v[6], v[7], inv)};
        if (t % 16 == 0) scales[(r0 + r) * scale_stride + c0 / kBlock] = (uint8_t)(e + 127);
    };
#pragma unroll
    for (int i = 0; i < kRowTurns; ++i) {
        const int r = t / 16 + kThreads / 16 * i;
        float v[8];
        load_eight(x + (r0 + r) * row_stride, c0 + c, r0 + r < rows ? cols : 0, v);
        float m = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j) m = fmaxf(m, scale_magnitude(v[j]));
        peak = fmaxf(peak, m);
        if (data && !square) {
            m = max_of_sixteen(m);
            if (r0 + r < rows) write_row(r, scale_exponent(m), v);
        }
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) tile[r * kRowWords<T> + c + j] = __float_as_uint(v[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                tile[r * kRowWords<T> + c / 2 + j] =
                    (unsigned int)__builtin_bit_cast(unsigned short, (T)v[2 * j]) |
                    (unsigned int)__builtin_bit_cast(unsigned short, (T)v[2 * j + 1]) << 16;
        }
    }
    if (square) {
        peak = wave_max(peak);
        if (t % kWave == 0) square_max[t / kWave] = peak;
    }
    __syncthreads();
    if (square) {
        peak = square_max[0];
        for (int w = 1; w < kThreads / kWave; ++w) peak = fmaxf(peak, square_max[w]);
    }
    const int square_exponent = scale_exponent(peak);
    if (data) {
        if (square) {
#pragma unroll
            for (int i = 0; i < kRowTurns; ++i) {
                const int r = t / 16 + kThreads / 16 * i;
                if (r0 + r >= rows) continue;
                float v[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = at(r, c + j);
                write_row(r, square_exponent, v);
            }
        }
        // (scales behind the last block)
        if (c0 + kTile >= cols && t < kTile && r0 + t < rows)
            for (int64_t b = c0 / kBlock + 1; b < scale_stride; ++b) scales[(r0 + t) * scale_stride + b] = 127;
    }
    if (data_t) {
        // Rows 16 (t % 8) ... + 16 of the columns in word t / 8, + kThreads / 8, ... of a row.
        const int r = t % 8 * 16;
#pragma unroll
        for (int i = 0; i < kColumnTurns<T>; ++i) {
            const int word = t / 8 + kThreads / 8 * i;
            float v[kPerWord<T>][16], m[kPerWord<T>] = {};
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const unsigned int w = tile[(r + j) * kRowWords<T> + word];
#pragma unroll
                for (int p = 0; p < kPerWord<T>; ++p) {
                    if constexpr (sizeof(T) == 4) v[p][j] = __uint_as_float(w);
                    else v[p][j] = value_of(__builtin_bit_cast(T, (unsigned short)(w >> (16 * p))));
                    m[p] = fmaxf(m[p], scale_magnitude(v[p][j]));
                }
            }
#pragma unroll
            for (int p = 0; p < kPerWord<T>; ++p) {
                const int64_t col = c0 + word * kPerWord<T> + p;
                const float most = max_of_eight(m[p]);
                if (col >= cols) continue;
                const int e = square ? square_exponent : scale_exponent(most);
                const float inv = inverse_scale(e);
                u32x4 q;
#pragma unroll
                for (int j = 0; j < 4; ++j) q[j] = pack4(v[p][4 * j], v[p][4 * j + 1], v[p][4 * j + 2], v[p][4 * j + 3], inv);
                *reinterpret_cast<u32x4 *>(data_t + col * data_t_stride + r0 + r) = q;
                if (t % 8 == 0) scales_t[col * scale_t_stride + r0 / kBlock] = (uint8_t)(e + 127);
            }
        }
        if (r0 + kTile >= rows && t < kTile && c0 + t < cols)
            for (int64_t b = r0 / kBlock + 1; b < scale_t_stride; ++b) scales_t[(c0 + t) * scale_t_stride + b] = 127;
    }
}

// Rows alone, whose blocks need nobody else's values: 16 threads a block, nothing in LDS.
template <typename T>
__global__ __launch_bounds__(256) void quantize_rows_kernel(const T *__restrict__ x, int64_t units, int64_t cols,
                                                            int64_t row_stride, uint8_t *__restrict__ data,
                                                            uint8_t *__restrict__ scales, unsigned int blocks,
                                                            int64_t scale_stride) {
    const int64_t u = (int64_t)blockIdx.x * (256 / 16) + threadIdx.x / 16;  // a row's block
    if (u >= units) return;
    const int64_t row = u / blocks;
    const unsigned int at = (unsigned int)(u - row * blocks);
    const int64_t c = (int64_t)at * kBlock + threadIdx.x % 16 * 8;
    float v[8];
    load_eight(x + row * row_stride, c, cols, v);
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, scale_magnitude(v[j]));
    const int e = scale_exponent(max_of_sixteen(m));
    const float inv = inverse_scale(e);
    *reinterpret_cast<u32x2 *>(data + row * blocks * kBlock + c) =
        u32x2{pack4(v[0], v[1], v[2], v[3], inv), pack4(v[4], v[5], v[6], v[7], inv)};
    if (threadIdx.x % 16 == 0) {
        uint8_t *const s = scales + row * scale_stride + at;
        *s = (uint8_t)(e + 127);
        if (at + 1 == blocks)  // (scales behind the last block)
            for (int64_t b = blocks; b < scale_stride; ++b) s[b - at] = 127;
    }
}

}  // namespace

int launch_quantize(const void *x, int type, int64_t rows, int64_t cols, int64_t row_stride, int square, uint8_t *data,
                    uint8_t *scales, uint8_t *data_t, uint8_t *scales_t, hipStream_t s) {
    const int64_t row_tiles = (rows + kTile - 1) / kTile, column_tiles = (cols + kTile - 1) / kTile;
    // (A launch's threads are fewer than 2^32.)
    TSNE_OPERATOR_REQUIRE(row_tiles <= 0xffffffff / kThreads / (column_tiles ? column_tiles : 1),
                          "quantize_blocks: %lld x %lld values are more than one launch holds", (long long)rows,
                          (long long)cols);
    if (row_tiles * column_tiles == 0) return 0;
    const int64_t units = rows * column_tiles;
    if (!square && !data_t && units < (int64_t)1 << 27) {
        return by_type(type, "quantize_blocks", [&](auto zero) {
            using T = decltype(zero);
            quantize_rows_kernel<T><<<div_up(units, 256 / 16), 256, 0, s>>>((const T *)x, units, cols, row_stride, data, scales,
                                                                           (unsigned int)column_tiles, block_scale_stride(cols));
            TSNE_LAUNCHED(s);
            return 0;
        });
    }
    return by_type(type, "quantize_blocks", [&](auto zero) {
        using T = decltype(zero);
        quantize_kernel<T><<<(unsigned int)(row_tiles * column_tiles), kThreads, 0, s>>>(
            (const T *)x, rows, cols, row_stride, square, data, scales, data_t, scales_t, block_data_stride(cols),
            block_scale_stride(cols), block_data_stride(rows), block_scale_stride(rows), (unsigned int)column_tiles);
        TSNE_LAUNCHED(s);
        return 0;
    });
}

}  // namespace tsnehip

using namespace tsnehip;

extern "C" int tsne_hip_quantize_blocks(const void *x, int type, int64_t rows, int64_t cols, int64_t row_stride,
                                        int square, uint8_t *data, uint8_t *scales, uint8_t *data_t, uint8_t *scales_t,
                                        void *stream) {
    TSNE_OPERATOR_REQUIRE(rows >= 0 && cols >= 0, "quantize_blocks: a matrix of %lld x %lld", (long long)rows,
                          (long long)cols);
    TSNE_OPERATOR_REQUIRE(row_stride >= cols, "quantize_blocks: rows of %lld values are only %lld apart",
                          (long long)cols, (long long)row_stride);
    TSNE_OPERATOR_REQUIRE(square == 0 || square == 1, "quantize_blocks: square must be 0 or 1 (got %d)", square);
    TSNE_OPERATOR_REQUIRE((data != nullptr) == (scales != nullptr) && (data_t != nullptr) == (scales_t != nullptr),
                          "quantize_blocks: data and scales go together");
    if (rows == 0 || cols == 0) return 0;
    TSNE_OPERATOR_REQUIRE(x && (data || data_t), "quantize_blocks: null argument");
    TSNE_OPERATOR_REQUIRE((reinterpret_cast<uintptr_t>(data) | reinterpret_cast<uintptr_t>(data_t)) % 16 == 0,
                          "quantize_blocks: data must be aligned to 16 bytes");
    TSNE_OPERATOR_REQUIRE((reinterpret_cast<uintptr_t>(scales) | reinterpret_cast<uintptr_t>(scales_t)) % 16 == 0,
                          "quantize_blocks: scales must be aligned to 16 bytes");
    return launch_quantize(x, type, rows, cols, row_stride, square, data, scales, data_t, scales_t,
                           (hipStream_t)stream);
}
