// dropout.cu -- dropout with a mask computed from a counter, and its VJP
// (geo/geo_b200.h section 5).
//
// y = [residual +] keep x / (1 - rate): one multiply-add a value and an eighth of a
// Philox block (forty instructions), so HBM bounds it as long as a block is worked
// out once for its eight values. Measured on two boards, calls in turn over three sets
// of arrays, host included: 8192^2 bfloat16 with a residual 62 and 66 us (6.1 TB/s, 94%
// of the copy bandwidth on the slower one), 2^18 x 64 float64 by whole multivectors 44
// and 45 us (6.0 TB/s, 92%); 8192 x 2001 bfloat16 with a residual, rows off 16 bytes,
// 34 us (2.9 TB/s: 420 instructions for eight values, on 72% of the issue slots).
#include "geo_runtime.h"
#include "layers.h"

namespace {

using namespace geo::layers;

constexpr int kThreads = 256;

struct Rows {
    const void *x, *residual;
    void *y;
    size_t x_stride, residual_stride, y_stride;
    size_t rows, cols;  // packed arrays: one row of all values
};

template <typename T>
__device__ __forceinline__ Wide<T> drop_value(bool kept, T x, Wide<T> scale, Wide<T> residual) {
    using W = Wide<T>;
    const W v = kept ? (W)widen(x) : W(0);  // selected, not multiplied: a dropped NaN is gone
    if constexpr (std::is_same_v<W, double>)
        return ::fma(v, scale, residual);
    else
        return fmaf(v, scale, residual);
}

// Vectors of 16 bytes. A warp takes 256 values at a time, kChunks times: lane l
// works out the block of values 8 l .. 8 l + 7, once for every eight values at
// every type, and the eight decisions go to the lanes that hold the values.
constexpr int kChunks = 4;
template <typename T, bool PACKED, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads) drop_vectors_kernel(const Rows a, const Drop drop) {
    using W = Wide<T>;
    constexpr int V = 16 / sizeof(T), R = 8 / V;
    const uint64_t offset = drop_offset(drop);
    const W scale = (W)drop.scale;
    const uint32_t lane = threadIdx.x & 31;
    const size_t count = a.rows * a.cols;
    const size_t warp = (blockIdx.x * (size_t)kThreads + threadIdx.x) / 32;
    Vec<T, V> x[kChunks][R], res[RESIDUAL ? kChunks : 1][R];
    size_t y_at[PACKED ? 1 : kChunks][R];
    auto value = [&](int m, int i) { return (warp * kChunks + m) * 256 + (i * 32 + lane) * V; };
#pragma unroll
    for (int m = 0; m < kChunks; ++m)
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const size_t e = value(m, i);
            x[m][i] = Vec<T, V>::zero();
            if constexpr (RESIDUAL) res[m][i] = Vec<T, V>::zero();
            if (e >= count) continue;
            if constexpr (PACKED) {
                if (e + V <= count) {
                    x[m][i] = load<T, V>((const T *)a.x + e);
                    if constexpr (RESIDUAL) res[m][i] = load<T, V>((const T *)a.residual + e);
                }
            } else {
                const size_t row = count <= 0xFFFFFFFFu ? (uint32_t)e / (uint32_t)a.cols : e / a.cols;
                const size_t c = e - row * a.cols;
                y_at[m][i] = row * a.y_stride + c;
                x[m][i] = load<T, V>((const T *)a.x + row * a.x_stride + c);
                if constexpr (RESIDUAL) res[m][i] = load<T, V>((const T *)a.residual + row * a.residual_stride + c);
            }
        }
#pragma unroll
    for (int m = 0; m < kChunks; ++m) {
        // 16-bit values: the eight of the vector. Wider ones: a block's decisions, handed round.
        uint32_t draws[4] = {}, mine = 0xFFu;
        if (drop.threshold != 0) {
            const size_t eight = (warp * kChunks + m) * 256 + lane * 8;
            if constexpr (R == 1)
                draws_of_pairs<8>(drop, offset, eight, draws);
            else
                mine = kept_of_eight(drop, offset, eight);
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const size_t e = value(m, i);
            uint32_t kept = mine;
            if constexpr (R > 1) kept = __shfl_sync(0xffffffffu, mine, (i * 32 + lane) / R) >> (lane % R * V);
            Vec<T, V> out;
#pragma unroll
            for (int q = 0; q < V / 2; ++q) {
                Pair<W> v = x[m][i].pair(q);
                if constexpr (R == 1) {
                    if (drop.threshold != 0) v = drop_pair(v, draws[q], drop.bound);
                } else {
                    v.x = (kept >> (2 * q)) & 1 ? v.x : W(0);
                    v.y = (kept >> (2 * q + 1)) & 1 ? v.y : W(0);
                }
                if constexpr (RESIDUAL)
                    v = fma(v, both(scale), res[m][i].pair(q));
                else
                    v = v * both(scale);
                out.set(q, v);
            }
            if (e >= count) continue;
            if constexpr (PACKED) {
                if (e + V <= count) {
                    store<T, V>((T *)a.y + e, out);
                } else {  // the last values of all, one by one
                    for (int j = 0; e + j < count; ++j) {
                        const W residual = RESIDUAL ? (W)widen(((const T *)a.residual)[e + j]) : W(0);
                        const bool live = drop.threshold == 0 || unit_kept(drop, offset, (e + j) >> drop.shift);
                        ((T *)a.y)[e + j] = narrow<T>(drop_value<T>(live, ((const T *)a.x)[e + j], scale, residual));
                    }
                }
            } else {
                store<T, V>((T *)a.y + y_at[m][i], out);
            }
        }
    }
}

// 16-bit rows that do not start on 16 bytes, or are not made of whole eights:
// `lanes` lanes (a power of two) put together lanes - 1 aligned chunks of eight
// values of y. Each loads the aligned chunk of x (and of the residual) in which
// its values start and takes the rest from its neighbour's; so it does with the
// draws, whose blocks lie as they like too. The last lane only lends. Chunks that
// reach over a row's ends are written, and those over the array's ends read,
// value by value.
template <typename T>
__device__ __forceinline__ Vec<T, 8> shifted(const Vec<T, 8> &low, const Vec<T, 8> &high, uint32_t values) {
    uint32_t w[8] = {low.w[0], low.w[1], low.w[2], low.w[3], high.w[0], high.w[1], high.w[2], high.w[3]};
#pragma unroll
    for (int k = 0; k < 6; ++k) w[k] = (values & 4) ? w[k + 2] : w[k];
#pragma unroll
    for (int k = 0; k < 5; ++k) w[k] = (values & 2) ? w[k + 1] : w[k];
    Vec<T, 8> r;
#pragma unroll
    for (int k = 0; k < 4; ++k) r.w[k] = __funnelshift_r(w[k], w[k + 1], (values & 1) * 16);
    return r;
}
template <typename T>
__device__ __forceinline__ Vec<T, 8> load_chunk(const T *base, const T *whole_end, const T *start, int cols, int column) {
    const int shift = (int)((((uintptr_t)start >> 1) + column) & 7), first = column - shift;
    Vec<T, 8> own = Vec<T, 8>::zero();
    if (first + 8 > 0 && first < cols) {
        const T *from = start + first;
        if ((first >= 0 && first + 8 <= cols) || (from >= base && from + 8 <= whole_end)) {
            own = load<T, 8>(from);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (first + j >= 0 && first + j < cols)
                    own.w[j / 2] |= (uint32_t) * (const unsigned short *)(from + j) << (j % 2 * 16);
        }
    }
    return own;
}
template <typename T>
__device__ __forceinline__ Vec<T, 8> join_chunk(const Vec<T, 8> &own, const T *start, int column) {
    Vec<T, 8> next;
#pragma unroll
    for (int k = 0; k < 4; ++k) next.w[k] = __shfl_down_sync(0xffffffffu, own.w[k], 1);
    return shifted(own, next, (uint32_t)((((uintptr_t)start >> 1) + column) & 7));
}
template <typename T, bool RESIDUAL>
__global__ void __launch_bounds__(kThreads) drop_chunks_kernel(const Rows a, const Drop drop, uint32_t lane_bits, uint32_t pieces) {
    const uint64_t offset = drop_offset(drop);
    const float scale = (float)drop.scale;
    const uint32_t lanes = 1u << lane_bits, lane = threadIdx.x & (lanes - 1);
    const int cols = (int)a.cols;
    const size_t count = a.rows * pieces, step = (size_t)gridDim.x * (kThreads >> lane_bits);
    const T *x_end = (const T *)a.x + (a.rows - 1) * a.x_stride + cols;
    const T *residual_end = (const T *)a.residual + (a.rows - 1) * a.residual_stride + cols;
    // A piece's row and first column, and its chunks, on their way while the piece before is worked on.
    struct Piece {
        size_t row;
        int c;
        Vec<T, 8> x, residual;
    };
    auto fetch = [&](size_t first) {
        const size_t piece = first + ((threadIdx.x & 31) >> lane_bits);
        const bool live = piece < count;
        Piece p;
        p.row = live ? piece : 0;
        if (pieces > 1) p.row = count <= 0xFFFFFFFFu ? (uint32_t)p.row / pieces : p.row / pieces;
        const int back = (int)((uintptr_t)((T *)a.y + p.row * a.y_stride) >> 1 & 7);
        p.c = live ? (int)((uint32_t)(piece - p.row * pieces) * (lanes - 1) + lane) * 8 - back : cols;
        p.x = load_chunk((const T *)a.x, x_end, (const T *)a.x + p.row * a.x_stride, cols, p.c);
        if constexpr (RESIDUAL)
            p.residual = load_chunk((const T *)a.residual, residual_end,
                                    (const T *)a.residual + p.row * a.residual_stride, cols, p.c);
        return p;
    };
    // The bound is the warp's first piece, so that all its lanes stay for the shuffles.
    const size_t begin = blockIdx.x * (size_t)(kThreads >> lane_bits) + (threadIdx.x >> 5 << (5 - lane_bits));
    Piece next = fetch(begin);
    for (size_t first = begin; first < count; first += step) {
        const Piece p = next;
        if (first + step < count) next = fetch(first + step);
        const size_t row = p.row;
        const int c = p.c;
        T *y = (T *)a.y + row * a.y_stride;
        const Vec<T, 8> x = join_chunk(p.x, (const T *)a.x + row * a.x_stride, c);
        Vec<T, 8> residual = x;
        if constexpr (RESIDUAL) residual = join_chunk(p.residual, (const T *)a.residual + row * a.residual_stride, c);
        const uint64_t e = row * (uint64_t)cols + (int64_t)c;
        const uint32_t mine = kept_of_eight(drop, offset, e & ~(uint64_t)7);
        const uint32_t kept = (mine | __shfl_down_sync(0xffffffffu, mine, 1) << 8) >> ((uint32_t)e & 7u);
        Vec<T, 8> out;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            Pair<float> v = x.pair(q);
            v.x = (kept >> (2 * q)) & 1 ? v.x : 0.0f;
            v.y = (kept >> (2 * q + 1)) & 1 ? v.y : 0.0f;
            out.set(q, RESIDUAL ? fma(v, both(scale), residual.pair(q)) : v * both(scale));
        }
        if (lane == lanes - 1 || c >= cols || c + 8 <= 0) continue;
        if (c >= 0 && c + 8 <= cols) {
            store<T, 8>(y + c, out);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (c + j >= 0 && c + j < cols)
                    *(unsigned short *)(y + c + j) = (unsigned short)(out.w[j / 2] >> (j % 2 * 16));
        }
    }
}

// Wider values off 16 bytes: a warp takes 256 values of one row, lane by lane.
template <typename T>
__global__ void __launch_bounds__(kThreads) drop_values_kernel(const Rows a, const Drop drop) {
    using W = Wide<T>;
    const uint64_t offset = drop_offset(drop);
    const W scale = (W)drop.scale;
    const uint32_t lane = threadIdx.x & 31;
    const size_t pieces = (a.cols + 255) / 256, count = a.rows * pieces;
    const size_t step = (size_t)gridDim.x * (kThreads / 32);
    for (size_t piece = (blockIdx.x * (size_t)kThreads + threadIdx.x) / 32; piece < count; piece += step) {
        const size_t row = piece / pieces, first = (piece - row * pieces) * 256;
        const T *x = (const T *)a.x + row * a.x_stride;
        const T *residual = a.residual != nullptr ? (const T *)a.residual + row * a.residual_stride : nullptr;
        T v[8], r[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t c = first + i * 32 + lane;
            v[i] = c < a.cols ? x[c] : T{};
            r[i] = residual != nullptr && c < a.cols ? residual[c] : T{};
        }
        const uint32_t kept = kept_by_warp<8>(drop, offset, row * a.cols + first, 32);
        T *y = (T *)a.y + row * a.y_stride;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const size_t c = first + i * 32 + lane;
            if (c < a.cols) y[c] = narrow<T>(drop_value<T>((kept >> i) & 1, v[i], scale, widen(r[i])));
        }
    }
}

cudaError_t launch(uint32_t type, const void *x, size_t x_stride, const void *residual, size_t residual_stride,
                   void *y, size_t y_stride, size_t rows, size_t cols, const Drop &drop, cudaStream_t stream) {
    Rows a = {x, residual, y, x_stride, residual_stride, y_stride, rows, cols};
    const bool packed = x_stride == cols && y_stride == cols && (residual == nullptr || residual_stride == cols);
    if (packed) a.cols = rows * cols, a.rows = 1;
    const size_t b = type_bytes(type), low = (uintptr_t)x | (uintptr_t)y | (uintptr_t)residual;
    const size_t strides = x_stride | y_stride | (residual != nullptr ? residual_stride : 0);
    const bool vectors = low % 16 == 0 && (packed || (cols % 8 == 0 && strides * b % 16 == 0));
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        if (vectors) {
            const size_t each = (size_t)kThreads * 8 * kChunks;
            const size_t grid = (rows * cols + each - 1) / each;
            if (grid > 0x7fffffff) return cudaErrorInvalidValue;
            if (packed && residual != nullptr)
                drop_vectors_kernel<T, true, true><<<(unsigned)grid, kThreads, 0, stream>>>(a, drop);
            else if (packed)
                drop_vectors_kernel<T, true, false><<<(unsigned)grid, kThreads, 0, stream>>>(a, drop);
            else if (residual != nullptr)
                drop_vectors_kernel<T, false, true><<<(unsigned)grid, kThreads, 0, stream>>>(a, drop);
            else
                drop_vectors_kernel<T, false, false><<<(unsigned)grid, kThreads, 0, stream>>>(a, drop);
        } else if constexpr (sizeof(T) == 2) {
            a.rows = rows, a.cols = cols;  // row by row, packed or not: a row's columns fit 32 bits
            uint32_t lane_bits = 1;
            while (lane_bits < 5 && (1u << lane_bits) - 1 < (cols + 14) / 8) ++lane_bits;
            const uint32_t whole = (1u << lane_bits) - 1, pieces = ((uint32_t)(cols + 14) / 8 + whole - 1) / whole;
            const size_t each = kThreads >> lane_bits, blocks = (rows * pieces + each - 1) / each;
            const size_t most = (size_t)geo::device_sm_count() * 12;  // twice the resident ones
            const unsigned grid = (unsigned)(blocks < most ? blocks : most);
            if (residual != nullptr)
                drop_chunks_kernel<T, true><<<grid, kThreads, 0, stream>>>(a, drop, lane_bits, pieces);
            else
                drop_chunks_kernel<T, false><<<grid, kThreads, 0, stream>>>(a, drop, lane_bits, pieces);
        } else {
            const size_t pieces = a.rows * ((a.cols + 255) / 256), blocks = (pieces + kThreads / 32 - 1) / (kThreads / 32);
            drop_values_kernel<T><<<(unsigned)(blocks < 0x7fffffff ? blocks : 0x7fffffff), kThreads, 0, stream>>>(a, drop);
        }
        return cudaGetLastError();
    });
}

}  // namespace

extern "C" geo_b200_status_t geo_b200_dropout(const geo_b200_dropout_config_t *config, const void *device_x,
                                              const void *device_residual, const uint64_t *device_offset,
                                              void *device_y, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.dropout");
    Drop drop;
    if (config == nullptr || device_x == nullptr || device_y == nullptr || !make_drop(*config, device_offset, &drop))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_dropout_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.residual_stride, &c.y_stride}) ||
        !same_or_apart(device_y, c.y_stride, device_x, c.x_stride) ||
        !same_or_apart(device_y, c.y_stride, device_residual, c.residual_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_residual, b}, {device_y, b}, {device_offset, 8}}))
        return GEO_B200_INVALID_ARGUMENT;
    return status_of(launch(c.type, device_x, c.x_stride, device_residual, c.residual_stride, device_y, c.y_stride,
                            c.rows, c.cols, drop, stream));
}

extern "C" geo_b200_status_t geo_b200_dropout_vjp(const geo_b200_dropout_config_t *config,
                                                  const uint64_t *device_offset, const void *device_y_cotangent,
                                                  void *device_x_cotangent, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.dropout_vjp");
    Drop drop;
    if (config == nullptr || device_y_cotangent == nullptr || device_x_cotangent == nullptr ||
        !make_drop(*config, device_offset, &drop))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_dropout_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.y_cotangent_stride, &c.x_cotangent_stride}) ||
        !same_or_apart(device_x_cotangent, c.x_cotangent_stride, device_y_cotangent, c.y_cotangent_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type);
    if (!arrays_usable({{device_y_cotangent, b}, {device_x_cotangent, b}, {device_offset, 8}}))
        return GEO_B200_INVALID_ARGUMENT;
    return status_of(launch(c.type, device_y_cotangent, c.y_cotangent_stride, nullptr, 0, device_x_cotangent,
                            c.x_cotangent_stride, c.rows, c.cols, drop, stream));
}
