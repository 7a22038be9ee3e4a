// feed_forward_plain.cu -- the feed-forward block's products that the tensor-core
// kernels do not take (geo/geo_b200.h section 5): float32 and float64, 16-bit arrays
// that do not start on 16 bytes, and few rows of any type.
#include "feed_forward.h"
#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

// ---- tiles in registers -----------------------------------------------------------

// C = A B, 256 threads a tile, TM x TN sums a thread in groups of 16 bytes along
// each side; 16 of K at a time through shared memory, the next 16 on their way in
// registers meanwhile. Multiply-adds bound it: float32 on the packed two-wide units.
constexpr int kSide = 16, kBK = 16, kTileThreads = kSide * kSide;

template <typename W, int KIND>
constexpr int rows_of_thread() {
    return sizeof(W) == 8 && KIND == kGated ? 4 : 8;
}
template <typename W, int KIND>
constexpr int columns_of_thread() {
    return sizeof(W) == 8 || KIND == kGated ? 4 : 8;
}

template <typename T, typename O, int KIND>
__global__ void __launch_bounds__(kTileThreads)
    tile_kernel(const __grid_constant__ Product p, int down, int across, int tiles) {
    using W = Wide<T>;
    constexpr bool kAMn = KIND == kWeights, kBMn = KIND == kHidden || KIND == kInput || KIND == kWeights;
    constexpr int TM = rows_of_thread<W, KIND>(), TN = columns_of_thread<W, KIND>(), V = 16 / (int)sizeof(W);
    constexpr int BM = kSide * TM, BN = kSide * TN, kOperands = KIND == kGated ? 2 : 1;
    constexpr int kLoadA = BM * kBK / kTileThreads, kLoadB = BN * kBK / kTileThreads;
    constexpr int kPitchA = BM + V, kPitchB = BN + V;
    __shared__ __align__(16) W sa[kBK * kPitchA], sb[kOperands][kBK * kPitchB];
    const int ty = threadIdx.x / kSide, tx = threadIdx.x % kSide;
    const int blocks_k = (p.k + kBK - 1) / kBK;

    for (int index = blockIdx.x; index < tiles; index += gridDim.x) {
        const int part = index / (down * across), rest = index % (down * across);
        const int problem = KIND == kWeights ? part / p.splits : 0, split = KIND == kWeights ? part % p.splits : 0;
        const int first = (int)((long long)blocks_k * split / p.splits);
        const int last = KIND == kInput ? 2 * blocks_k : (int)((long long)blocks_k * (split + 1) / p.splits);
        const int row0 = rest % down * BM, col0 = rest / down * BN;
        Pair<W> sum[kOperands][TM][TN / 2];
#pragma unroll
        for (int o = 0; o < kOperands; ++o)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
                for (int j = 0; j < TN / 2; ++j) sum[o][i][j] = both(W(0));
        W next_a[kLoadA], next_b[kOperands][kLoadB];
        auto fetch = [&](int step) {
            const int second = KIND == kInput && step >= blocks_k ? 1 : 0, k0 = (step - second * blocks_k) * kBK;
            const Matrix &a = p.a[KIND == kWeights ? problem : second];
#pragma unroll
            for (int e = 0; e < kLoadA; ++e) {
                const int n = threadIdx.x + e * kTileThreads;
                const int k = k0 + (kAMn ? n / BM : n % kBK), m = row0 + (kAMn ? n % BM : n / kBK);
                const bool in = k < p.k && m < p.m;
                const size_t at = kAMn ? (size_t)k * a.stride + m : (size_t)m * a.stride + k;
                next_a[e] = in ? widen(((const T *)a.p)[at]) : W(0);
                if constexpr (KIND == kWeights && sizeof(O) > sizeof(T))
                    if (in) next_a[e] += widen(((const T *)p.low[problem].p)[at]);
            }
#pragma unroll
            for (int o = 0; o < kOperands; ++o) {
                const Matrix &b = p.b[KIND == kGated ? o : (KIND == kWeights ? problem : second)];
#pragma unroll
                for (int e = 0; e < kLoadB; ++e) {
                    const int n = threadIdx.x + e * kTileThreads;
                    const int k = k0 + (kBMn ? n / BN : n % kBK), c = col0 + (kBMn ? n % BN : n / kBK);
                    const bool in = k < p.k && c < p.n;
                    next_b[o][e] =
                        in ? widen(((const T *)b.p)[kBMn ? (size_t)k * b.stride + c : (size_t)c * b.stride + k]) : W(0);
                }
            }
        };
        fetch(first);
        for (int step = first; step < last; ++step) {
            __syncthreads();  // the tiles before have been read
#pragma unroll
            for (int e = 0; e < kLoadA; ++e) {
                const int n = threadIdx.x + e * kTileThreads;
                sa[(kAMn ? n / BM : n % kBK) * kPitchA + (kAMn ? n % BM : n / kBK)] = next_a[e];
            }
#pragma unroll
            for (int o = 0; o < kOperands; ++o)
#pragma unroll
                for (int e = 0; e < kLoadB; ++e) {
                    const int n = threadIdx.x + e * kTileThreads;
                    sb[o][(kBMn ? n / BN : n % kBK) * kPitchB + (kBMn ? n % BN : n / kBK)] = next_b[o][e];
                }
            __syncthreads();
            if (step + 1 < last) fetch(step + 1);
#pragma unroll
            for (int k = 0; k < kBK; ++k) {
                W a[TM];
#pragma unroll
                for (int i = 0; i < TM / V; ++i) {
                    const Vec<W, V> piece = load<W, V>(&sa[k * kPitchA + i * kSide * V + ty * V]);
#pragma unroll
                    for (int q = 0; q < V / 2; ++q) {
                        const Pair<W> v = piece.pair(q);
                        a[i * V + 2 * q] = v.x;
                        a[i * V + 2 * q + 1] = v.y;
                    }
                }
#pragma unroll
                for (int o = 0; o < kOperands; ++o) {
                    Pair<W> b[TN / 2];
#pragma unroll
                    for (int j = 0; j < TN / V; ++j) {
                        const Vec<W, V> piece = load<W, V>(&sb[o][k * kPitchB + j * kSide * V + tx * V]);
#pragma unroll
                        for (int q = 0; q < V / 2; ++q) b[j * V / 2 + q] = piece.pair(q);
                    }
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN / 2; ++j) sum[o][i][j] = fma(both(a[i]), b[j], sum[o][i][j]);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < TM; ++i) {
            const int row = row0 + i / V * kSide * V + ty * V + i % V;
            if (row >= p.m) continue;
#pragma unroll
            for (int j = 0; j < TN; ++j) {
                const int col = col0 + j / V * kSide * V + tx * V + j % V;
                if (col >= p.n) continue;
                auto value = [&](int o) { return j & 1 ? sum[o][i][j / 2].y : sum[o][i][j / 2].x; };
                auto put = [&](const OutMatrix &out, W v) {
                    if (out.p != nullptr) ((T *)out.p)[(size_t)row * out.stride + col] = narrow<T>(v);
                };
                const W v = value(0);
                if constexpr (KIND == kGated) {
                    const W u = value(kOperands - 1);
                    put(p.out[0], v);
                    put(p.out[1], u);
                    put(p.out[2], activation<sizeof(T) == 2>(p.activation, v, (W *)nullptr) * u);
                } else if constexpr (KIND == kHidden) {
                    const W g = widen(((const T *)p.saved[0].p)[(size_t)row * p.saved[0].stride + col]);
                    const W u = widen(((const T *)p.saved[1].p)[(size_t)row * p.saved[1].stride + col]);
                    W slope;
                    const W f = activation<sizeof(T) == 2>(p.activation, g, &slope);
                    auto put_two = [&](int n, W x) {
                        put(p.out[n], x);
                        if constexpr (sizeof(T) == 2) put(p.out_low[n], lost_to<T>(x));
                    };
                    put_two(0, v * u * slope);
                    put_two(1, v * f);
                    put_two(2, f * u);
                } else if constexpr (KIND == kWeights) {
                    const OutMatrix &out = p.out[problem];
                    if (p.splits > 1)
                        ((W *)p.partial)[((size_t)part * p.m + row) * (((size_t)p.n + 3) / 4 * 4) + col] = v;
                    else if (p.transposed[problem])
                        ((O *)out.p)[(size_t)col * out.stride + row] = narrow<O>((Wide<O>)v);
                    else
                        ((O *)out.p)[(size_t)row * out.stride + col] = narrow<O>((Wide<O>)v);
                } else {
                    put(p.out[0], v);
                }
            }
        }
    }
}

template <typename T, typename O, int KIND>
cudaError_t launch_tile(const Product &p, cudaStream_t stream) {
    using W = Wide<T>;
    constexpr int BM = kSide * rows_of_thread<W, KIND>(), BN = kSide * columns_of_thread<W, KIND>();
    const int down = (p.m + BM - 1) / BM, across = (p.n + BN - 1) / BN;
    const long long tiles = (long long)down * across * p.problems * p.splits;
    if (tiles > INT32_MAX) return cudaErrorInvalidValue;
    tile_kernel<T, O, KIND><<<(unsigned)tiles, kTileThreads, 0, stream>>>(p, down, across, (int)tiles);
    return cudaGetLastError();
}

// ---- parts of K -----------------------------------------------------------------------

template <typename W, typename O>
__global__ void __launch_bounds__(256) join_splits_kernel(const __grid_constant__ Product p, size_t stride) {
    const size_t each = (size_t)p.m * p.n;
    for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < each * p.problems; i += (size_t)gridDim.x * 256) {
        const int problem = (int)(i / each);
        const size_t row = (i - problem * each) / p.n, col = (i - problem * each) % p.n;
        const W *from = (const W *)p.partial + ((size_t)problem * p.splits * p.m + row) * stride + col;
        W sum = 0;
#pragma unroll 8
        for (int s = 0; s < p.splits; ++s) sum += from[(size_t)s * p.m * stride];
        const OutMatrix &out = p.out[problem];
        ((O *)out.p)[p.transposed[problem] ? col * out.stride + row : row * out.stride + col] = narrow<O>((Wide<O>)sum);
    }
}

// ---- few rows -----------------------------------------------------------------------

// A token or a few: every weight is read once and that is all the time it takes. A
// column of the result (kGated: of gate and up) is `split` warps' work, each along its
// part of K, vectors of 16 bytes side by side; the rows of x come from L1. `split`
// grows until there are warps enough to keep HBM busy.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;

template <typename T, int KIND, int ROWS, bool ALIGNED>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const __grid_constant__ Product p, int split) {
    using W = Wide<T>;
    constexpr int kOperands = KIND == kGated ? 2 : 1, V = ALIGNED ? 16 / (int)sizeof(T) : 1;
    __shared__ W parts[kFewWarps][kOperands * ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = warp % split, columns = kFewWarps / split;
    const int col = (int)blockIdx.x * columns + warp / split;
    W sum[kOperands][ROWS];
#pragma unroll
    for (int o = 0; o < kOperands; ++o)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) sum[o][r] = W(0);
    if (col < p.n) {
        const T *x = (const T *)p.a[0].p, *w[kOperands];
#pragma unroll
        for (int o = 0; o < kOperands; ++o) w[o] = (const T *)p.b[o].p + (size_t)col * p.b[o].stride;
        const int step = 32 * V * split;
#pragma unroll 4
        for (int k = (part * 32 + lane) * V; k < p.k; k += step) {
            if constexpr (ALIGNED) {
                Vec<T, V> piece[kOperands];
#pragma unroll
                for (int o = 0; o < kOperands; ++o) piece[o] = load<T, V>(w[o] + k);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    if (r >= p.m) break;
                    const Vec<T, V> xs = load<T, V>(x + (size_t)r * p.a[0].stride + k);
#pragma unroll
                    for (int o = 0; o < kOperands; ++o) {
                        Pair<W> two = both(W(0));
#pragma unroll
                        for (int q = 0; q < V / 2; ++q) two = fma(xs.pair(q), piece[o].pair(q), two);
                        sum[o][r] += two.x + two.y;
                    }
                }
            } else {
                W v[kOperands];
#pragma unroll
                for (int o = 0; o < kOperands; ++o) v[o] = widen(w[o][k]);
#pragma unroll
                for (int r = 0; r < ROWS; ++r) {
                    if (r >= p.m) break;
                    const W xs = widen(x[(size_t)r * p.a[0].stride + k]);
#pragma unroll
                    for (int o = 0; o < kOperands; ++o) sum[o][r] += xs * v[o];
                }
            }
        }
    }
#pragma unroll
    for (int o = 0; o < kOperands; ++o)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) {
            W v = sum[o][r];
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(0xffffffffu, v, d);
            if (lane == 0) parts[warp][o * ROWS + r] = v;
        }
    __syncthreads();
    const int t = threadIdx.x, row = t % ROWS, c = t / ROWS;
    if (c >= columns || row >= p.m || (int)blockIdx.x * columns + c >= p.n) return;
    W total[kOperands];
#pragma unroll
    for (int o = 0; o < kOperands; ++o) {
        total[o] = W(0);
        for (int s = 0; s < split; ++s) total[o] += parts[c * split + s][o * ROWS + row];
    }
    const size_t at = (size_t)blockIdx.x * columns + c;
    auto put = [&](const OutMatrix &out, W v) {
        if (out.p != nullptr) ((T *)out.p)[(size_t)row * out.stride + at] = narrow<T>(v);
    };
    if constexpr (KIND == kGated) {
        put(p.out[0], total[0]);
        put(p.out[1], total[kOperands - 1]);
        put(p.out[2], activation<sizeof(T) == 2>(p.activation, total[0], (W *)nullptr) * total[kOperands - 1]);
    } else {
        put(p.out[0], total[0]);
    }
}

template <typename T, int KIND, int ROWS>
cudaError_t launch_rows(const Product &p, cudaStream_t stream) {
    bool aligned = p.k % (16 / sizeof(T)) == 0;
    auto look = [&](const Matrix &x, int rows) {
        aligned = aligned && (uintptr_t)x.p % 16 == 0 && (rows == 1 || x.stride * sizeof(T) % 16 == 0);
    };
    look(p.a[0], p.m);
    for (int o = 0; o < (KIND == kGated ? 2 : 1); ++o) look(p.b[o], p.n);
    int split = 1;
    const long long wanted = (long long)geo::device_sm_count() * 32;  // warps
    while (split < kFewWarps && (long long)p.n * split < wanted && p.k > split * 512) split *= 2;
    const int columns = kFewWarps / split;
    const unsigned grid = (unsigned)((p.n + columns - 1) / columns);
    if (aligned)
        few_kernel<T, KIND, ROWS, true><<<grid, kFewThreads, 0, stream>>>(p, split);
    else
        few_kernel<T, KIND, ROWS, false><<<grid, kFewThreads, 0, stream>>>(p, split);
    return cudaGetLastError();
}

template <typename T, int KIND>
cudaError_t launch_few(const Product &p, cudaStream_t stream) {
    if (p.m == 1) return launch_rows<T, KIND, 1>(p, stream);
    if (p.m == 2) return launch_rows<T, KIND, 2>(p, stream);
    if (p.m <= 4) return launch_rows<T, KIND, 4>(p, stream);
    return launch_rows<T, KIND, kFewRows>(p, stream);
}

// ---- rows that start on 16 bytes -----------------------------------------------------

__global__ void __launch_bounds__(256) pack_kernel(Matrix from, size_t rows, int cols, void *to, size_t to_stride) {
    const size_t pieces = to_stride / 8, n = rows * pieces;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
        const size_t row = i / pieces;
        const int col = (int)(i - row * pieces) * 8;
        const unsigned short *x = (const unsigned short *)from.p + row * from.stride + col;
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t low = col + 2 * q < cols ? x[2 * q] : 0, high = col + 2 * q + 1 < cols ? x[2 * q + 1] : 0;
            w[q] = low | high << 16;
        }
        ((uint4 *)to)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

}  // namespace

int weight_splits(size_t m, size_t n, size_t k, int tile_m, int tile_n, size_t least) {
    const size_t tiles = 3 * ((m + tile_m - 1) / tile_m) * ((n + tile_n - 1) / tile_n), sms = geo::device_sm_count();
    const size_t wanted = sms / tiles, most = k / least;
    const size_t splits = wanted < most ? wanted : most;
    return splits < 1 ? 1 : (splits < (size_t)kSplitMost ? (int)splits : kSplitMost);
}
int weight_splits_plain(uint32_t type, size_t m, size_t n, size_t k) {
    return type == GEO_B200_F64 ? weight_splits(m, n, k, kSide * rows_of_thread<double, kWeights>(),
                                                kSide * columns_of_thread<double, kWeights>(), 128)
                                : weight_splits(m, n, k, kSide * rows_of_thread<float, kWeights>(),
                                                kSide * columns_of_thread<float, kWeights>(), 128);
}

cudaError_t launch_join_splits(uint32_t type, uint32_t out_type, const Product &p, cudaStream_t stream) {
    const size_t n = (size_t)p.m * p.n * p.problems, blocks = (n + 255) / 256, most = (size_t)geo::device_sm_count() * 8;
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        using W = Wide<T>;
        const size_t stride = partial_stride(p.n);
        if (sizeof(T) == 2 && out_type == GEO_B200_F32)
            join_splits_kernel<W, W><<<grid, 256, 0, stream>>>(p, stride);
        else
            join_splits_kernel<W, T><<<grid, 256, 0, stream>>>(p, stride);
        return cudaGetLastError();
    });
}

cudaError_t launch_product_plain(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p,
                                 cudaStream_t stream) {
    return by_type(type, [&](auto t) -> cudaError_t {
        using T = decltype(t);
        switch (kind) {
            case kGated: return launch_tile<T, T, kGated>(p, stream);
            case kDown: return launch_tile<T, T, kDown>(p, stream);
            case kHidden: return launch_tile<T, T, kHidden>(p, stream);
            case kInput: return launch_tile<T, T, kInput>(p, stream);
            default: break;
        }
        cudaError_t e;
        if constexpr (sizeof(T) == 2)
            e = out_type == GEO_B200_F32 ? launch_tile<T, float, kWeights>(p, stream) : launch_tile<T, T, kWeights>(p, stream);
        else
            e = launch_tile<T, T, kWeights>(p, stream);
        return e != cudaSuccess || p.splits == 1 ? e : launch_join_splits(type, out_type, p, stream);
    });
}

cudaError_t launch_product_few(ProductKind kind, uint32_t type, const Product &p, cudaStream_t stream) {
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        return kind == kGated ? launch_few<T, kGated>(p, stream) : launch_few<T, kDown>(p, stream);
    });
}

cudaError_t launch_pack_rows(const Matrix &from, size_t rows, size_t cols, void *to, size_t to_stride,
                             cudaStream_t stream) {
    const size_t n = rows * (to_stride / 8), blocks = (n + 255) / 256, most = (size_t)geo::device_sm_count() * 32;
    pack_kernel<<<(unsigned)(blocks < most ? blocks : most), 256, 0, stream>>>(from, rows, (int)cols, to, to_stride);
    return cudaGetLastError();
}

}  // namespace layers
}  // namespace geo
