// feed_forward_plain.cu -- the feed-forward block's products that the other kernels do
// not take (geo/geo_b200.h section 5): few rows of any type, and 16-bit arrays that do
// not start on 16 bytes; the joining of sums over parts of K; copies of 16-bit rows to
// where the tensor cores' copies can start.
#include "feed_forward.h"
#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

// ---- tiles in registers -----------------------------------------------------------

// For 16-bit arrays of any alignment, value by value and simple: C = A B, 256 threads a
// tile, TM x TN float32 sums a thread in groups of 16 bytes along each side; 16 of K at a
// time through shared memory, the next 16 on their way in registers meanwhile.
constexpr int kSide = 16, kBK = 16, kTileThreads = kSide * kSide;

template <int KIND>
constexpr int rows_of_thread() {
    return 8;
}
template <int KIND>
constexpr int columns_of_thread() {
    return KIND == kGated ? 4 : 8;
}

template <typename T, typename O, int KIND>
__global__ void __launch_bounds__(kTileThreads)
    tile_kernel(const __grid_constant__ Product p, int down, int across, int tiles) {
    using W = Wide<T>;
    constexpr bool kAMn = KIND == kWeights, kBMn = KIND == kHidden || KIND == kInput || KIND == kWeights;
    constexpr int TM = rows_of_thread<KIND>(), TN = columns_of_thread<KIND>(), V = 16 / (int)sizeof(W);
    constexpr int BM = kSide * TM, BN = kSide * TN, kOperands = KIND == kGated ? 2 : 1;
    constexpr int kLoadA = BM * kBK / kTileThreads, kLoadB = BN * kBK / kTileThreads;
    constexpr int kPitchA = BM + V, kPitchB = BN + V;
    __shared__ __align__(16) W sa[kBK * kPitchA], sb[kOperands][kBK * kPitchB];
    const int ty = threadIdx.x / kSide, tx = threadIdx.x % kSide;
    const int blocks_k = (p.k + kBK - 1) / kBK;
    after_previous();
    let_next_start();

    for (int index = blockIdx.x; index < tiles; index += gridDim.x) {
        const int part = index / (down * across), rest = index % (down * across);
        const int problem = part / p.splits, split = part - problem * p.splits;
        const int all = (KIND == kInput ? 2 : 1) * blocks_k;
        const int first = (int)((long long)all * split / p.splits), last = (int)((long long)all * (split + 1) / p.splits);
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
                if (p.splits > 1) {
                    const size_t stride = partial_stride(p.n), each = (size_t)p.splits * p.m * stride;
                    W *to = (W *)p.partial + problem * each + ((size_t)split * p.m + row) * stride + col;
#pragma unroll
                    for (int o = 0; o < kOperands; ++o) to[o * each] = value(o);
                } else {
                    finish<T, O, KIND>(p, problem, row, col, value(0), value(kOperands - 1));
                }
            }
        }
    }
}

template <typename T, typename O, int KIND>
cudaError_t launch_tile(const Product &p, cudaStream_t stream) {
    using W = Wide<T>;
    constexpr int BM = kSide * rows_of_thread<KIND>(), BN = kSide * columns_of_thread<KIND>();
    const int down = (p.m + BM - 1) / BM, across = (p.n + BN - 1) / BN;
    const long long tiles = (long long)down * across * p.problems * p.splits;
    if (tiles > INT32_MAX) return cudaErrorInvalidValue;
    return launch_after(tile_kernel<T, O, KIND>, (unsigned)tiles, kTileThreads, 0, 1, stream, p, down, across, (int)tiles);
}

// ---- parts of K -----------------------------------------------------------------------

// Adds the parts of K up, four columns a thread, and does with the sums what the kernel
// that made them does where K is whole. LANES: that many threads share the parts of a
// place, each every so many in order, and add theirs up as a tree (three results of 256 x
// 64 float64 in 49 parts: 28 us by one thread each).
template <typename T, typename O, int KIND, int LANES>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Product p) {
    using W = Wide<T>;
    constexpr int kSums = KIND == kGated ? 2 : 1, V = 16 / (int)sizeof(W), kPlaces = 256 / LANES;
    after_previous();
    let_next_start();
    const size_t stride = partial_stride(p.n), groups = stride / 4, each = (size_t)p.m * groups;
    const size_t part = (size_t)p.m * stride, all = each * p.problems;
    // The threads of a place are neighbours in a warp; all of them go through the same rounds.
    const int lane = threadIdx.x % LANES;
    for (size_t first = (size_t)blockIdx.x * kPlaces; first < all; first += (size_t)gridDim.x * kPlaces) {
        const size_t i = first + threadIdx.x / LANES;
        const bool live = i < all;
        const int problem = live ? (int)(i / each) : 0;
        const size_t place = live ? i - problem * each : 0, row = place / groups, col = place % groups * 4;
        W sum[kSums][4];
#pragma unroll
        for (int z = 0; z < kSums; ++z) {
            const W *from = (const W *)p.partial + (size_t)(KIND == kWeights ? problem : z) * p.splits * part + row * stride + col;
#pragma unroll
            for (int j = 0; j < 4; ++j) sum[z][j] = W(0);
#pragma unroll 4
            for (int s = lane; s < p.splits; s += LANES)
#pragma unroll
                for (int v = 0; v < 4 / V; ++v) {
                    const Vec<W, V> piece = load<W, V>(from + s * part + v * V);
#pragma unroll
                    for (int q = 0; q < V / 2; ++q) {
                        sum[z][v * V + 2 * q] += piece.pair(q).x;
                        sum[z][v * V + 2 * q + 1] += piece.pair(q).y;
                    }
                }
#pragma unroll
            for (int o = LANES / 2; o > 0; o /= 2)
#pragma unroll
                for (int j = 0; j < 4; ++j) sum[z][j] += __shfl_xor_sync(0xffffffffu, sum[z][j], o);
        }
        const int held = !live || lane != 0 ? 0 : ((size_t)p.n - col < 4 ? (int)((size_t)p.n - col) : 4);
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (j < held) finish<T, O, KIND>(p, problem, row, col + j, sum[0][j], sum[kSums - 1][j]);
    }
}

// ---- few rows -----------------------------------------------------------------------

// A token or a few: every weight is read once and that is all the time it takes. A
// column of the result (kGated: of gate and up) is `split` warps' work, each along its
// part of K, vectors of 16 bytes side by side; a lane has kBatch of them on their way,
// past L1, which is left to the rows of x. `split` grows until
// there are warps enough to keep HBM busy. kDown's weights are asked for before the
// kernel that makes its rows has ended: whatever wrote them had ended before that one
// read anything, and L1 is not asked.
constexpr int kFewThreads = 256, kFewWarps = kFewThreads / 32;

// Volatile: all of a batch before anything waits for one. EARLY: before the kernel before
// this one has ended; L1, which might hold what was there before, is passed by. (Later
// loads only do not stay in it: .cg for all of them takes 64 us for one token of 4096 x
// 12288 bfloat16, 58 so.)
template <bool EARLY, typename T, int V>
__device__ __forceinline__ Vec<T, V> load_once(const T *p) {
    Vec<T, V> r;
    if constexpr (Vec<T, V>::kBytes == 16 && EARLY) {
        asm volatile("ld.global.cg.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                     : "l"(p));
    } else if constexpr (Vec<T, V>::kBytes == 16) {
        asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
                     : "=r"(r.w[0]), "=r"(r.w[1]), "=r"(r.w[2]), "=r"(r.w[3])
                     : "l"(p));
    } else if constexpr (Vec<T, V>::kBytes == 8) {
        const uint2 v = __ldcg(reinterpret_cast<const uint2 *>(p));
        r.w[0] = v.x, r.w[1] = v.y;
    } else if constexpr (Vec<T, V>::kBytes == 4) {
        r.w[0] = __ldcg(reinterpret_cast<const uint32_t *>(p));
    } else {
        r.w[0] = __ldcg(reinterpret_cast<const unsigned short *>(p));
    }
    return r;
}

template <typename T, int KIND, int ROWS, bool ALIGNED>
__global__ void __launch_bounds__(kFewThreads) few_kernel(const __grid_constant__ Product p, int split) {
    using W = Wide<T>;
    // Several rows: as many columns a warp as make four streams of weights, which share what is read of the rows.
    constexpr int kOperands = KIND == kGated ? 2 : 1, kColumns = ROWS == 1 ? 1 : 4 / kOperands;
    constexpr int kStreams = kOperands * kColumns, V = ALIGNED ? 16 / (int)sizeof(T) : 1, kBatch = 8 / kStreams;
    // Up to two rows: the next vector as soon as one is used; more: a batch at a time (4096 x 12288 bfloat16, 2 rows 69
    // and 79 us; 2048 x 4096 float64, 4 rows 72 and 66).
    constexpr bool kRoll = ROWS <= 2;
    __shared__ W parts[kFewWarps][kStreams * ROWS];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int part = warp % split, columns = kFewWarps / split * kColumns;  // of the block
    const int col = (int)blockIdx.x * columns + warp / split * kColumns;
    W sum[kStreams][ROWS];
#pragma unroll
    for (int o = 0; o < kStreams; ++o)
#pragma unroll
        for (int r = 0; r < ROWS; ++r) sum[o][r] = W(0);
    const T *x = (const T *)p.a[0].p, *w[kStreams];
#pragma unroll
    for (int o = 0; o < kStreams; ++o) {
        const int c = col + o / kOperands;
        w[o] = (const T *)p.b[o % kOperands].p + (size_t)(c < p.n ? c : 0) * p.b[o % kOperands].stride;
    }
    const int step = 32 * V * split, first = (part * 32 + lane) * V, last = col < p.n ? p.k : 0;
    Vec<T, V> piece[kBatch][kStreams];
    auto ask = [&](auto early, int i, int k) {
#pragma unroll
        for (int o = 0; o < kStreams; ++o)
            piece[i][o] = k < last ? load_once<decltype(early)::value, T, V>(w[o] + k) : Vec<T, V>::zero();
    };
    if (KIND == kGated) after_previous();
#pragma unroll
    for (int i = 0; i < kBatch; ++i) ask(std::bool_constant<KIND == kDown>{}, i, first + i * step);
    if (KIND == kDown) after_previous();
    let_next_start();
    for (int k = first; k < last; k += kBatch * step) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (k + i * step >= last) break;
#pragma unroll
            for (int r = 0; r < ROWS; ++r) {
                if (r >= p.m) break;
                const Vec<T, V> xs = load<T, V>(x + (size_t)r * p.a[0].stride + k + i * step);
#pragma unroll
                for (int o = 0; o < kStreams; ++o) {
                    if constexpr (V == 1) {
                        sum[o][r] += xs.one() * piece[i][o].one();
                    } else {
                        Pair<W> two = both(W(0));
#pragma unroll
                        for (int q = 0; q < V / 2; ++q) two = fma(xs.pair(q), piece[i][o].pair(q), two);
                        sum[o][r] += two.x + two.y;
                    }
                }
            }
            if constexpr (kRoll) ask(std::false_type{}, i, k + (i + kBatch) * step);
        }
        if constexpr (!kRoll)
            if (k + kBatch * step < last) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) ask(std::false_type{}, i, k + (i + kBatch) * step);
            }
    }
#pragma unroll
    for (int o = 0; o < kStreams; ++o)
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
        for (int s = 0; s < split; ++s)
            total[o] += parts[c / kColumns * split + s][(c % kColumns * kOperands + o) * ROWS + row];
    }
    finish<T, T, KIND>(p, 0, row, (size_t)blockIdx.x * columns + c, total[0], total[kOperands - 1]);
}

template <typename T, int KIND, int ROWS>
cudaError_t launch_rows(const Product &p, cudaStream_t stream) {
    bool aligned = p.k % (16 / sizeof(T)) == 0;
    auto look = [&](const Matrix &x, int rows) {
        aligned = aligned && (uintptr_t)x.p % 16 == 0 && (rows == 1 || x.stride * sizeof(T) % 16 == 0);
    };
    look(p.a[0], p.m);
    for (int o = 0; o < (KIND == kGated ? 2 : 1); ++o) look(p.b[o], p.n);
    constexpr int kColumns = ROWS == 1 ? 1 : (KIND == kGated ? 2 : 4);
    int split = 1;
    const long long wanted = (long long)geo::device_sm_count() * 32;  // warps
    while (split < kFewWarps && (long long)p.n * split < wanted * kColumns && p.k > split * 512) split *= 2;
    const int columns = kFewWarps / split * kColumns;
    const unsigned grid = (unsigned)((p.n + columns - 1) / columns);
    return aligned ? launch_after(few_kernel<T, KIND, ROWS, true>, grid, kFewThreads, 0, 1, stream, p, split)
                   : launch_after(few_kernel<T, KIND, ROWS, false>, grid, kFewThreads, 0, 1, stream, p, split);
}

template <typename T, int KIND>
cudaError_t launch_few(const Product &p, cudaStream_t stream) {
    if (p.m == 1) return launch_rows<T, KIND, 1>(p, stream);
    if (p.m == 2) return launch_rows<T, KIND, 2>(p, stream);
    if (p.m <= 4) return launch_rows<T, KIND, 4>(p, stream);
    return launch_rows<T, KIND, kFewRows>(p, stream);
}

// ---- rows that start on 16 bytes -----------------------------------------------------

__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Pack pack) {
    after_previous();
    let_next_start();
    const size_t n = pack.arrays[pack.count - 1].end;
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (size_t)gridDim.x * blockDim.x) {
        int which = 0;
        while (i >= pack.arrays[which].end) ++which;
        const Pack::Array &a = pack.arrays[which];
        const size_t piece = i - (which > 0 ? pack.arrays[which - 1].end : 0), pieces = a.to_stride / 8;
        const size_t row = piece / pieces;
        const int col = (int)(piece - row * pieces) * 8;
        const unsigned short *x = (const unsigned short *)a.from.p + row * a.from.stride + col;
        uint32_t w[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t low = col + 2 * q < a.cols ? x[2 * q] : 0, high = col + 2 * q + 1 < a.cols ? x[2 * q + 1] : 0;
            w[q] = low | high << 16;
        }
        ((uint4 *)a.to)[piece] = make_uint4(w[0], w[1], w[2], w[3]);
    }
}

}  // namespace

// As many parts as give every multiprocessor a tile, none under 128 of K.
Cut cut_plain(ProductKind kind, size_t m, size_t n, size_t k) {
    const size_t high = kSide * rows_of_thread<kDown>();
    const size_t wide = kSide * (kind == kGated ? columns_of_thread<kGated>() : columns_of_thread<kDown>());
    const size_t tiles = (kind == kWeights ? 3 : 1) * ((m + high - 1) / high) * ((n + wide - 1) / wide);
    const size_t wanted = (size_t)geo::device_sm_count() / tiles, most = k * (kind == kInput ? 2 : 1) / 128;
    const size_t splits = wanted < most ? wanted : most;
    return {(int)wide, false, splits < 1 ? 1 : (splits < 64 ? (int)splits : 64)};
}

template <typename T, typename O, int KIND>
cudaError_t launch_join_kind(const Product &p, cudaStream_t stream) {
    const size_t n = (size_t)p.m * (partial_stride(p.n) / 4) * p.problems, most = (size_t)geo::device_sm_count() * 8;
    // Threads that share a place where there are parts for them and threads to spare.
    const bool share = p.splits >= 16 && n * 8 <= most * 256;
    const size_t blocks = (n * (share ? 8 : 1) + 255) / 256;
    const unsigned grid = (unsigned)(blocks < most ? blocks : most);
    return share ? launch_after(join_kernel<T, O, KIND, 8>, grid, 256, 0, 1, stream, p)
                 : launch_after(join_kernel<T, O, KIND, 1>, grid, 256, 0, 1, stream, p);
}
cudaError_t launch_join(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p, cudaStream_t stream) {
    return by_type(type, [&](auto t) -> cudaError_t {
        using T = decltype(t);
        switch (kind) {
            case kGated: return launch_join_kind<T, T, kGated>(p, stream);
            case kDown: return launch_join_kind<T, T, kDown>(p, stream);
            case kHidden: return launch_join_kind<T, T, kHidden>(p, stream);
            case kInput: return launch_join_kind<T, T, kInput>(p, stream);
            default: break;
        }
        if constexpr (sizeof(T) == 2) {
            if (out_type == GEO_B200_F32) return launch_join_kind<T, float, kWeights>(p, stream);
        }
        return launch_join_kind<T, T, kWeights>(p, stream);
    });
}

cudaError_t launch_product_plain(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p,
                                 cudaStream_t stream) {
    auto launch = [&](auto t) -> cudaError_t {
        using T = decltype(t);
        switch (kind) {
            case kGated: return launch_tile<T, T, kGated>(p, stream);
            case kDown: return launch_tile<T, T, kDown>(p, stream);
            case kHidden: return launch_tile<T, T, kHidden>(p, stream);
            case kInput: return launch_tile<T, T, kInput>(p, stream);
            default: break;
        }
        return out_type == GEO_B200_F32 ? launch_tile<T, float, kWeights>(p, stream) : launch_tile<T, T, kWeights>(p, stream);
    };
    const cudaError_t e = type == GEO_B200_BF16 ? launch(__nv_bfloat16{}) : launch(__half{});
    return e != cudaSuccess || p.splits == 1 ? e : launch_join(kind, type, out_type, p, stream);
}

cudaError_t launch_product_few(ProductKind kind, uint32_t type, const Product &p, cudaStream_t stream) {
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        return kind == kGated ? launch_few<T, kGated>(p, stream) : launch_few<T, kDown>(p, stream);
    });
}

cudaError_t launch_pack(const Pack &pack, cudaStream_t stream) {
    if (pack.count == 0) return cudaSuccess;
    const size_t blocks = (pack.arrays[pack.count - 1].end + 255) / 256, most = (size_t)geo::device_sm_count() * 32;
    return launch_after(pack_kernel, (unsigned)(blocks < most ? blocks : most), 256, 0, 1, stream, pack);
}

}  // namespace layers
}  // namespace geo
