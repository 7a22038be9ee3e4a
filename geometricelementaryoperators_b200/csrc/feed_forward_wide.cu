// feed_forward_wide.cu -- the feed-forward block's products of float32 and float64
// (geo/geo_b200.h section 5).
//
// C = A B over tiles of 128 rows (32 where there are no more than 64, whose time is the
// weights' and what is multiplied for nothing) by 64 (float64) or 128 (float32) columns,
// 256 threads a tile, 16 of K at a time through a ring of three or four stages that asynchronous
// copies fill (16 bytes each, 8 or 4 where rows are off 16 bytes; zeros past the ends).
// Multiply-adds bound both types. What they need from shared memory comes next, so each
// type's tiles are read in the way that takes the fewest bytes a multiply-add:
//   float64  the FP64 tensor cores (mma.sync m8n8k4, 32 x 32 a warp): 16 multiply-adds a
//            value read, where 8 x 4 sums a thread would give 2.7;
//   float32  8 x 8 sums a thread, packed two-wide: along K where both operands lie that
//            way (even and odd k apart, added at the end), along the columns otherwise.
// Operands lie in shared memory as they do outside, [row][K] or [K][row], rows padded so
// that a warp's reads fall on distinct banks. Measured: 1024 x 2048 x 4096 float64 VJP 3.8
// ms (27 TFLOP/s, the FP64 pipe three quarters busy; the plain form's library products
// 3.2 ms), 2048 x 2048 x 4096 float32 forward 2.65 ms (39 TFLOP/s; 1.9 ms).
#include "feed_forward.h"
#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

constexpr int kThreads = 256, kBK = 16;
constexpr int tile_rows(size_t m) { return m <= 64 ? 32 : 128; }
template <typename T>
constexpr int kBN = sizeof(T) == 8 ? 64 : 128;
template <typename T>
constexpr int kStages = sizeof(T) == 8 ? 3 : 4;
constexpr int kPitchK = kBK + 4;           // values of a row of K
constexpr int pitch_mn(int rows) { return rows + 4; }  // of a row along M or N
constexpr int held(int rows) {             // values of an operand's part of a stage, either way
    return rows * kPitchK > kBK * pitch_mn(rows) ? rows * kPitchK : kBK * pitch_mn(rows);
}
// The ring, or the tile of sums that is left there at the end.
template <typename T, int BM>
constexpr size_t kShared =
    ((size_t)kStages<T> * (held(BM) + held(kBN<T>)) > (size_t)BM * (kBN<T> + 1)
         ? (size_t)kStages<T> * (held(BM) + held(kBN<T>))
         : (size_t)BM * (kBN<T> + 1)) * sizeof(T);

// BYTES at most, `valid` of them (zeros else).
template <int BYTES>
__device__ __forceinline__ void copy_part(uint32_t to, const void *from, int valid) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(valid) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES), "r"(valid)
                     : "memory");
}

// Starts the copies of ROWS x 16 values of an operand: rows row0 ... of `rows`, K from k0 of `k`.
// ROW_OF maps the tile's row to the array and its row (kGated's B is two arrays).
template <typename T, int ROWS, bool K_MAJOR, int BYTES, typename F>
__device__ __forceinline__ void fetch(uint32_t to, int k0, int k, int rows, F &&row_of) {
    constexpr int V = BYTES / (int)sizeof(T), kPerLine = (K_MAJOR ? kBK : ROWS) / V, kPieces = ROWS * kBK / V;
#pragma unroll
    for (int e = 0; e < (kPieces + kThreads - 1) / kThreads; ++e) {
        const int n = threadIdx.x + e * kThreads;
        if (kPieces % kThreads != 0 && n >= kPieces) break;
        const int line = n / kPerLine, at = n % kPerLine * V;
        const int tile_row = K_MAJOR ? line : at, kk = k0 + (K_MAJOR ? at : line);
        const Matrix *m;
        int row;
        row_of(tile_row, m, row);
        const int left = K_MAJOR ? (row < rows ? k - kk : 0) : (kk < k ? rows - row : 0);
        const int valid = (left < 0 ? 0 : (left < V ? left : V)) * (int)sizeof(T);
        const T *from = (const T *)m->p + (K_MAJOR ? (size_t)row * m->stride + kk : (size_t)kk * m->stride + row);
        copy_part<BYTES>(to + (uint32_t)((K_MAJOR ? line * kPitchK : line * pitch_mn(ROWS)) + at) * sizeof(T),
                         valid > 0 ? from : (const T *)m->p, valid);
    }
}

__device__ __forceinline__ void multiply(double (&c)[2], double a, double b) {
    asm volatile("mma.sync.aligned.m8n8k4.row.col.f64.f64.f64.f64 {%0,%1}, {%2}, {%3}, {%0,%1};"
                 : "+d"(c[0]), "+d"(c[1])
                 : "d"(a), "d"(b));
}

// The sums of one thread, kCount of them, and where they stand in the tile. add(): a stage's 16 of K.
template <typename T, int BM, bool A_K, bool B_K>
struct Sums;

// A warp holds 32 rows by 32 columns (8 where the tile has 32 rows).
template <int BM, bool A_K, bool B_K>
struct Sums<double, BM, A_K, B_K> {
    static constexpr int kJ = BM == 128 ? 4 : 1, kCount = 4 * kJ * 2;
    static constexpr int kTurn = 8;  // kGated: eight columns of gate, eight of up in turn
    double c[4][kJ][2];
    int lane, row, col;
    __device__ __forceinline__ Sums() : lane(threadIdx.x & 31) {
        const int warp = threadIdx.x >> 5;
        row = warp % (BM / 32) * 32;
        col = warp / (BM / 32) * kJ * 8;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < kJ; ++j) c[i][j][0] = c[i][j][1] = 0.0;
    }
    __device__ __forceinline__ void add(const double *a, const double *b) {
#pragma unroll
        for (int k = 0; k < kBK; k += 4) {
            double fa[4], fb[kJ];
            const int kk = k + lane % 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int m = row + i * 8 + lane / 4;
                fa[i] = a[A_K ? m * kPitchK + kk : kk * pitch_mn(BM) + m];
            }
#pragma unroll
            for (int j = 0; j < kJ; ++j) {
                const int n = col + j * 8 + lane / 4;
                fb[j] = b[B_K ? n * kPitchK + kk : kk * pitch_mn(kBN<double>) + n];
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < kJ; ++j) multiply(c[i][j], fa[i], fb[j]);
        }
    }
    __device__ __forceinline__ int row_at(int n) const { return row + n / (2 * kJ) * 8 + lane / 4; }
    __device__ __forceinline__ int column_at(int n) const { return col + n % (2 * kJ) / 2 * 8 + lane % 4 * 2 + n % 2; }
    __device__ __forceinline__ double at(int n) const { return c[n / (2 * kJ)][n % (2 * kJ) / 2][n % 2]; }
};

// A thread holds 8 x 8 (4 x 4 where the tile has 32 rows), in groups of four either way.
template <int BM, bool A_K, bool B_K>
struct Sums<float, BM, A_K, B_K> {
    static constexpr bool kAlongK = A_K && B_K;
    static constexpr int kI = BM == 128 ? 8 : 4, kJ = kI, kCount = kI * kJ;
    static constexpr int kTurn = 64;  // kGated: 64 columns of gate, then 64 of up
    Pair<float> c[kI][kAlongK ? kJ : kJ / 2];
    int lane, row, col;
    __device__ __forceinline__ Sums() : lane(threadIdx.x & 31) {
        const int warp = threadIdx.x >> 5;
        row = BM == 128 ? warp % 2 * 64 : 0;
        col = BM == 128 ? warp / 2 * 16 : warp * 16;
#pragma unroll
        for (int i = 0; i < kI; ++i)
#pragma unroll
            for (int j = 0; j < (kAlongK ? kJ : kJ / 2); ++j) c[i][j] = both(0.0f);
    }
    __device__ __forceinline__ int row_of(int i) const {
        return row + i / 4 * 32 + (A_K ? i % 4 * 8 + lane / 4 : lane / 4 * 4 + i % 4);
    }
    __device__ __forceinline__ int col_of(int j) const {
        return j / 4 * 64 + col + (B_K ? j % 4 * 4 + lane % 4 : lane % 4 * 4 + j % 4);
    }
    __device__ __forceinline__ void add(const float *a, const float *b) {
#pragma unroll
        for (int k = 0; k < kBK; k += 4) {
            Vec<float, 4> fa[kI];  // A_K: four of K of each row; else four rows (and four more) of each of four k
#pragma unroll
            for (int i = 0; i < kI; ++i)
                fa[i] = A_K ? load<float, 4>(a + row_of(i) * kPitchK + k)
                            : load<float, 4>(a + (k + i / (kI / 4)) * pitch_mn(BM) + row_of(i % (kI / 4) * 4));
            if constexpr (kAlongK) {
#pragma unroll
                for (int j = 0; j < kJ; ++j) {
                    const Vec<float, 4> fb = load<float, 4>(b + col_of(j) * kPitchK + k);
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int i = 0; i < kI; ++i) c[i][j] = fma(fa[i].pair(q), fb.pair(q), c[i][j]);
                }
            } else {
                static_assert(!B_K, "columns lie side by side");
#pragma unroll
                for (int kk = 0; kk < 4; ++kk) {
                    Vec<float, 4> fb[kJ / 4];
#pragma unroll
                    for (int h = 0; h < kJ / 4; ++h)
                        fb[h] = load<float, 4>(b + (k + kk) * pitch_mn(kBN<float>) + col_of(4 * h));
#pragma unroll
                    for (int i = 0; i < kI; ++i) {
                        const Pair<float> two = A_K ? fa[i].pair(kk / 2) : fa[kk * (kI / 4) + i / 4].pair(i % 4 / 2);
                        const float v = (A_K ? kk : i) % 2 ? two.y : two.x;
#pragma unroll
                        for (int j = 0; j < kJ / 2; ++j) c[i][j] = fma(both(v), fb[j / 2].pair(j % 2), c[i][j]);
                    }
                }
            }
        }
    }
    __device__ __forceinline__ int row_at(int n) const { return row_of(n / kJ); }
    __device__ __forceinline__ int column_at(int n) const { return col_of(n % kJ); }
    __device__ __forceinline__ float at(int n) const {
        if constexpr (kAlongK)
            return c[n / kJ][n % kJ].x + c[n / kJ][n % kJ].y;
        else
            return n % 2 ? c[n / kJ][n % kJ / 2].y : c[n / kJ][n % kJ / 2].x;
    }
};

// Up to 128 registers a thread in float64, so that two blocks share a multiprocessor.
template <typename T, int KIND, int BYTES, int kBM>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 8 ? 2 : 1)
    wide_kernel(const __grid_constant__ Product p, int down, int across, int tiles) {
    constexpr bool kAK = KIND != kWeights, kBK_ = KIND == kGated || KIND == kDown;
    constexpr int BN = kBN<T>, kColumns = KIND == kGated ? BN / 2 : BN;
    using S = Sums<T, kBM, kAK, kBK_>;
    extern __shared__ __align__(16) unsigned char memory[];
    T *const stages = (T *)memory;
    constexpr int kStage = held(kBM) + held(BN);
    const int blocks_k = (p.k + kBK - 1) / kBK, all = (KIND == kInput ? 2 : 1) * blocks_k;
    after_previous();
    let_next_start();

    for (int index = blockIdx.x; index < tiles; index += gridDim.x) {
        const int part = index / (down * across), rest = index - part * (down * across);
        const int problem = part / p.splits, split = part - problem * p.splits;
        const int row0 = rest % down * kBM, col0 = rest / down * kColumns;
        const int first = (int)((long long)all * split / p.splits), last = (int)((long long)all * (split + 1) / p.splits);
        auto next = [&](int step, int stage) {
            if (step < last) {
                const int second = KIND == kInput && step >= blocks_k ? 1 : 0, k0 = (step - second * blocks_k) * kBK;
                const int which = KIND == kWeights ? problem : second;
                const uint32_t to = shared_address(stages + stage * kStage);
                fetch<T, kBM, kAK, BYTES>(to, k0, p.k, p.m, [&](int r, const Matrix *&m, int &row) {
                    m = &p.a[which];
                    row = row0 + r;
                });
                fetch<T, BN, kBK_, BYTES>(to + held(kBM) * sizeof(T), k0, p.k, p.n, [&](int r, const Matrix *&m, int &row) {
                    if constexpr (KIND == kGated) {
                        m = &p.b[r / S::kTurn % 2];
                        row = col0 + r / (2 * S::kTurn) * S::kTurn + r % S::kTurn;
                    } else {
                        m = &p.b[which];
                        row = col0 + r;
                    }
                });
            }
            commit_async();
        };
        S sums;
#pragma unroll
        for (int s = 0; s < kStages<T> - 1; ++s) next(first + s, s);
        int stage = 0;
        for (int step = first; step < last; ++step) {
            wait_async<kStages<T> - 2>();
            __syncthreads();  // this stage is there for all, and the one before it read
            next(step + kStages<T> - 1, stage == 0 ? kStages<T> - 1 : stage - 1);
            sums.add(stages + stage * kStage, stages + stage * kStage + held(kBM));
            stage = stage == kStages<T> - 1 ? 0 : stage + 1;
        }
        // The sums to where the ring was, then value by value, neighbours by neighbouring
        // threads: what is done with them stands in the code once, not once for each of a
        // thread's sums (float64's functions are long: the VJP's first product of 16384 x 64
        // through 256 hidden values, GELU, 192 us so).
        constexpr int kPitch = BN + 1;
        static_assert((size_t)kBM * kPitch * sizeof(T) <= kShared<T, kBM>, "the tile fits the ring");
        wait_async<0>();
        __syncthreads();
#pragma unroll
        for (int n = 0; n < S::kCount; ++n) stages[sums.row_at(n) * kPitch + sums.column_at(n)] = sums.at(n);
        __syncthreads();
        const size_t stride = partial_stride(p.n), each = (size_t)p.splits * p.m * stride;
        T *const partial = (T *)p.partial + problem * each + (size_t)split * p.m * stride;
        const bool turned = KIND == kWeights && p.splits == 1 && p.transposed[problem];
#pragma unroll 2
        for (int n = threadIdx.x; n < kBM * kColumns; n += kThreads) {
            const int r = turned ? n % kBM : n / kColumns, c = turned ? n / kBM : n % kColumns;
            const int row = row0 + r, col = col0 + c;
            if (row >= p.m || col >= p.n) continue;
            const T *at = stages + r * kPitch + (KIND == kGated ? c / S::kTurn * 2 * S::kTurn + c % S::kTurn : c);
            const T v = at[0], other = KIND == kGated ? at[S::kTurn] : v;
            if (p.splits > 1) {
                partial[row * stride + col] = v;
                if constexpr (KIND == kGated) partial[each + row * stride + col] = other;
            } else {
                finish<T, T, KIND>(p, problem, row, col, v, other);
            }
        }
        __syncthreads();  // before the next tile's first copies
    }
}

template <typename T, int KIND, int BYTES, int kBM>
cudaError_t launch_tiles(const Product &p, cudaStream_t stream) {
    constexpr int kColumns = KIND == kGated ? kBN<T> / 2 : kBN<T>;
    const int down = (p.m + kBM - 1) / kBM, across = (p.n + kColumns - 1) / kColumns;
    const long long tiles = (long long)down * across * p.problems * p.splits;
    if (tiles > INT32_MAX) return cudaErrorInvalidValue;
    const auto kernel = wide_kernel<T, KIND, BYTES, kBM>;
    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kShared<T, kBM>);
    if (e != cudaSuccess) return e;
    const long long most = (long long)geo::device_sm_count() * (sizeof(T) == 8 ? 2 : 1);
    return launch_after(kernel, (unsigned)(tiles < most ? tiles : most), kThreads, kShared<T, kBM>, 1, stream, p, down, across,
                        (int)tiles);
}

// Whether every operand can be copied by 16 bytes.
template <typename T, int KIND>
cudaError_t launch_kind(const Product &p, cudaStream_t stream) {
    bool whole = true;
    auto look = [&](const Matrix &x) {
        whole = whole && (uintptr_t)x.p % 16 == 0 && x.stride * sizeof(T) % 16 == 0;
    };
    for (int i = 0; i < (KIND == kInput ? 2 : p.problems); ++i) look(p.a[i]);
    for (int i = 0; i < (KIND == kInput || KIND == kGated ? 2 : p.problems); ++i) look(p.b[i]);
    auto launch = [&](auto bytes) {
        constexpr int kBytes = decltype(bytes)::value;
        return tile_rows(p.m) == 32 ? launch_tiles<T, KIND, kBytes, 32>(p, stream)
                                    : launch_tiles<T, KIND, kBytes, 128>(p, stream);
    };
    return whole ? launch(std::integral_constant<int, 16>{}) : launch(std::integral_constant<int, (int)sizeof(T)>{});
}

template <typename T>
cudaError_t launch_type(ProductKind kind, const Product &p, cudaStream_t stream) {
    switch (kind) {
        case kGated: return launch_kind<T, kGated>(p, stream);
        case kDown: return launch_kind<T, kDown>(p, stream);
        case kHidden: return launch_kind<T, kHidden>(p, stream);
        case kInput: return launch_kind<T, kInput>(p, stream);
        default: return launch_kind<T, kWeights>(p, stream);
    }
}

}  // namespace

// As many parts as give every multiprocessor its tiles, none under 128 of K. (Two tiles a
// multiprocessor in float64, although they share its multiply-adds: a single one's eight
// warps do not keep them busy. x_bar of 16384 x 64 from 256 hidden values, 128 tiles: 30
// us more whole than in two parts.)
Cut cut_wide(ProductKind kind, uint32_t type, size_t m, size_t n, size_t k) {
    const bool f64 = type == GEO_B200_F64;
    const size_t wide = (f64 ? kBN<double> : kBN<float>) / (kind == kGated ? 2 : 1);
    const size_t tiles = (kind == kWeights ? 3 : 1) * ((m + tile_rows(m) - 1) / tile_rows(m)) * ((n + wide - 1) / wide);
    const size_t wanted = (size_t)geo::device_sm_count() * (f64 ? 2 : 1) / tiles, most = k * (kind == kInput ? 2 : 1) / 128;
    const size_t splits = wanted < most ? wanted : most;
    return {(int)wide, false, splits < 1 ? 1 : (splits < 64 ? (int)splits : 64)};
}

cudaError_t launch_product_wide(ProductKind kind, uint32_t type, const Product &p, cudaStream_t stream) {
    const cudaError_t e =
        type == GEO_B200_F64 ? launch_type<double>(kind, p, stream) : launch_type<float>(kind, p, stream);
    return e != cudaSuccess || p.splits == 1 ? e : launch_join(kind, type, type, p, stream);
}

}  // namespace layers
}  // namespace geo
