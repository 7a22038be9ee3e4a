// layer_norm.cu -- layer norm over rows, alone and behind residual + dropout,
// and their VJPs (geo/geo_b200.h section 5).
//
// Forward, per row of C values: m = sum x / C, v = sum (x - m)^2 / C,
// y = (x - m) rstd w + b. VJP with xh = (x - m) rstd, g = y_bar w:
//   x_bar = rstd (g - mean(g) - xh mean(g xh)),
//   w_bar = sum_rows y_bar xh, b_bar = sum_rows y_bar.
// Every variant does a few multiply-adds per value, so HBM bounds it.
#include <cooperative_groups.h>

#include <cmath>

#include "geo_runtime.h"
#include "layers.h"

namespace {

using namespace geo::layers;

constexpr int kThreads = 256;

// Sum over the block, the same on every thread, in a fixed order. Leaves
// `scratch` free for the next call.
template <typename W>
__device__ W block_sum(W v, W *scratch) {
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
    __syncthreads();
    W sum = 0;
    for (int i = 0; i < (int)blockDim.x / 32; ++i) sum += scratch[i];
    __syncthreads();
    return sum;
}

struct ForwardArgs {
    const void *x, *residual, *weight, *bias;
    void *z, *y, *mean, *rstd;
    size_t rows, x_stride, residual_stride, z_stride, y_stride;
    int cols;
    double epsilon;
    Drop drop;
};

struct BackwardArgs {
    const void *x, *weight, *mean, *rstd, *dy, *dz;
    void *dsum, *dx, *dweight, *dbias;  // dsum: layer norm's x_bar (+ dz); dx: dropout's x_bar
    size_t rows, x_stride, dy_stride, dz_stride, dsum_stride, dx_stride;
    int cols;
    Drop drop;
};

// ---- rows held on chip ---------------------------------------------------------

// A team of lanes holds one row, thread `lane` the vectors lane, lane + lanes, ...
// (K of them, V values each; pair q of the thread's values is 2q, 2q + 1 in that
// order): part of a warp (lanes a power of two up to 32, several rows a warp), a
// whole block, or (backward) the blocks of a cluster.

template <typename W>
__device__ __forceinline__ W team_sum(W v, int lanes) {
    for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Pairs of weight or bias for values [first, first + G) of the thread, of the
// value type or (16-bit values only) float32; `absent` past the row or without
// the array. G: whole vectors, at least two values.
template <typename T, int V, int G>
__device__ __forceinline__ void load_parameters(const void *p, bool is_float, int first_vector, int lane, int threads,
                                                int cols, Wide<T> absent, Pair<Wide<T>> (&out)[G / 2]) {
    using W = Wide<T>;
#pragma unroll
    for (int i = 0; i < G / V; ++i) {
        const int c = (lane + (first_vector + i) * threads) * V;
        const bool there = p != nullptr && c < cols;
        if constexpr (V == 1) {
            W v = absent;
            if (there) {
                if (sizeof(T) == 2 && is_float)
                    v = (W)((const float *)p)[c];
                else
                    v = load<T, 1>((const T *)p + c).one();
            }
            (i & 1 ? out[i / 2].y : out[i / 2].x) = v;
        } else {
#pragma unroll
            for (int q = 0; q < V / 2; ++q) out[i * V / 2 + q] = both(absent);
            if (!there) continue;
            if (sizeof(T) == 2 && is_float) {
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int j = 0; j < V; j += 4) {
                        const Vec<float, 4> w = load<float, 4>((const float *)p + c + j);
                        out[i * V / 2 + j / 2] = w.pair(0);
                        out[i * V / 2 + j / 2 + 1] = w.pair(1);
                    }
                }
            } else {
                const Vec<T, V> w = load<T, V>((const T *)p + c);
#pragma unroll
                for (int q = 0; q < V / 2; ++q) out[i * V / 2 + q] = w.pair(q);
            }
        }
    }
}

template <typename T, int V, int K>
__device__ __forceinline__ Pair<Wide<T>> pair_at(const Vec<T, V> (&raw)[K], int q) {
    if constexpr (V == 1)
        return {raw[2 * q].one(), raw[2 * q + 1].one()};
    else
        return raw[2 * q / V].pair(q % (V / 2));
}

template <typename T, int V, int K>
__device__ __forceinline__ void set_pair(Vec<T, V> (&raw)[K], int q, Pair<Wide<T>> v) {
    if constexpr (V == 1) {
        raw[2 * q].set_one(v.x);
        raw[2 * q + 1].set_one(v.y);
    } else {
        raw[2 * q / V].set(q % (V / 2), v);
    }
}

// Which of the thread's values dropout keeps, bit i V + j.
template <int V, int K>
__device__ __forceinline__ uint32_t kept_of_row(const Drop &drop, uint64_t offset, uint64_t row_start, int lane,
                                                int threads, int cols) {
    if constexpr (V == 1) {
        return kept_by_warp<K>(drop, offset, row_start + (lane & ~31), threads);
    } else {
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int c = (lane + i * threads) * V;
            if (c >= cols) continue;
            bits |= (kept_values<V>(drop, offset, row_start + c) & ((1u << V) - 1u)) << (i * V);
        }
        return bits;
    }
}

template <typename T, int V, int K, bool DROP, bool BLOCK, int THREADS>
__global__ void __launch_bounds__(THREADS, THREADS == 1024 ? 1 : 768 / THREADS) norm_kernel(const ForwardArgs a, int lanes, bool float_parameters) {
    using W = Wide<T>;
    constexpr int Q = K * V / 2;
    __shared__ W sums[2][BLOCK ? 32 : 1][2];
    const int threads = BLOCK ? (int)blockDim.x : lanes;
    const int lane = BLOCK ? (int)threadIdx.x : (int)threadIdx.x & (lanes - 1);
    const int warp = (int)threadIdx.x >> 5, wlane = (int)threadIdx.x & 31;
    const int teams = BLOCK ? 1 : 128 / lanes;
    const size_t step = (size_t)gridDim.x * teams;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const W scale = (W)a.drop.scale, over = W(1) / (W)a.cols;
    // BLOCK: how many values of the row warp w holds.
    auto held_by = [&](int w) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int left = a.cols / V - (w * 32 + i * threads);
            n += left < 0 ? 0 : (left < 32 ? left : 32);
        }
        return (W)(n * V);
    };
    const W held = BLOCK ? held_by(warp) : (W)a.cols;
    const W over_held = held > W(0) ? W(1) / held : W(0);
    // BLOCK: thread `wlane` of every warp joins what warp `wlane` held.
    const W joined = BLOCK && wlane < threads / 32 ? held_by(wlane) : W(0);
    const W over_joined = joined > W(0) ? W(1) / joined : W(0);
    const bool ragged = threads * K * V != a.cols;
    int flip = 0;
    // The bound is the warp's first row, so that all its lanes stay for the shuffles.
    for (size_t first = (size_t)blockIdx.x * teams + (BLOCK ? 0 : warp * (32 / lanes)); first < a.rows;
         first += step, flip ^= 1) {
        const size_t row = BLOCK ? first : first + wlane / lanes;
        const bool live = BLOCK || row < a.rows;
        Pair<W> v[Q];
        {
            Vec<T, V> raw[K], res[DROP ? K : 1];
            const T *x = (const T *)a.x + row * a.x_stride;
            const T *r = DROP ? (const T *)a.residual + row * a.residual_stride : nullptr;
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const int c = (lane + i * threads) * V;
                raw[i] = Vec<T, V>::zero();
                if constexpr (DROP) res[i] = Vec<T, V>::zero();
                if (live && c < a.cols) {
                    raw[i] = load<T, V>(x + c);
                    if constexpr (DROP) res[i] = load<T, V>(r + c);
                }
            }
            if constexpr (DROP) {
                const uint32_t kept = kept_of_row<V, K>(a.drop, offset, row * (size_t)a.cols, lane, threads, a.cols);
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    Pair<W> p = pair_at(raw, q);
                    p.x = (kept >> (2 * q)) & 1 ? p.x : W(0);
                    p.y = (kept >> (2 * q + 1)) & 1 ? p.y : W(0);
                    v[q] = fma(p, both(scale), pair_at(res, q));
                }
            } else {
#pragma unroll
                for (int q = 0; q < Q; ++q) v[q] = pair_at(raw, q);
            }
        }
        // Two sweeps over registers: the mean of what the warp (or its team)
        // holds, then the squares about it. Values past the row are 0 in the
        // first, the mean itself in the second.
        Pair<W> two = both(W(0));
#pragma unroll
        for (int q = 0; q < Q; ++q) two = two + v[q];
        W sum = team_sum(two.x + two.y, BLOCK ? 32 : lanes);
        W mean = BLOCK ? sum * over_held : sum / held;
        if (ragged)
#pragma unroll
            for (int i = 0; i < K; ++i) {
                if ((lane + i * threads) * V < a.cols) continue;
                if constexpr (V == 1) {
                    (i & 1 ? v[i / 2].y : v[i / 2].x) = mean;
                } else {
#pragma unroll
                    for (int q = i * V / 2; q < (i + 1) * V / 2; ++q) v[q] = both(mean);
                }
            }
        two = both(W(0));
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const Pair<W> d = v[q] + both(-mean);
            two = fma(d, d, two);
        }
        W squares = team_sum(two.x + two.y, BLOCK ? 32 : lanes);
        if constexpr (BLOCK) {
            // Warps joined about the row's mean: squares + held (warp's mean - mean)^2. Two buffers, one barrier a row.
            if (wlane == 0) {
                sums[flip][warp][0] = sum;
                sums[flip][warp][1] = squares;
            }
            __syncthreads();
            const W other = wlane < threads / 32 ? sums[flip][wlane][0] : W(0);
            mean = team_sum(other, 32) / (W)a.cols;  // divided, so that a row of one value has no spread
            const W d = other * over_joined - mean;
            squares = team_sum(wlane < threads / 32 ? sums[flip][wlane][1] + joined * d * d : W(0), 32);
        }
        const W rstd = rsqrt(squares * over + (W)a.epsilon);
        if (live && lane == 0) {
            if (a.mean != nullptr) ((W *)a.mean)[row] = mean;
            if (a.rstd != nullptr) ((W *)a.rstd)[row] = rstd;
        }
        // A vector (or two single values) at a time, so that few parameters are held.
        constexpr int G = V > 1 ? V : 2;
#pragma unroll
        for (int m = 0; m < K * V / G; ++m) {
            Vec<T, V> z[G / V], y[G / V];
            Pair<W> w[G / 2], b[G / 2];
            load_parameters<T, V, G>(a.weight, float_parameters, m * G / V, lane, threads, a.cols, W(1), w);
            load_parameters<T, V, G>(a.bias, float_parameters, m * G / V, lane, threads, a.cols, W(0), b);
#pragma unroll
            for (int q = 0; q < G / 2; ++q) {
                const Pair<W> p = v[m * G / 2 + q];
                if constexpr (DROP) set_pair(z, q, p);
                const Pair<W> hat = (p + both(-mean)) * both(rstd);
                set_pair(y, q, fma(hat, w[q], b[q]));
            }
#pragma unroll
            for (int i = 0; i < G / V; ++i) {
                const int c = (lane + (m * G / V + i) * threads) * V;
                if (!live || c >= a.cols) continue;
                if constexpr (DROP) store<T, V>((T *)a.z + row * a.z_stride + c, z[i]);
                store<T, V>((T *)a.y + row * a.y_stride + c, y[i]);
            }
        }
    }
}

// ---- backward ------------------------------------------------------------------

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

template <int BYTES>
__device__ __forceinline__ void copy_async(uint32_t to, const void *from, bool live) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2, %3;" ::"r"(to), "l"(from), "n"(BYTES),
                     "r"(live ? BYTES : 0)
                     : "memory");
}
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void wait_async() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}

// Bytes of shared memory behind one vector of one thread: 16, or a whole copy
// of 4 or 8 bytes for single values.
template <typename T, int V>
constexpr int kSlot = V > 1 ? 16 : (sizeof(T) == 8 ? 8 : 4);

// Copies a vector into its slot (zeros when not `live`). A single 16-bit value
// travels as the aligned 4-byte word around it, whose other half is not used;
// where that word would reach over an end of the array (`edge`: the array's
// first or last value), the value alone is loaded and stored.
template <typename T, int V>
__device__ __forceinline__ void fetch(uint32_t slot, const T *from, bool live, bool edge) {
    if constexpr (kSlot<T, V> > sizeof(T) * V) {
        if (edge) {
            const uint16_t v = *reinterpret_cast<const uint16_t *>(from);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(slot + (uint32_t)((uintptr_t)from & 2)), "h"(v) : "memory");
        } else {
            copy_async<4>(slot, (const void *)((uintptr_t)from & ~(uintptr_t)3), live);
        }
    } else {
        copy_async<kSlot<T, V>>(slot, from, live);
    }
}

// One pass over x and y_bar (and z_bar): x_bar row by row, and the column sums
// of y_bar xh and y_bar in the registers of the thread that owns the column; at
// the end partial[cluster][0: weight, 1: bias][col]. Rows come through a ring of
// `stages` in shared memory, each thread copying and waiting for its own vectors
// only, stages - 1 rows ahead. CLUSTER: the row is cut into the cluster's blocks,
// which hand each other their warps' sums through distributed shared memory.
template <typename T, int V, int K, bool DROP, bool BLOCK, bool CLUSTER, int STAGES>
__global__ void __launch_bounds__(BLOCK ? 256 : 128, BLOCK ? 2 : 4)
    vjp_kernel(const BackwardArgs a, int lanes, bool float_parameters, Wide<T> *partial) {
    using W = Wide<T>;
    constexpr int Q = K * V / 2;
    constexpr int kColumns = BLOCK ? 1 : (V == 1 ? 32 * K : 32 * K * V);
    constexpr int S = kSlot<T, V>;
    extern __shared__ __align__(16) unsigned char ring[];
    __shared__ W sums[2][CLUSTER ? 64 : 8][2];
    __shared__ W columns[2][kColumns];
    namespace cg = cooperative_groups;
    const int rank = CLUSTER ? (int)cg::this_cluster().block_rank() : 0;
    const int ranks = CLUSTER ? (int)cg::this_cluster().num_blocks() : 1;
    const int threads = BLOCK ? (int)blockDim.x * ranks : lanes;
    const int lane = BLOCK ? (int)threadIdx.x + rank * (int)blockDim.x : (int)threadIdx.x & (lanes - 1);
    const int warp = (int)threadIdx.x >> 5, wlane = (int)threadIdx.x & 31;
    const int teams = BLOCK ? 1 : 128 / lanes;
    const int warps = BLOCK ? (int)blockDim.x / 32 : 1;
    const size_t cluster = blockIdx.x / ranks;
    const size_t step = (size_t)(gridDim.x / ranks) * teams;
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const W scale = (W)a.drop.scale, over = W(1) / (W)a.cols;
    const bool has_dz = DROP && a.dz != nullptr;
    const int arrays = has_dz ? 3 : 2;

    Pair<W> weight[Q], dw[Q], db[Q];
    load_parameters<T, V, K * V>(a.weight, float_parameters, 0, lane, threads, a.cols, W(1), weight);
#pragma unroll
    for (int q = 0; q < Q; ++q) dw[q] = db[q] = both(W(0));

    const uint32_t slots = shared_address(ring) + threadIdx.x * S;
    const uint32_t next_vector = blockDim.x * S, next_array = K * next_vector, next_stage = arrays * next_array;
    auto enqueue = [&](size_t row, uint32_t stage) {
        const bool live = row < a.rows;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int c = (lane + i * threads) * V;
            const bool inside = live && c < a.cols;
            const bool edge = inside && ((row == 0 && c == 0) || (row == a.rows - 1 && c == a.cols - 1));
            const size_t r = inside ? row : 0, at = inside ? c : 0;
            const uint32_t slot = slots + stage * next_stage + i * next_vector;
            fetch<T, V>(slot, (const T *)a.x + r * a.x_stride + at, inside, edge);
            fetch<T, V>(slot + next_array, (const T *)a.dy + r * a.dy_stride + at, inside, edge);
            if constexpr (DROP)
                if (has_dz) fetch<T, V>(slot + 2 * next_array, (const T *)a.dz + r * a.dz_stride + at, inside, edge);
        }
        commit_async();
    };
    auto vectors = [&](Vec<T, V> (&out)[K], uint32_t stage, int array, const T *row_start) {
        const unsigned char *from = ring + threadIdx.x * S + stage * next_stage + array * next_array;
        // Where in its word a single 16-bit value is: the same for all of a thread's, which are 32 n apart.
        if constexpr (S > sizeof(T) * V) from += (uintptr_t)(row_start + lane) & 2;
#pragma unroll
        for (int i = 0; i < K; ++i) out[i] = load<T, V>((const T *)(from + i * next_vector));
    };

    const size_t begin = cluster * teams + (BLOCK ? 0 : warp * (32 / lanes));
    const size_t within = BLOCK ? 0 : wlane / lanes;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s) enqueue(begin + within + s * step, s);
    W next_mean = 0, next_rstd = 0;
    if (begin + within < a.rows) {
        next_mean = ((const W *)a.mean)[begin + within];
        next_rstd = ((const W *)a.rstd)[begin + within];
    }
    if constexpr (CLUSTER) cg::this_cluster().sync();  // every block runs before its memory is written
    int flip = 0;
    uint32_t stage = 0;
    for (size_t first = begin; first < a.rows; first += step, flip ^= 1) {
        const size_t row = first + within;
        const bool live = row < a.rows;
        const W mean = next_mean, rstd = next_rstd;
        next_mean = next_rstd = 0;
        if (row + step < a.rows) {
            next_mean = ((const W *)a.mean)[row + step];
            next_rstd = ((const W *)a.rstd)[row + step];
        }
        // Into the slot that this thread read in the last round.
        enqueue(row + (STAGES - 1) * step, stage == 0 ? STAGES - 1 : stage - 1);
        wait_async<STAGES - 1>();
        const T *x_row = (const T *)a.x + (live ? row : 0) * a.x_stride;
        const T *dy_row = (const T *)a.dy + (live ? row : 0) * a.dy_stride;
        const T *dz_row = has_dz ? (const T *)a.dz + (live ? row : 0) * a.dz_stride : nullptr;
        Vec<T, V> x[K], dy[K];
        vectors(x, stage, 0, x_row);
        vectors(dy, stage, 1, dy_row);
        Pair<W> sum2 = both(W(0)), along2 = both(W(0));
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const Pair<W> d = pair_at(dy, q), xh = (pair_at(x, q) + both(-mean)) * both(rstd), g = d * weight[q];
            sum2 = sum2 + g;
            along2 = fma(g, xh, along2);
            dw[q] = fma(d, xh, dw[q]);
            db[q] = db[q] + d;
        }
        W sum = team_sum(sum2.x + sum2.y, BLOCK ? 32 : lanes);
        W along = team_sum(along2.x + along2.y, BLOCK ? 32 : lanes);
        if constexpr (BLOCK) {
            if constexpr (CLUSTER) {
                if (wlane < ranks) {
                    W *there = cg::this_cluster().map_shared_rank(&sums[flip][rank * warps + warp][0], wlane);
                    there[0] = sum;
                    there[1] = along;
                }
                cg::this_cluster().sync();
            } else {
                if (wlane == 0) {
                    sums[flip][warp][0] = sum;
                    sums[flip][warp][1] = along;
                }
                __syncthreads();
            }
            const int n = ranks * warps;
            sum = wlane < n ? sums[flip][wlane][0] : W(0);
            along = wlane < n ? sums[flip][wlane][1] : W(0);
            if (CLUSTER && wlane + 32 < n) {
                sum += sums[flip][wlane + 32][0];
                along += sums[flip][wlane + 32][1];
            }
            sum = team_sum(sum, 32);
            along = team_sum(along, 32);
        }
        sum *= over;
        along *= over;
        if (BLOCK) {
            vectors(x, stage, 0, x_row);
            vectors(dy, stage, 1, dy_row);
        }
        Pair<W> v[Q];
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            const Pair<W> xh = (pair_at(x, q) + both(-mean)) * both(rstd);
            v[q] = (fma(xh, both(-along), pair_at(dy, q) * weight[q]) + both(-sum)) * both(rstd);
        }
        if constexpr (DROP)
            if (has_dz) {
                vectors(x, stage, 2, dz_row);
#pragma unroll
                for (int q = 0; q < Q; ++q) v[q] = v[q] + pair_at(x, q);
            }
        if (a.dsum != nullptr) {
#pragma unroll
            for (int q = 0; q < Q; ++q) set_pair(x, q, v[q]);
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const int c = (lane + i * threads) * V;
                if (live && c < a.cols) store<T, V>((T *)a.dsum + row * a.dsum_stride + c, x[i]);
            }
        }
        if constexpr (DROP) {
            if (a.dx != nullptr) {
                const uint32_t kept = kept_of_row<V, K>(a.drop, offset, row * (size_t)a.cols, lane, threads, a.cols);
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    v[q] = v[q] * both(scale);
                    v[q].x = (kept >> (2 * q)) & 1 ? v[q].x : W(0);
                    v[q].y = (kept >> (2 * q + 1)) & 1 ? v[q].y : W(0);
                    set_pair(x, q, v[q]);
                }
#pragma unroll
                for (int i = 0; i < K; ++i) {
                    const int c = (lane + i * threads) * V;
                    if (live && c < a.cols) store<T, V>((T *)a.dx + row * a.dx_stride + c, x[i]);
                }
            }
        }
        stage = stage == STAGES - 1 ? 0 : stage + 1;
    }
    if (partial == nullptr) return;
    W *mine = partial + cluster * 2 * a.cols;
    W flat[2][K * V];
#pragma unroll
    for (int q = 0; q < Q; ++q) {
        flat[0][2 * q] = dw[q].x, flat[0][2 * q + 1] = dw[q].y;
        flat[1][2 * q] = db[q].x, flat[1][2 * q + 1] = db[q].y;
    }
    if constexpr (BLOCK) {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int c = (lane + i * threads) * V;
            if (c < a.cols)
#pragma unroll
                for (int j = 0; j < V; ++j) {
                    mine[c + j] = flat[0][i * V + j];
                    mine[a.cols + c + j] = flat[1][i * V + j];
                }
        }
    } else {
        // The block's teams in order.
        for (int team = 0; team < teams; ++team) {
            if ((int)threadIdx.x / lanes == team)
#pragma unroll
                for (int i = 0; i < K; ++i)
#pragma unroll
                    for (int j = 0; j < V; ++j) {
                        const int c = (lane + i * threads) * V + j;
                        columns[0][c] = flat[0][i * V + j] + (team > 0 ? columns[0][c] : W(0));
                        columns[1][c] = flat[1][i * V + j] + (team > 0 ? columns[1][c] : W(0));
                    }
            __syncthreads();
        }
        for (int c = threadIdx.x; c < a.cols; c += 128) {
            mine[c] = columns[0][c];
            mine[a.cols + c] = columns[1][c];
        }
    }
}

// ---- any row length ----------------------------------------------------------

// One CTA per row, three sweeps over it (the second and third hit L2).
template <typename T, typename P, bool DROP>
__global__ void __launch_bounds__(kThreads) norm_any_kernel(const ForwardArgs a) {
    using W = Wide<T>;
    __shared__ W scratch[kThreads / 32];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const W scale = (W)a.drop.scale;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride;
        const T *res = DROP ? (const T *)a.residual + row * a.residual_stride : nullptr;
        T *z = DROP ? (T *)a.z + row * a.z_stride : nullptr;
        T *y = (T *)a.y + row * a.y_stride;
        auto value = [&](int c) -> W {
            if constexpr (DROP) {
                const bool kept =
                    a.drop.threshold == 0 || unit_kept(a.drop, offset, (row * (size_t)a.cols + c) >> a.drop.shift);
                return widen(res[c]) + (kept ? widen(x[c]) * scale : W(0));
            } else {
                return widen(x[c]);
            }
        };
        W sum = 0;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) sum += value(c);
        const W mean = block_sum(sum, scratch) / (W)a.cols;
        W squares = 0;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const W d = value(c) - mean;
            squares += d * d;
        }
        const W rstd = W(1) / sqrt(block_sum(squares, scratch) / (W)a.cols + (W)a.epsilon);
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const W v = value(c);
            W out = (v - mean) * rstd;
            if (a.weight != nullptr) out *= (W)widen(((const P *)a.weight)[c]);
            if (a.bias != nullptr) out += (W)widen(((const P *)a.bias)[c]);
            if constexpr (DROP) z[c] = narrow<T>(v);
            y[c] = narrow<T>(out);
        }
        if (threadIdx.x == 0) {
            if (a.mean != nullptr) ((W *)a.mean)[row] = mean;
            if (a.rstd != nullptr) ((W *)a.rstd)[row] = rstd;
        }
    }
}

// x_bar of one row per CTA, two sweeps.
template <typename T, typename P, bool DROP>
__global__ void __launch_bounds__(kThreads) vjp_rows_any_kernel(const BackwardArgs a) {
    using W = Wide<T>;
    __shared__ W scratch[kThreads / 32];
    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const W scale = (W)a.drop.scale;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride;
        const T *dy = (const T *)a.dy + row * a.dy_stride;
        const T *dz = DROP && a.dz != nullptr ? (const T *)a.dz + row * a.dz_stride : nullptr;
        T *dsum = a.dsum != nullptr ? (T *)a.dsum + row * a.dsum_stride : nullptr;
        T *dx = DROP && a.dx != nullptr ? (T *)a.dx + row * a.dx_stride : nullptr;
        const W mean = ((const W *)a.mean)[row], rstd = ((const W *)a.rstd)[row];
        auto scaled = [&](int c) -> W {
            const W v = widen(dy[c]);
            return a.weight != nullptr ? v * (W)widen(((const P *)a.weight)[c]) : v;
        };
        W sum = 0, along = 0;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const W g = scaled(c);
            sum += g;
            along += g * ((widen(x[c]) - mean) * rstd);
        }
        sum = block_sum(sum, scratch) / (W)a.cols;
        along = block_sum(along, scratch) / (W)a.cols;
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            W v = rstd * (scaled(c) - sum - (widen(x[c]) - mean) * rstd * along);
            if (dz != nullptr) v += widen(dz[c]);
            if (dx != nullptr) {
                const bool kept =
                    a.drop.threshold == 0 || unit_kept(a.drop, offset, (row * (size_t)a.cols + c) >> a.drop.shift);
                dx[c] = narrow<T>(kept ? v * scale : W(0));
            }
            if (dsum != nullptr) dsum[c] = narrow<T>(v);
        }
    }
}

// Partial sums over rows [first, last) of block column range blockIdx.x:
// partial[blockIdx.y][0: weight, 1: bias][col].
template <typename T>
__global__ void __launch_bounds__(kThreads) vjp_columns_any_kernel(const BackwardArgs a, Wide<T> *partial,
                                                                   size_t rows_per_block) {
    using W = Wide<T>;
    __shared__ W sums[2][8][33];
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    const int c = (int)blockIdx.x * 32 + lane;
    const size_t first = blockIdx.y * rows_per_block;
    const size_t last = first + rows_per_block < a.rows ? first + rows_per_block : a.rows;
    W dw = 0, db = 0;
    if (c < a.cols)
        for (size_t row = first + group; row < last; row += 8) {
            const W v = widen(((const T *)a.dy)[row * a.dy_stride + c]);
            const W xh = (widen(((const T *)a.x)[row * a.x_stride + c]) - ((const W *)a.mean)[row]) *
                         ((const W *)a.rstd)[row];
            dw += v * xh;
            db += v;
        }
    sums[0][group][lane] = dw;
    sums[1][group][lane] = db;
    __syncthreads();
    if (group < 2 && c < a.cols) {
        W total = 0;
        for (int i = 0; i < 8; ++i) total += sums[group][i][lane];
        partial[((size_t)blockIdx.y * 2 + group) * a.cols + c] = total;
    }
}

// out[c] = sum over the blocks of partial[block][which][c]. `wide` columns a
// block of threads, 1024 / wide threads a column, each over every so many
// blocks in order, then those in order.
template <typename W, typename P>
__global__ void __launch_bounds__(1024) join_columns_kernel(const W *partial, int blocks, int cols, int wide,
                                                            void *dweight, void *dbias) {
    __shared__ W sums[1024];
    P *out = (P *)(blockIdx.y == 0 ? dweight : dbias);
    if (out == nullptr) return;
    const int column = threadIdx.x & (wide - 1), part = threadIdx.x / wide, parts = 1024 / wide;
    const int c = (int)blockIdx.x * wide + column;
    W sum = 0;
    if (c < cols) {
#pragma unroll 8
        for (int i = part; i < blocks; i += parts) sum += partial[((size_t)i * 2 + blockIdx.y) * cols + c];
    }
    sums[threadIdx.x] = sum;
    for (int n = parts / 2; n > 0; n /= 2) {
        __syncthreads();
        if (part < n) sums[threadIdx.x] += sums[threadIdx.x + n * wide];
    }
    if (part == 0 && c < cols) out[c] = narrow<P>((Wide<P>)sums[threadIdx.x]);
}

// ---- launches ----------------------------------------------------------------

// How a row is held: values a thread loads at once, vectors a thread, threads.
struct Shape {
    int vector;   // 16 bytes of values, or one value
    int vectors;  // K; 0: rows too long, the kernels for any row length
    int lanes;    // threads of a row in a block: a power of two up to 32, or a whole block
    int blocks;   // blocks of a row (backward)
    int grid;     // backward: clusters of `blocks`, each with a partial sum of the columns
};

// Single values are spread over whole warps, which work their draws out together.
int threads_for(size_t vectors, int k, bool aligned) {
    const size_t lanes = (vectors + k - 1) / k;
    if (lanes > 32 || !aligned) return (int)((lanes + 31) / 32 * 32);
    int n = 1;
    while (n < (int)lanes) n *= 2;
    return n;
}

// Forward: the fewest threads a row that still fill the device, because sums
// across threads cost a fixed number of instructions a thread; with few rows as
// many threads as vectors, because then the chain of one row is the time.
Shape forward_shape(size_t rows, size_t cols, uint32_t type, bool aligned) {
    const int b = (int)type_bytes(type);
    Shape s = {aligned ? 16 / b : 1, 0, 0, 1, 0};
    const size_t vectors = cols / s.vector;
    const int most = !aligned ? 16 : (type == GEO_B200_F64 ? 8 : 4);
    for (int k = aligned ? 1 : 4; k <= most; k *= aligned ? 2 : 4) {
        const int lanes = threads_for(vectors, k, aligned);
        if (lanes > 1024) continue;
        if (k == 8 && s.vectors != 0) break;  // 8: only where 4 cannot hold the row
        s.vectors = k;
        s.lanes = lanes;
        if (rows * lanes <= (size_t)geo::device_sm_count() * 2048) break;
    }
    return s;
}

constexpr int kBackwardThreads = 256;

// Backward: 16 values a thread (8 in float64), whose two column sums and weight
// fit 128 registers beside the arithmetic; 512 threads a multiprocessor.
Shape backward_shape(size_t rows, size_t cols, uint32_t type, bool aligned) {
    const int b = (int)type_bytes(type);
    const int each = type == GEO_B200_F64 ? 8 : 16;
    Shape s = {aligned ? 16 / b : 1, 0, 0, 1, 0};
    const int k = each / s.vector;
    int lanes = threads_for(cols / s.vector, k, aligned);
    while (lanes > kBackwardThreads * s.blocks) s.blocks *= 2;
    if (s.blocks > 8) return s;
    if (s.blocks > 1) lanes = (lanes / s.blocks + 31) / 32 * 32;
    if (s.blocks * lanes * (size_t)k < cols / s.vector) lanes += 32;
    s.vectors = k;
    s.lanes = lanes;
    const size_t teams = lanes <= 32 ? 128 / lanes : 1;
    const size_t wanted = (rows + teams - 1) / teams;
    const size_t resident = lanes <= 128 ? 4 : 2;  // blocks a multiprocessor
    const size_t most = geo::device_sm_count() * resident / s.blocks;
    s.grid = (int)(wanted < most ? wanted : most);
    return s;
}

// Row blocks of the column sums: enough for four CTAs per SM, at least 64 rows each.
size_t column_blocks(size_t rows, size_t cols) {
    const size_t wide = (cols + 31) / 32, want = ((size_t)geo::device_sm_count() * 4 + wide - 1) / wide;
    const size_t most = (rows + 63) / 64;
    return want < most ? want : most;
}

unsigned row_grid(size_t rows) { return (unsigned)(rows < (1u << 20) ? rows : (1u << 20)); }

template <typename F>
cudaError_t by_types(uint32_t type, uint32_t parameter_type, F &&f) {
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2) {
            if (parameter_type == GEO_B200_F32) return f(t, float{});
        }
        return f(t, t);
    });
}

// f(V, K) as compile-time constants.
template <typename T, typename F>
void by_shape(const Shape &s, F &&f) {
    constexpr int V = 16 / (int)sizeof(T);
    using std::integral_constant;
    if (s.vector == 1) {
        if (s.vectors == 4) f(integral_constant<int, 1>{}, integral_constant<int, 4>{});
        if (s.vectors == 8) f(integral_constant<int, 1>{}, integral_constant<int, 8>{});
        if (s.vectors == 16) f(integral_constant<int, 1>{}, integral_constant<int, 16>{});
    } else {
        if (s.vectors == 1) f(integral_constant<int, V>{}, integral_constant<int, 1>{});
        if (s.vectors == 2) f(integral_constant<int, V>{}, integral_constant<int, 2>{});
        if (s.vectors == 4) f(integral_constant<int, V>{}, integral_constant<int, 4>{});
        if constexpr (V == 2)
            if (s.vectors == 8) f(integral_constant<int, V>{}, integral_constant<int, 8>{});
    }
}

// Whether every array starts on, and every row is a multiple of, 16 bytes.
struct Rows {
    const void *pointer;
    size_t stride;
};
bool aligned16(size_t cols, size_t bytes, size_t parameter_bytes, std::initializer_list<Rows> arrays,
               std::initializer_list<const void *> parameters) {
    if (cols * bytes % 16 != 0) return false;
    for (const Rows &r : arrays)
        if (r.pointer != nullptr && ((uintptr_t)r.pointer % 16 != 0 || r.stride * bytes % 16 != 0)) return false;
    // A thread's parameters are loaded by up to 16 bytes at multiples of the same.
    const size_t need = 16 / bytes * parameter_bytes < 16 ? 16 / bytes * parameter_bytes : 16;
    for (const void *p : parameters)
        if ((uintptr_t)p % need != 0) return false;
    return true;
}

template <bool DROP>
cudaError_t launch_forward(const geo_b200_layer_norm_config_t &c, const ForwardArgs &a, cudaStream_t stream) {
    const bool aligned = aligned16(a.cols, type_bytes(c.type), type_bytes(c.parameter_type),
                                   {{a.x, a.x_stride}, {a.residual, a.residual_stride}, {a.z, a.z_stride}, {a.y, a.y_stride}},
                                   {a.weight, a.bias});
    const Shape s = forward_shape(a.rows, a.cols, c.type, aligned);
    if (s.vectors == 0)
        return by_types(c.type, c.parameter_type, [&](auto t, auto p) {
            norm_any_kernel<decltype(t), decltype(p), DROP><<<row_grid(a.rows), kThreads, 0, stream>>>(a);
            return cudaGetLastError();
        });
    const bool float_parameters = c.parameter_type == GEO_B200_F32;
    return by_type(c.type, [&](auto t) {
        using T = decltype(t);
        by_shape<T>(s, [&](auto v, auto k) {
            constexpr int V = decltype(v)::value, K = decltype(k)::value;
            if constexpr (V > 1 || K != 8) {  // 8 single values a thread: the backward pass only
                // As many blocks as are resident, each over several rows.
                const size_t teams = s.lanes <= 32 ? 128 / s.lanes : 1, threads = s.lanes <= 32 ? 128 : s.lanes;
                const size_t wanted = (a.rows + teams - 1) / teams;
                const size_t most = (size_t)geo::device_sm_count() * (threads > 256 ? 1024 / threads : 768 / threads);
                const unsigned grid = (unsigned)(wanted < most ? wanted : most);
                if (s.lanes <= 32)
                    norm_kernel<T, V, K, DROP, false, 128><<<grid, 128, 0, stream>>>(a, s.lanes, float_parameters);
                else if (s.lanes <= 256)
                    norm_kernel<T, V, K, DROP, true, 256><<<grid, s.lanes, 0, stream>>>(a, s.lanes, float_parameters);
                else
                    norm_kernel<T, V, K, DROP, true, 1024><<<grid, s.lanes, 0, stream>>>(a, s.lanes, float_parameters);
            }
        });
        return cudaGetLastError();
    });
}

template <typename T, int V, int K, bool DROP, bool BLOCK, bool CLUSTER, int STAGES>
cudaError_t launch_vjp(const Shape &s, const BackwardArgs &a, bool float_parameters, size_t ring, Wide<T> *partial,
                       cudaStream_t stream) {
    auto kernel = vjp_kernel<T, V, K, DROP, BLOCK, CLUSTER, STAGES>;
    if (ring > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(s.grid * s.blocks));
    config.blockDim = dim3((unsigned)(BLOCK ? s.lanes : 128));
    config.dynamicSmemBytes = ring;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim = {(unsigned)s.blocks, 1, 1};
    config.attrs = &attribute;
    config.numAttrs = CLUSTER ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, a, s.lanes, float_parameters, partial);
}

template <bool DROP>
cudaError_t launch_backward(const geo_b200_layer_norm_config_t &c, const BackwardArgs &a, void *workspace,
                            cudaStream_t stream) {
    const bool sums = a.dweight != nullptr || a.dbias != nullptr;
    const bool aligned =
        aligned16(a.cols, type_bytes(c.type), type_bytes(c.parameter_type),
                  {{a.x, a.x_stride}, {a.dy, a.dy_stride}, {a.dz, a.dz_stride}, {a.dsum, a.dsum_stride}, {a.dx, a.dx_stride}},
                  {a.weight});
    const Shape s = backward_shape(a.rows, a.cols, c.type, aligned);
    const bool float_parameters = c.parameter_type == GEO_B200_F32;
    return by_types(c.type, c.parameter_type, [&](auto t, auto p) {
        using T = decltype(t);
        using P = decltype(p);
        using W = Wide<T>;
        int blocks = s.grid;
        cudaError_t e = cudaSuccess;
        if (s.vectors != 0) {
            W *partial = sums ? (W *)workspace : nullptr;
            by_shape<T>(s, [&](auto v, auto k) {
                constexpr int V = decltype(v)::value, K = decltype(k)::value;
                if constexpr (V * K == (sizeof(T) == 8 ? 8 : 16)) {
                    // Four rows in flight where shared memory holds them at 512 threads a multiprocessor, else two.
                    const int threads = s.lanes <= 32 ? 128 : s.lanes;
                    const size_t stage = (size_t)(a.dz != nullptr ? 3 : 2) * K * threads * kSlot<T, V>;
                    const size_t room = (size_t)208 * 1024 * (threads <= 128 ? 128 : 256) / 512;
                    const bool deep = 4 * stage <= room;
                    const size_t ring = (deep ? 4 : 2) * stage;
                    auto go = [&](auto block, auto cluster) {
                        constexpr bool B = decltype(block)::value, C = decltype(cluster)::value;
                        e = deep ? launch_vjp<T, V, K, DROP, B, C, 4>(s, a, float_parameters, ring, partial, stream)
                                 : launch_vjp<T, V, K, DROP, B, C, 2>(s, a, float_parameters, ring, partial, stream);
                    };
                    if (s.lanes <= 32 && s.blocks == 1)
                        go(std::false_type{}, std::false_type{});
                    else if (s.blocks == 1)
                        go(std::true_type{}, std::false_type{});
                    else
                        go(std::true_type{}, std::true_type{});
                }
            });
        } else {
            // Columns first: the row kernel may overwrite x or y_bar.
            if (sums) {
                blocks = (int)column_blocks(a.rows, a.cols);
                const dim3 grid((unsigned)((a.cols + 31) / 32), (unsigned)blocks);
                vjp_columns_any_kernel<T>
                    <<<grid, kThreads, 0, stream>>>(a, (W *)workspace, (a.rows + blocks - 1) / blocks);
            }
            if (a.dsum != nullptr || a.dx != nullptr)
                vjp_rows_any_kernel<T, P, DROP><<<row_grid(a.rows), kThreads, 0, stream>>>(a);
            e = cudaGetLastError();
        }
        if (e != cudaSuccess || !sums) return e;
        const int wide = a.cols >= 2048 ? 32 : 8;
        const dim3 join((unsigned)((a.cols + wide - 1) / wide), 2);
        join_columns_kernel<W, P><<<join, 1024, 0, stream>>>((const W *)workspace, blocks, a.cols, wide, a.dweight,
                                                             a.dbias);
        return cudaGetLastError();
    });
}

bool config_valid(const geo_b200_layer_norm_config_t *c) {
    if (c == nullptr || type_bytes(c->type) == 0) return false;
    if (c->parameter_type != c->type && !(type_bytes(c->type) == 2 && c->parameter_type == GEO_B200_F32)) return false;
    return c->rows != 0 && c->cols != 0 && c->rows <= GEO_B200_LAYER_MAX_ROWS && c->cols <= GEO_B200_LAYER_MAX_COLS &&
           std::isfinite(c->epsilon) && c->epsilon >= 0.0;
}

// Enough for whatever alignment the arrays turn out to have.
size_t workspace_bytes_of(const geo_b200_layer_norm_config_t &c) {
    size_t blocks = 0;
    for (const bool aligned : {false, true}) {
        if (aligned && c.cols * type_bytes(c.type) % 16 != 0) continue;
        const Shape s = backward_shape(c.rows, c.cols, c.type, aligned);
        const size_t n = s.vectors != 0 ? (size_t)s.grid : column_blocks(c.rows, c.cols);
        if (n > blocks) blocks = n;
    }
    return blocks * 2 * c.cols * wide_bytes(c.type);
}

bool workspace_usable(const geo_b200_layer_norm_config_t &c, const void *workspace, size_t bytes) {
    return workspace != nullptr && bytes >= workspace_bytes_of(c) && arrays_usable({{workspace, 16}});
}

// The dropout config of a fused call agrees with the norm's.
bool pair_valid(const geo_b200_layer_norm_config_t &n, const geo_b200_dropout_config_t &d) {
    return n.type == d.type && n.rows == d.rows && n.cols == d.cols;
}

}  // namespace

extern "C" geo_b200_status_t geo_b200_layer_norm(const geo_b200_layer_norm_config_t *config, const void *device_x,
                                                 const void *device_weight, const void *device_bias, void *device_y,
                                                 void *device_mean, void *device_rstd, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.layer_norm");
    if (!config_valid(config) || device_x == nullptr || device_y == nullptr) return GEO_B200_INVALID_ARGUMENT;
    geo_b200_layer_norm_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_stride}) ||
        !same_or_apart(device_y, c.y_stride, device_x, c.x_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_y, b}, {device_weight, p}, {device_bias, p}, {device_mean, w},
                        {device_rstd, w}}))
        return GEO_B200_INVALID_ARGUMENT;
    ForwardArgs a = {};
    a.x = device_x;
    a.weight = device_weight;
    a.bias = device_bias;
    a.y = device_y;
    a.mean = device_mean;
    a.rstd = device_rstd;
    a.rows = c.rows;
    a.cols = (int)c.cols;
    a.x_stride = c.x_stride;
    a.y_stride = c.y_stride;
    a.epsilon = c.epsilon;
    return status_of(launch_forward<false>(c, a, stream));
}

extern "C" size_t geo_b200_layer_norm_vjp_workspace(const geo_b200_layer_norm_config_t *config) {
    return config_valid(config) ? workspace_bytes_of(*config) : 0;
}

extern "C" geo_b200_status_t geo_b200_layer_norm_vjp(const geo_b200_layer_norm_config_t *config, const void *device_x,
                                                     const void *device_weight, const void *device_mean,
                                                     const void *device_rstd, const void *device_y_cotangent,
                                                     void *device_x_cotangent, void *device_weight_cotangent,
                                                     void *device_bias_cotangent, void *device_workspace,
                                                     size_t workspace_bytes, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.layer_norm_vjp");
    if (!config_valid(config) || device_x == nullptr || device_mean == nullptr || device_rstd == nullptr ||
        device_y_cotangent == nullptr ||
        (device_x_cotangent == nullptr && device_weight_cotangent == nullptr && device_bias_cotangent == nullptr))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_layer_norm_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_cotangent_stride, &c.x_cotangent_stride}) ||
        !same_or_apart(device_x_cotangent, c.x_cotangent_stride, device_x, c.x_stride) ||
        !same_or_apart(device_x_cotangent, c.x_cotangent_stride, device_y_cotangent, c.y_cotangent_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_weight, p}, {device_mean, w}, {device_rstd, w}, {device_y_cotangent, b},
                        {device_x_cotangent, b}, {device_weight_cotangent, p}, {device_bias_cotangent, p}}))
        return GEO_B200_INVALID_ARGUMENT;
    if ((device_weight_cotangent != nullptr || device_bias_cotangent != nullptr) &&
        !workspace_usable(c, device_workspace, workspace_bytes))
        return GEO_B200_INVALID_ARGUMENT;
    BackwardArgs a = {};
    a.x = device_x;
    a.weight = device_weight;
    a.mean = device_mean;
    a.rstd = device_rstd;
    a.dy = device_y_cotangent;
    a.dsum = device_x_cotangent;
    a.dweight = device_weight_cotangent;
    a.dbias = device_bias_cotangent;
    a.rows = c.rows;
    a.cols = (int)c.cols;
    a.x_stride = c.x_stride;
    a.dy_stride = c.y_cotangent_stride;
    a.dsum_stride = c.x_cotangent_stride;
    return status_of(launch_backward<false>(c, a, device_workspace, stream));
}

extern "C" geo_b200_status_t geo_b200_residual_dropout_layer_norm(
    const geo_b200_layer_norm_config_t *norm, const geo_b200_dropout_config_t *dropout, const void *device_x,
    const void *device_residual, const uint64_t *device_offset, const void *device_weight, const void *device_bias,
    void *device_z, void *device_y, void *device_mean, void *device_rstd, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.residual_dropout_layer_norm");
    ForwardArgs a = {};
    if (!config_valid(norm) || dropout == nullptr || !make_drop(*dropout, device_offset, &a.drop) ||
        !pair_valid(*norm, *dropout) || device_x == nullptr || device_residual == nullptr || device_z == nullptr ||
        device_y == nullptr || device_y == device_z)
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_layer_norm_config_t c = *norm;
    geo_b200_dropout_config_t d = *dropout;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_stride, &d.x_stride, &d.residual_stride, &d.y_stride}) ||
        c.x_stride != d.y_stride || !same_or_apart(device_z, d.y_stride, device_x, d.x_stride) ||
        !same_or_apart(device_z, d.y_stride, device_residual, d.residual_stride) ||
        !same_or_apart(device_y, c.y_stride, device_x, d.x_stride) ||
        !same_or_apart(device_y, c.y_stride, device_residual, d.residual_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_residual, b}, {device_offset, 8}, {device_weight, p}, {device_bias, p},
                        {device_z, b}, {device_y, b}, {device_mean, w}, {device_rstd, w}}))
        return GEO_B200_INVALID_ARGUMENT;
    a.x = device_x;
    a.residual = device_residual;
    a.weight = device_weight;
    a.bias = device_bias;
    a.z = device_z;
    a.y = device_y;
    a.mean = device_mean;
    a.rstd = device_rstd;
    a.rows = c.rows;
    a.cols = (int)c.cols;
    a.x_stride = d.x_stride;
    a.residual_stride = d.residual_stride;
    a.z_stride = d.y_stride;
    a.y_stride = c.y_stride;
    a.epsilon = c.epsilon;
    return status_of(launch_forward<true>(c, a, stream));
}

extern "C" geo_b200_status_t geo_b200_residual_dropout_layer_norm_vjp(
    const geo_b200_layer_norm_config_t *norm, const geo_b200_dropout_config_t *dropout,
    const uint64_t *device_offset, const void *device_z, const void *device_weight, const void *device_mean,
    const void *device_rstd, const void *device_y_cotangent, const void *device_z_cotangent,
    void *device_residual_cotangent, void *device_x_cotangent, void *device_weight_cotangent,
    void *device_bias_cotangent, void *device_workspace, size_t workspace_bytes, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.residual_dropout_layer_norm_vjp");
    BackwardArgs a = {};
    if (!config_valid(norm) || dropout == nullptr || !make_drop(*dropout, device_offset, &a.drop) ||
        !pair_valid(*norm, *dropout) || device_z == nullptr || device_mean == nullptr || device_rstd == nullptr ||
        device_y_cotangent == nullptr ||
        (device_residual_cotangent == nullptr && device_x_cotangent == nullptr && device_weight_cotangent == nullptr &&
         device_bias_cotangent == nullptr) ||
        (device_x_cotangent != nullptr && device_x_cotangent == device_residual_cotangent))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_layer_norm_config_t c = *norm;
    geo_b200_dropout_config_t d = *dropout;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_cotangent_stride, &c.x_cotangent_stride, &d.y_stride,
                                          &d.y_cotangent_stride, &d.x_cotangent_stride}) ||
        c.x_stride != d.y_stride)
        return GEO_B200_INVALID_ARGUMENT;
    const struct {
        const void *out;
        size_t stride;
    } outs[2] = {{device_residual_cotangent, c.x_cotangent_stride}, {device_x_cotangent, d.x_cotangent_stride}};
    for (const auto &o : outs)
        if (!same_or_apart(o.out, o.stride, device_z, c.x_stride) ||
            !same_or_apart(o.out, o.stride, device_y_cotangent, c.y_cotangent_stride) ||
            !same_or_apart(o.out, o.stride, device_z_cotangent, d.y_cotangent_stride))
            return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_offset, 8}, {device_z, b}, {device_weight, p}, {device_mean, w}, {device_rstd, w},
                        {device_y_cotangent, b}, {device_z_cotangent, b}, {device_residual_cotangent, b},
                        {device_x_cotangent, b}, {device_weight_cotangent, p}, {device_bias_cotangent, p}}))
        return GEO_B200_INVALID_ARGUMENT;
    if ((device_weight_cotangent != nullptr || device_bias_cotangent != nullptr) &&
        !workspace_usable(c, device_workspace, workspace_bytes))
        return GEO_B200_INVALID_ARGUMENT;
    a.x = device_z;
    a.weight = device_weight;
    a.mean = device_mean;
    a.rstd = device_rstd;
    a.dy = device_y_cotangent;
    a.dz = device_z_cotangent;
    a.dsum = device_residual_cotangent;
    a.dx = device_x_cotangent;
    a.dweight = device_weight_cotangent;
    a.dbias = device_bias_cotangent;
    a.rows = c.rows;
    a.cols = (int)c.cols;
    a.x_stride = c.x_stride;
    a.dy_stride = c.y_cotangent_stride;
    a.dz_stride = d.y_cotangent_stride;
    a.dsum_stride = c.x_cotangent_stride;
    a.dx_stride = d.x_cotangent_stride;
    return status_of(launch_backward<true>(c, a, device_workspace, stream));
}
