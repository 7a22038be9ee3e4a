// layer_norm.h -- what layer norm's forward (layer_norm.cu) and backward
// (layer_norm_vjp.cu) kernels share.
//
// A row lives on chip between the two sweeps that its sums need. A team of
// threads holds it: part of a warp (a power of two up to 32 lanes, several rows a
// warp), a block of up to 256 threads, or a cluster of up to eight such blocks
// that exchange their warps' sums through distributed shared memory. Thread
// `lane` of the team holds K vectors of V values
// (16 bytes, or single values where rows are not aligned; a warp's vectors are
// adjacent: lane, lane + 32, ... of its part), 16 values in all (8 in
// float64), so that a column belongs to one thread: weight, bias and the column
// sums of the backward pass stay in its registers over all its rows. Rows come
// through a ring in shared memory filled by asynchronous copies, each thread
// copying and waiting for its own vectors only (no barrier), one to four rows
// ahead: with few warps (registers) that keeps enough bytes in flight. What is
// left to wait for is the sums' way across the team, so teams of several warps
// take two rows of 16-bit values at a time: one barrier for both, two chains of
// additions side by side.
#pragma once

#include <cooperative_groups.h>

#include "layers.h"

namespace geo {
namespace layers {

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


// Launches (layer_norm.cu, layer_norm_vjp.cu). `partial` is the workspace of
// vjp_workspace() bytes, or null without column sums.
struct NormTypes {
    uint32_t type, parameter_type;
};
cudaError_t launch_norm(NormTypes t, const ForwardArgs &a, bool drop, cudaStream_t stream);
cudaError_t launch_norm_vjp(NormTypes t, const BackwardArgs &a, bool drop, void *partial, cudaStream_t stream);
size_t vjp_workspace(NormTypes t, size_t rows, size_t cols);

// How a row is held.
enum Team : int { kWarp = 0, kBlock = 1, kCluster = 2 };
constexpr int kTeamThreads = 256;  // of a block, at most
constexpr int kWarpBlock = 128;    // threads of a block of kWarp teams
struct Shape {
    int vector;  // values a thread moves at once: 16 bytes, or one value
    int lanes;   // threads of the team in a block; 0: rows too long for a team
    int blocks;  // blocks of the team
    bool full;   // the team's threads hold the row exactly
    Team team() const { return lanes > 32 || blocks > 1 ? (blocks > 1 ? kCluster : kBlock) : kWarp; }
    int threads() const { return team() == kWarp ? kWarpBlock : lanes; }
    size_t teams() const { return team() == kWarp ? kWarpBlock / lanes : 1; }  // of a block
};
constexpr int values_per_thread(size_t bytes) { return bytes == 8 ? 8 : 16; }
Shape shape_of(size_t cols, size_t bytes, bool aligned);

// Whether every array starts on, and every row is a multiple of, 16 bytes.
struct RowArray {
    const void *pointer;
    size_t stride;
};
bool aligned16(size_t cols, size_t bytes, size_t parameter_bytes, std::initializer_list<RowArray> arrays,
               std::initializer_list<const void *> parameters);

// Rows that a team takes at a time.
constexpr int rows_at_once(size_t bytes, int vector, int team) { return bytes == 2 && vector > 1 && team != kWarp ? 2 : 1; }

// Rows in the ring: up to four beyond those being read, where the
// multiprocessor's shared memory holds them for `resident` threads, at least as
// many as are read at once.
inline int ring_stages(size_t row_bytes, int at_once, int threads, int resident) {
    const int most = at_once == 2 ? 6 : 4;
    const int n = (int)((size_t)220 * 1024 * threads / resident / row_bytes) / at_once * at_once;
    return n >= most ? most : (n > 2 * at_once ? n : 2 * at_once);
}

#ifdef __CUDACC__

constexpr int kThreads = 256;  // of the kernels for any row length

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


// Sum over 2, 4, ... `lanes` adjacent lanes, the same on each.
template <typename W>
__device__ __forceinline__ W team_sum(W v, int lanes) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1)
        if (o < lanes) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Pairs of weight or bias for the thread's values, which start at column `first`
// and go on every `gap` columns, of the value type or (16-bit values only)
// float32; `absent` past the row or without the array.
template <typename T, int V, int K>
__device__ __forceinline__ void load_parameters(const void *p, bool is_float, int first, int gap, int cols,
                                                Wide<T> absent, Pair<Wide<T>> (&out)[K * V / 2]) {
    using W = Wide<T>;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int c = first + i * gap;
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

template <typename T, int V>
__device__ __forceinline__ uint32_t word_offset(const T *p) {
    return kSlot<T, V> > (int)sizeof(T) * V ? (uint32_t)((uintptr_t)p & 2) : 0u;
}

// Copies a vector into its slot (zeros when not `live`). A single 16-bit value
// travels as the aligned 4-byte word around it, whose other half is not used;
// where that word would reach over an end of the array (`edge`: the array's
// first or last value), the value alone is loaded and stored.
template <typename T, int V>
__device__ __forceinline__ void fetch(uint32_t slot, const T *from, bool live, bool edge) {
    if constexpr (kSlot<T, V> > (int)sizeof(T) * V) {
        if (edge) {
            const uint16_t v = *reinterpret_cast<const uint16_t *>(from);
            asm volatile("st.shared.u16 [%0], %1;" ::"r"(slot + word_offset<T, V>(from)), "h"(v) : "memory");
        } else {
            copy_async<4>(slot, (const void *)((uintptr_t)from & ~(uintptr_t)3), live);
        }
    } else {
        copy_async<kSlot<T, V>>(slot, from, live);
    }
}

// Where this thread stands.
template <int TEAM, int V, int K>
struct Place {
    int threads, lane, warp, wlane, rank, ranks, entries;  // entries: warps of the team
    int first, gap;                                        // its vectors' columns: first, first + gap, ...
    size_t team, step, begin, within;  // rows begin + within, + step, ...: `begin` is the warp's
    __device__ __forceinline__ explicit Place(int lanes) {
        namespace cg = cooperative_groups;
        rank = TEAM == kCluster ? (int)cg::this_cluster().block_rank() : 0;
        ranks = TEAM == kCluster ? (int)cg::this_cluster().num_blocks() : 1;
        threads = TEAM == kWarp ? lanes : (int)blockDim.x * ranks;
        lane = TEAM == kWarp ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x + rank * (int)blockDim.x;
        wlane = (int)threadIdx.x & 31;
        warp = TEAM == kWarp ? (int)threadIdx.x >> 5 : lane >> 5;
        entries = threads / 32;
        first = (TEAM == kWarp ? lane : warp * 32 * K + wlane) * V;
        gap = (TEAM == kWarp ? lanes : 32) * V;
        const size_t teams = TEAM == kWarp ? kWarpBlock / lanes : 1;
        team = blockIdx.x / ranks;
        step = gridDim.x / ranks * teams;
        begin = team * teams + (TEAM == kWarp ? warp * (32 / lanes) : 0);
        within = TEAM == kWarp ? wlane / lanes : 0;
    }
    __device__ __forceinline__ int column(int i) const { return first + i * (TEAM == kWarp ? gap : 32 * V); }
};

// The slots of one thread, for `arrays` arrays of rows.
template <typename T, int V, int K, int TEAM, bool FULL, int R>
struct Ring {
    static constexpr uint32_t kVector = 32 * kSlot<T, V>;  // bytes between a thread's vectors: its warp's lie together
    const Place<TEAM, V, K> &at;
    const unsigned char *slots;
    uint32_t next_array, next_stage;
    int stages, read, write, cols;
    size_t row, rows;  // row: the next to fetch

    __device__ __forceinline__ Ring(unsigned char *memory, int stages, int arrays, const Place<TEAM, V, K> &at,
                                    size_t rows, int cols)
        : at(at), slots(memory + ((threadIdx.x >> 5) * (32 * K) + (threadIdx.x & 31)) * kSlot<T, V>), stages(stages),
          read(0), write(0), cols(cols), row(at.begin + at.within), rows(rows) {
        next_array = K * blockDim.x * kSlot<T, V>;
        next_stage = arrays * next_array;
    }
    // Starts the copies of array `array` of the row to fetch; zeros past the last row.
    __device__ __forceinline__ void copy(int array, const void *base, size_t stride) {
        const bool live = row < rows;
        const T *start = (const T *)base + (live ? row : 0) * stride + at.first;
        const uint32_t slot = shared_address(slots) + write * next_stage + array * next_array;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int c = at.column(i);
            const bool inside = live && (FULL || c < cols);
            const bool edge = kSlot<T, V> > (int)sizeof(T) * V && inside &&
                              ((row == 0 && c == 0) || (row == rows - 1 && c == cols - 1));
            fetch<T, V>(slot + i * kVector, FULL || inside ? start + (c - at.first) : (const T *)base, inside, edge);
        }
    }
    __device__ __forceinline__ void fetched() {
        commit_async();
        row += at.step;
        write = write == stages - 1 ? 0 : write + 1;
    }
    // All but the newest stages - R rows have arrived.
    __device__ __forceinline__ void wait() const {
        switch (stages - R) {
            case 1: wait_async<1>(); break;
            case 2: wait_async<2>(); break;
            case 3: wait_async<3>(); break;
            default: wait_async<4>(); break;
        }
    }
    // This thread's part of row u of those being read; row_start: where it lies in global memory.
    __device__ __forceinline__ void get(Vec<T, V> (&out)[K], int u, int array, const T *row_start) const {
        const unsigned char *from = slots + (read + u) * next_stage + array * next_array;
        // A thread's single 16-bit values are 32 apart: all in the same half of their words.
        from += word_offset<T, V>(row_start + at.first);
#pragma unroll
        for (int i = 0; i < K; ++i) out[i] = load<T, V>((const T *)(from + i * kVector));
    }
    __device__ __forceinline__ void done() { read = read == stages - R ? 0 : read + R; }
};

// One step of a sum that leaves two values in the two halves of 2 o lanes.
template <typename W>
__device__ __forceinline__ W fold(W low, W high, int o) {
    const bool upper = threadIdx.x & o;
    return (upper ? high : low) + __shfl_xor_sync(0xffffffffu, upper ? low : high, o);
}

// Warp sums of N = 2 or 4 values: lanes 32 / N n and on hold value n.
template <typename W, int N>
__device__ __forceinline__ W folded_sums(const W (&v)[N]) {
    W s;
    if constexpr (N == 4)
        s = fold(fold(v[0], v[2], 16), fold(v[1], v[3], 16), 8);
    else
        s = fold(v[0], v[1], 16);
    return team_sum(s, 32 / N);
}

// Every warp's N values, value n in lanes 32 / N n and on, to where all the
// team's threads find them after the barrier (of the block or the cluster) in
// here, sums[n][warp]. Two buffers in turn, so that one barrier is enough.
template <int TEAM>
constexpr int kSums = TEAM == kCluster ? 64 : (TEAM == kBlock ? 8 : 1);
template <int N, typename W, int TEAM, int V, int K>
__device__ __forceinline__ void publish(W (*sums)[kSums<TEAM>], const Place<TEAM, V, K> &at, W value) {
    namespace cg = cooperative_groups;
    const int n = at.wlane / (32 / N), sub = at.wlane % (32 / N);
    if constexpr (TEAM == kCluster) {
        if (sub < at.ranks) *cg::this_cluster().map_shared_rank(&sums[n][at.warp], sub) = value;
        cg::this_cluster().sync();
    } else {
        if (sub == 0) sums[n][at.warp] = value;
        __syncthreads();
    }
}

// Zeroes the values that dropout drops.
template <typename T, int V, int K, bool FULL, int TEAM>
__device__ __forceinline__ void drop_row(const Drop &drop, uint64_t offset, uint64_t row_start,
                                         const Place<TEAM, V, K> &at, int cols, Pair<Wide<T>> (&v)[K * V / 2]) {
    using W = Wide<T>;
    if (drop.threshold == 0) return;
    if constexpr (V == 1) {
        const uint32_t kept = kept_by_warp<K>(drop, offset, row_start + at.first - at.wlane, 32);
#pragma unroll
        for (int q = 0; q < K / 2; ++q) {
            v[q].x = (kept >> (2 * q)) & 1 ? v[q].x : W(0);
            v[q].y = (kept >> (2 * q + 1)) & 1 ? v[q].y : W(0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            if (!FULL && at.column(i) >= cols) continue;
            uint32_t draws[V / 2];
            draws_of_pairs<V>(drop, offset, row_start + at.column(i), draws);
#pragma unroll
            for (int q = 0; q < V / 2; ++q) v[i * V / 2 + q] = drop_pair(v[i * V / 2 + q], draws[q], drop.bound);
        }
    }
}

// The thread's part of a row to global memory.
template <typename T, int V, int K, bool FULL, int TEAM>
__device__ __forceinline__ void store_row(T *row_start, const Place<TEAM, V, K> &at, bool live, int cols,
                                          const Vec<T, V> (&v)[K]) {
    T *to = row_start + at.first;
#pragma unroll
    for (int i = 0; i < K; ++i)
        if (live && (FULL || at.column(i) < cols)) store<T, V>(to + (at.column(i) - at.first), v[i]);
}

// f(V, K, TEAM, FULL) of a shape as compile-time constants, as far as they occur.
template <typename T, typename F>
cudaError_t by_shape(const Shape &s, F &&f) {
    using std::integral_constant;
    constexpr int E = values_per_thread(sizeof(T)), V = 16 / (int)sizeof(T);
    auto team = [&](auto v, auto k, auto full) {
        if (s.team() == kWarp) return f(v, k, integral_constant<int, kWarp>{}, full);
        if (s.team() == kBlock) return f(v, k, integral_constant<int, kBlock>{}, full);
        return f(v, k, integral_constant<int, kCluster>{}, full);
    };
    if (s.vector == 1) return team(integral_constant<int, 1>{}, integral_constant<int, E>{}, std::false_type{});
    if (s.full) return team(integral_constant<int, V>{}, integral_constant<int, E / V>{}, std::true_type{});
    return team(integral_constant<int, V>{}, integral_constant<int, E / V>{}, std::false_type{});
}

template <typename F>
cudaError_t by_types(NormTypes n, F &&f) {
    return by_type(n.type, [&](auto t) {
        using T = decltype(t);
        if constexpr (sizeof(T) == 2) {
            if (n.parameter_type == GEO_B200_F32) return f(t, float{});
        }
        return f(t, t);
    });
}

// Launches a team kernel: shared memory above the default allowance, clusters.
template <typename... A>
cudaError_t launch_team(void (*kernel)(A...), const Shape &s, size_t grid, size_t ring, cudaStream_t stream,
                        const A &...args) {
    if (ring > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(grid * s.blocks));
    config.blockDim = dim3((unsigned)s.threads());
    config.dynamicSmemBytes = ring;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = (unsigned)s.blocks;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = s.blocks > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

#endif

}  // namespace layers
}  // namespace geo
