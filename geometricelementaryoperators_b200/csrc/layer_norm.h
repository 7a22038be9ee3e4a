// layer_norm.h -- what layer norm's forward (layer_norm.cu) and backward
// (layer_norm_vjp.cu) kernels share.
//
// A row lives on chip between the two sweeps that its sums need. A team of
// threads holds it: part of a warp (a power of two up to 32 lanes, several rows a
// warp), a block of up to 256 threads, or a cluster of up to eight such blocks
// that exchange their warps' sums through distributed shared memory. Thread
// `lane` of the team holds the K vectors lane, lane + threads, ... of V values
// (16 bytes, or single values where rows are not aligned), 16 values in all (8 in
// float64), so that a column belongs to one thread: weight, bias and the column
// sums of the backward pass stay in its registers over all its rows. Rows come
// through a ring in shared memory filled by asynchronous copies, each thread
// copying and waiting for its own vectors only (no barrier), one to three rows
// ahead: with few warps (registers) that keeps enough bytes in flight.
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

// Rows in the ring: four where the multiprocessor's shared memory holds them for
// `resident` threads, at least two.
inline int ring_stages(size_t stage_bytes, int threads, int resident) {
    const size_t room = (size_t)220 * 1024 * threads / resident;
    const size_t n = room / stage_bytes;
    return n >= 4 ? 4 : (n >= 3 ? 3 : 2);
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
template <int TEAM>
struct Place {
    int threads, lane, warp, wlane, rank, ranks, warps;
    size_t teams, team, step, begin, within;  // rows begin + within, + step, ...: `begin` is the warp's
    __device__ __forceinline__ explicit Place(int lanes) {
        namespace cg = cooperative_groups;
        rank = TEAM == kCluster ? (int)cg::this_cluster().block_rank() : 0;
        ranks = TEAM == kCluster ? (int)cg::this_cluster().num_blocks() : 1;
        threads = TEAM == kWarp ? lanes : (int)blockDim.x * ranks;
        lane = TEAM == kWarp ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x + rank * (int)blockDim.x;
        warp = (int)threadIdx.x >> 5;
        wlane = (int)threadIdx.x & 31;
        warps = (int)blockDim.x / 32;
        teams = TEAM == kWarp ? kWarpBlock / lanes : 1;
        team = blockIdx.x / ranks;
        step = gridDim.x / ranks * teams;
        begin = team * teams + (TEAM == kWarp ? warp * (32 / lanes) : 0);
        within = TEAM == kWarp ? wlane / lanes : 0;
    }
};

// The slots of one thread, for `arrays` arrays of rows.
template <typename T, int V, int K, int TEAM, bool FULL>
struct Ring {
    const unsigned char *slots;
    uint32_t address, next_vector, next_array, next_stage;
    int stages, read, write;
    size_t row, step, rows;  // of the next row to fetch
    int cols, lane, threads;

    __device__ __forceinline__ Ring(unsigned char *memory, int stages, int arrays, const Place<TEAM> &at, size_t rows,
                                    int cols)
        : slots(memory + threadIdx.x * kSlot<T, V>), stages(stages), read(0), write(0), row(at.begin + at.within),
          step(at.step), rows(rows), cols(cols), lane(at.lane), threads(at.threads) {
        address = shared_address(slots);
        next_vector = blockDim.x * kSlot<T, V>;
        next_array = K * next_vector;
        next_stage = arrays * next_array;
    }
    // Starts the copies of array `array` of the row to fetch, which begins at `start`.
    __device__ __forceinline__ void copy(int array, const void *base, size_t stride) {
        if (TEAM != kWarp && row >= rows) return;
        const bool live = TEAM != kWarp || row < rows;
        const T *start = (const T *)base + (live ? row : 0) * stride;
        const uint32_t slot = address + write * next_stage + array * next_array;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int c = (lane + i * threads) * V;
            const bool inside = live && (FULL || c < cols);
            const bool edge = kSlot<T, V> > (int)sizeof(T) * V && inside &&
                              ((row == 0 && c == 0) || (row == rows - 1 && c == cols - 1));
            fetch<T, V>(slot + i * next_vector, FULL || inside ? start + c : (const T *)base, inside, edge);
        }
    }
    __device__ __forceinline__ void fetched() {
        commit_async();
        row += step;
        write = write == stages - 1 ? 0 : write + 1;
    }
    // All but the newest stages - 1 rows have arrived.
    __device__ __forceinline__ void wait() const {
        if (stages == 4)
            wait_async<3>();
        else if (stages == 3)
            wait_async<2>();
        else
            wait_async<1>();
    }
    // This thread's part of the row being read; row_start: where it lies in global memory.
    __device__ __forceinline__ void get(Vec<T, V> (&out)[K], int array, const T *row_start) const {
        const unsigned char *from = slots + read * next_stage + array * next_array;
        // A thread's single 16-bit values are 32 n apart: all in the same half of their words.
        from += word_offset<T, V>(row_start + lane);
#pragma unroll
        for (int i = 0; i < K; ++i) out[i] = load<T, V>((const T *)(from + i * next_vector));
    }
    __device__ __forceinline__ void done() { read = read == stages - 1 ? 0 : read + 1; }
};

// Two sums of every warp of the team, where all its threads find them after the
// barrier (of the block or the cluster) in here. Two buffers in turn, so that one
// barrier a row is enough.
template <typename W, int TEAM>
__device__ __forceinline__ void publish(W (*sums)[2], const Place<TEAM> &at, W a, W b) {
    namespace cg = cooperative_groups;
    const int mine = at.rank * at.warps + at.warp;
    if constexpr (TEAM == kCluster) {
        if (at.wlane < at.ranks) {
            W *there = cg::this_cluster().map_shared_rank(&sums[mine][0], at.wlane);
            there[0] = a;
            there[1] = b;
        }
        cg::this_cluster().sync();
    } else {
        if (at.wlane == 0) {
            sums[mine][0] = a;
            sums[mine][1] = b;
        }
        __syncthreads();
    }
}
template <int TEAM>
constexpr int kSums = TEAM == kCluster ? 64 : (TEAM == kBlock ? 8 : 1);
// Lanes that add the published sums up: a block has at most eight, a cluster 64, two a lane.
template <int TEAM>
constexpr int kJoiners = TEAM == kCluster ? 32 : 8;

// Zeroes the values that dropout drops.
template <typename T, int V, int K, bool FULL>
__device__ __forceinline__ void drop_row(const Drop &drop, uint64_t offset, uint64_t row_start, int lane, int threads,
                                         int cols, Pair<Wide<T>> (&v)[K * V / 2]) {
    using W = Wide<T>;
    if (drop.threshold == 0) return;
    if constexpr (V == 1) {
        const uint32_t kept = kept_by_warp<K>(drop, offset, row_start + (lane & ~31), (uint32_t)threads);
#pragma unroll
        for (int q = 0; q < K / 2; ++q) {
            v[q].x = (kept >> (2 * q)) & 1 ? v[q].x : W(0);
            v[q].y = (kept >> (2 * q + 1)) & 1 ? v[q].y : W(0);
        }
    } else {
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const int c = (lane + i * threads) * V;
            if (!FULL && c >= cols) continue;
            uint32_t draws[V / 2];
            draws_of_pairs<V>(drop, offset, row_start + c, draws);
#pragma unroll
            for (int q = 0; q < V / 2; ++q) v[i * V / 2 + q] = drop_pair(v[i * V / 2 + q], draws[q], drop.bound);
        }
    }
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
