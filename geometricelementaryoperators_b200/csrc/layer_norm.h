// layer_norm.h -- what layer norm's forward (layer_norm.cu) and backward
// (layer_norm_vjp.cu) kernels share.
//
// A row lives on chip between the two sweeps that its sums need. A team of
// threads holds it: part of a warp (a power of two up to 32 lanes, several rows a
// warp), several warps of a block (up to 256 threads; smaller teams share a
// block, each with a barrier of its own), or a cluster of up to eight blocks that
// send each other their warps' sums through distributed shared memory. A thread
// holds K vectors of V values, 16 bytes each, 16 values in all (8 in float64), so
// that a column belongs to one thread: weight, bias and the column sums of the
// backward pass stay in its registers over all its rows. A warp's vectors lie side
// by side (lane, lane + 32, ...), which leaves constant offsets between them. (Half
// as many values a thread and twice the threads: 16384 x 4096 bfloat16 fused VJP
// 176 instead of 166 us at the time, the sums across threads being a fixed cost.)
//
// Rows come through a ring in shared memory filled by asynchronous copies, each
// thread copying and waiting for its own vectors only (no barrier), one to four
// rows ahead: with few warps (registers) that keeps enough bytes in flight. What
// is left to wait for is the sums' way across the team, so teams of several warps
// take two rows of 16-bit values at a time: one barrier for both, two chains of
// additions side by side (the same VJP: 166 us a row at a time, 127 two). Within a
// warp there is no barrier to share and the second row's registers cost more than
// it gives (65536 x 256 bfloat16 VJP: 25 us a row at a time, 44 two).
//
// Rows that do not start on 16 bytes (SHIFT) are moved in words of 4 bytes (8 in
// float64), neighbouring lanes neighbouring words, into and out of shared memory,
// where a unit's part starts on 16 bytes and threads find their vectors. Only a
// 16-bit row that starts in the middle of a word needs shifting, by one value;
// the half of a word that belongs to someone else is not written, and a word that
// reaches over an end of the array is read value by value.
#pragma once

#include <cooperative_groups.h>

#include "layers.h"

namespace geo {
namespace layers {

// For the self-test of the clusters' waits alone: the round in which the last block
// of every cluster sends nothing, and how often a wait looks.
struct Starve {
    uint32_t round, polls;
};

struct ForwardArgs {
    const void *x, *residual, *weight, *bias;
    void *z, *y, *mean, *rstd;
    size_t rows, x_stride, residual_stride, z_stride, y_stride;
    int cols;
    double epsilon;
    Drop drop;
    Starve starve;
};

struct BackwardArgs {
    const void *x, *weight, *mean, *rstd, *dy, *dz;
    void *dsum, *dx, *dweight, *dbias;  // dsum: layer norm's x_bar (+ dz); dx: dropout's x_bar
    size_t rows, x_stride, dy_stride, dz_stride, dsum_stride, dx_stride;
    int cols;
    Drop drop;
    Starve starve;
};

// Launches (layer_norm.cu, layer_norm_vjp.cu). `partial` is the workspace of
// vjp_workspace() bytes, or null without column sums.
struct NormTypes {
    uint32_t type, parameter_type;
};
cudaError_t launch_norm(NormTypes t, const ForwardArgs &a, bool drop, cudaStream_t stream);
cudaError_t launch_norm_vjp(NormTypes t, const BackwardArgs &a, bool drop, void *partial, cudaStream_t stream);
// float32 rows that fill a cluster of blocks, with a.starve.
cudaError_t launch_norm_starved(const ForwardArgs &a, cudaStream_t stream);
cudaError_t launch_norm_vjp_starved(const BackwardArgs &a, void *partial, cudaStream_t stream);
size_t vjp_workspace(NormTypes t, size_t rows, size_t cols);

// How a row is held.
constexpr int values_per_thread(size_t bytes) { return bytes == 8 ? 8 : 16; }
enum Team : int { kWarp = 0, kPart = 1, kBlock = 2, kCluster = 3 };  // part of a warp, of a block; a block; several
constexpr int kTeamThreads = 256;  // of a block, at most
constexpr int kWarpBlock = 128;    // threads of a block of kWarp teams
struct Shape {
    bool shift;  // rows are not whole aligned vectors
    int lanes;   // threads of the team in a block; 0: rows too long for a team
    int blocks;  // blocks of the team
    bool full;   // the team's threads hold the row exactly
    Team team() const {
        return blocks > 1 ? kCluster : (lanes <= 32 ? kWarp : (lanes <= kTeamThreads / 2 ? kPart : kBlock));
    }
    int threads() const { return (int)teams() * lanes; }  // of a block
    // Bytes of one array's part of a row in a block's ring.
    size_t part(size_t bytes) const {
        const size_t units = team() == kWarp ? teams() : threads() / 32;
        return (size_t)threads() * values_per_thread(bytes) * bytes + (shift ? units * 16 : 0);
    }
    size_t teams() const {  // of a block
        return team() == kWarp ? kWarpBlock / lanes : (team() == kPart ? kTeamThreads / lanes : 1);
    }
};
Shape shape_of(size_t cols, size_t bytes, bool aligned);

// Whether every array starts on, and every row is a multiple of, 16 bytes.
struct RowArray {
    const void *pointer;
    size_t stride;
};
bool aligned16(size_t cols, size_t bytes, size_t parameter_bytes, std::initializer_list<RowArray> arrays,
               std::initializer_list<const void *> parameters);

// Rows that a team takes at a time.
constexpr int rows_at_once(size_t bytes, bool shift, int team) { return bytes == 2 && !shift && team != kWarp ? 2 : 1; }

// Rows in the ring: up to four beyond those being read, where the
// multiprocessor's shared memory holds them for `resident` threads, at least as
// many as are read at once.
inline int ring_stages(size_t row_bytes, int at_once, int threads, int resident) {
    const int most = at_once == 2 ? 6 : 4;
    const int n = (int)((size_t)220 * 1024 * threads / resident / row_bytes) / at_once * at_once;
    return n >= most ? most : (n > 2 * at_once ? n : 2 * at_once);
}
// No ring is larger: half of a multiprocessor's 220 KB for the largest blocks (256 of 512 threads), and the fewest rows,
// 2 at_once, of three arrays take 96 KB and the 16 bytes a unit of rows off 16 bytes.
constexpr int kRingMost = 110 * 1024;

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

// What add(sum, i) adds up over i = first, first + step, ... below last: 64 values
// one after another, then 64 of those sums, then the rest. In one chain of float32
// additions the errors of equal values add up too: the mean of a row of 2^22 times
// 0.1 was 2590 roundings off. float64 has the bits for one chain. Unrolled by eight,
// since no loads are in flight at the end of a chain (256 x 65536 float32 VJP 245 us,
// 308 by four, 279 as one chain).
template <typename V, typename I, typename F>
__device__ __forceinline__ V long_sum(I first, I last, I step, F &&add) {
    V sum = {};
    if constexpr (std::is_same_v<V, double> || std::is_same_v<V, Pair<double>>) {
        for (; first < last; first += step) add(sum, first);
    } else {
        while (first < last) {
            V middle = {};
            for (int j = 0; j < 64 && first < last; ++j) {
                const I end = last - first > 64 * step ? first + 64 * step : last;
                V inner = {};
#pragma unroll 8
                for (; first < end; first += step) add(inner, first);
                middle = middle + inner;
            }
            sum = sum + middle;
        }
    }
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

// Where this thread stands. A unit is what lies side by side in a ring: a team
// within a warp, or a warp's part of the row.
template <int TEAM, int V, int K>
struct Place {
    int threads, lane, warp, wlane, rank, ranks;  // threads: of the team
    int teams, team, entries, first_entry;        // in the block; entries: warps of the team, in order from first_entry
    int unit, unit_lanes, unit_lane, unit_first;  // of the block; the unit's first column
    size_t slice, step, begin, within;  // rows begin + within, + step, ...: `begin` is the warp's; slice: block or cluster
    __device__ __forceinline__ explicit Place(int lanes) {
        namespace cg = cooperative_groups;
        rank = TEAM == kCluster ? (int)cg::this_cluster().block_rank() : 0;
        ranks = TEAM == kCluster ? (int)cg::this_cluster().num_blocks() : 1;
        threads = lanes * ranks;
        teams = TEAM == kWarp ? kWarpBlock / lanes : (TEAM == kPart ? kTeamThreads / lanes : 1);
        team = TEAM <= kPart ? (int)threadIdx.x / lanes : 0;
        lane = (int)threadIdx.x + (TEAM == kCluster ? rank * lanes : -team * lanes);
        wlane = (int)threadIdx.x & 31;
        warp = lane >> 5;
        entries = threads / 32;
        first_entry = TEAM == kPart ? team * entries : 0;
        unit = TEAM == kWarp ? team : (int)threadIdx.x >> 5;
        unit_lanes = TEAM == kWarp ? lanes : 32;
        unit_lane = TEAM == kWarp ? lane : wlane;
        unit_first = TEAM == kWarp ? 0 : warp * 32 * K * V;
        slice = blockIdx.x / ranks;
        step = gridDim.x / ranks * (size_t)teams;
        begin = slice * teams + (TEAM == kWarp ? (threadIdx.x >> 5) * (32 / lanes) : team);
        within = TEAM == kWarp ? wlane / lanes : 0;
    }
    // First column of the thread's vector i.
    __device__ __forceinline__ int column(int i) const {
        return unit_first + (i * (TEAM == kWarp ? unit_lanes : 32) + unit_lane) * V;
    }
};

// Weight or bias of the thread's values as pairs, of the value type or (16-bit
// values only) float32; `absent` past the row or without the array.
template <typename T, int V, int K, bool SHIFT, int TEAM>
__device__ __forceinline__ void load_parameters(const void *p, bool is_float, const Place<TEAM, V, K> &at, int cols,
                                                Wide<T> absent, Pair<Wide<T>> (&out)[K * V / 2]) {
    using W = Wide<T>;
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int c = at.column(i);
#pragma unroll
        for (int q = 0; q < V / 2; ++q) out[i * V / 2 + q] = both(absent);
        if (p == nullptr || c >= cols) continue;
        if constexpr (SHIFT) {
#pragma unroll
            for (int j = 0; j < V; ++j)
                if (c + j < cols) {
                    const W v = sizeof(T) == 2 && is_float ? (W)((const float *)p)[c + j] : (W)widen(((const T *)p)[c + j]);
                    (j & 1 ? out[i * V / 2 + j / 2].y : out[i * V / 2 + j / 2].x) = v;
                }
        } else if (sizeof(T) == 2 && is_float) {
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

template <typename T, int V, int K>
__device__ __forceinline__ Pair<Wide<T>> pair_at(const Vec<T, V> (&raw)[K], int q) {
    return raw[2 * q / V].pair(q % (V / 2));
}

template <typename T, int V, int K>
__device__ __forceinline__ void set_pair(Vec<T, V> (&raw)[K], int q, Pair<Wide<T>> v) {
    raw[2 * q / V].set(q % (V / 2), v);
}

// Sets the thread's values past the row's end (all of them when not `live`) to `value`.
template <int V, int K, int TEAM, typename W>
__device__ __forceinline__ void set_past(Pair<W> (&v)[K * V / 2], const Place<TEAM, V, K> &at, bool live, int cols,
                                         W value) {
#pragma unroll
    for (int i = 0; i < K; ++i) {
        const int left = live ? cols - at.column(i) : 0;
        if (left >= V) continue;
#pragma unroll
        for (int q = 0; q < V / 2; ++q) {
            Pair<W> &p = v[i * V / 2 + q];
            p.x = 2 * q < left ? p.x : value;
            p.y = 2 * q + 1 < left ? p.y : value;
        }
    }
}

// SHIFT: the word that moves values, how many a thread moves (one more where a
// row of 16-bit values starts in the middle of a word), and whether it does.
template <typename T>
using Word = std::conditional_t<sizeof(T) == 8, uint64_t, uint32_t>;
template <typename T, int V, int K>
constexpr int kWords = K * V * (int)sizeof(T) / (int)sizeof(Word<T>) + (sizeof(T) == 2 ? 1 : 0);
template <typename T>
__device__ __forceinline__ int half_word(const T *p) {
    return sizeof(T) == 2 ? (int)((uintptr_t)p >> 1 & 1) : 0;
}

// The slots of one thread, for `arrays` arrays of rows.
template <typename T, int V, int K, int TEAM, bool SHIFT, bool FULL, int R>
struct Ring {
    const Place<TEAM, V, K> &at;
    const unsigned char *slots;  // 16 bytes each; the unit's lie together
    uint32_t next_array, next_stage;
    int stages, read, write, cols;
    size_t row, rows;  // row: the next to fetch

    // Bytes of one array's part of a row, in a block of so many units of so many lanes.
    __host__ __device__ static constexpr uint32_t part(int units, int lanes) {
        return (uint32_t)units * (lanes * K + (SHIFT ? 1 : 0)) * 16;
    }
    __device__ __forceinline__ Ring(unsigned char *memory, int stages, int arrays, const Place<TEAM, V, K> &at,
                                    size_t rows, int cols)
        : at(at), slots(memory + part(at.unit, at.unit_lanes) + at.unit_lane * 16), stages(stages), read(0), write(0),
          cols(cols), row(at.begin + at.within), rows(rows) {
        next_array = part(TEAM == kWarp ? at.teams : (int)blockDim.x / 32, at.unit_lanes);
        next_stage = arrays * next_array;
    }
    __device__ __forceinline__ uint32_t vector_gap() const { return TEAM == kWarp ? at.unit_lanes * 16 : 512; }

    // Starts the copies of array `array` of the row to fetch (not SHIFT: zeros past the last row).
    __device__ __forceinline__ void copy(int array, const T *base, size_t stride) {
        const bool live = row < rows;
        const uint32_t slot = shared_address(slots) + write * next_stage + array * next_array;
        if constexpr (SHIFT) {
            const int left = cols - at.unit_first;
            if (!live || left <= 0) return;
            constexpr int kPerWord = (int)(sizeof(Word<T>) / sizeof(T)), kBytes = (int)sizeof(Word<T>);
            const T *first = base + row * stride + at.unit_first;
            const int part = at.unit_lanes * K * V, held = left < part ? left : part, half = half_word(first);
            const int words = (held + half + kPerWord - 1) / kPerWord, gap = TEAM == kWarp ? at.unit_lanes : 32;
            const Word<T> *from = (const Word<T> *)(first - half) + at.unit_lane;
            const uint32_t to = slot + at.unit_lane * (kBytes - 16);
            // The array's first and last word may reach over its ends.
            const bool ends = sizeof(T) == 2 && (row == 0 || row == rows - 1);
            if (!ends) {
#pragma unroll
                for (int k = 0; k < kWords<T, V, K>; ++k)
                    if (k * gap + at.unit_lane < words) copy_async<kBytes>(to + k * gap * kBytes, from + k * gap);
            } else {
                const T *whole_end = base + (rows - 1) * stride + cols;
#pragma unroll 1
                for (int w = 0; w + at.unit_lane < words; w += gap) {
                    const T *word = (const T *)(from + w);
                    if (word >= base && word + kPerWord <= whole_end) {
                        copy_async<kBytes>(to + w * kBytes, word);
                    } else {
                        for (int j = 0; j < kPerWord; ++j)
                            if (word + j >= base && word + j < whole_end)
                                asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + w * kBytes + j * (int)sizeof(T)),
                                             "h"(*(const unsigned short *)(word + j))
                                             : "memory");
                    }
                }
            }
        } else {
            const T *start = base + (live ? row : 0) * stride + at.column(0);
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const int c = at.column(i);
                const bool inside = live && (FULL || c < cols);
                copy_async(slot + i * vector_gap(), FULL || inside ? start + (c - at.column(0)) : base, inside);
            }
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
            case 0: wait_async<0>(); break;
            case 1: wait_async<1>(); break;
            case 2: wait_async<2>(); break;
            case 3: wait_async<3>(); break;
            default: wait_async<4>(); break;
        }
        if constexpr (SHIFT) __syncwarp();  // chunks of the neighbours
    }
    // This thread's part of row u of those being read; row_start: where it lies in
    // global memory. SHIFT: what is past the row's end is anything.
    __device__ __forceinline__ void get(Vec<T, V> (&out)[K], int u, int array, const T *row_start) const {
        const unsigned char *from = slots + (read + u) * next_stage + array * next_array;
        const uint32_t shift = SHIFT ? 16u * half_word(row_start + at.unit_first) : 0;
#pragma unroll
        for (int i = 0; i < K; ++i) {
            out[i] = load<T, V>((const T *)(from + i * vector_gap()));
            if constexpr (SHIFT && sizeof(T) == 2) {
                const uint32_t next = *(const uint32_t *)(from + i * vector_gap() + 16);
#pragma unroll
                for (int w = 0; w < 4; ++w)
                    out[i].w[w] = __funnelshift_r(out[i].w[w], w < 3 ? out[i].w[w + 1] : next, shift);
            }
        }
    }
    // Vector i alone.
    __device__ __forceinline__ Vec<T, V> get_one(int i, int u, int array, const T *row_start) const {
        const unsigned char *from = slots + (read + u) * next_stage + array * next_array + i * vector_gap();
        Vec<T, V> out = load<T, V>((const T *)from);
        if constexpr (SHIFT && sizeof(T) == 2) {
            const uint32_t shift = 16u * half_word(row_start + at.unit_first), next = *(const uint32_t *)(from + 16);
#pragma unroll
            for (int w = 0; w < 4; ++w) out.w[w] = __funnelshift_r(out.w[w], w < 3 ? out.w[w + 1] : next, shift);
        }
        return out;
    }
    // The thread's part of a row to global memory; SHIFT: through the place of
    // array `array` of row u, which has been read (every lane of the warp takes part).
    __device__ __forceinline__ void put(T *row_start, bool live, int u, int array, const Vec<T, V> (&v)[K]) const {
        if constexpr (SHIFT) {
            constexpr int kPerWord = (int)(sizeof(Word<T>) / sizeof(T));
            unsigned char *vectors = const_cast<unsigned char *>(slots) + (read + u) * next_stage + array * next_array;
            __syncwarp();  // the neighbours have read their vectors
#pragma unroll
            for (int i = 0; i < K; ++i) store<T, V>((T *)(vectors + i * vector_gap()), v[i]);
            __syncwarp();
            const int part = at.unit_lanes * K * V, left = cols - at.unit_first, held = left < part ? left : part;
            if (!live || held <= 0) return;
            T *first = row_start + at.unit_first;
            const int half = half_word(first), gap = TEAM == kWarp ? at.unit_lanes : 32;
            const Word<T> *words = (const Word<T> *)(vectors - at.unit_lane * 16) + at.unit_lane;
            Word<T> *to = (Word<T> *)(first - half) + at.unit_lane;
            // Word w of the row holds values w kPerWord - half and on: with half, the
            // upper half of word w - 1 here and the lower half of word w. Whole ones:
            const int begin = half, end = (held + half) / kPerWord;
#pragma unroll
            for (int k = 0; k < kWords<T, V, K>; ++k) {
                const int w = k * gap + at.unit_lane;
                if (w >= end || (k == 0 && w < begin)) continue;
                if constexpr (sizeof(T) == 2)
                    to[k * gap] = __funnelshift_r(words[k * gap - half], words[k * gap], 16 * half);
                else
                    to[k * gap] = words[k * gap];
            }
            if constexpr (sizeof(T) == 2) {  // and the halves at both ends
                const unsigned short *values = (const unsigned short *)(words - at.unit_lane);
                if (half && at.unit_lane == 0) *(unsigned short *)first = values[0];
                if (((held + half) & 1) && at.unit_lane == at.unit_lanes - 1)
                    *(unsigned short *)(first + held - 1) = values[held - 1];
            }
        } else {
            T *to = row_start + at.column(0);
#pragma unroll
            for (int i = 0; i < K; ++i)
                if (live && (FULL || at.column(i) < cols)) store<T, V>(to + (at.column(i) - at.column(0)), v[i]);
        }
    }
    __device__ __forceinline__ void done() {
        if constexpr (SHIFT) __syncwarp();  // the neighbours have read this thread's chunks
        read = read == stages - R ? 0 : read + R;
    }
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

// Where the warps of a team leave N values for one another: values[n][entry]
// of the block's (or cluster's) warps. Two of them in turn, so that one wait a
// round is enough: a warp writes round t + 2 only after every warp has sent its
// values of round t + 1, for which it has read those of round t.
template <int TEAM>
constexpr int kEntries = TEAM == kCluster ? 64 : (TEAM == kWarp ? 1 : 8);
template <typename W, int N, int TEAM>
struct Exchange {
    W values[2][N][kEntries<TEAM>];
    uint64_t arrived[2];  // kCluster: mbarriers that count the bytes which other blocks send
};
constexpr uint32_t kWaitPolls = 1u << 22;  // 16 seconds (3.9 us each); a round takes microseconds

template <typename W, int N, int TEAM>
__device__ __forceinline__ void open_exchange(Exchange<W, N, TEAM> &x) {
    if constexpr (TEAM == kCluster) {
        if (threadIdx.x == 0) {
            for (int i = 0; i < 2; ++i)
                asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(&x.arrived[i])) : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        cooperative_groups::this_cluster().sync();  // every block runs, its barriers ready, before it is sent anything
    }
}
// A block leaves only when nothing is on its way to it.
template <int TEAM>
__device__ __forceinline__ void close_exchange() {
    if constexpr (TEAM == kCluster) cooperative_groups::this_cluster().sync();
}

// Sends the warp's values (value n in lanes 32 / N n and on) and waits for those
// of all the team's warps. A cluster's blocks send straight into each other's
// shared memory, where a barrier counts the bytes: unlike a barrier of the
// cluster, this does not wait for the stores of the row before.
// `complete`: what the round before returned. False, for the whole warp, when this
// wait or one before gave up (never, unless a block of the cluster failed). Such a
// warp sends and waits no more: its barriers' phases are no longer those of its
// rounds. The other warps of the cluster miss its values in the next round and give
// up in turn. Nothing is on its way to a block that leaves: after what it sent last
// every warp waited for that round to be complete, or a wait's whole length.
// `silent`: sends nothing (the self-test).
template <typename W, int N, int TEAM, int V, int K>
__device__ __forceinline__ bool exchange(Exchange<W, N, TEAM> &x, uint32_t round, const Place<TEAM, V, K> &at, W value,
                                         bool complete, uint32_t polls = kWaitPolls, bool silent = false) {
    const int n = at.wlane / (32 / N), sub = at.wlane % (32 / N), flip = round & 1;
    if constexpr (TEAM == kCluster) {
        if (!complete) return false;
        const uint32_t barrier = shared_address(&x.arrived[flip]);
        if (threadIdx.x == 0)
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(barrier),
                         "r"((uint32_t)(at.entries * N * (int)sizeof(W)))
                         : "memory");
        if (sub < at.ranks && !silent) {
            uint32_t to, there;
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;"
                         : "=r"(to)
                         : "r"(shared_address(&x.values[flip][n][at.warp])), "r"(sub));
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(barrier), "r"(sub));
            if constexpr (sizeof(W) == 8)
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b64 [%0], %1, [%2];" ::"r"(to),
                             "l"(__double_as_longlong(value)), "r"(there)
                             : "memory");
            else
                asm volatile("st.async.shared::cluster.mbarrier::complete_tx::bytes.b32 [%0], %1, [%2];" ::"r"(to),
                             "r"(__float_as_uint(value)), "r"(there)
                             : "memory");
        }
        uint32_t done = 0;
        for (uint32_t poll = 0; poll < polls && !done; ++poll)
            asm volatile(
                "{\n.reg .pred p;\nmbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
                "selp.u32 %0, 1, 0, p;\n}"
                : "=r"(done)
                : "r"(barrier), "r"((round >> 1) & 1u)
                : "memory");
        return __all_sync(0xffffffffu, done);
    } else {
        if (sub == 0) x.values[flip][n][at.first_entry + at.warp] = value;
        if constexpr (TEAM == kPart)
            asm volatile("bar.sync %0, %1;" ::"r"(1 + at.team), "r"(at.threads) : "memory");
        else
            __syncthreads();
        return true;
    }
}

// Zeroes the values that dropout drops. SHIFT: a vector's values are of two
// blocks; the unit's blocks are worked out once, their decisions (a byte each) in
// `bytes` of shared memory.
constexpr int kDropBytes = 576;  // eight warps' 65, or 128 threads' 3 and fewer
template <typename T, int V, int K, bool SHIFT, bool FULL, int TEAM>
__device__ __forceinline__ void drop_row(const Drop &drop, uint64_t offset, uint64_t row_start,
                                         const Place<TEAM, V, K> &at, int cols, unsigned char *bytes,
                                         Pair<Wide<T>> (&v)[K * V / 2]) {
    if (drop.threshold == 0) return;
    if constexpr (SHIFT) {
        const uint64_t first = row_start + at.unit_first;
        const uint32_t in_block = (uint32_t)first & 7u;
        const int blocks = at.unit_lanes * K * V / 8 + 1, left = cols - at.unit_first;
        unsigned char *mine = bytes + at.unit * blocks;
        __syncwarp();
        for (int n = at.unit_lane; n < blocks && 8 * n < left + (int)in_block; n += at.unit_lanes)
            mine[n] = (unsigned char)kept_of_eight(drop, offset, (first & ~(uint64_t)7) + 8 * n);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < K; ++i) {
            const uint32_t place = in_block + (uint32_t)(at.column(i) - at.unit_first);
            // The vector's last value is in the next block only if the first is not the block's first.
            const uint32_t low = mine[place >> 3], high = mine[(place + V - 1) >> 3];
            const uint32_t kept = (low | high << 8) >> (place & 7u);
#pragma unroll
            for (int q = 0; q < V / 2; ++q) {
                Pair<Wide<T>> &p = v[i * V / 2 + q];
                p.x = (kept >> (2 * q)) & 1 ? p.x : Wide<T>(0);
                p.y = (kept >> (2 * q + 1)) & 1 ? p.y : Wide<T>(0);
            }
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

// The end of a VJP's pass: the two column sums of every thread, in the registers of the
// thread that owns the column, to partial[block or cluster][0, 1][col], the teams of a
// block added up in `memory` (where the ring was). `alone`: the grid is one cluster,
// whose blocks add the partial sums up themselves, and no second kernel is needed.
constexpr int kAloneBlocks = 8;
template <typename T, int TEAM, int V, int K>
__device__ __forceinline__ void leave_column_sums(const Place<TEAM, V, K> &at, const Pair<Wide<T>> (&dw)[K * V / 2],
                                                  const Pair<Wide<T>> (&db)[K * V / 2], Wide<T> *memory,
                                                  Wide<T> *partial, bool alone, int lanes, int cols, void *dweight,
                                                  void *dbias, bool float_parameters) {
    using W = Wide<T>;
    constexpr int Q = K * V / 2;
    // The kernel that joins the partial sums may be set up from here on.
    if (!alone) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto value = [&](const Pair<W> (&p)[Q], int e) { return e & 1 ? p[e / 2].y : p[e / 2].x; };
    // Every thread's sums to where the ring was (two rows of it hold two sums of a
    // row; value e of thread t at e threads + (t ^ e): no bank twice), then a
    // column's, the block's teams in order, in whole lines to global memory.
    const int each = blockDim.x, first_column = at.rank * lanes * K * V;
    const int columns = cols - first_column < lanes * K * V ? cols - first_column : lanes * K * V;
    W *found = memory, *mine = partial + at.slice * 2 * cols + first_column;
    auto place = [&](int e, int thread) { return e * each + (thread ^ (e & 31)); };
    __syncthreads();
#pragma unroll
    for (int e = 0; e < K * V; ++e) {
        found[place(e, threadIdx.x)] = value(dw, e);
        found[each * K * V + place(e, threadIdx.x)] = value(db, e);
    }
    __syncthreads();
    const int kinds = dbias != nullptr ? 2 : 1;
    for (int which = 0; which < kinds; ++which)
        for (int c = threadIdx.x; c < columns; c += each) {
            const int vector = c / V, unit = TEAM == kWarp ? 0 : vector / (32 * K), in_unit = vector - unit * 32 * K;
            const int round = TEAM == kWarp ? in_unit / at.unit_lanes : in_unit / 32;
            const int e = round * V + c % V, lane = unit * 32 + in_unit - round * at.unit_lanes;
            W sum = 0;
            for (int team = 0; team < at.teams; ++team)
                sum += found[which * each * K * V + place(e, team * lanes + lane)];
            mine[(size_t)which * cols + c] = sum;
        }
    if constexpr (TEAM != kCluster) {
        if (!alone) return;
        cooperative_groups::this_cluster().sync();  // makes the blocks' sums visible to one another
        for (int n = blockIdx.x * each + threadIdx.x; n < kinds * cols; n += gridDim.x * each) {
            W sum = 0;
#pragma unroll
            for (int block = 0; block < kAloneBlocks; ++block)
                if (block < (int)gridDim.x) sum += partial[(size_t)block * 2 * cols + n];
            const int c = n < cols ? n : n - cols;
            void *out = n < cols ? dweight : dbias;
            if (out == nullptr) continue;
            if (sizeof(T) == 2 && float_parameters)
                ((float *)out)[c] = (float)sum;
            else
                ((T *)out)[c] = narrow<T>(sum);
        }
    }
}

// out[c] = sum over the blocks of partial[block][which][c]: 32 columns a block of
// threads, so that whole 128-byte lines are read, blockDim / 32 threads a column, each
// over every so many blocks in order, then those as a tree. (With 16 columns 16384 x
// 4096 bfloat16 takes as long, 74.0 and 74.5 us.)
constexpr int kJoinColumns = 32;
template <typename W, typename P>
__global__ void __launch_bounds__(1024) join_columns_kernel(const W *partial, int blocks, int cols, void *dweight,
                                                            void *dbias) {
    __shared__ W sums[1024];
    P *out = (P *)(blockIdx.y == 0 ? dweight : dbias);
    const int column = threadIdx.x % kJoinColumns, part = threadIdx.x / kJoinColumns, parts = blockDim.x / kJoinColumns;
    const int c = (int)blockIdx.x * kJoinColumns + column;
    W sum = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");  // for the kernel before to end
    if (c < cols) {
#pragma unroll 8
        for (int i = part; i < blocks; i += parts) sum += partial[((size_t)i * 2 + blockIdx.y) * cols + c];
    }
    sums[threadIdx.x] = sum;
    for (int n = parts / 2; n > 0; n /= 2) {
        __syncthreads();
        if (part < n) sums[threadIdx.x] += sums[threadIdx.x + n * kJoinColumns];
    }
    if (part == 0 && c < cols && out != nullptr) out[c] = narrow<P>((Wide<P>)sums[threadIdx.x]);
}

// f(TEAM, SHIFT, FULL) of a shape as compile-time constants, as far as they occur.
template <typename F>
cudaError_t by_shape(const Shape &s, F &&f) {
    using std::integral_constant;
    auto team = [&](auto shift, auto full) {
        if (s.team() == kWarp) return f(integral_constant<int, kWarp>{}, shift, full);
        if (s.team() == kPart) return f(integral_constant<int, kPart>{}, shift, full);
        if (s.team() == kBlock) return f(integral_constant<int, kBlock>{}, shift, full);
        return f(integral_constant<int, kCluster>{}, shift, full);
    };
    if (s.shift) return team(std::true_type{}, std::false_type{});
    if (s.full) return team(std::false_type{}, std::true_type{});
    return team(std::false_type{}, std::false_type{});
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

// Launches `grid` teams' worth of blocks of a team kernel, in clusters of
// `cluster`. Shared memory above the default allowance is a property of the kernel,
// not of the launch, and other host threads launch the same kernel with rings of
// their own: what is allowed is the same for all, kRingMost. A cluster lies within
// one group of multiprocessors, so fewer clusters may be resident than the
// multiprocessors' total allows (of four blocks, two a multiprocessor: 71 of 74):
// `grid` is cut to those, or the rest would start when the first have taken all
// their rows (4096 x 16384 bfloat16: forward 81 us with 74 clusters, 53 with 71;
// VJP 117 and 90). The question costs 0.4 us on the host.
template <typename... A>
cudaError_t launch_team(void (*kernel)(A...), const Shape &s, size_t &grid, size_t cluster, size_t ring,
                        cudaStream_t stream, const A &...args) {
    if (ring > 40 * 1024) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingMost);
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)(grid * s.blocks));
    config.blockDim = dim3((unsigned)s.threads());
    config.dynamicSmemBytes = ring;
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeClusterDimension;
    attribute.val.clusterDim.x = (unsigned)cluster;
    attribute.val.clusterDim.y = attribute.val.clusterDim.z = 1;
    config.attrs = &attribute;
    config.numAttrs = cluster > 1 ? 1 : 0;
    if (s.team() == kCluster) {
        int resident = 0;
        const cudaError_t e = cudaOccupancyMaxActiveClusters(&resident, kernel, &config);
        if (e != cudaSuccess) return e;
        if (resident > 0 && grid > (size_t)resident) grid = (size_t)resident;
        config.gridDim.x = (unsigned)(grid * s.blocks);
    }
    return cudaLaunchKernelEx(&config, kernel, args...);
}

// Launched while the pass still runs: its start-up is over when the sums are there.
// About eight partial sums a thread, more where 1024 threads a multiprocessor do not reach: with 32 threads a
// column always 8192 x 5120 bfloat16 60.0 us, so 57.1; 300 x 4096 10.8, so 9.9; with 8 always 8192 x 2048 27.4,
// so 26.0.
template <typename W, typename P>
cudaError_t launch_join(const W *partial, size_t blocks, int cols, void *dweight, void *dbias, int sms,
                        cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((cols + kJoinColumns - 1) / kJoinColumns), dbias != nullptr ? 2 : 1);
    const size_t columns = (size_t)config.gridDim.x * config.gridDim.y * kJoinColumns, threads = (size_t)sms * 1024;
    int parts = 8;
    while (parts < 1024 / kJoinColumns && (size_t)parts * 8 < blocks && columns * parts * 2 <= threads) parts *= 2;
    config.blockDim = dim3((unsigned)(kJoinColumns * parts));
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, join_columns_kernel<W, P>, partial, (int)blocks, cols, dweight, dbias);
}

#endif

}  // namespace layers
}  // namespace geo
