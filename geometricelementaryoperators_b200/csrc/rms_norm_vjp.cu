// rms_norm_vjp.cu -- VJPs of RMS norm and of the norms before and after a block
// (geo/geo_b200.h section 5); entry points in rms_norm.cu.
//
// RMS norm, xh = x r, g = y_bar w: x_bar = r (g - xh mean(g xh)), w_bar = sum y_bar xh.
// Block norm, zh = z rz, g = y_bar pre, s = beta act(gate), q = s xh post:
//   dz = rz (g - zh c1) + z_bar,  c1 = mean(g zh),
//   x_bar = rx (s post dz - xh c2),  c2 = mean(q dz).
// dz is linear in c1, so c2 = mean(q (rz g + z_bar)) - rz c1 mean(q zh): three sums and
// one exchange across a row's team instead of two. (Nothing is lost to it: where the
// difference cancels, dz itself is the difference of the same terms.) Every array is read
// and written once; HBM bounds it. The weights' cotangents are summed as in layer norm:
// in the registers of the thread that owns the column, then over teams and blocks.
// Measured: block norm with a sigmoid gate 16384 x 4096 bfloat16 224 us (73% of the copy
// bandwidth: 70 instructions a value, a third of them the gate's, on 62% of the issue
// slots of 16 warps); RMS norm 3001 x 1003 float32 off 16 bytes 18.4 us.
#include "rms_norm.h"

#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

// Zeroes the values of the thread's vector i that lie past the row's end (all when not `live`).
template <typename T, int V, int K, int TEAM>
__device__ __forceinline__ void cut(Vec<T, V> &v, int i, const Place<TEAM, V, K> &at, bool live, int cols) {
    const int left = live ? cols - at.column(i) : 0;
    if (left >= V) return;
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
        const Pair<Wide<T>> p = v.pair(q);
        v.set(q, {2 * q < left ? p.x : Wide<T>(0), 2 * q + 1 < left ? p.y : Wide<T>(0)});
    }
}

// Blocks a multiprocessor holds: 512 threads of up to 128 registers. A block norm's
// passes within a warp, whose columns' places vary, want 170 of them.
constexpr int resident_blocks(int mode, int team) {
    return team == kWarp ? (mode == kRms ? 4 : 3) : 2;
}

// The arrays in the ring: x, y_bar, then (block norm) z, the gate, z_bar, as far as they are there.
template <typename T, int MODE, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
__global__ void __launch_bounds__(TEAM == kWarp ? kWarpBlock : kTeamThreads, resident_blocks(MODE, TEAM))
    rms_vjp_kernel(const RmsBackwardArgs a, int lanes, bool float_parameters, int stages, Wide<T> *partial, bool alone) {
    using W = Wide<T>;
    constexpr int V = 16 / (int)sizeof(T), K = values_per_thread(sizeof(T)) / V, Q = K * V / 2;
    constexpr int R = MODE == kRms ? rows_at_once(sizeof(T), SHIFT, TEAM) : 1, N = MODE == kRms ? R : 4;
    constexpr bool kBlocks = MODE >= kBlockNorm, kGates = MODE == kGatedNorm, kFast = sizeof(T) == 2;
    extern __shared__ __align__(128) unsigned char memory[];
    __shared__ Exchange<W, N, TEAM> sums;
    const Place<TEAM, V, K> at(lanes);
    const bool has_dz = kBlocks && a.dz != nullptr;
    constexpr int kDz = kGates ? 4 : 3;
    Ring<T, V, K, TEAM, SHIFT, FULL, R> ring(memory, stages, kBlocks ? kDz + (has_dz ? 1 : 0) : 2, at, a.rows, a.cols);
    auto next = [&] {
        ring.copy(0, (const T *)a.x, a.x_stride);
        ring.copy(1, (const T *)a.dy, a.dy_stride);
        if constexpr (kBlocks) {
            ring.copy(2, (const T *)a.z, a.z_stride);
            if constexpr (kGates) ring.copy(3, (const T *)a.gate, a.gate_stride);
            if (has_dz) ring.copy(kDz, (const T *)a.dz, a.dz_stride);
        }
        ring.fetched();
    };
    for (int s = 0; s < stages - R; ++s) next();

    const W over = W(1) / (W)a.cols, alpha = (W)a.residual_scale, beta = (W)a.block_scale;
    Pair<W> w[Q], dw[Q], post[kBlocks ? Q : 1], dpost[Q];
    load_parameters<T, V, K, SHIFT>(a.weight, float_parameters, at, a.cols, W(1), w);
    if constexpr (kBlocks) {
        load_parameters<T, V, K, SHIFT>(a.post, float_parameters, at, a.cols, W(1), post);
#pragma unroll
        for (int q = 0; q < Q; ++q) post[q] = post[q] * both(beta);  // wherever it stands below, block_scale does too
    }
#pragma unroll
    for (int q = 0; q < Q; ++q) dw[q] = dpost[q] = both(W(0));

    // A row past the last one is zeros with rstd zero: it adds nothing.
    W next_rstd[R], next_x_rstd = W(0);
    auto statistics = [&](size_t first) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = first + at.within + u * at.step;
            next_rstd[u] = row < a.rows ? ((const W *)a.rstd)[row] : W(0);
            if constexpr (kBlocks) next_x_rstd = row < a.rows ? ((const W *)a.x_rstd)[row] : W(0);
        }
    };
    statistics(at.begin);
    open_exchange(sums);
    uint32_t round = 0;
    bool complete = true;  // no wait for the cluster gave up
    for (size_t first = at.begin; first < a.rows; first += R * at.step, ++round) {
        W rstd[R], part[N];
        const W x_rstd = next_x_rstd;
#pragma unroll
        for (int u = 0; u < R; ++u) rstd[u] = next_rstd[u];
        statistics(first + R * at.step);
        for (int u = 0; u < R; ++u) next();
        ring.wait();
        auto row_of = [&](int u) { return first + at.within + u * at.step; };
        // Vector i of an array of row u, zeros past the row's end.
        auto vector = [&](int i, int u, int array, const void *p, size_t stride) {
            const size_t row = row_of(u), r = row < a.rows ? row : 0;
            Vec<T, V> v = ring.get_one(i, u, array, (const T *)p + r * stride);
            if constexpr (SHIFT) cut(v, i, at, row < a.rows, a.cols);
            return v;
        };
        if constexpr (!kBlocks) {
#pragma unroll
            for (int u = 0; u < R; ++u) {
                Pair<W> along = both(W(0));
#pragma unroll
                for (int i = 0; i < K; ++i) {
                    const Vec<T, V> x = vector(i, u, 0, a.x, a.x_stride), dy = vector(i, u, 1, a.dy, a.dy_stride);
#pragma unroll
                    for (int q = 0; q < V / 2; ++q) {
                        const int n = i * V / 2 + q;
                        const Pair<W> xh = x.pair(q) * both(rstd[u]), d = dy.pair(q);
                        along = fma(d * w[n], xh, along);
                        dw[n] = fma(d, xh, dw[n]);
                    }
                }
                part[u] = along.x + along.y;
            }
        } else {
            Pair<W> s1 = both(W(0)), s2 = both(W(0)), s3 = both(W(0));
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const Vec<T, V> x = vector(i, 0, 0, a.x, a.x_stride), dy = vector(i, 0, 1, a.dy, a.dy_stride),
                                z = vector(i, 0, 2, a.z, a.z_stride);
                Vec<T, V> gate = Vec<T, V>::zero(), dz = Vec<T, V>::zero();
                if constexpr (kGates) gate = vector(i, 0, 3, a.gate, a.gate_stride);
                if (has_dz) dz = vector(i, 0, kDz, a.dz, a.dz_stride);
                Pair<W> act[V / 2], none[V / 2];
                if constexpr (kGates) gate_values<kFast, false>(a.gate_kind, gate, act, none);
#pragma unroll
                for (int q = 0; q < V / 2; ++q) {
                    const int n = i * V / 2 + q;
                    const Pair<W> zh = z.pair(q) * both(rstd[0]), d = dy.pair(q), g = d * w[n];
                    Pair<W> f = x.pair(q) * both(x_rstd) * post[n];
                    if constexpr (kGates) f = f * act[q];
                    s1 = fma(g, zh, s1);
                    s2 = fma(f, fma(g, both(rstd[0]), dz.pair(q)), s2);
                    s3 = fma(f, zh, s3);
                    dw[n] = fma(d, zh, dw[n]);
                }
            }
            part[0] = s1.x + s1.y;
            part[1] = s2.x + s2.y;
            part[2] = s3.x + s3.y;
            part[3] = W(0);
        }
        complete = team_sums<N>(sums, round, at, part, complete, STARVE ? a.starve.polls : kWaitPolls,
                                STARVE && round == a.starve.round && at.rank == at.ranks - 1);
        if constexpr (!kBlocks) {
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const size_t row = row_of(u);
                const bool live = (TEAM != kWarp && u == 0) || row < a.rows;
                if (a.dx == nullptr) continue;
                Vec<T, V> out[K];
#pragma unroll
                for (int i = 0; i < K; ++i) {
                    const Vec<T, V> x = vector(i, u, 0, a.x, a.x_stride), dy = vector(i, u, 1, a.dy, a.dy_stride);
#pragma unroll
                    for (int q = 0; q < V / 2; ++q) {
                        const Pair<W> xh = x.pair(q) * both(rstd[u]);
                        out[i].set(q, fma(xh, both(-part[u] * over), dy.pair(q) * w[i * V / 2 + q]) * both(rstd[u]));
                    }
                }
                ring.put((T *)a.dx + row * a.dx_stride, live, u, 0, out);
            }
        } else {
            const size_t row = row_of(0);
            const bool live = TEAM != kWarp || row < a.rows;
            const W c1 = part[0] * over, c2 = ::fma(-rstd[0] * c1, part[2] * over, part[1] * over);
            // Off 16 bytes outputs go through the inputs' places, once every lane has read them.
            Vec<T, V> kept[3][SHIFT ? K : 1];
            auto put = [&](int which, int i, void *p, size_t stride, const Vec<T, V> &v) {
                if constexpr (SHIFT) {
                    kept[which][i] = v;
                } else {
                    if (p != nullptr && live && (FULL || at.column(i) < a.cols))
                        store<T, V>((T *)p + row * stride + at.column(i), v);
                }
            };
#pragma unroll
            for (int i = 0; i < K; ++i) {
                const Vec<T, V> x = vector(i, 0, 0, a.x, a.x_stride), dy = vector(i, 0, 1, a.dy, a.dy_stride),
                                z = vector(i, 0, 2, a.z, a.z_stride);
                Vec<T, V> gate = Vec<T, V>::zero(), dzs = Vec<T, V>::zero(), dresidual, dx, dgate;
                if constexpr (kGates) gate = vector(i, 0, 3, a.gate, a.gate_stride);
                if (has_dz) dzs = vector(i, 0, kDz, a.dz, a.dz_stride);
                Pair<W> act[V / 2], slope[V / 2];
                if constexpr (kGates) gate_values<kFast, true>(a.gate_kind, gate, act, slope);
#pragma unroll
                for (int q = 0; q < V / 2; ++q) {
                    const int n = i * V / 2 + q;
                    const Pair<W> zh = z.pair(q) * both(rstd[0]);
                    const Pair<W> dz = fma(fma(zh, both(-c1), dy.pair(q) * w[n]), both(rstd[0]), dzs.pair(q));
                    const Pair<W> xh = x.pair(q) * both(x_rstd);
                    Pair<W> dn = dz;  // without block_scale
                    dresidual.set(q, dz * both(alpha));
                    if constexpr (kGates) {
                        dgate.set(q, dn * (xh * post[n]) * slope[q]);
                        dn = dn * act[q];
                    }
                    dpost[n] = fma(dn, xh, dpost[n]);
                    dx.set(q, fma(xh, both(-c2), dn * post[n]) * both(x_rstd));
                }
                put(0, i, a.dresidual, a.dresidual_stride, dresidual);
                put(1, i, a.dx, a.dx_stride, dx);
                if constexpr (kGates) put(2, i, a.dgate, a.dgate_stride, dgate);
            }
            if constexpr (SHIFT) {
                if (a.dresidual != nullptr)
                    ring.put((T *)a.dresidual + row * a.dresidual_stride, live, 0, 0, kept[0]);
                if (a.dx != nullptr) ring.put((T *)a.dx + row * a.dx_stride, live, 0, 1, kept[1]);
                if constexpr (kGates)
                    if (a.dgate != nullptr) ring.put((T *)a.dgate + row * a.dgate_stride, live, 0, 2, kept[2]);
            }
        }
        ring.done();
    }
    wait_async<0>();
    close_exchange<TEAM>();
    if (partial == nullptr) return;
    if constexpr (kBlocks) {
#pragma unroll
        for (int q = 0; q < Q; ++q) dpost[q] = dpost[q] * both(beta);
    }
    if (!complete) {
#pragma unroll
        for (int q = 0; q < Q; ++q) dw[q] = dpost[q] = both((W)NAN);
    }
    leave_column_sums<T, TEAM, V, K>(at, dw, dpost, (W *)memory, partial, alone, lanes, a.cols, a.dweight, a.dpost,
                                     float_parameters);
}

// ---- rows of any length --------------------------------------------------------

// For rows beyond eight blocks of threads (32768 values, 16384 in float64): one CTA a
// row. What a row's sums come to, on every thread of its CTA.
template <typename W>
struct RowSums {
    W c1, c2;  // kRms: c1 alone, mean(g xh)
};
template <typename T, typename P, int MODE>
struct AnyRow {
    using W = Wide<T>;
    const RmsBackwardArgs &a;
    size_t row;
    W rstd, x_rstd, beta;
    __device__ __forceinline__ AnyRow(const RmsBackwardArgs &a, size_t row)
        : a(a), row(row), rstd(((const W *)a.rstd)[row]),
          x_rstd(MODE == kRms ? rstd : ((const W *)a.x_rstd)[row]), beta((W)a.block_scale) {}
    __device__ __forceinline__ W at(const void *p, size_t stride, int c) const {
        return widen(((const T *)p)[row * stride + c]);
    }
    __device__ __forceinline__ W parameter(const void *p, int c) const {
        return p != nullptr ? (W)widen(((const P *)p)[c]) : W(1);
    }
    __device__ __forceinline__ W xh(int c) const { return at(a.x, a.x_stride, c) * x_rstd; }
    __device__ __forceinline__ W zh(int c) const { return MODE == kRms ? xh(c) : at(a.z, a.z_stride, c) * rstd; }
    __device__ __forceinline__ W g(int c) const { return at(a.dy, a.dy_stride, c) * parameter(a.weight, c); }
    __device__ __forceinline__ W dz_in(int c) const { return a.dz != nullptr ? at(a.dz, a.dz_stride, c) : W(0); }
    __device__ __forceinline__ W gate(int c, W *slope) const {
        if constexpr (MODE != kGatedNorm) return W(1);
        return gate_value<sizeof(T) == 2>(a.gate_kind, at(a.gate, a.gate_stride, c), slope);
    }
    __device__ __forceinline__ W dz(int c, W c1) const { return ::fma(g(c) - zh(c) * c1, rstd, dz_in(c)); }
    __device__ RowSums<W> sums(W *scratch) const {
        if constexpr (MODE == kRms) {
            const W sum = long_sum<W>((int)threadIdx.x, a.cols, kThreads, [&](W &s, int c) { s += g(c) * xh(c); });
            return {block_sum(sum, scratch) / (W)a.cols, W(0)};
        } else {
            const W first = long_sum<W>((int)threadIdx.x, a.cols, kThreads, [&](W &s, int c) { s += g(c) * zh(c); });
            const W c1 = block_sum(first, scratch) / (W)a.cols;
            const W second = long_sum<W>((int)threadIdx.x, a.cols, kThreads, [&](W &s, int c) {
                s += gate(c, nullptr) * beta * parameter(a.post, c) * xh(c) * dz(c, c1);
            });
            return {c1, block_sum(second, scratch) / (W)a.cols};
        }
    }
};

template <typename T, typename P, int MODE>
__global__ void __launch_bounds__(kThreads, 4) rms_vjp_rows_any_kernel(const RmsBackwardArgs a) {
    using W = Wide<T>;
    __shared__ W scratch[kThreads / 32];
    for (size_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        const AnyRow<T, P, MODE> row(a, n);
        const RowSums<W> s = row.sums(scratch);
        auto put = [&](void *p, size_t stride, int c, W v) {
            if (p != nullptr) ((T *)p)[n * stride + c] = narrow<T>(v);
        };
        for (int c = threadIdx.x; c < a.cols; c += kThreads) {
            const W xh = row.xh(c);
            if constexpr (MODE == kRms) {
                put(a.dx, a.dx_stride, c, (row.g(c) - xh * s.c1) * row.rstd);
            } else {
                W slope = W(0);
                const W dz = row.dz(c, s.c1), f = row.gate(c, &slope), post = row.parameter(a.post, c),
                        dn = dz * row.beta;
                put(a.dx, a.dx_stride, c, (dn * f * post - xh * s.c2) * row.x_rstd);
                if constexpr (MODE == kGatedNorm) put(a.dgate, a.dgate_stride, c, dn * (xh * post) * slope);
                put(a.dresidual, a.dresidual_stride, c, dz * (W)a.residual_scale);
            }
        }
    }
}

// c1 of every row, which the columns' sums need.
template <typename T, typename P, int MODE>
__global__ void __launch_bounds__(kThreads, 4) rms_vjp_means_any_kernel(const RmsBackwardArgs a, Wide<T> *means) {
    using W = Wide<T>;
    __shared__ W scratch[kThreads / 32];
    for (size_t n = blockIdx.x; n < a.rows; n += gridDim.x) {
        const AnyRow<T, P, MODE> row(a, n);
        const W sum = long_sum<W>((int)threadIdx.x, a.cols, kThreads,
                                  [&](W &s, int c) { s += row.g(c) * row.zh(c); });
        const W total = block_sum(sum, scratch);
        if (threadIdx.x == 0) means[n] = total / (W)a.cols;
    }
}

// Partial sums over rows [first, last) of block column range blockIdx.x:
// partial[blockIdx.y][0: weight, 1: post weight][col].
template <typename T, typename P, int MODE>
__global__ void __launch_bounds__(kThreads) rms_vjp_columns_any_kernel(const RmsBackwardArgs a, const Wide<T> *means,
                                                                       Wide<T> *partial, size_t rows_per_block) {
    using W = Wide<T>;
    __shared__ W sums[2][8][33];
    const int lane = threadIdx.x & 31, group = threadIdx.x >> 5;
    const int c = (int)blockIdx.x * 32 + lane;
    const size_t first = blockIdx.y * rows_per_block;
    const size_t last = first + rows_per_block < a.rows ? first + rows_per_block : a.rows;
    Pair<W> found = {};
    if (c < a.cols)
        found = long_sum<Pair<W>>(first + group, last, (size_t)8, [&](Pair<W> &s, size_t n) {
            const AnyRow<T, P, MODE> row(a, n);
            s.x += row.at(a.dy, a.dy_stride, c) * row.zh(c);
            if constexpr (MODE != kRms) s.y += row.gate(c, nullptr) * row.beta * row.dz(c, means[n]) * row.xh(c);
        });
    sums[0][group][lane] = found.x;
    sums[1][group][lane] = found.y;
    __syncthreads();
    if (group < 2 && c < a.cols) {
        W total = 0;
        for (int i = 0; i < 8; ++i) total += sums[group][i][lane];
        partial[((size_t)blockIdx.y * 2 + group) * a.cols + c] = total;
    }
}

// Row blocks of the column sums: enough for four CTAs per SM, at least 64 rows each.
size_t column_blocks(size_t rows, size_t cols) {
    const size_t wide = (cols + 31) / 32, want = ((size_t)geo::device_sm_count() * 4 + wide - 1) / wide;
    const size_t most = (rows + 63) / 64;
    return want < most ? want : most;
}

// Rows that a team takes at a time, and teams (blocks of teams) of the pass.
int at_once_of(NormMode mode, size_t bytes, const Shape &s) {
    return mode == kRms ? rows_at_once(bytes, s.shift, s.team()) : 1;
}
size_t team_grid(NormMode mode, const Shape &s, size_t bytes, size_t rows) {
    const size_t each = s.teams() * at_once_of(mode, bytes, s), wanted = (rows + each - 1) / each;
    const int resident = s.team() == kWarp ? resident_blocks(mode, kWarp) : 512 / s.threads();
    const size_t most = (size_t)geo::device_sm_count() * resident / s.blocks;
    return wanted < most ? wanted : most;
}

// Rows in the ring. A block norm has up to five arrays: of float32 and float64 rows
// only the one being read fits (the multiprocessor's other block is then what loads
// meanwhile).
int stages_of(NormMode mode, int at_once, size_t stage, int threads) {
    if (mode == kRms) return ring_stages(stage, at_once, threads, 512);
    const int n = (int)((size_t)110 * 1024 * threads / 256 / stage);
    return n > 4 ? 4 : (n > 1 ? n : 1);
}

template <typename T, int MODE, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
cudaError_t launch_shape(const Shape &s, const RmsBackwardArgs &a, bool float_parameters, Wide<T> *partial, bool alone,
                         size_t &blocks, cudaStream_t stream) {
    const int arrays = MODE == kRms ? 2 : 3 + (MODE == kGatedNorm) + (a.dz != nullptr);
    const size_t stage = arrays * s.part(sizeof(T));
    const int stages = stages_of((NormMode)MODE, at_once_of((NormMode)MODE, sizeof(T), s), stage, s.threads());
    return launch_team(rms_vjp_kernel<T, MODE, TEAM, SHIFT, FULL, STARVE>, s, blocks, alone ? blocks : s.blocks, stages * stage,
                       stream, a, s.lanes, float_parameters, stages, partial, alone);
}

}  // namespace

// Enough for whatever alignment the arrays turn out to have.
size_t rms_vjp_workspace(NormTypes t, NormMode mode, size_t rows, size_t cols) {
    const size_t bytes = type_bytes(t.type), wide = wide_bytes(t.type);
    size_t blocks = 0, means = 0;
    for (const bool aligned : {false, true}) {
        if (aligned && cols * bytes % 16 != 0) continue;
        const Shape s = shape_of(cols, bytes, aligned);
        const size_t n = s.lanes != 0 ? team_grid(mode, s, bytes, rows) : column_blocks(rows, cols);
        if (n > blocks) blocks = n;
        if (s.lanes == 0 && mode != kRms) means = rows * wide;
    }
    return blocks * 2 * cols * wide + means;
}

cudaError_t launch_rms_vjp(NormTypes n, NormMode mode, const RmsBackwardArgs &a, void *workspace, cudaStream_t stream) {
    const bool sums = a.dweight != nullptr || a.dpost != nullptr;
    const size_t bytes = type_bytes(n.type);
    const bool aligned = aligned16(a.cols, bytes, type_bytes(n.parameter_type),
                                   {{a.x, a.x_stride}, {a.z, a.z_stride}, {a.gate, a.gate_stride}, {a.dy, a.dy_stride},
                                    {a.dz, a.dz_stride}, {a.dresidual, a.dresidual_stride}, {a.dx, a.dx_stride},
                                    {a.dgate, a.dgate_stride}},
                                   {a.post, a.weight});
    const Shape s = shape_of(a.cols, bytes, aligned);
    const bool float_parameters = n.parameter_type == GEO_B200_F32;
    return by_mode(mode, [&](auto m) {
        constexpr int MODE = decltype(m)::value;
        return by_types(n, [&](auto t, auto p) {
            using T = decltype(t);
            using P = decltype(p);
            using W = Wide<T>;
            W *partial = sums ? (W *)workspace : nullptr;
            size_t blocks = 0;
            bool alone = false;
            cudaError_t e = cudaSuccess;
            if (s.lanes != 0) {
                blocks = team_grid(mode, s, bytes, a.rows);
                // A grid of at most eight blocks is one cluster and joins its own sums.
                alone = sums && s.team() != kCluster && blocks <= kAloneBlocks;
                e = by_shape(s, [&](auto team, auto shift, auto full) {
                    return launch_shape<T, MODE, decltype(team)::value, decltype(shift)::value, decltype(full)::value>(
                        s, a, float_parameters, partial, alone, blocks, stream);
                });
            } else {
                const unsigned grid = (unsigned)(a.rows < (1u << 20) ? a.rows : (1u << 20));
                // Columns first: the row kernel may overwrite what they read.
                if (sums) {
                    blocks = column_blocks(a.rows, a.cols);
                    W *means = partial + blocks * 2 * a.cols;
                    if constexpr (MODE != kRms)
                        rms_vjp_means_any_kernel<T, P, MODE><<<grid, kThreads, 0, stream>>>(a, means);
                    const dim3 columns((unsigned)((a.cols + 31) / 32), (unsigned)blocks);
                    rms_vjp_columns_any_kernel<T, P, MODE>
                        <<<columns, kThreads, 0, stream>>>(a, means, partial, (a.rows + blocks - 1) / blocks);
                }
                if (a.dx != nullptr || a.dresidual != nullptr || a.dgate != nullptr)
                    rms_vjp_rows_any_kernel<T, P, MODE><<<grid, kThreads, 0, stream>>>(a);
                e = cudaGetLastError();
            }
            if (e != cudaSuccess || !sums || alone) return e;
            return launch_join<W, P>(partial, blocks, a.cols, a.dweight, a.dpost, geo::device_sm_count(), stream);
        });
    });
}

cudaError_t launch_rms_vjp_starved(const RmsBackwardArgs &a, void *workspace, cudaStream_t stream) {
    const Shape s = shape_of(a.cols, 4, true);
    float *const partial = (float *)workspace;
    size_t blocks = team_grid(kBlockNorm, s, 4, a.rows);
    const cudaError_t e = launch_shape<float, kBlockNorm, kCluster, false, true, true>(s, a, true, partial, false, blocks,
                                                                                      stream);
    return e != cudaSuccess ? e : launch_join<float, float>(partial, blocks, a.cols, a.dweight, a.dpost,
                                                             geo::device_sm_count(), stream);
}

}  // namespace layers
}  // namespace geo
