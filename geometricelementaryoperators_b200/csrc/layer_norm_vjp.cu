// layer_norm_vjp.cu -- VJPs of layer norm, alone and behind residual + dropout
// (geo/geo_b200.h section 5); entry points in layer_norm.cu.
//
// With xh = (x - m) rstd and g = y_bar w (means over the row):
//   x_bar = rstd (g - mean(g) - xh mean(g xh)),
//   w_bar = sum_rows y_bar xh, b_bar = sum_rows y_bar.
// One pass reads x and y_bar once and writes x_bar once: HBM bounds it. The column
// sums stay with the thread that owns the column over all rows of its team, so
// what is added up at the end is one partial sum a block, in a fixed order.
// Measured on two boards, calls in turn over three sets of arrays, host included:
// 2^19 x 64 float64 136 and 140 us (5.8 TB/s, 89% of the copy bandwidth on the slower
// one), 16384 x 4096 bfloat16 behind residual + dropout 120 and 129 us (5.2 TB/s, 80%:
// 35 instructions a value, a third of them dropout's, on 61% of the issue slots),
// 3001 x 1003 float32 off 16 bytes 20 us (two and a half rows a team: start-up and
// joining are half of it).
#include "layer_norm.h"

#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

// One pass over x and y_bar (and z_bar): x_bar row by row, and the column sums
// of y_bar xh and y_bar in the registers of the thread that owns the column; at
// the end partial[block or cluster][0: weight, 1: bias][col], the teams of a
// block added up in shared memory. `alone`: the grid is one cluster, whose blocks
// add the partial sums up themselves, and no second kernel is needed.
constexpr int kAloneBlocks = 8;
template <typename T, bool DROP, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
__global__ void __launch_bounds__(TEAM == kWarp ? kWarpBlock : kTeamThreads, TEAM == kWarp ? 4 : 2)
    vjp_kernel(const BackwardArgs a, int lanes, bool float_parameters, int stages, Wide<T> *partial, bool alone) {
    using W = Wide<T>;
    constexpr int V = 16 / (int)sizeof(T), K = values_per_thread(sizeof(T)) / V, Q = K * V / 2;
    constexpr int R = rows_at_once(sizeof(T), SHIFT, TEAM);
    extern __shared__ __align__(128) unsigned char memory[];  // a row of copies or reads is whole 128-byte lines
    __shared__ Exchange<W, 2 * R, TEAM> sums;
    __shared__ unsigned char drop_bytes[SHIFT && DROP ? kDropBytes : 1];
    const Place<TEAM, V, K> at(lanes);
    const bool has_dz = DROP && a.dz != nullptr;
    Ring<T, V, K, TEAM, SHIFT, FULL, R> ring(memory, stages, has_dz ? 3 : 2, at, a.rows, a.cols);
    auto next = [&] {
        ring.copy(0, (const T *)a.x, a.x_stride);
        ring.copy(1, (const T *)a.dy, a.dy_stride);
        if constexpr (DROP)
            if (has_dz) ring.copy(2, (const T *)a.dz, a.dz_stride);
        ring.fetched();
    };
    for (int s = 0; s < stages - R; ++s) next();

    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const W scale = (W)a.drop.scale, over = W(1) / (W)a.cols;
    Pair<W> w[Q], dw[Q], db[Q];
    load_parameters<T, V, K, SHIFT>(a.weight, float_parameters, at, a.cols, W(1), w);
#pragma unroll
    for (int q = 0; q < Q; ++q) dw[q] = db[q] = both(W(0));

    // A row past the last one is zeros with mean and rstd zero: it adds nothing.
    W next_mean[R], next_rstd[R];
    auto statistics = [&](size_t first) {
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = first + at.within + u * at.step;
            next_mean[u] = row < a.rows ? ((const W *)a.mean)[row] : W(0);
            next_rstd[u] = row < a.rows ? ((const W *)a.rstd)[row] : W(0);
        }
    };
    statistics(at.begin);
    open_exchange(sums);
    uint32_t round = 0;
    bool complete = true;  // no wait for the cluster gave up
    for (size_t first = at.begin; first < a.rows; first += R * at.step, ++round) {
        W mean[R], rstd[R], part[2 * R];
#pragma unroll
        for (int u = 0; u < R; ++u) mean[u] = next_mean[u], rstd[u] = next_rstd[u];
        statistics(first + R * at.step);
        for (int u = 0; u < R; ++u) next();
        ring.wait();
        Vec<T, V> x[K], dy[K];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = first + at.within + u * at.step, r = row < a.rows ? row : 0;
            ring.get(x, u, 0, (const T *)a.x + r * a.x_stride);
            ring.get(dy, u, 1, (const T *)a.dy + r * a.dy_stride);
            Pair<W> sum = both(W(0)), along = both(W(0));
            auto add = [&](int q, Pair<W> d, Pair<W> xh) {
                const Pair<W> g = d * w[q];
                sum = sum + g;
                along = fma(g, xh, along);
                dw[q] = fma(d, xh, dw[q]);
                db[q] = db[q] + d;
            };
            if constexpr (SHIFT) {
                Pair<W> d[Q], xh[Q];
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    d[q] = pair_at(dy, q);
                    xh[q] = (pair_at(x, q) + both(-mean[u])) * both(rstd[u]);
                }
                set_past(d, at, row < a.rows, a.cols, W(0));
                set_past(xh, at, row < a.rows, a.cols, W(0));
#pragma unroll
                for (int q = 0; q < Q; ++q) add(q, d[q], xh[q]);
            } else {
#pragma unroll
                for (int q = 0; q < Q; ++q) {
                    // Past the row x and y_bar are 0, but (0 - mean) rstd may overflow where no value of the row does,
                    // and 0 inf would reach the sums: it is left out in float64 within a warp (2^18 x 72: 84 us, 100
                    // with rstd 0), elsewhere worked out with rstd 0 (the fused pass there 169 us, 188 left out; 65536 x
                    // 200 float16 fused 43.7, 47.3).
                    constexpr bool kLeave = TEAM == kWarp && sizeof(T) == 8 && !DROP;
                    const bool inside = FULL || at.column(2 * q / V) < a.cols;
                    if (kLeave && !inside) continue;
                    const W r = kLeave || inside ? rstd[u] : W(0);
                    add(q, pair_at(dy, q), (pair_at(x, q) + both(-mean[u])) * both(r));
                }
            }
            part[2 * u] = sum.x + sum.y;
            part[2 * u + 1] = along.x + along.y;
        }
        if constexpr (TEAM == kWarp) {
            part[0] = team_sum(part[0], at.threads) * over;
            part[1] = team_sum(part[1], at.threads) * over;
        } else {
            complete = exchange(sums, round, at, folded_sums(part), complete, STARVE ? a.starve.polls : kWaitPolls,
                                STARVE && round == a.starve.round && at.rank == at.ranks - 1);
            constexpr int kJoin = 32 / (2 * R);  // lanes that add one value up
            W total = 0;
#pragma unroll
            for (int j = 0; j < (TEAM == kCluster ? 64 / kJoin : 1); ++j) {
                const int e = at.wlane % kJoin + j * kJoin;
                if (e < at.entries) total += sums.values[round & 1][at.wlane / kJoin][at.first_entry + e];
            }
            total = team_sum(total, kJoin) * over;
            if (!complete) total = (W)NAN;
#pragma unroll
            for (int n = 0; n < 2 * R; ++n) part[n] = __shfl_sync(0xffffffffu, total, n * kJoin);
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = first + at.within + u * at.step, r = row < a.rows ? row : 0;
            const bool live = (TEAM != kWarp && u == 0) || row < a.rows;
            if constexpr (TEAM != kWarp) {  // read again rather than held over the barrier: registers
                ring.get(x, u, 0, (const T *)a.x + r * a.x_stride);
                ring.get(dy, u, 1, (const T *)a.dy + r * a.dy_stride);
            }
            Pair<W> v[Q];
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const Pair<W> xh = (pair_at(x, q) + both(-mean[u])) * both(rstd[u]);
                v[q] = (fma(xh, both(-part[2 * u + 1]), pair_at(dy, q) * w[q]) + both(-part[2 * u])) * both(rstd[u]);
            }
            if constexpr (DROP)
                if (has_dz) {
                    ring.get(x, u, 2, (const T *)a.dz + r * a.dz_stride);
#pragma unroll
                    for (int q = 0; q < Q; ++q) v[q] = v[q] + pair_at(x, q);
                }
            if (a.dsum != nullptr) {
#pragma unroll
                for (int q = 0; q < Q; ++q) set_pair(x, q, v[q]);
                ring.put((T *)a.dsum + row * a.dsum_stride, live, u, 0, x);
            }
            if constexpr (DROP) {
                if (a.dx != nullptr) {
                    drop_row<T, V, K, SHIFT, FULL>(a.drop, offset, row * (size_t)a.cols, at, a.cols, drop_bytes, v);
#pragma unroll
                    for (int q = 0; q < Q; ++q) set_pair(x, q, v[q] * both(scale));
                    ring.put((T *)a.dx + row * a.dx_stride, live, u, 1, x);
                }
            }
        }
        ring.done();
    }
    wait_async<0>();
    close_exchange<TEAM>();
    if (partial == nullptr) return;
    if (!complete) {
#pragma unroll
        for (int q = 0; q < Q; ++q) dw[q] = db[q] = both((W)NAN);
    }
    // The kernel that joins the partial sums may be set up from here on.
    if (!alone) asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    auto value = [&](const Pair<W> (&p)[Q], int e) { return e & 1 ? p[e / 2].y : p[e / 2].x; };
    // Every thread's sums to where the ring was (two rows of it hold two sums of a
    // row; value e of thread t at e threads + (t ^ e): no bank twice), then a
    // column's, the block's teams in order, in whole lines to global memory.
    const int each = blockDim.x, first_column = at.rank * lanes * K * V;
    const int columns = a.cols - first_column < lanes * K * V ? a.cols - first_column : lanes * K * V;
    W *found = (W *)memory, *mine = partial + at.slice * 2 * a.cols + first_column;
    auto place = [&](int e, int thread) { return e * each + (thread ^ (e & 31)); };
    __syncthreads();
#pragma unroll
    for (int e = 0; e < K * V; ++e) {
        found[place(e, threadIdx.x)] = value(dw, e);
        found[each * K * V + place(e, threadIdx.x)] = value(db, e);
    }
    __syncthreads();
    for (int which = 0; which < 2; ++which)
        for (int c = threadIdx.x; c < columns; c += each) {
            const int vector = c / V, unit = TEAM == kWarp ? 0 : vector / (32 * K), in_unit = vector - unit * 32 * K;
            const int round = TEAM == kWarp ? in_unit / at.unit_lanes : in_unit / 32;
            const int e = round * V + c % V, lane = unit * 32 + in_unit - round * at.unit_lanes;
            W sum = 0;
            for (int team = 0; team < at.teams; ++team)
                sum += found[which * each * K * V + place(e, team * lanes + lane)];
            mine[(size_t)which * a.cols + c] = sum;
        }
    if constexpr (TEAM != kCluster) {
        if (!alone) return;
        cooperative_groups::this_cluster().sync();  // makes the blocks' sums visible to one another
        for (int n = blockIdx.x * each + threadIdx.x; n < 2 * a.cols; n += gridDim.x * each) {
            W sum = 0;
#pragma unroll
            for (int block = 0; block < kAloneBlocks; ++block)
                if (block < (int)gridDim.x) sum += partial[(size_t)block * 2 * a.cols + n];
            const int c = n < a.cols ? n : n - a.cols;
            void *out = n < a.cols ? a.dweight : a.dbias;
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

// ---- rows of any length --------------------------------------------------------

// For rows beyond eight blocks of threads (32768 values, 16384 in float64).
// x_bar of one row per CTA, two sweeps; eight CTAs a multiprocessor (4096 x 40000
// bfloat16 559 us, 629 without that bound).
template <typename T, typename P, bool DROP>
__global__ void __launch_bounds__(kThreads, 8) vjp_rows_any_kernel(const BackwardArgs a) {
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
        const Pair<W> both_sums = long_sum<Pair<W>>((int)threadIdx.x, a.cols, kThreads, [&](Pair<W> &s, int c) {
            const W g = scaled(c);
            s.x += g;
            s.y += g * ((widen(x[c]) - mean) * rstd);
        });
        const W sum = block_sum(both_sums.x, scratch) / (W)a.cols;
        const W along = block_sum(both_sums.y, scratch) / (W)a.cols;
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
    Pair<W> found = {};
    if (c < a.cols)
        found = long_sum<Pair<W>>(first + group, last, (size_t)8, [&](Pair<W> &s, size_t row) {
            const W v = widen(((const T *)a.dy)[row * a.dy_stride + c]);
            const W xh = (widen(((const T *)a.x)[row * a.x_stride + c]) - ((const W *)a.mean)[row]) *
                         ((const W *)a.rstd)[row];
            s.x += v * xh;
            s.y += v;
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

// Teams (blocks of teams, kWarp) of the pass: as many as 512 threads a
// multiprocessor make, each with a partial sum of the columns.
size_t team_grid(const Shape &s, size_t bytes, size_t rows) {
    const size_t each = s.teams() * rows_at_once(bytes, s.shift, s.team()), wanted = (rows + each - 1) / each;
    const size_t most = (size_t)geo::device_sm_count() * (512 / s.threads()) / s.blocks;
    return wanted < most ? wanted : most;
}

// The pass of a team kernel; `blocks`: the partial sums it leaves.
template <typename T, bool DROP, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
cudaError_t launch_shape(const Shape &s, const BackwardArgs &a, bool float_parameters, Wide<T> *partial, bool alone,
                         size_t &blocks, cudaStream_t stream) {
    const size_t stage = (a.dz != nullptr ? 3 : 2) * s.part(sizeof(T));
    const int stages = ring_stages(stage, rows_at_once(sizeof(T), SHIFT, TEAM), s.threads(), 512);
    return launch_team(vjp_kernel<T, DROP, TEAM, SHIFT, FULL, STARVE>, s, blocks, alone ? blocks : s.blocks,
                       stages * stage, stream, a, s.lanes, float_parameters, stages, partial, alone);
}

// Launched while the pass still runs: its start-up is over when the sums are there.
// About eight partial sums a thread, more where 1024 threads a multiprocessor do not reach: with 32 threads a
// column always 8192 x 5120 bfloat16 60.0 us, so 57.1; 300 x 4096 10.8, so 9.9; with 8 always 8192 x 2048 27.4,
// so 26.0.
template <typename W, typename P>
cudaError_t launch_join(const BackwardArgs &a, const W *partial, size_t blocks, cudaStream_t stream) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3((unsigned)((a.cols + kJoinColumns - 1) / kJoinColumns), 2);
    const size_t columns = (size_t)config.gridDim.x * 2 * kJoinColumns, threads = (size_t)geo::device_sm_count() * 1024;
    int parts = 8;
    while (parts < 1024 / kJoinColumns && (size_t)parts * 8 < blocks && columns * parts * 2 <= threads) parts *= 2;
    config.blockDim = dim3((unsigned)(kJoinColumns * parts));
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, join_columns_kernel<W, P>, partial, (int)blocks, a.cols, a.dweight, a.dbias);
}

template <bool DROP>
cudaError_t launch(NormTypes n, const BackwardArgs &a, void *workspace, cudaStream_t stream) {
    const bool sums = a.dweight != nullptr || a.dbias != nullptr;
    const size_t bytes = type_bytes(n.type);
    const bool aligned = aligned16(a.cols, bytes, type_bytes(n.parameter_type),
                                   {{a.x, a.x_stride}, {a.dy, a.dy_stride}, {a.dz, a.dz_stride},
                                    {a.dsum, a.dsum_stride}, {a.dx, a.dx_stride}},
                                   {a.weight});
    const Shape s = shape_of(a.cols, bytes, aligned);
    const bool float_parameters = n.parameter_type == GEO_B200_F32;
    return by_types(n, [&](auto t, auto p) {
        using T = decltype(t);
        using P = decltype(p);
        using W = Wide<T>;
        W *partial = sums ? (W *)workspace : nullptr;
        size_t blocks = 0;
        bool alone = false;
        cudaError_t e = cudaSuccess;
        if (s.lanes != 0) {
            blocks = team_grid(s, bytes, a.rows);
            // A grid of at most eight blocks is one cluster (64 x 1024 bfloat16: 5.6 us on the device and one launch, 6.0
            // us and two with a second kernel).
            alone = sums && s.team() != kCluster && blocks <= kAloneBlocks;
            e = by_shape(s, [&](auto team, auto shift, auto full) {
                return launch_shape<T, DROP, decltype(team)::value, decltype(shift)::value, decltype(full)::value>(
                    s, a, float_parameters, partial, alone, blocks, stream);
            });
        } else {
            // Columns first: the row kernel may overwrite x or y_bar.
            if (sums) {
                blocks = column_blocks(a.rows, a.cols);
                const dim3 grid((unsigned)((a.cols + 31) / 32), (unsigned)blocks);
                vjp_columns_any_kernel<T><<<grid, kThreads, 0, stream>>>(a, partial, (a.rows + blocks - 1) / blocks);
            }
            const unsigned grid = (unsigned)(a.rows < (1u << 20) ? a.rows : (1u << 20));
            if (a.dsum != nullptr || a.dx != nullptr)
                vjp_rows_any_kernel<T, P, DROP><<<grid, kThreads, 0, stream>>>(a);
            e = cudaGetLastError();
        }
        if (e != cudaSuccess || !sums || alone) return e;
        return launch_join<W, P>(a, partial, blocks, stream);
    });
}

}  // namespace

// Enough for whatever alignment the arrays turn out to have.
size_t vjp_workspace(NormTypes t, size_t rows, size_t cols) {
    const size_t bytes = type_bytes(t.type);
    size_t blocks = 0;
    for (const bool aligned : {false, true}) {
        if (aligned && cols * bytes % 16 != 0) continue;
        const Shape s = shape_of(cols, bytes, aligned);
        const size_t n = s.lanes != 0 ? team_grid(s, bytes, rows) : column_blocks(rows, cols);
        if (n > blocks) blocks = n;
    }
    return blocks * 2 * cols * wide_bytes(t.type);
}

cudaError_t launch_norm_vjp(NormTypes t, const BackwardArgs &a, bool drop, void *partial, cudaStream_t stream) {
    return drop ? launch<true>(t, a, partial, stream) : launch<false>(t, a, partial, stream);
}

cudaError_t launch_norm_vjp_starved(const BackwardArgs &a, void *partial, cudaStream_t stream) {
    const Shape s = shape_of(a.cols, 4, true);
    size_t blocks = team_grid(s, 4, a.rows);
    const cudaError_t e = launch_shape<float, false, kCluster, false, true, true>(s, a, true, (float *)partial, false,
                                                                                 blocks, stream);
    return e != cudaSuccess ? e : launch_join<float, float>(a, (float *)partial, blocks, stream);
}

}  // namespace layers
}  // namespace geo
