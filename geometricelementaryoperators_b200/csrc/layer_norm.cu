// layer_norm.cu -- layer norm over rows, alone and behind residual + dropout
// (geo/geo_b200.h section 5): entry points and the forward kernels; the backward
// ones are in layer_norm_vjp.cu, what they share in layer_norm.h.
//
// Per row of C values: m = sum x / C, v = sum (x - m)^2 / C,
// y = (x - m) rsqrt(v + epsilon) w + b. A few multiply-adds a value, so HBM bounds
// it; but a 16-bit value comes and goes in four bytes, and at 6.5 TB/s a
// multiprocessor has 22 instructions for each, hence the packed arithmetic, the
// parameters in registers and the few exchanges between threads (11 instructions a
// value, 25 with residual and dropout). What is left to wait for are shared memory
// and fixed latencies, at 16 warps a multiprocessor (half the issue slots are used).
// Measured on two boards, calls in turn over three sets of arrays, host included:
// 8192 x 4096 bfloat16 25 us (5.3 TB/s, 82% of the copy bandwidth), with residual
// and dropout 16384 x 4096 94 and 101 us (5.3 TB/s, 81% on the slower one).
#include "layer_norm.h"

#include <cmath>

#include "geo_runtime.h"

namespace geo {
namespace layers {

Shape shape_of(size_t cols, size_t bytes, bool aligned) {
    Shape s = {!aligned, 0, 1, false};
    const size_t held = values_per_thread(bytes), threads = (cols + held - 1) / held;
    if (threads <= 32) {
        s.lanes = 1;
        while (s.lanes < (int)threads) s.lanes *= 2;
    } else {
        while (threads > (size_t)kTeamThreads * s.blocks) s.blocks *= 2;
        if (s.blocks > 8) return s;
        s.lanes = (int)((threads + s.blocks * 32 - 1) / (s.blocks * 32) * 32);
    }
    s.full = aligned && s.lanes * s.blocks * held == cols;
    return s;
}

bool aligned16(size_t cols, size_t bytes, size_t parameter_bytes, std::initializer_list<RowArray> arrays,
               std::initializer_list<const void *> parameters) {
    if (cols * bytes % 16 != 0) return false;
    for (const RowArray &r : arrays)
        if (r.pointer != nullptr && ((uintptr_t)r.pointer % 16 != 0 || r.stride * bytes % 16 != 0)) return false;
    // Parameters are loaded by 16 bytes at most, at multiples of a vector's worth.
    const size_t need = 16 / bytes * parameter_bytes < 16 ? 16 / bytes * parameter_bytes : 16;
    for (const void *p : parameters)
        if ((uintptr_t)p % need != 0) return false;
    return true;
}

namespace {

// Threads that a multiprocessor holds: 512 of up to 128 registers each. With 768 of
// 80 most kernels spill, and the deeper ring that 512 leave room for feeds them as
// well: 65536 x 200 float64 37.0 us with 512, 46.7 with 768; 2^18 x 65 float64 fused
// 146, 180; 2^19 x 64 bfloat16 fused 50.3, 62.4; 16384 x 3000 float32 68.0, 78.2; 4096
// x 8192 float64 101, 113; 8192 x 4001 float16 fused 96, 105. float32 rows in clusters
// wait for the exchange and want the warps: 4096 x 8192 52.1 us with 512, 48.8 with
// 768; 2048 x 32768 113, 105; with dropout to work on meanwhile they do not (96.5,
// 100.7).
constexpr int resident_threads(size_t bytes, bool drop, bool shift, int team) {
    return bytes == 4 && team == kCluster && !drop && !shift ? 768 : 512;
}

template <typename T, bool DROP, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
__global__ void __launch_bounds__(TEAM == kWarp ? kWarpBlock : kTeamThreads,
                                  resident_threads(sizeof(T), DROP, SHIFT, TEAM) / (TEAM == kWarp ? kWarpBlock : kTeamThreads))
    norm_kernel(const ForwardArgs a, int lanes, bool float_parameters, int stages) {
    using W = Wide<T>;
    constexpr int V = 16 / (int)sizeof(T), K = values_per_thread(sizeof(T)) / V, Q = K * V / 2;
    constexpr int R = rows_at_once(sizeof(T), SHIFT, TEAM);
    extern __shared__ __align__(128) unsigned char memory[];  // a row of copies or reads is whole 128-byte lines
    __shared__ Exchange<W, 2 * R, TEAM> sums;
    __shared__ unsigned char drop_bytes[SHIFT && DROP ? kDropBytes : 1];
    const Place<TEAM, V, K> at(lanes);
    Ring<T, V, K, TEAM, SHIFT, FULL, R> ring(memory, stages, DROP ? 2 : 1, at, a.rows, a.cols);
    auto next = [&] {
        ring.copy(0, (const T *)a.x, a.x_stride);
        if constexpr (DROP) ring.copy(1, (const T *)a.residual, a.residual_stride);
        ring.fetched();
    };
    for (int s = 0; s < stages - R; ++s) next();

    const uint64_t offset = DROP ? drop_offset(a.drop) : 0;
    const W scale = (W)a.drop.scale, over = W(1) / (W)a.cols;
    Pair<W> w[Q], b[Q];
    load_parameters<T, V, K, SHIFT>(a.weight, float_parameters, at, a.cols, W(1), w);
    load_parameters<T, V, K, SHIFT>(a.bias, float_parameters, at, a.cols, W(0), b);

    // How many values of the row warp `n` of the team holds.
    auto held_by = [&](int n) {
        if (FULL) return (W)(32 * K * V);
        const int left = a.cols - n * (32 * K * V);
        return (W)(left < 0 ? 0 : (left < 32 * K * V ? left : 32 * K * V));
    };
    // The team's warps are joined by 8 lanes a row in a block, 32 / R in a cluster, each over every so many warps.
    constexpr int kJoin = TEAM == kCluster ? 32 / R : 8, kEach = TEAM == kCluster ? 64 / kJoin : 1;
    const int joiner = at.wlane % kJoin, joined_row = at.wlane / kJoin % R;
    const W held = TEAM == kWarp ? (W)a.cols : held_by(at.warp);
    const W over_held = held > W(0) ? W(1) / held : W(0);
    W joined[kEach], over_joined[kEach];
#pragma unroll
    for (int j = 0; j < kEach; ++j) {
        joined[j] = joiner + j * kJoin < at.entries ? held_by(joiner + j * kJoin) : W(0);
        over_joined[j] = joined[j] > W(0) ? W(1) / joined[j] : W(0);
    }
    open_exchange(sums);

    uint32_t round = 0;
    bool complete = true;  // no wait for the cluster gave up
    for (size_t first = at.begin; first < a.rows; first += R * at.step, ++round) {
        for (int u = 0; u < R; ++u) next();
        ring.wait();
        Pair<W> v[R][Q];
        W sum[R], mean[R], squares[R];
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = first + at.within + u * at.step, r = row < a.rows ? row : 0;
            Vec<T, V> raw[K];
            ring.get(raw, u, 0, (const T *)a.x + r * a.x_stride);
#pragma unroll
            for (int q = 0; q < Q; ++q) v[u][q] = pair_at(raw, q);
            if constexpr (DROP) {
                drop_row<T, V, K, SHIFT, FULL>(a.drop, offset, row * (size_t)a.cols, at, a.cols, drop_bytes, v[u]);
                ring.get(raw, u, 1, (const T *)a.residual + r * a.residual_stride);
#pragma unroll
                for (int q = 0; q < Q; ++q) v[u][q] = fma(v[u][q], both(scale), pair_at(raw, q));
            }
            if constexpr (SHIFT) set_past(v[u], at, row < a.rows, a.cols, W(0));
            Pair<W> two = both(W(0));
#pragma unroll
            for (int q = 0; q < Q; ++q) two = two + v[u][q];
            sum[u] = two.x + two.y;
        }
        // Two sweeps over registers: the mean of what the warp (or its team)
        // holds, then the squares about it. Values past the row are 0 in the
        // first, the mean itself in the second.
        if constexpr (R == 2) {
            sum[0] = folded_sums(sum);  // rows in halves of the warp
            mean[0] = __shfl_sync(0xffffffffu, sum[0], 0) * over_held;
            mean[1] = __shfl_sync(0xffffffffu, sum[0], 16) * over_held;
        } else {
            sum[0] = team_sum(sum[0], TEAM == kWarp ? at.threads : 32);
            mean[0] = TEAM == kWarp ? sum[0] / held : sum[0] * over_held;
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            if constexpr (!FULL) set_past(v[u], at, true, a.cols, mean[u]);
            Pair<W> two = both(W(0));
#pragma unroll
            for (int q = 0; q < Q; ++q) {
                const Pair<W> d = v[u][q] + both(-mean[u]);
                two = fma(d, d, two);
            }
            squares[u] = two.x + two.y;
        }
        W rstd[R];
        if constexpr (TEAM == kWarp) {
            rstd[0] = rsqrt(team_sum(squares[0], at.threads) * over + (W)a.epsilon);
        } else {
            squares[0] = R == 2 ? folded_sums(squares) : team_sum(squares[0], 32);
            // Values 2 u: sum of row u, 2 u + 1: its squares.
            complete = exchange(sums, round, at, at.wlane / (16 / R) % 2 ? squares[0] : sum[0], complete,
                                STARVE ? a.starve.polls : kWaitPolls,
                                STARVE && round == a.starve.round && at.rank == at.ranks - 1);
            auto found = [&](int n, int j) { return sums.values[round & 1][n][at.first_entry + joiner + j * kJoin]; };
            // Warps joined about the row's mean: squares + held (warp's mean - mean)^2.
            W total = 0, other[kEach];
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                other[j] = joined[j] > W(0) ? found(2 * joined_row, j) : W(0);
                total += other[j];
            }
            // Divided, so that a row of one value has no spread.
            W middle = team_sum(total, kJoin) / (W)a.cols;
            if (!complete) middle = (W)NAN;
            W spread = 0;
#pragma unroll
            for (int j = 0; j < kEach; ++j) {
                const W d = other[j] * over_joined[j] - middle;
                if (joined[j] > W(0)) spread += found(2 * joined_row + 1, j) + joined[j] * d * d;
            }
            const W inverse = rsqrt(team_sum(spread, kJoin) * over + (W)a.epsilon);
#pragma unroll
            for (int u = 0; u < R; ++u) {
                mean[u] = R == 1 ? middle : __shfl_sync(0xffffffffu, middle, u * kJoin);
                rstd[u] = R == 1 ? inverse : __shfl_sync(0xffffffffu, inverse, u * kJoin);
            }
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = first + at.within + u * at.step;
            const bool live = (TEAM != kWarp && u == 0) || row < a.rows;
            if (live && at.lane == 0) {
                if (a.mean != nullptr) ((W *)a.mean)[row] = mean[u];
                if (a.rstd != nullptr) ((W *)a.rstd)[row] = rstd[u];
            }
            Vec<T, V> out[K];
            if constexpr (DROP) {
#pragma unroll
                for (int q = 0; q < Q; ++q) set_pair(out, q, v[u][q]);
                ring.put((T *)a.z + row * a.z_stride, live, u, 0, out);
            }
#pragma unroll
            for (int q = 0; q < Q; ++q)
                set_pair(out, q, fma((v[u][q] + both(-mean[u])) * both(rstd[u]), w[q], b[q]));
            ring.put((T *)a.y + row * a.y_stride, live, u, DROP ? 1 : 0, out);
        }
        ring.done();
    }
    wait_async<0>();
    close_exchange<TEAM>();
}

// ---- rows of any length --------------------------------------------------------

// For rows beyond eight blocks of threads (32768 values, 16384 in float64).
// One CTA per row, three sweeps over it (the second and third hit L2). Eight CTAs a
// multiprocessor (256 x 65536 bfloat16 116 us, 128 without that bound); with dropout
// they would spill (fused 355 us, 325 without).
template <typename T, typename P, bool DROP>
__global__ void __launch_bounds__(kThreads, DROP ? 4 : 8) norm_any_kernel(const ForwardArgs a) {
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
        const W sum = long_sum<W>((int)threadIdx.x, a.cols, kThreads, [&](W &s, int c) { s += value(c); });
        const W mean = block_sum(sum, scratch) / (W)a.cols;
        const W squares = long_sum<W>((int)threadIdx.x, a.cols, kThreads, [&](W &s, int c) {
            const W d = value(c) - mean;
            s += d * d;
        });
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

// `stages` rows of `stage` bytes in the ring, and the grid, of a team kernel.
template <typename T, bool DROP, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
cudaError_t launch_shape(const Shape &s, const ForwardArgs &a, bool float_parameters, cudaStream_t stream) {
    constexpr int resident = resident_threads(sizeof(T), DROP, SHIFT, TEAM), at_once = rows_at_once(sizeof(T), SHIFT, TEAM);
    const size_t stage = (DROP ? 2 : 1) * s.part(sizeof(T));
    const int stages = ring_stages(stage, at_once, s.threads(), resident);
    const size_t each = s.teams() * at_once, wanted = (a.rows + each - 1) / each;
    const size_t most = (size_t)geo::device_sm_count() * (resident / s.threads()) / s.blocks;
    size_t grid = wanted < most ? wanted : most;
    return launch_team(norm_kernel<T, DROP, TEAM, SHIFT, FULL, STARVE>, s, grid, s.blocks, stages * stage, stream, a,
                       s.lanes, float_parameters, stages);
}

template <bool DROP>
cudaError_t launch(NormTypes n, const ForwardArgs &a, cudaStream_t stream) {
    const size_t bytes = type_bytes(n.type);
    const bool aligned =
        aligned16(a.cols, bytes, type_bytes(n.parameter_type),
                  {{a.x, a.x_stride}, {a.residual, a.residual_stride}, {a.z, a.z_stride}, {a.y, a.y_stride}},
                  {a.weight, a.bias});
    const Shape s = shape_of(a.cols, bytes, aligned);
    if (s.lanes == 0)
        return by_types(n, [&](auto t, auto p) {
            const unsigned grid = (unsigned)(a.rows < (1u << 20) ? a.rows : (1u << 20));
            norm_any_kernel<decltype(t), decltype(p), DROP><<<grid, kThreads, 0, stream>>>(a);
            return cudaGetLastError();
        });
    const bool float_parameters = n.parameter_type == GEO_B200_F32;
    return by_type(n.type, [&](auto t) {
        using T = decltype(t);
        return by_shape(s, [&](auto team, auto shift, auto full) {
            return launch_shape<T, DROP, decltype(team)::value, decltype(shift)::value, decltype(full)::value>(
                s, a, float_parameters, stream);
        });
    });
}

}  // namespace

cudaError_t launch_norm(NormTypes t, const ForwardArgs &a, bool drop, cudaStream_t stream) {
    return drop ? launch<true>(t, a, stream) : launch<false>(t, a, stream);
}

cudaError_t launch_norm_starved(const ForwardArgs &a, cudaStream_t stream) {
    return launch_shape<float, false, kCluster, false, true, true>(shape_of(a.cols, 4, true), a, true, stream);
}

}  // namespace layers
}  // namespace geo

namespace {

using namespace geo::layers;

bool config_valid(const geo_b200_layer_norm_config_t *c) {
    if (c == nullptr || type_bytes(c->type) == 0) return false;
    if (c->parameter_type != c->type && !(type_bytes(c->type) == 2 && c->parameter_type == GEO_B200_F32)) return false;
    return c->rows != 0 && c->cols != 0 && c->rows <= GEO_B200_LAYER_MAX_ROWS && c->cols <= GEO_B200_LAYER_MAX_COLS &&
           std::isfinite(c->epsilon) && c->epsilon >= 0.0;
}

size_t workspace_bytes_of(const geo_b200_layer_norm_config_t &c) {
    return vjp_workspace({c.type, c.parameter_type}, c.rows, c.cols);
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
    return status_of(launch_norm({c.type, c.parameter_type}, a, false, stream));
}

extern "C" size_t geo_b200_layer_norm_vjp_workspace(const geo_b200_layer_norm_config_t *config) {
    if (!config_valid(config)) return 0;
    geo_b200_layer_norm_config_t c = *config;
    return resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_cotangent_stride, &c.x_cotangent_stride})
               ? workspace_bytes_of(c)
               : 0;
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
    return status_of(launch_norm_vjp({c.type, c.parameter_type}, a, false, device_workspace, stream));
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
    return status_of(launch_norm({c.type, c.parameter_type}, a, true, stream));
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
    return status_of(launch_norm_vjp({c.type, c.parameter_type}, a, true, device_workspace, stream));
}

extern "C" geo_b200_status_t geo_b200_layer_norm_wait_selftest(
    const geo_b200_layer_norm_config_t *config, const void *device_x, const void *device_y_cotangent, void *device_out,
    void *device_mean, void *device_rstd, void *device_weight_cotangent, void *device_bias_cotangent,
    void *device_workspace, size_t workspace_bytes, uint32_t round, uint32_t wait_limit, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.layer_norm_wait_selftest");
    if (!config_valid(config) || config->type != GEO_B200_F32 || config->x_stride != 0 || config->y_stride != 0 ||
        config->y_cotangent_stride != 0 || config->x_cotangent_stride != 0 || wait_limit == 0 || wait_limit > kWaitPolls || device_x == nullptr ||
        device_out == nullptr || device_mean == nullptr || device_rstd == nullptr)
        return GEO_B200_INVALID_ARGUMENT;
    const Shape s = shape_of(config->cols, 4, true);
    if (s.team() != kCluster || s.lanes == 0 || !s.full ||
        !arrays_usable({{device_x, 16}, {device_y_cotangent, 16}, {device_out, 16}, {device_mean, 4}, {device_rstd, 4},
                        {device_weight_cotangent, 4}, {device_bias_cotangent, 4}}))
        return GEO_B200_INVALID_ARGUMENT;
    if (device_y_cotangent == nullptr) {
        ForwardArgs a = {};
        a.x = device_x;
        a.y = device_out;
        a.mean = device_mean;
        a.rstd = device_rstd;
        a.rows = config->rows;
        a.cols = (int)config->cols;
        a.x_stride = a.y_stride = config->cols;
        a.epsilon = config->epsilon;
        a.starve = {round, wait_limit};
        return status_of(launch_norm_starved(a, stream));
    }
    if (device_weight_cotangent == nullptr || device_bias_cotangent == nullptr ||
        !workspace_usable(*config, device_workspace, workspace_bytes))
        return GEO_B200_INVALID_ARGUMENT;
    BackwardArgs a = {};
    a.x = device_x;
    a.mean = device_mean;
    a.rstd = device_rstd;
    a.dy = device_y_cotangent;
    a.dsum = device_out;
    a.dweight = device_weight_cotangent;
    a.dbias = device_bias_cotangent;
    a.rows = config->rows;
    a.cols = (int)config->cols;
    a.x_stride = a.dy_stride = a.dsum_stride = config->cols;
    a.starve = {round, wait_limit};
    return status_of(launch_norm_vjp_starved(a, device_workspace, stream));
}
