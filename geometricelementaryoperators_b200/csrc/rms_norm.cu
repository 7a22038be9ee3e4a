// rms_norm.cu -- RMS norm over rows, and the norms before and after a block with its
// gate and residual (geo/geo_b200.h section 5): entry points and the forward kernels;
// the backward ones are in rms_norm_vjp.cu.
//
// r = rsqrt(mean(x^2) + epsilon), y = x r w; a block norm joins n = x r w to the
// residual stream, z = alpha residual + beta act(gate) n, and normalises z. HBM
// bounds both: every array is read or written once. Rows are held, moved and joined as
// in layer norm (layer_norm.h): a team of threads holds a row in registers between the
// sweeps, rows arrive through a ring of asynchronous copies. A block norm's second
// statistic depends on the first, so a row takes two exchanges across its team (one
// statistic from sums over x, residual and gate alone would be a difference of large
// squares where the block nearly cancels the residual). Measured, host included: 8192 x
// 4096 bfloat16 RMS norm 24.8 us (83% of the copy bandwidth), block norm with a sigmoid
// gate 16384 x 4096 bfloat16 110 us (93%).
#include "rms_norm.h"

#include <cmath>

#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

template <typename T, int MODE, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
__global__ void __launch_bounds__(TEAM == kWarp ? kWarpBlock : kTeamThreads, TEAM == kWarp ? 4 : 2)
    rms_kernel(const RmsForwardArgs a, int lanes, bool float_parameters, int stages) {
    using W = Wide<T>;
    constexpr int V = 16 / (int)sizeof(T), K = values_per_thread(sizeof(T)) / V, Q = K * V / 2;
    constexpr int R = rows_at_once(sizeof(T), SHIFT, TEAM), kArrays = MODE + 1;
    extern __shared__ __align__(128) unsigned char memory[];
    __shared__ Exchange<W, R, TEAM> sums;
    const Place<TEAM, V, K> at(lanes);
    Ring<T, V, K, TEAM, SHIFT, FULL, R> ring(memory, stages, kArrays, at, a.rows, a.cols);
    auto next = [&] {
        ring.copy(0, (const T *)a.x, a.x_stride);
        if constexpr (MODE >= kBlockNorm) ring.copy(1, (const T *)a.residual, a.residual_stride);
        if constexpr (MODE == kGatedNorm) ring.copy(2, (const T *)a.gate, a.gate_stride);
        ring.fetched();
    };
    for (int s = 0; s < stages - R; ++s) next();

    const W over = W(1) / (W)a.cols, alpha = (W)a.residual_scale, beta = (W)a.block_scale;
    Pair<W> w[Q], post[MODE >= kBlockNorm ? Q : 1];
    load_parameters<T, V, K, SHIFT>(a.weight, float_parameters, at, a.cols, W(1), w);
    if constexpr (MODE >= kBlockNorm) {
        load_parameters<T, V, K, SHIFT>(a.post, float_parameters, at, a.cols, W(1), post);
#pragma unroll
        for (int q = 0; q < Q; ++q) post[q] = post[q] * both(beta);
    }
    open_exchange(sums);

    uint32_t round = 0;
    bool complete = true;  // no wait for the cluster gave up
    for (size_t first = at.begin; first < a.rows; first += R * at.step) {
        for (int u = 0; u < R; ++u) next();
        ring.wait();
        Pair<W> v[R][Q];
        W part[R];
        auto square = [&](int u) {
            Pair<W> two = both(W(0));
#pragma unroll
            for (int q = 0; q < Q; ++q) two = fma(v[u][q], v[u][q], two);
            part[u] = two.x + two.y;
        };
        auto row_of = [&](int u) { return first + at.within + u * at.step; };
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = row_of(u), r = row < a.rows ? row : 0;
            Vec<T, V> raw[K];
            ring.get(raw, u, 0, (const T *)a.x + r * a.x_stride);
#pragma unroll
            for (int q = 0; q < Q; ++q) v[u][q] = pair_at(raw, q);
            if constexpr (SHIFT) set_past(v[u], at, row < a.rows, a.cols, W(0));
            square(u);
        }
        auto join = [&] {
            const bool silent = STARVE && round == a.starve.round && at.rank == at.ranks - 1;
            complete = team_sums<R>(sums, round++, at, part, complete, STARVE ? a.starve.polls : kWaitPolls, silent);
        };
        join();
        W rstd[R];
#pragma unroll
        for (int u = 0; u < R; ++u) rstd[u] = rsqrt(part[u] * over + (W)a.epsilon);
        if constexpr (MODE >= kBlockNorm) {
#pragma unroll
            for (int u = 0; u < R; ++u) {
                const size_t row = row_of(u), r = row < a.rows ? row : 0;
                const bool live = (TEAM != kWarp && u == 0) || row < a.rows;
                if (live && at.lane == 0 && a.x_rstd != nullptr) ((W *)a.x_rstd)[row] = rstd[u];
                Vec<T, V> raw[K];
#pragma unroll
                for (int q = 0; q < Q; ++q) v[u][q] = v[u][q] * both(rstd[u]) * post[q];
                if constexpr (MODE == kGatedNorm) {
                    ring.get(raw, u, 2, (const T *)a.gate + r * a.gate_stride);
#pragma unroll
                    for (int i = 0; i < K; ++i) {
                        Pair<W> f[V / 2], none[V / 2];
                        gate_values<sizeof(T) == 2, false>(a.gate_kind, raw[i], f, none);
#pragma unroll
                        for (int q = 0; q < V / 2; ++q) v[u][i * V / 2 + q] = v[u][i * V / 2 + q] * f[q];
                    }
                }
                ring.get(raw, u, 1, (const T *)a.residual + r * a.residual_stride);
#pragma unroll
                for (int q = 0; q < Q; ++q) v[u][q] = fma(both(alpha), pair_at(raw, q), v[u][q]);
                if constexpr (SHIFT) set_past(v[u], at, row < a.rows, a.cols, W(0));
                square(u);
            }
            join();
#pragma unroll
            for (int u = 0; u < R; ++u) rstd[u] = rsqrt(part[u] * over + (W)a.epsilon);
        }
#pragma unroll
        for (int u = 0; u < R; ++u) {
            const size_t row = row_of(u);
            const bool live = (TEAM != kWarp && u == 0) || row < a.rows;
            if (live && at.lane == 0 && a.rstd != nullptr) ((W *)a.rstd)[row] = rstd[u];
            Vec<T, V> out[K];
            if constexpr (MODE >= kBlockNorm) {
#pragma unroll
                for (int q = 0; q < Q; ++q) set_pair(out, q, v[u][q]);
                ring.put((T *)a.z + row * a.z_stride, live, u, 0, out);
            }
#pragma unroll
            for (int q = 0; q < Q; ++q) set_pair(out, q, v[u][q] * both(rstd[u]) * w[q]);
            ring.put((T *)a.y + row * a.y_stride, live, u, MODE >= kBlockNorm ? 1 : 0, out);
        }
        ring.done();
    }
    wait_async<0>();
    close_exchange<TEAM>();
}

// ---- rows of any length --------------------------------------------------------

// For rows beyond eight blocks of threads (32768 values, 16384 in float64): one CTA a
// row, a sweep for each statistic and one that writes (all but the first hit L2).
template <typename T, typename P, int MODE>
__global__ void __launch_bounds__(kThreads, 4) rms_any_kernel(const RmsForwardArgs a) {
    using W = Wide<T>;
    __shared__ W scratch[kThreads / 32];
    const W alpha = (W)a.residual_scale, beta = (W)a.block_scale;
    for (size_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const T *x = (const T *)a.x + row * a.x_stride;
        T *y = (T *)a.y + row * a.y_stride;
        auto root = [&](auto &&value) {
            const W sum = long_sum<W>((int)threadIdx.x, a.cols, kThreads, [&](W &s, int c) {
                const W v = value(c);
                s += v * v;
            });
            return W(1) / sqrt(block_sum(sum, scratch) / (W)a.cols + (W)a.epsilon);
        };
        auto parameter = [&](const void *p, int c) { return p != nullptr ? (W)widen(((const P *)p)[c]) : W(1); };
        W rstd = root([&](int c) { return widen(x[c]); });
        if constexpr (MODE >= kBlockNorm) {
            const T *residual = (const T *)a.residual + row * a.residual_stride;
            const T *gate = MODE == kGatedNorm ? (const T *)a.gate + row * a.gate_stride : nullptr;
            T *z = (T *)a.z + row * a.z_stride;
            const W x_rstd = rstd;
            auto joined = [&](int c) {
                W n = widen(x[c]) * x_rstd * (parameter(a.post, c) * beta);
                if constexpr (MODE == kGatedNorm)
                    n *= gate_value<sizeof(T) == 2>(a.gate_kind, widen(gate[c]), (W *)nullptr);
                return ::fma(alpha, widen(residual[c]), n);
            };
            rstd = root(joined);
            for (int c = threadIdx.x; c < a.cols; c += kThreads) {
                const W v = joined(c);
                z[c] = narrow<T>(v);
                y[c] = narrow<T>(v * rstd * parameter(a.weight, c));
            }
            if (threadIdx.x == 0 && a.x_rstd != nullptr) ((W *)a.x_rstd)[row] = x_rstd;
        } else {
            for (int c = threadIdx.x; c < a.cols; c += kThreads)
                y[c] = narrow<T>(widen(x[c]) * rstd * parameter(a.weight, c));
        }
        if (threadIdx.x == 0 && a.rstd != nullptr) ((W *)a.rstd)[row] = rstd;
    }
}

template <typename T, int MODE, int TEAM, bool SHIFT, bool FULL, bool STARVE = false>
cudaError_t launch_shape(const Shape &s, const RmsForwardArgs &a, bool float_parameters, cudaStream_t stream) {
    constexpr int at_once = rows_at_once(sizeof(T), SHIFT, TEAM);
    const size_t stage = (MODE + 1) * s.part(sizeof(T));
    const int stages = ring_stages(stage, at_once, s.threads(), 512);
    const size_t each = s.teams() * at_once, wanted = (a.rows + each - 1) / each;
    const size_t most = (size_t)geo::device_sm_count() * (512 / s.threads()) / s.blocks;
    size_t grid = wanted < most ? wanted : most;
    return launch_team(rms_kernel<T, MODE, TEAM, SHIFT, FULL, STARVE>, s, grid, s.blocks, stages * stage, stream, a, s.lanes,
                       float_parameters, stages);
}

}  // namespace

cudaError_t launch_rms(NormTypes n, NormMode mode, const RmsForwardArgs &a, cudaStream_t stream) {
    const size_t bytes = type_bytes(n.type);
    const bool aligned = aligned16(a.cols, bytes, type_bytes(n.parameter_type),
                                   {{a.x, a.x_stride}, {a.residual, a.residual_stride}, {a.gate, a.gate_stride},
                                    {a.z, a.z_stride}, {a.y, a.y_stride}},
                                   {a.post, a.weight});
    const Shape s = shape_of(a.cols, bytes, aligned);
    if (s.lanes == 0)
        return by_mode(mode, [&](auto m) {
            return by_types(n, [&](auto t, auto p) {
                const unsigned grid = (unsigned)(a.rows < (1u << 20) ? a.rows : (1u << 20));
                rms_any_kernel<decltype(t), decltype(p), decltype(m)::value><<<grid, kThreads, 0, stream>>>(a);
                return cudaGetLastError();
            });
        });
    return by_mode(mode, [&](auto m) {
        return by_type(n.type, [&](auto t) {
            return by_shape(s, [&](auto team, auto shift, auto full) {
                return launch_shape<decltype(t), decltype(m)::value, decltype(team)::value, decltype(shift)::value,
                                    decltype(full)::value>(s, a, n.parameter_type == GEO_B200_F32, stream);
            });
        });
    });
}

cudaError_t launch_rms_starved(const RmsForwardArgs &a, cudaStream_t stream) {
    return launch_shape<float, kBlockNorm, kCluster, false, true, true>(shape_of(a.cols, 4, true), a, true, stream);
}

}  // namespace layers
}  // namespace geo

namespace {

using namespace geo::layers;

bool types_valid(uint32_t type, uint32_t parameter_type) {
    return type_bytes(type) != 0 &&
           (parameter_type == type || (type_bytes(type) == 2 && parameter_type == GEO_B200_F32));
}
bool shape_valid(size_t rows, size_t cols, double epsilon) {
    return rows != 0 && cols != 0 && rows <= GEO_B200_LAYER_MAX_ROWS && cols <= GEO_B200_LAYER_MAX_COLS &&
           std::isfinite(epsilon) && epsilon >= 0.0;
}
bool config_valid(const geo_b200_layer_norm_config_t *c) {
    return c != nullptr && types_valid(c->type, c->parameter_type) && shape_valid(c->rows, c->cols, c->epsilon);
}
bool config_valid(const geo_b200_block_norm_config_t *c) {
    return c != nullptr && types_valid(c->type, c->parameter_type) && shape_valid(c->rows, c->cols, c->epsilon) &&
           c->reserved == 0 && c->gate <= GEO_B200_GATE_TANH && std::isfinite(c->residual_scale) &&
           std::isfinite(c->block_scale);
}
NormMode mode_of(const geo_b200_block_norm_config_t &c) { return c.gate == GEO_B200_GATE_NONE ? kBlockNorm : kGatedNorm; }

bool vjp_strides(geo_b200_block_norm_config_t &c) {
    return resolve_strides(c.rows, c.cols, {&c.x_stride, &c.gate_stride, &c.z_stride, &c.y_cotangent_stride,
                                            &c.z_cotangent_stride, &c.residual_cotangent_stride,
                                            &c.x_cotangent_stride, &c.gate_cotangent_stride});
}

struct Rows {
    const void *p;
    size_t stride;
};
// Outputs apart from one another, and the same as an input only with its stride.
bool outputs_apart(std::initializer_list<Rows> outs, std::initializer_list<Rows> ins) {
    for (auto o = outs.begin(); o != outs.end(); ++o) {
        if (o->p == nullptr) continue;
        for (const Rows &i : ins)
            if (!same_or_apart(o->p, o->stride, i.p, i.stride)) return false;
        for (auto other = o + 1; other != outs.end(); ++other)
            if (o->p == other->p) return false;
    }
    return true;
}

bool workspace_usable(size_t need, const void *workspace, size_t bytes) {
    return workspace != nullptr && bytes >= need && arrays_usable({{workspace, 16}});
}

}  // namespace

extern "C" geo_b200_status_t geo_b200_rms_norm(const geo_b200_layer_norm_config_t *config, const void *device_x,
                                               const void *device_weight, void *device_y, void *device_rstd,
                                               cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.rms_norm");
    if (!config_valid(config) || device_x == nullptr || device_y == nullptr) return GEO_B200_INVALID_ARGUMENT;
    geo_b200_layer_norm_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_stride}) ||
        !same_or_apart(device_y, c.y_stride, device_x, c.x_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_y, b}, {device_weight, p}, {device_rstd, w}}))
        return GEO_B200_INVALID_ARGUMENT;
    RmsForwardArgs a = {};
    a.x = device_x;
    a.weight = device_weight;
    a.y = device_y;
    a.rstd = device_rstd;
    a.rows = c.rows;
    a.cols = (int)c.cols;
    a.x_stride = c.x_stride;
    a.y_stride = c.y_stride;
    a.epsilon = c.epsilon;
    return status_of(launch_rms({c.type, c.parameter_type}, kRms, a, stream));
}

extern "C" size_t geo_b200_rms_norm_vjp_workspace(const geo_b200_layer_norm_config_t *config) {
    if (!config_valid(config)) return 0;
    geo_b200_layer_norm_config_t c = *config;
    return resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_cotangent_stride, &c.x_cotangent_stride})
               ? rms_vjp_workspace({c.type, c.parameter_type}, kRms, c.rows, c.cols)
               : 0;
}

extern "C" geo_b200_status_t geo_b200_rms_norm_vjp(const geo_b200_layer_norm_config_t *config, const void *device_x,
                                                   const void *device_weight, const void *device_rstd,
                                                   const void *device_y_cotangent, void *device_x_cotangent,
                                                   void *device_weight_cotangent, void *device_workspace,
                                                   size_t workspace_bytes, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.rms_norm_vjp");
    if (!config_valid(config) || device_x == nullptr || device_rstd == nullptr || device_y_cotangent == nullptr ||
        (device_x_cotangent == nullptr && device_weight_cotangent == nullptr))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_layer_norm_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.y_cotangent_stride, &c.x_cotangent_stride}) ||
        !outputs_apart({{device_x_cotangent, c.x_cotangent_stride}},
                       {{device_x, c.x_stride}, {device_y_cotangent, c.y_cotangent_stride}}))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_weight, p}, {device_rstd, w}, {device_y_cotangent, b},
                        {device_x_cotangent, b}, {device_weight_cotangent, p}}))
        return GEO_B200_INVALID_ARGUMENT;
    if (device_weight_cotangent != nullptr &&
        !workspace_usable(rms_vjp_workspace({c.type, c.parameter_type}, kRms, c.rows, c.cols), device_workspace,
                          workspace_bytes))
        return GEO_B200_INVALID_ARGUMENT;
    RmsBackwardArgs a = {};
    a.x = device_x;
    a.weight = device_weight;
    a.rstd = device_rstd;
    a.dy = device_y_cotangent;
    a.dx = device_x_cotangent;
    a.dweight = device_weight_cotangent;
    a.rows = c.rows;
    a.cols = (int)c.cols;
    a.x_stride = c.x_stride;
    a.dy_stride = c.y_cotangent_stride;
    a.dx_stride = c.x_cotangent_stride;
    return status_of(launch_rms_vjp({c.type, c.parameter_type}, kRms, a, device_workspace, stream));
}

extern "C" geo_b200_status_t geo_b200_block_norm(const geo_b200_block_norm_config_t *config, const void *device_x,
                                                 const void *device_residual, const void *device_gate,
                                                 const void *device_post_weight, const void *device_pre_weight,
                                                 void *device_z, void *device_y, void *device_x_rstd,
                                                 void *device_z_rstd, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.block_norm");
    if (!config_valid(config) || device_x == nullptr || device_residual == nullptr ||
        (device_gate == nullptr) != (config->gate == GEO_B200_GATE_NONE) || device_z == nullptr || device_y == nullptr)
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_block_norm_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols,
                         {&c.x_stride, &c.residual_stride, &c.gate_stride, &c.z_stride, &c.y_stride}) ||
        !outputs_apart({{device_z, c.z_stride}, {device_y, c.y_stride}},
                       {{device_x, c.x_stride}, {device_residual, c.residual_stride}, {device_gate, c.gate_stride}}))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_residual, b}, {device_gate, b}, {device_post_weight, p},
                        {device_pre_weight, p}, {device_z, b}, {device_y, b}, {device_x_rstd, w}, {device_z_rstd, w}}))
        return GEO_B200_INVALID_ARGUMENT;
    RmsForwardArgs a = {};
    a.x = device_x;
    a.residual = device_residual;
    a.gate = device_gate;
    a.post = device_post_weight;
    a.weight = device_pre_weight;
    a.z = device_z;
    a.y = device_y;
    a.x_rstd = device_x_rstd;
    a.rstd = device_z_rstd;
    a.rows = c.rows;
    a.x_stride = c.x_stride;
    a.residual_stride = c.residual_stride;
    a.gate_stride = c.gate_stride;
    a.z_stride = c.z_stride;
    a.y_stride = c.y_stride;
    a.cols = (int)c.cols;
    a.gate_kind = (int)c.gate;
    a.epsilon = c.epsilon;
    a.residual_scale = c.residual_scale;
    a.block_scale = c.block_scale;
    return status_of(launch_rms({c.type, c.parameter_type}, mode_of(c), a, stream));
}

extern "C" size_t geo_b200_block_norm_vjp_workspace(const geo_b200_block_norm_config_t *config) {
    if (!config_valid(config)) return 0;
    geo_b200_block_norm_config_t c = *config;
    return vjp_strides(c) ? rms_vjp_workspace({c.type, c.parameter_type}, mode_of(c), c.rows, c.cols) : 0;
}

extern "C" geo_b200_status_t geo_b200_block_norm_vjp(
    const geo_b200_block_norm_config_t *config, const void *device_x, const void *device_gate, const void *device_z,
    const void *device_post_weight, const void *device_pre_weight, const void *device_x_rstd,
    const void *device_z_rstd, const void *device_y_cotangent, const void *device_z_cotangent,
    void *device_residual_cotangent, void *device_x_cotangent, void *device_gate_cotangent,
    void *device_post_weight_cotangent, void *device_pre_weight_cotangent, void *device_workspace,
    size_t workspace_bytes, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.block_norm_vjp");
    if (!config_valid(config) || device_x == nullptr || device_z == nullptr || device_x_rstd == nullptr ||
        device_z_rstd == nullptr || device_y_cotangent == nullptr ||
        (device_gate == nullptr) != (config->gate == GEO_B200_GATE_NONE) ||
        (device_gate_cotangent != nullptr && device_gate == nullptr) ||
        (device_residual_cotangent == nullptr && device_x_cotangent == nullptr && device_gate_cotangent == nullptr &&
         device_post_weight_cotangent == nullptr && device_pre_weight_cotangent == nullptr))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_block_norm_config_t c = *config;
    if (!vjp_strides(c) ||
        !outputs_apart({{device_residual_cotangent, c.residual_cotangent_stride},
                        {device_x_cotangent, c.x_cotangent_stride},
                        {device_gate_cotangent, c.gate_cotangent_stride}},
                       {{device_x, c.x_stride},
                        {device_gate, c.gate_stride},
                        {device_z, c.z_stride},
                        {device_y_cotangent, c.y_cotangent_stride},
                        {device_z_cotangent, c.z_cotangent_stride}}))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), p = type_bytes(c.parameter_type), w = wide_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_gate, b}, {device_z, b}, {device_post_weight, p}, {device_pre_weight, p},
                        {device_x_rstd, w}, {device_z_rstd, w}, {device_y_cotangent, b}, {device_z_cotangent, b},
                        {device_residual_cotangent, b}, {device_x_cotangent, b}, {device_gate_cotangent, b},
                        {device_post_weight_cotangent, p}, {device_pre_weight_cotangent, p}}))
        return GEO_B200_INVALID_ARGUMENT;
    if ((device_post_weight_cotangent != nullptr || device_pre_weight_cotangent != nullptr) &&
        !workspace_usable(rms_vjp_workspace({c.type, c.parameter_type}, mode_of(c), c.rows, c.cols), device_workspace,
                          workspace_bytes))
        return GEO_B200_INVALID_ARGUMENT;
    RmsBackwardArgs a = {};
    a.x = device_x;
    a.z = device_z;
    a.gate = device_gate;
    a.post = device_post_weight;
    a.weight = device_pre_weight;
    a.x_rstd = device_x_rstd;
    a.rstd = device_z_rstd;
    a.dy = device_y_cotangent;
    a.dz = device_z_cotangent;
    a.dresidual = device_residual_cotangent;
    a.dx = device_x_cotangent;
    a.dgate = device_gate_cotangent;
    a.dpost = device_post_weight_cotangent;
    a.dweight = device_pre_weight_cotangent;
    a.rows = c.rows;
    a.x_stride = c.x_stride;
    a.z_stride = c.z_stride;
    a.gate_stride = c.gate_stride;
    a.dy_stride = c.y_cotangent_stride;
    a.dz_stride = c.z_cotangent_stride;
    a.dresidual_stride = c.residual_cotangent_stride;
    a.dx_stride = c.x_cotangent_stride;
    a.dgate_stride = c.gate_cotangent_stride;
    a.cols = (int)c.cols;
    a.gate_kind = (int)c.gate;
    a.residual_scale = c.residual_scale;
    a.block_scale = c.block_scale;
    return status_of(launch_rms_vjp({c.type, c.parameter_type}, mode_of(c), a, device_workspace, stream));
}

extern "C" geo_b200_status_t geo_b200_block_norm_wait_selftest(
    const geo_b200_block_norm_config_t *config, const void *device_x, const void *device_residual,
    const void *device_y_cotangent, void *device_out, void *device_y, void *device_x_rstd, void *device_z_rstd,
    void *device_post_weight_cotangent, void *device_pre_weight_cotangent, void *device_workspace,
    size_t workspace_bytes, uint32_t round, uint32_t wait_limit, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.block_norm_wait_selftest");
    if (!config_valid(config) || config->type != GEO_B200_F32 || config->gate != GEO_B200_GATE_NONE || wait_limit == 0 ||
        wait_limit > kWaitPolls || device_x == nullptr || device_residual == nullptr || device_out == nullptr ||
        device_y == nullptr || device_x_rstd == nullptr || device_z_rstd == nullptr)
        return GEO_B200_INVALID_ARGUMENT;
    const geo_b200_block_norm_config_t &c = *config;
    for (const size_t stride : {c.x_stride, c.residual_stride, c.z_stride, c.y_stride, c.y_cotangent_stride,
                                c.residual_cotangent_stride, c.x_cotangent_stride})
        if (stride != 0) return GEO_B200_INVALID_ARGUMENT;
    const Shape s = shape_of(c.cols, 4, true);
    if (s.team() != kCluster || s.lanes == 0 || !s.full ||
        !arrays_usable({{device_x, 16}, {device_residual, 16}, {device_y_cotangent, 16}, {device_out, 16}, {device_y, 16},
                        {device_x_rstd, 4}, {device_z_rstd, 4}, {device_post_weight_cotangent, 4},
                        {device_pre_weight_cotangent, 4}}))
        return GEO_B200_INVALID_ARGUMENT;
    if (device_y_cotangent == nullptr) {
        RmsForwardArgs a = {};
        a.x = device_x;
        a.residual = device_residual;
        a.z = device_out;
        a.y = device_y;
        a.x_rstd = device_x_rstd;
        a.rstd = device_z_rstd;
        a.rows = c.rows;
        a.x_stride = a.residual_stride = a.z_stride = a.y_stride = c.cols;
        a.cols = (int)c.cols;
        a.epsilon = c.epsilon;
        a.residual_scale = c.residual_scale;
        a.block_scale = c.block_scale;
        a.starve = {round, wait_limit};
        return status_of(launch_rms_starved(a, stream));
    }
    if (device_post_weight_cotangent == nullptr || device_pre_weight_cotangent == nullptr ||
        !workspace_usable(rms_vjp_workspace({c.type, c.parameter_type}, kBlockNorm, c.rows, c.cols), device_workspace,
                          workspace_bytes))
        return GEO_B200_INVALID_ARGUMENT;
    RmsBackwardArgs a = {};
    a.x = device_x;
    a.z = device_residual;
    a.x_rstd = device_x_rstd;
    a.rstd = device_z_rstd;
    a.dy = device_y_cotangent;
    a.dresidual = device_out;
    a.dx = device_y;
    a.dpost = device_post_weight_cotangent;
    a.dweight = device_pre_weight_cotangent;
    a.rows = c.rows;
    a.x_stride = a.z_stride = a.dy_stride = a.dresidual_stride = a.dx_stride = c.cols;
    a.cols = (int)c.cols;
    a.residual_scale = c.residual_scale;
    a.block_scale = c.block_scale;
    a.starve = {round, wait_limit};
    return status_of(launch_rms_vjp_starved(a, device_workspace, stream));
}
