// rms_norm.h -- what RMS norm's and the block norm's forward (rms_norm.cu) and
// backward (rms_norm_vjp.cu) kernels share. How rows are held, moved and joined is
// layer norm's (layer_norm.h).
#pragma once

#include "layer_norm.h"

namespace geo {
namespace layers {

// What a pass works on. kRms: one norm of x. kBlock: x, its norm, a residual and a
// second norm; kGated: with a gate.
enum NormMode : int { kRms = 0, kBlockNorm = 1, kGatedNorm = 2 };

struct RmsForwardArgs {
    const void *x, *residual, *gate, *post, *weight;  // weight: of the norm that gives y
    void *z, *y, *x_rstd, *rstd;                      // rstd: of z (kRms: of x)
    size_t rows, x_stride, residual_stride, gate_stride, z_stride, y_stride;
    int cols, gate_kind;
    double epsilon, residual_scale, block_scale;
    Starve starve;
};

struct RmsBackwardArgs {
    const void *x, *z, *gate, *post, *weight, *x_rstd, *rstd, *dy, *dz;
    void *dresidual, *dx, *dgate, *dpost, *dweight;
    size_t rows, x_stride, z_stride, gate_stride, dy_stride, dz_stride, dresidual_stride, dx_stride, dgate_stride;
    int cols, gate_kind;
    double residual_scale, block_scale;
    Starve starve;
};

cudaError_t launch_rms(NormTypes t, NormMode mode, const RmsForwardArgs &a, cudaStream_t stream);
cudaError_t launch_rms_vjp(NormTypes t, NormMode mode, const RmsBackwardArgs &a, void *workspace, cudaStream_t stream);
// Block norms without a gate of float32 rows that fill a cluster of blocks, with a.starve.
cudaError_t launch_rms_starved(const RmsForwardArgs &a, cudaStream_t stream);
cudaError_t launch_rms_vjp_starved(const RmsBackwardArgs &a, void *workspace, cudaStream_t stream);
size_t rms_vjp_workspace(NormTypes t, NormMode mode, size_t rows, size_t cols);

#ifdef __CUDACC__

// The gate's value and, where asked for, its slope.
template <bool FAST, typename W>
__device__ __forceinline__ W gate_value(int kind, W g, W *slope) {
    if (kind == GEO_B200_GATE_LINEAR) {
        if (slope != nullptr) *slope = g == g ? W(1) : g;
        return g;
    }
    W s, rest;
    if (kind == GEO_B200_GATE_SIGMOID) {
        if (slope == nullptr) return logistic<FAST>(g);
        logistic<FAST>(g, s, rest);
        *slope = s * rest;
        return s;
    }
    if (slope != nullptr) {  // 1 - tanh^2 = 4 s (1 - s) at twice the argument, which does not cancel
        logistic<FAST>(g + g, s, rest);
        *slope = W(4) * s * rest;
    }
    return tanh(g);
}

// The gate's values, and where asked for their slopes, of a vector; the kind is looked
// at once for all of them, whose functions are then worked out side by side (the
// VJP of 16384 x 4096 bfloat16, sigmoid: 236 us with a look at each value).
template <bool FAST, bool SLOPES, typename T, int V>
__device__ __forceinline__ void gate_values(int kind, const Vec<T, V> &gate, Pair<Wide<T>> (&f)[V / 2],
                                            Pair<Wide<T>> (&slope)[V / 2]) {
    using W = Wide<T>;
    auto all = [&](auto k) {
#pragma unroll
        for (int q = 0; q < V / 2; ++q) {
            const Pair<W> g = gate.pair(q);
            f[q].x = gate_value<FAST>(decltype(k)::value, g.x, SLOPES ? &slope[q].x : (W *)nullptr);
            f[q].y = gate_value<FAST>(decltype(k)::value, g.y, SLOPES ? &slope[q].y : (W *)nullptr);
        }
    };
    if (kind == GEO_B200_GATE_SIGMOID)
        all(std::integral_constant<int, GEO_B200_GATE_SIGMOID>{});
    else if (kind == GEO_B200_GATE_TANH)
        all(std::integral_constant<int, GEO_B200_GATE_TANH>{});
    else
        all(std::integral_constant<int, GEO_B200_GATE_LINEAR>{});
}

// What the warps of a team sum up together: N values a warp (1, 2 or 4), from every
// lane of it; the sums, the same on every thread. False: a wait gave up, sums are NaN.
template <int N, int TEAM, int V, int K, typename W>
__device__ __forceinline__ bool team_sums(Exchange<W, N, TEAM> &sums, uint32_t round, const Place<TEAM, V, K> &at,
                                          W (&part)[N], bool complete, uint32_t polls = kWaitPolls,
                                          bool silent = false) {
    if constexpr (TEAM == kWarp) {
#pragma unroll
        for (int n = 0; n < N; ++n) part[n] = team_sum(part[n], at.threads);
    } else {
        W mine;
        if constexpr (N == 1)
            mine = team_sum(part[0], 32);
        else
            mine = folded_sums(part);
        complete = exchange(sums, round, at, mine, complete, polls, silent);
        constexpr int kJoin = 32 / N;  // lanes that add one value up
        W total = 0;
#pragma unroll
        for (int j = 0; j < (TEAM == kCluster ? 64 / kJoin : 1); ++j) {
            const int e = at.wlane % kJoin + j * kJoin;
            if (e < at.entries) total += sums.values[round & 1][at.wlane / kJoin][at.first_entry + e];
        }
        total = team_sum(total, kJoin);
        if (!complete) total = (W)NAN;
#pragma unroll
        for (int n = 0; n < N; ++n) part[n] = __shfl_sync(0xffffffffu, total, n * kJoin);
    }
    return complete;
}

// f(MODE) as a compile-time constant.
template <typename F>
cudaError_t by_mode(NormMode mode, F &&f) {
    using std::integral_constant;
    if (mode == kRms) return f(integral_constant<int, kRms>{});
    if (mode == kBlockNorm) return f(integral_constant<int, kBlockNorm>{});
    return f(integral_constant<int, kGatedNorm>{});
}

#endif

}  // namespace layers
}  // namespace geo
