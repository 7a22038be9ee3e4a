// layer_norm.cu -- layer norm over rows, alone and behind residual + dropout,
// and their VJPs (geo/geo_b200.h section 5).
//
// Forward, per row of C values: m = sum x / C, v = sum (x - m)^2 / C,
// y = (x - m) rstd w + b. VJP with xh = (x - m) rstd, g = y_bar w:
//   x_bar = rstd (g - mean(g) - xh mean(g xh)),
//   w_bar = sum_rows y_bar xh, b_bar = sum_rows y_bar.
// Every variant does a few multiply-adds per value, so HBM bounds it.
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

// out[c] = sum over the blocks of partial[block][which][c], in block order.
template <typename W, typename P>
__global__ void __launch_bounds__(kThreads) join_columns_kernel(const W *partial, int blocks, int cols, void *dweight,
                                                                void *dbias) {
    const int c = (int)blockIdx.x * kThreads + threadIdx.x;
    if (c >= cols) return;
    P *out = (P *)(blockIdx.y == 0 ? dweight : dbias);
    if (out == nullptr) return;
    W sum = 0;
    for (int i = 0; i < blocks; ++i) sum += partial[((size_t)i * 2 + blockIdx.y) * cols + c];
    out[c] = narrow<P>((Wide<P>)sum);
}

// ---- launches ----------------------------------------------------------------

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

template <bool DROP>
cudaError_t launch_forward(const geo_b200_layer_norm_config_t &c, const ForwardArgs &a, cudaStream_t stream) {
    return by_types(c.type, c.parameter_type, [&](auto t, auto p) {
        norm_any_kernel<decltype(t), decltype(p), DROP><<<row_grid(a.rows), kThreads, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

template <bool DROP>
cudaError_t launch_backward(const geo_b200_layer_norm_config_t &c, const BackwardArgs &a, void *workspace,
                            cudaStream_t stream) {
    return by_types(c.type, c.parameter_type, [&](auto t, auto p) {
        using T = decltype(t);
        using P = decltype(p);
        using W = Wide<T>;
        // Columns first: the row kernel may overwrite x or y_bar.
        if (a.dweight != nullptr || a.dbias != nullptr) {
            const size_t blocks = column_blocks(a.rows, a.cols);
            const dim3 grid((unsigned)((a.cols + 31) / 32), (unsigned)blocks);
            vjp_columns_any_kernel<T>
                <<<grid, kThreads, 0, stream>>>(a, (W *)workspace, (a.rows + blocks - 1) / blocks);
            const dim3 join((unsigned)((a.cols + kThreads - 1) / kThreads), 2);
            join_columns_kernel<W, P><<<join, kThreads, 0, stream>>>((const W *)workspace, (int)blocks, a.cols,
                                                                     a.dweight, a.dbias);
        }
        if (a.dsum != nullptr || a.dx != nullptr)
            vjp_rows_any_kernel<T, P, DROP><<<row_grid(a.rows), kThreads, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

bool config_valid(const geo_b200_layer_norm_config_t *c) {
    if (c == nullptr || type_bytes(c->type) == 0) return false;
    if (c->parameter_type != c->type && !(type_bytes(c->type) == 2 && c->parameter_type == GEO_B200_F32)) return false;
    return c->rows != 0 && c->cols != 0 && c->rows <= GEO_B200_LAYER_MAX_ROWS && c->cols <= GEO_B200_LAYER_MAX_COLS &&
           std::isfinite(c->epsilon) && c->epsilon >= 0.0;
}

size_t workspace_bytes_of(const geo_b200_layer_norm_config_t &c) {
    return column_blocks(c.rows, c.cols) * 2 * c.cols * wide_bytes(c.type);
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
