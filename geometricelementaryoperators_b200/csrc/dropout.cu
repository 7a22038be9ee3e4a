// dropout.cu -- dropout with a mask computed from a counter, and its VJP
// (geo/geo_b200.h section 5).
#include "geo_runtime.h"
#include "layers.h"

namespace {

using namespace geo::layers;

constexpr int kThreads = 256;

// One value per thread.
template <typename T>
__global__ void __launch_bounds__(kThreads)
    drop_kernel(const T *x, size_t x_stride, const T *residual, size_t residual_stride, T *y, size_t y_stride,
                size_t rows, uint32_t cols, const Drop drop) {
    using W = Wide<T>;
    const uint64_t offset = drop_offset(drop);
    const W scale = (W)drop.scale;
    const size_t count = rows * cols;
    for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < count; i += (size_t)gridDim.x * kThreads) {
        const size_t row = i / cols, c = i - row * cols;
        W v = drop.threshold == 0 || unit_kept(drop, offset, i >> drop.shift) ? widen(x[row * x_stride + c]) * scale
                                                                              : W(0);
        if (residual != nullptr) v += widen(residual[row * residual_stride + c]);
        y[row * y_stride + c] = narrow<T>(v);
    }
}

cudaError_t launch(uint32_t type, const void *x, size_t x_stride, const void *residual, size_t residual_stride,
                   void *y, size_t y_stride, size_t rows, size_t cols, const Drop &drop, cudaStream_t stream) {
    return by_type(type, [&](auto t) {
        using T = decltype(t);
        const size_t blocks = (rows * cols + kThreads - 1) / kThreads, most = (size_t)geo::device_sm_count() * 32;
        drop_kernel<T><<<(unsigned)(blocks < most ? blocks : most), kThreads, 0, stream>>>(
            (const T *)x, x_stride, (const T *)residual, residual_stride, (T *)y, y_stride, rows, (uint32_t)cols,
            drop);
        return cudaGetLastError();
    });
}

}  // namespace

extern "C" geo_b200_status_t geo_b200_dropout(const geo_b200_dropout_config_t *config, const void *device_x,
                                              const void *device_residual, const uint64_t *device_offset,
                                              void *device_y, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.dropout");
    Drop drop;
    if (config == nullptr || device_x == nullptr || device_y == nullptr || !make_drop(*config, device_offset, &drop))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_dropout_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.x_stride, &c.residual_stride, &c.y_stride}) ||
        !same_or_apart(device_y, c.y_stride, device_x, c.x_stride) ||
        !same_or_apart(device_y, c.y_stride, device_residual, c.residual_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_residual, b}, {device_y, b}, {device_offset, 8}}))
        return GEO_B200_INVALID_ARGUMENT;
    return status_of(launch(c.type, device_x, c.x_stride, device_residual, c.residual_stride, device_y, c.y_stride,
                            c.rows, c.cols, drop, stream));
}

extern "C" geo_b200_status_t geo_b200_dropout_vjp(const geo_b200_dropout_config_t *config,
                                                  const uint64_t *device_offset, const void *device_y_cotangent,
                                                  void *device_x_cotangent, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.dropout_vjp");
    Drop drop;
    if (config == nullptr || device_y_cotangent == nullptr || device_x_cotangent == nullptr ||
        !make_drop(*config, device_offset, &drop))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_dropout_config_t c = *config;
    if (!resolve_strides(c.rows, c.cols, {&c.y_cotangent_stride, &c.x_cotangent_stride}) ||
        !same_or_apart(device_x_cotangent, c.x_cotangent_stride, device_y_cotangent, c.y_cotangent_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type);
    if (!arrays_usable({{device_y_cotangent, b}, {device_x_cotangent, b}, {device_offset, 8}}))
        return GEO_B200_INVALID_ARGUMENT;
    return status_of(launch(c.type, device_y_cotangent, c.y_cotangent_stride, nullptr, 0, device_x_cotangent,
                            c.x_cotangent_stride, c.rows, c.cols, drop, stream));
}
