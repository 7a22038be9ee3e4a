// layers.cpp -- argument checks of the layer operators (layers.h).
#include "layers.h"

#include <cmath>

namespace geo {
namespace layers {

bool arrays_usable(std::initializer_list<Array> arrays) {
    int device = -1;
    for (const Array &a : arrays) {
        if (a.pointer == nullptr) continue;
        if ((uintptr_t)a.pointer % a.bytes != 0) return false;
        if (device < 0 && cudaGetDevice(&device) != cudaSuccess) {
            (void)cudaGetLastError();
            return false;
        }
        cudaPointerAttributes attr = {};
        if (cudaPointerGetAttributes(&attr, a.pointer) != cudaSuccess) {
            (void)cudaGetLastError();
            return false;
        }
        const bool usable = attr.type == cudaMemoryTypeManaged ||
                            (attr.type == cudaMemoryTypeDevice && attr.device == device) ||
                            (attr.type == cudaMemoryTypeHost && attr.devicePointer == a.pointer);
        if (!usable) return false;
    }
    return true;
}

bool resolve_strides(size_t rows, size_t cols, std::initializer_list<size_t *> strides) {
    for (size_t *s : strides) {
        if (*s == 0) *s = cols;
        size_t last;
        if (*s < cols || __builtin_mul_overflow(rows, *s, &last) || last > ((size_t)1 << 59)) return false;
    }
    return true;
}

bool make_drop(const geo_b200_dropout_config_t &config, const uint64_t *device_offset, Drop *out) {
    if (type_bytes(config.type) == 0 || config.dimension > 6 || !(config.rate >= 0.0 && config.rate <= 1.0) ||
        config.rows == 0 || config.cols == 0 || config.rows > GEO_B200_LAYER_MAX_ROWS ||
        config.cols > GEO_B200_LAYER_MAX_COLS || (config.cols & (((size_t)1 << config.dimension) - 1)) != 0)
        return false;
    const double threshold = std::nearbyint(config.rate * 65536.0);
    for (uint32_t round = 0; round < 10; ++round) {
        out->key[round][0] = (uint32_t)config.seed + round * 0x9E3779B9u;
        out->key[round][1] = (uint32_t)(config.seed >> 32) + round * 0xBB67AE85u;
    }
    out->offset = config.offset;
    out->device_offset = device_offset;
    out->threshold = (uint32_t)threshold;
    out->bound = (uint32_t)((uint64_t)out->threshold * 65536u - 1u);  // 2^32 - 1 when everything is dropped
    out->scale = threshold < 65536.0 ? 65536.0 / (65536.0 - threshold) : 0.0;
    out->shift = config.dimension;
    return true;
}

}  // namespace layers
}  // namespace geo
