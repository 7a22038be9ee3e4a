// layers.h -- what the layer operators (layer_norm.cu, dropout.cu, rotary.cu;
// geo/geo_b200.h section 5) share: value types, argument checks, the
// counter-based draws of dropout.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <initializer_list>
#include <type_traits>

#include "geo/geo_b200.h"

namespace geo {
namespace layers {

// ---- value types -------------------------------------------------------------

#ifdef __CUDACC__
// Arithmetic type of a value type: float64 for float64, else float32 (every
// 16-bit value is exact in it; only a result's final conversion rounds).
template <typename T>
using Wide = std::conditional_t<std::is_same_v<T, double>, double, float>;

__device__ __forceinline__ double widen(double v) { return v; }
__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T narrow(Wide<T> v) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        return __float2bfloat16_rn(v);
    else if constexpr (std::is_same_v<T, __half>)
        return __float2half_rn(v);
    else
        return v;
}

#endif

inline size_t type_bytes(uint32_t type) {
    switch (type) {
        case GEO_B200_F64: return 8;
        case GEO_B200_F32: return 4;
        case GEO_B200_BF16:
        case GEO_B200_F16: return 2;
        default: return 0;
    }
}
inline size_t wide_bytes(uint32_t type) { return type == GEO_B200_F64 ? 8 : 4; }

#ifdef __CUDACC__
// f(T{}) for the value type `type`, which the caller has checked.
template <typename F>
cudaError_t by_type(uint32_t type, F &&f) {
    switch (type) {
        case GEO_B200_F64: return f(double{});
        case GEO_B200_F32: return f(float{});
        case GEO_B200_BF16: return f(__nv_bfloat16{});
        default: return f(__half{});
    }
}

#endif

// ---- argument checks ---------------------------------------------------------

struct Array {
    const void *pointer;
    size_t bytes;  // of one value
};
// Every non-null array is aligned to its values and readable by kernels of the
// current device: its own memory, managed memory or pinned host memory. A
// pointer of another device or of pageable memory would fault in the kernel.
bool arrays_usable(std::initializer_list<Array> arrays);

// Row length and strides (0 = packed, replaced by cols) of up to `count` arrays;
// false when a stride is below cols or an offset would not fit 63 bits.
bool resolve_strides(size_t rows, size_t cols, std::initializer_list<size_t *> strides);

// An output may be an input only with the same stride.
inline bool same_or_apart(const void *out, size_t out_stride, const void *in, size_t in_stride) {
    return out == nullptr || out != in || out_stride == in_stride;
}

inline geo_b200_status_t status_of(cudaError_t e) {
    if (e == cudaSuccess) return GEO_B200_OK;
    (void)cudaGetLastError();  // launch errors do not stay behind for the caller's next check
    return GEO_B200_RUNTIME_FAILURE;
}

// ---- dropout's draws ---------------------------------------------------------

// What a kernel needs of a geo_b200_dropout_config_t.
struct Drop {
    uint64_t seed;
    uint64_t offset;
    const uint64_t *device_offset;
    double scale;        // 65536 / (65536 - threshold); 0 when everything is dropped
    uint32_t threshold;  // drop when draw < threshold, 0 .. 65536
    uint32_t shift;      // a unit is 2^shift values
};
// Checks everything but strides and arrays; false when a field is out of range.
bool make_drop(const geo_b200_dropout_config_t &config, const uint64_t *device_offset, Drop *out);

#ifdef __CUDACC__
struct Block {
    uint32_t word[4];
};

// Philox4x32-10: ten rounds of two 32 x 32 -> 64 bit products whose high halves
// are mixed with the key (Salmon et al., SC 2011).
__device__ __forceinline__ Block philox(uint64_t index, uint64_t offset, uint64_t seed) {
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32);
    uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0;
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
        c3 = (uint32_t)p0;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ uint64_t drop_offset(const Drop &drop) {
    return drop.offset + (drop.device_offset != nullptr ? *drop.device_offset : 0);
}

// Whether the unit is kept; for callers that look at one unit at a time.
__device__ __forceinline__ bool unit_kept(const Drop &drop, uint64_t offset, uint64_t unit) {
    const Block b = philox(unit >> 3, offset, drop.seed);
    const uint32_t word = (unit & 4) ? ((unit & 2) ? b.word[3] : b.word[2]) : ((unit & 2) ? b.word[1] : b.word[0]);
    return ((unit & 1) ? word >> 16 : word & 0xFFFFu) >= drop.threshold;
}
#endif

}  // namespace layers
}  // namespace geo
