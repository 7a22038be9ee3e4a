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

// Two values of the arithmetic type. float32 pairs go through the packed
// two-wide add, multiply and multiply-add of sm_100a: half the instructions of
// kernels that would otherwise issue more than HBM lets them.
template <typename W>
struct alignas(2 * sizeof(W)) Pair {
    W x, y;
};

__device__ __forceinline__ uint64_t bits_of(Pair<float> a) {
    return (uint64_t)__float_as_uint(a.x) | (uint64_t)__float_as_uint(a.y) << 32;
}
__device__ __forceinline__ Pair<float> pair_of(uint64_t b) {
    return {__uint_as_float((uint32_t)b), __uint_as_float((uint32_t)(b >> 32))};
}
__device__ __forceinline__ Pair<float> operator+(Pair<float> a, Pair<float> b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return pair_of(r);
}
__device__ __forceinline__ Pair<float> operator*(Pair<float> a, Pair<float> b) {
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)));
    return pair_of(r);
}
__device__ __forceinline__ Pair<float> fma(Pair<float> a, Pair<float> b, Pair<float> c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(bits_of(a)), "l"(bits_of(b)), "l"(bits_of(c)));
    return pair_of(r);
}
__device__ __forceinline__ Pair<double> operator+(Pair<double> a, Pair<double> b) { return {a.x + b.x, a.y + b.y}; }
__device__ __forceinline__ Pair<double> operator*(Pair<double> a, Pair<double> b) { return {a.x * b.x, a.y * b.y}; }
__device__ __forceinline__ Pair<double> fma(Pair<double> a, Pair<double> b, Pair<double> c) {
    return {::fma(a.x, b.x, c.x), ::fma(a.y, b.y, c.y)};
}
template <typename W>
__device__ __forceinline__ Pair<W> both(W v) {
    return {v, v};
}

// One value from, and to, its bits in the low half of a word.
template <typename T>
__device__ __forceinline__ float half_of_word(uint32_t w) {
    if constexpr (std::is_same_v<T, __nv_bfloat16>)
        return __uint_as_float(w << 16);
    else
        return __half2float(__ushort_as_half((unsigned short)w));
}

// V adjacent values, moved as one access and held as 32-bit words: 16-bit values
// are taken from and put into a word two at a time (a bfloat16's float32 is its
// own bits: one instruction a value).
template <typename T, int V>
struct Vec {
    static constexpr int kBytes = (int)sizeof(T) * V;
    uint32_t w[kBytes < 4 ? 1 : kBytes / 4];

    __device__ __forceinline__ static Vec zero() {
        Vec r;
#pragma unroll
        for (uint32_t &x : r.w) x = 0;
        return r;
    }
    // Values 2q and 2q + 1.
    __device__ __forceinline__ Pair<Wide<T>> pair(int q) const {
        if constexpr (sizeof(T) == 8) {
            return {__hiloint2double((int)w[4 * q + 1], (int)w[4 * q]),
                    __hiloint2double((int)w[4 * q + 3], (int)w[4 * q + 2])};
        } else if constexpr (sizeof(T) == 4) {
            return {__uint_as_float(w[2 * q]), __uint_as_float(w[2 * q + 1])};
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            return {__uint_as_float(w[q] << 16), __uint_as_float(w[q] & 0xFFFF0000u)};
        } else {
            return {half_of_word<T>(w[q]), half_of_word<T>(w[q] >> 16)};
        }
    }
    __device__ __forceinline__ void set(int q, Pair<Wide<T>> v) {
        if constexpr (sizeof(T) == 8) {
            w[4 * q] = (uint32_t)__double2loint(v.x), w[4 * q + 1] = (uint32_t)__double2hiint(v.x);
            w[4 * q + 2] = (uint32_t)__double2loint(v.y), w[4 * q + 3] = (uint32_t)__double2hiint(v.y);
        } else if constexpr (sizeof(T) == 4) {
            w[2 * q] = __float_as_uint(v.x), w[2 * q + 1] = __float_as_uint(v.y);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            const __nv_bfloat162 r = __floats2bfloat162_rn(v.x, v.y);
            w[q] = *reinterpret_cast<const uint32_t *>(&r);
        } else {
            const __half2 r = __floats2half2_rn(v.x, v.y);
            w[q] = *reinterpret_cast<const uint32_t *>(&r);
        }
    }
    // The value of a Vec of one.
    __device__ __forceinline__ Wide<T> one() const {
        static_assert(V == 1, "one value");
        if constexpr (sizeof(T) == 8)
            return __hiloint2double((int)w[1], (int)w[0]);
        else if constexpr (sizeof(T) == 4)
            return __uint_as_float(w[0]);
        else
            return half_of_word<T>(w[0]);
    }
    __device__ __forceinline__ void set_one(Wide<T> v) {
        static_assert(V == 1, "one value");
        if constexpr (sizeof(T) == 8)
            w[0] = (uint32_t)__double2loint(v), w[1] = (uint32_t)__double2hiint(v);
        else if constexpr (sizeof(T) == 4)
            w[0] = __float_as_uint(v);
        else if constexpr (std::is_same_v<T, __nv_bfloat16>)
            w[0] = __bfloat16_as_ushort(__float2bfloat16_rn(v));
        else
            w[0] = __half_as_ushort(__float2half_rn(v));
    }
};
template <typename T, int V>
__device__ __forceinline__ Vec<T, V> load(const T *p) {
    Vec<T, V> r;
    if constexpr (Vec<T, V>::kBytes == 16) {
        const uint4 v = *reinterpret_cast<const uint4 *>(p);
        r.w[0] = v.x, r.w[1] = v.y, r.w[2] = v.z, r.w[3] = v.w;
    } else if constexpr (Vec<T, V>::kBytes == 8) {
        const uint2 v = *reinterpret_cast<const uint2 *>(p);
        r.w[0] = v.x, r.w[1] = v.y;
    } else if constexpr (Vec<T, V>::kBytes == 4) {
        r.w[0] = *reinterpret_cast<const uint32_t *>(p);
    } else {
        r.w[0] = *reinterpret_cast<const unsigned short *>(p);
    }
    return r;
}
template <typename T, int V>
__device__ __forceinline__ void store(T *p, const Vec<T, V> &v) {
    if constexpr (Vec<T, V>::kBytes == 16)
        *reinterpret_cast<uint4 *>(p) = make_uint4(v.w[0], v.w[1], v.w[2], v.w[3]);
    else if constexpr (Vec<T, V>::kBytes == 8)
        *reinterpret_cast<uint2 *>(p) = make_uint2(v.w[0], v.w[1]);
    else if constexpr (Vec<T, V>::kBytes == 4)
        *reinterpret_cast<uint32_t *>(p) = v.w[0];
    else
        *reinterpret_cast<unsigned short *>(p) = (unsigned short)v.w[0];
}
#endif

#ifdef __CUDACC__
// s = 1 / (1 + e^-a) and rest = 1 - s, each to its own relative accuracy: both from
// e^-|a|. FAST: float32's fast exponential and division (a few 2^-22 relative for
// |a| of a few units, |a| 2^-23 beyond), for results that are rounded to 16 bits.
template <bool FAST, typename W>
__device__ __forceinline__ void logistic(W a, W &s, W &rest) {
    W e, d;
    if constexpr (FAST && sizeof(W) == 4) {
        e = __expf(-fabsf(a));
        d = __fdividef(1.0f, 1.0f + e);
    } else {
        e = exp(-fabs(a));
        d = W(1) / (W(1) + e);
    }
    s = a < W(0) ? e * d : d;
    rest = a < W(0) ? d : e * d;
}
// s alone: 0 where e^-a leaves the type's range (FAST: below -87).
template <bool FAST, typename W>
__device__ __forceinline__ W logistic(W a) {
    if constexpr (FAST && sizeof(W) == 4)
        return __fdividef(1.0f, 1.0f + __expf(-a));
    else
        return W(1) / (W(1) + exp(-a));
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

// Strides of rows x cols arrays, 0 (packed) replaced by cols; false when one is
// below cols or an offset in bytes would not fit 63 bits.
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

#ifdef __CUDACC__
// ---- asynchronous copies into shared memory -----------------------------------

__device__ __forceinline__ uint32_t shared_address(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// 16 bytes (zeros when not `live`), or a word of 4 or 8.
template <int BYTES = 16>
__device__ __forceinline__ void copy_async(uint32_t to, const void *from, bool live = true) {
    if constexpr (BYTES == 16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
    else
        asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}
__device__ __forceinline__ void commit_async() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void wait_async() {
    asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
#endif

// ---- dropout's draws ---------------------------------------------------------

// What a kernel needs of a geo_b200_dropout_config_t.
struct Drop {
    uint32_t key[10][2];  // the seed's two words, advanced for each round
    uint64_t offset;
    const uint64_t *device_offset;
    double scale;        // 65536 / (65536 - threshold); 0 when everything is dropped
    uint32_t threshold;  // drop when draw < threshold, 0 .. 65536
    uint32_t bound;      // (threshold << 16) - 1: keep when draw << 16 is above it (threshold > 0)
    uint32_t shift;      // a unit is 2^shift values
};
// Checks everything but strides and arrays; false when a field is out of range.
bool make_drop(const geo_b200_dropout_config_t &config, const uint64_t *device_offset, Drop *out);

#ifdef __CUDACC__
struct Block {
    uint32_t word[4];
};

// Philox4x32-10: ten rounds of two 32 x 32 -> 64 bit products whose high halves
// are mixed with the key (Salmon et al., SC 2011). The keys of the rounds come
// from the host: as kernel parameters they cost the kernel no instruction.
__device__ __forceinline__ Block philox(uint64_t index, uint64_t offset, const uint32_t (&key)[10][2]) {
    uint32_t c0 = (uint32_t)index, c1 = (uint32_t)(index >> 32);
    uint32_t c2 = (uint32_t)offset, c3 = (uint32_t)(offset >> 32);
#pragma unroll
    for (int round = 0; round < 10; ++round) {
        const uint64_t p0 = (uint64_t)c0 * 0xD2511F53u, p1 = (uint64_t)c2 * 0xCD9E8D57u;
        c0 = (uint32_t)(p1 >> 32) ^ c1 ^ key[round][0];
        c1 = (uint32_t)p1;
        c2 = (uint32_t)(p0 >> 32) ^ c3 ^ key[round][1];
        c3 = (uint32_t)p0;
    }
    return {{c0, c1, c2, c3}};
}

__device__ __forceinline__ uint64_t drop_offset(const Drop &drop) {
    return drop.offset + (drop.device_offset != nullptr ? *drop.device_offset : 0);
}

// Bit i: whether draw i of the block is kept.
__device__ __forceinline__ uint32_t kept_of_block(const Drop &drop, uint64_t offset, uint64_t index) {
    const Block b = philox(index, offset, drop.key);
    uint32_t bits = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        bits |= (uint32_t)((b.word[i] << 16) > drop.bound) << (2 * i);
        bits |= (uint32_t)(b.word[i] > drop.bound) << (2 * i + 1);
    }
    return bits;
}

// Bit j: whether value e + j is kept, j < 8, e a multiple of 8: their units are
// draws of one block.
__device__ __forceinline__ uint32_t kept_of_eight(const Drop &drop, uint64_t offset, uint64_t e) {
    if (drop.threshold == 0) return 0xFFu;
    const uint64_t unit = e >> drop.shift;
    const uint32_t bits = kept_of_block(drop, offset, unit >> 3);
    if (drop.shift == 0) return bits;
    uint32_t out = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) out |= ((bits >> (((uint32_t)unit + ((uint32_t)j >> drop.shift)) & 7u)) & 1u) << j;
    return out;
}

// Words whose low and high halves are the draws of values e + 2q and e + 2q + 1,
// V = 2, 4 or 8 values, V dividing e.
template <int V>
__device__ __forceinline__ void draws_of_pairs(const Drop &drop, uint64_t offset, uint64_t e, uint32_t (&out)[V / 2]) {
    const uint64_t unit = e >> drop.shift;
    const Block b = philox(unit >> 3, offset, drop.key);
    if (drop.shift == 0) {
#pragma unroll
        for (int q = 0; q < V / 2; ++q) {
            out[q] = b.word[q];
            if (V == 4) out[q] = (e & 4) ? b.word[q + 2] : out[q];
            if (V == 2) out[q] = (e & 4) ? ((e & 2) ? b.word[3] : b.word[2]) : ((e & 2) ? b.word[1] : b.word[0]);
        }
    } else {  // both values of a pair are of one unit
#pragma unroll
        for (int q = 0; q < V / 2; ++q) {
            const uint32_t i = (uint32_t)unit + (2u * q >> drop.shift);
            const uint32_t w = (i & 4) ? ((i & 2) ? b.word[3] : b.word[2]) : ((i & 2) ? b.word[1] : b.word[0]);
            out[q] = __byte_perm(w, 0, (i & 1) ? 0x3232 : 0x1010);
        }
    }
}

// Zero where the draw is below the threshold (threshold > 0): selected, not
// multiplied, so that a dropped NaN is gone.
template <typename W>
__device__ __forceinline__ Pair<W> drop_pair(Pair<W> v, uint32_t draws, uint32_t bound) {
    return {(draws << 16) > bound ? v.x : W(0), draws > bound ? v.y : W(0)};
}

// For values spread over a warp: bit i of the result is whether value
// base + i step + lane is kept (i < K), lane = thread of the warp, the same base
// and step on every lane, all lanes taking part. The 32 values of one i lie in at
// most five blocks, so each lane works one block out for six i at a time and
// hands its eight decisions round: a sixth of a block a value instead of one.
template <int K>
__device__ __forceinline__ uint32_t kept_by_warp(const Drop &drop, uint64_t offset, uint64_t base, uint32_t step) {
    if (drop.threshold == 0) return 0xFFFFFFFFu;
    // Places relative to the start of the first value's block, in 32 bits.
    const uint32_t lane = threadIdx.x & 31, whole = drop.shift + 3;
    const uint64_t block = base >> whole;
    const uint32_t in_block = (uint32_t)base & ((8u << drop.shift) - 1u);
    uint32_t kept = 0;
#pragma unroll
    for (int i0 = 0; i0 < K; i0 += 6) {
        const uint32_t from = (in_block + (i0 + lane / 5) * step) >> whole;
        const uint32_t mine = kept_of_block(drop, offset, block + from + lane % 5);
#pragma unroll
        for (int m = 0; m < 6 && i0 + m < K; ++m) {
            const uint32_t first = in_block + (i0 + m) * step, place = first + lane;
            const uint32_t bits = __shfl_sync(0xffffffffu, mine, m * 5 + (place >> whole) - (first >> whole));
            kept |= ((bits >> ((place >> drop.shift) & 7u)) & 1u) << (i0 + m);
        }
    }
    return kept;
}

// Whether the unit is kept; for callers that look at one unit at a time.
__device__ __forceinline__ bool unit_kept(const Drop &drop, uint64_t offset, uint64_t unit) {
    const Block b = philox(unit >> 3, offset, drop.key);
    const uint32_t word = (unit & 4) ? ((unit & 2) ? b.word[3] : b.word[2]) : ((unit & 2) ? b.word[1] : b.word[0]);
    return ((unit & 1) ? word : word << 16) > drop.bound;
}
#endif

}  // namespace layers
}  // namespace geo
