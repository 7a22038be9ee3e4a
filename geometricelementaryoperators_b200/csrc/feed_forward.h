// feed_forward.h -- what the gated feed-forward block's entry points
// (feed_forward.cu) and products (feed_forward_tensor.cu: 16-bit types on the tensor
// cores; feed_forward_wide.cu: float32 and float64; feed_forward_plain.cu: few rows, and
// 16-bit arrays that the tensor cores cannot be given; feed_forward_scale.cu: float16's
// powers of two) share.
#pragma once

#include "layers.h"

namespace geo {
namespace layers {

// A row-major array; stride in values.
struct Matrix {
    const void *p;
    size_t stride;
};
struct OutMatrix {
    void *p;
    size_t stride;
};

// The products of the block. M x N results, sums over K:
enum ProductKind : int {
    kGated = 0,   // gate = x Wg^T, up = x Wu^T, h = act(gate) up:   a[0] [M][K], b[0], b[1] [N][K]
    kDown = 1,    // y = h Wd^T:                                     a[0] [M][K], b[0] [N][K]
    kHidden = 2,  // h_bar = y_bar Wd, from it the cotangents of gate and up, and h: a[0] [M][K], b[0] [K][N]
    kInput = 3,   // x_bar = gate_bar Wg + up_bar Wu:                a[0], a[1] [M][K], b[0], b[1] [K][N]
    kWeights = 4  // up to three results of one size, a[z]^T b[z]:   a[z] [K][M], b[z] [K][N]
};

struct Product {
    int m, n, k;
    int activation;    // geo_b200_activation_t
    int problems;      // kWeights: how many results; else 1
    int splits;        // parts of K, each with sums of its own in `partial`, which are then joined; mostly 1
    Matrix a[3], b[3];
    Matrix low[3];     // kWeights to float32 from 16-bit types: what a[z] lost to rounding
    Matrix saved[2];   // kHidden: gate, up
    OutMatrix out[3];  // kGated: gate, up (may be null), h; kHidden: cotangents of gate and up, h; kWeights: [M][N], or
    bool transposed[3];     // ... [N][M]
    OutMatrix out_low[3];  // kHidden: what those lost to rounding, or null
    const float *times[3]; // float16's VJP: device memory of what out[i] is multiplied by, a power of two; or null
    void *partial;     // splits > 1: [sum][split][M][partial_stride(N)] of the arithmetic type
};
__host__ __device__ inline size_t partial_stride(size_t n) { return (n + 3) / 4 * 4; }
// How many sums a result takes (kGated: gate and up), as `problems` are asked for.
constexpr int sums_of(ProductKind kind, int problems) { return kind == kGated ? 2 : (kind == kWeights ? problems : 1); }

// How a product is cut into tiles, and K into parts: by its sizes and the
// multiprocessors alone, for the kernels that take it. Counts all three results of kWeights, whichever are asked for.
struct Cut {
    int columns;  // of a tile of sums
    bool pair;    // two blocks a tile
    int splits;
};
Cut cut_tensor(ProductKind kind, uint32_t type, bool twice, size_t m, size_t n, size_t k);
Cut cut_wide(ProductKind kind, uint32_t type, size_t m, size_t n, size_t k);
Cut cut_plain(ProductKind kind, size_t m, size_t n, size_t k);
// Values of `partial`.
inline size_t partial_values(ProductKind kind, int splits, size_t m, size_t n) {
    return splits > 1 ? (size_t)sums_of(kind, 3) * splits * m * partial_stride(n) : 0;
}
// Adds the parts up, in their order, and does with the sums what the product's kernel does otherwise.
cudaError_t launch_join(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p, cudaStream_t stream);

// For the self-test of the pipeline's waits alone: the block of K at which the
// producer of every CTA stops (never: UINT32_MAX), and how often a wait looks.
struct PipelineStarve {
    uint32_t block, polls;
};
constexpr uint32_t kPipelinePolls = 1u << 20;  // seconds, where a stage takes microseconds

// `type`: of the operands; `out_type`: of kWeights' results. A stream-ordered launch.
cudaError_t launch_product_tensor(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p,
                                  PipelineStarve starve, cudaStream_t stream);
cudaError_t launch_product_wide(ProductKind kind, uint32_t type, const Product &p, cudaStream_t stream);
cudaError_t launch_product_plain(ProductKind kind, uint32_t type, uint32_t out_type, const Product &p,
                                 cudaStream_t stream);
// kGated, kDown with at most kFewRows rows.
constexpr int kFewRows = 8;
cudaError_t launch_product_few(ProductKind kind, uint32_t type, const Product &p, cudaStream_t stream);
// Copies arrays of 16-bit values to rows of `to_stride` (a multiple of 8), zeros behind each row's end.
constexpr int kPackMost = 5;
struct Pack {
    int count;
    struct Array {
        Matrix from;
        size_t rows;
        int cols;
        void *to;
        size_t to_stride;
        size_t end;  // of its pieces of 8 values, all arrays counted one after another
    } arrays[kPackMost];
};
cudaError_t launch_pack(const Pack &pack, cudaStream_t stream);
// float16's VJP: found[0] = the power of two for the cotangents of gate and up, its
// inverse, that for h, its inverse; behind it room for kScaleBlocks more.
constexpr int kScaleBlocks = 1024;
struct InnerScale {
    Matrix dy, wd, gate, up;  // dy, wd: null where only h is wanted
    size_t rows, cols, hidden;
    int activation;
    float4 *found;
};
cudaError_t launch_scale(const InnerScale &scale, cudaStream_t stream);
// Whether the tensor-core products can run at all (the driver's tensor map encoder).
bool tensor_products_available();

#ifdef __CUDACC__
// A kernel whose start-up overlaps the end of the one before it in the stream; before
// it reads or writes anything it waits for that one (after_previous).
__device__ __forceinline__ void after_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, unsigned threads, size_t shared, unsigned cluster,
                         cudaStream_t stream, const A &...args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute attributes[2] = {};
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = cluster;
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

// What v loses to its rounding to T, itself to be rounded to T: together they hold
// twice T's digits as far as T's range goes (float16's inner values are brought into it
// first, feed_forward_scale.cu). (What T has no finite value for loses an infinity or NaN.)
template <typename T>
__device__ __forceinline__ float lost_to(float v) {
    return v - widen(narrow<T>(v));
}

// ---- the activation ------------------------------------------------------------

// act(a) and, where `slope` is asked for, act'(a). FAST: logistic()'s, next to the
// 16-bit rounding of what it enters.
template <bool FAST, typename W>
__device__ __forceinline__ W activation(int kind, W a, W *slope) {
    switch (kind) {
        case GEO_B200_ACTIVATION_RELU:
            if (slope != nullptr) *slope = a > W(0) ? W(1) : (a == a ? W(0) : a);  // NaN stays
            return a > W(0) ? a : (a == a ? W(0) : a);
        case GEO_B200_ACTIVATION_GELU: {
            // Phi by the complementary error function, whose far tail keeps its relative accuracy.
            const W below = W(0.5) * erfc(a * W(-0.70710678118654752440));
            if (slope != nullptr) *slope = below + a * (exp(W(-0.5) * a * a) * W(0.39894228040143267794));
            return a * below;
        }
        default: {
            if (slope == nullptr) {
                const W alone = logistic<FAST>(a);
                return kind == GEO_B200_ACTIVATION_SIGMOID ? alone : a * alone;
            }
            W s, rest;
            logistic<FAST>(a, s, rest);
            *slope = kind == GEO_B200_ACTIVATION_SIGMOID ? s * rest : s * (W(1) + a * rest);
            if (kind == GEO_B200_ACTIVATION_SIGMOID) return s;
            return a * s;
        }
    }
}
// f(kind as a compile-time constant): chosen once for many values, whose functions can
// then be worked out side by side.
template <typename F>
__device__ __forceinline__ void by_activation(int kind, F &&f) {
    using std::integral_constant;
    switch (kind) {
        case GEO_B200_ACTIVATION_SILU: f(integral_constant<int, GEO_B200_ACTIVATION_SILU>{}); break;
        case GEO_B200_ACTIVATION_GELU: f(integral_constant<int, GEO_B200_ACTIVATION_GELU>{}); break;
        case GEO_B200_ACTIVATION_SIGMOID: f(integral_constant<int, GEO_B200_ACTIVATION_SIGMOID>{}); break;
        default: f(integral_constant<int, GEO_B200_ACTIVATION_RELU>{}); break;
    }
}

// What result n is multiplied by.
template <typename T>
__device__ __forceinline__ Wide<T> times_of(const Product &p, int n) {
    if constexpr (std::is_same_v<T, __half>)
        return p.times[n] != nullptr ? *p.times[n] : 1.0f;
    else
        return Wide<T>(1);
}

// What is done with the sums of one place of a product's result: gate and up (kGated), or one.
template <typename T, typename O, int KIND>
__device__ __forceinline__ void finish(const Product &p, int problem, size_t row, size_t col, Wide<T> v, Wide<T> other) {
    using W = Wide<T>;
    constexpr bool kFast = sizeof(T) == 2;
    auto put = [&](const OutMatrix &out, W x) {
        if (out.p != nullptr) ((T *)out.p)[row * out.stride + col] = narrow<T>(x);
    };
    auto scaled = [&](int n, W x) { return x * times_of<T>(p, n); };
    if constexpr (KIND == kGated) {
        put(p.out[0], v);
        put(p.out[1], other);
        put(p.out[2], activation<kFast>(p.activation, v, (W *)nullptr) * other);
    } else if constexpr (KIND == kHidden) {
        const W g = widen(((const T *)p.saved[0].p)[row * p.saved[0].stride + col]);
        const W u = widen(((const T *)p.saved[1].p)[row * p.saved[1].stride + col]);
        W slope;
        const W f = activation<kFast>(p.activation, g, &slope);
        auto put_two = [&](int n, W x) {
            x = scaled(n, x);
            put(p.out[n], x);
            if constexpr (sizeof(T) == 2) put(p.out_low[n], lost_to<T>(x));
        };
        put_two(0, v * u * slope);
        put_two(1, v * f);
        put_two(2, f * u);
    } else if constexpr (KIND == kWeights) {
        const OutMatrix &out = p.out[problem];
        ((O *)out.p)[p.transposed[problem] ? col * out.stride + row : row * out.stride + col] =
            narrow<O>((Wide<O>)scaled(problem, v));
    } else {
        put(p.out[0], scaled(0, v));
    }
}
#endif

}  // namespace layers
}  // namespace geo
