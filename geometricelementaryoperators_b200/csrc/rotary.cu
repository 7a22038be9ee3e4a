// rotary.cu -- rotary positions and their VJP (geo/geo_b200.h section 5).
//
// Pair i of a head at position p is turned by t = p f_i. The angle is taken in
// turns, p (hi + lo), with the rounding error of p hi recovered by a fused
// multiply-add, and its whole quarter turns are dropped in float64 before the
// sine and cosine are taken in the arithmetic type: what is left is at most an
// eighth of a turn, so its conversion to float32 costs 2^-28 turns and far
// positions lose nothing.
#include <cmath>

#include "geo_runtime.h"
#include "layers.h"

namespace {

using namespace geo::layers;

constexpr int kThreads = 256;

struct RotaryArgs {
    const void *x, *positions;
    void *y;
    size_t batch, tokens, heads, head_dim;
    size_t xb, xt, xh, yb, yt, yh, pb;
    int64_t first_position;
};

template <typename W>
__device__ __forceinline__ void rotor(int64_t position, double hi, double lo, W amplitude, W &c, W &s) {
    const double p = (double)position;
    const double turns = p * hi;
    const double rest = fma(p, lo, fma(p, hi, -turns));
    const double quarters = rint(turns * 4.0);
    const double left = (turns - quarters * 0.25) + rest;
    W sine, cosine;
    if constexpr (std::is_same_v<W, double>)
        sincospi(2.0 * left, &sine, &cosine);
    else
        sincospif((float)(2.0 * left), &sine, &cosine);
    const int q = (int)((long long)quarters & 3);
    c = amplitude * ((q & 1) ? (q == 1 ? -sine : sine) : (q == 0 ? cosine : -cosine));
    s = amplitude * ((q & 1) ? (q == 1 ? cosine : -cosine) : (q == 0 ? sine : -sine));
}

// One pair (or one copied coordinate past rotary_dim) of one token per thread,
// all heads.
template <typename T, typename I>
__global__ void __launch_bounds__(kThreads)
    rotary_kernel(const RotaryArgs a, const __grid_constant__ geo_b200_rotary_plan_t plan, int backward) {
    using W = Wide<T>;
    const size_t pairs = plan.rotary_dim / 2, columns = a.head_dim - pairs;
    const size_t count = a.batch * a.tokens * columns;
    for (size_t i = blockIdx.x * (size_t)kThreads + threadIdx.x; i < count; i += (size_t)gridDim.x * kThreads) {
        const size_t bt = i / columns, column = i - bt * columns;
        const size_t b = bt / a.tokens, t = bt - b * a.tokens;
        const T *x = (const T *)a.x + b * a.xb + t * a.xt;
        T *y = (T *)a.y + b * a.yb + t * a.yt;
        if (column >= pairs) {
            const size_t at = column + pairs;
            for (size_t h = 0; h < a.heads; ++h) y[h * a.yh + at] = x[h * a.xh + at];
            continue;
        }
        const int64_t position = a.positions != nullptr ? (int64_t)((const I *)a.positions)[b * a.pb + t]
                                                        : a.first_position + (int64_t)t;
        W c, s;
        rotor<W>(position, plan.turns[column], plan.turns_low[column], (W)plan.amplitude, c, s);
        if (backward) s = -s;
        const bool half = plan.layout == GEO_B200_ROTARY_HALF;
        const size_t ia = half ? column : 2 * column, ib = half ? column + pairs : 2 * column + 1;
        for (size_t h = 0; h < a.heads; ++h) {
            const W u = widen(x[h * a.xh + ia]), v = widen(x[h * a.xh + ib]);
            y[h * a.yh + ia] = narrow<T>(u * c - v * s);
            y[h * a.yh + ib] = narrow<T>(u * s + v * c);
        }
    }
}

// Strides (0 = packed) of one array; false when an offset would not fit.
bool resolve(const geo_b200_rotary_shape_t &s, size_t *sb, size_t *st, size_t *sh) {
    const size_t limit = (size_t)1 << 59;
    size_t span;
    if (*sh == 0) *sh = s.head_dim;
    if (*st == 0 && (__builtin_mul_overflow(s.heads, *sh, st) || *st > limit)) return false;
    if (*sb == 0 && (__builtin_mul_overflow(s.tokens, *st, sb) || *sb > limit)) return false;
    size_t total = s.head_dim;
    const size_t counts[3] = {s.batch, s.tokens, s.heads}, strides[3] = {*sb, *st, *sh};
    for (int i = 0; i < 3; ++i) {
        if (__builtin_mul_overflow(counts[i] - 1, strides[i], &span) || span > limit) return false;
        total += span;
    }
    return total <= limit;
}

// Whether the heads of an array are apart: ordered by stride, each step clears
// everything below it.
bool apart(const geo_b200_rotary_shape_t &s, size_t sb, size_t st, size_t sh) {
    size_t counts[3] = {s.batch, s.tokens, s.heads}, strides[3] = {sb, st, sh};
    size_t span = s.head_dim;
    for (int round = 0; round < 3; ++round) {
        int least = -1;
        for (int i = 0; i < 3; ++i)
            if (counts[i] > 1 && (least < 0 || strides[i] < strides[least])) least = i;
        if (least < 0) break;
        if (strides[least] < span) return false;
        span += (counts[least] - 1) * strides[least];
        counts[least] = 1;
    }
    return true;
}

geo_b200_status_t rotary(const geo_b200_rotary_plan_t *plan, const geo_b200_rotary_shape_t *shape,
                         const void *device_x, const void *device_positions, void *device_y, bool backward,
                         cudaStream_t stream) {
    if (plan == nullptr || shape == nullptr || device_x == nullptr || device_y == nullptr ||
        plan->abi_version != GEO_B200_ABI_VERSION || plan->layout > GEO_B200_ROTARY_HALF || plan->rotary_dim < 2 ||
        plan->rotary_dim > GEO_B200_ROTARY_MAX_DIM || plan->rotary_dim % 2 != 0 || !std::isfinite(plan->amplitude))
        return GEO_B200_INVALID_ARGUMENT;
    geo_b200_rotary_shape_t s = *shape;
    const size_t b = type_bytes(s.type);
    if (b == 0 || (s.position_type != GEO_B200_I32 && s.position_type != GEO_B200_I64) || s.batch == 0 ||
        s.tokens == 0 || s.heads == 0 || s.head_dim < plan->rotary_dim || s.head_dim > 65536)
        return GEO_B200_INVALID_ARGUMENT;
    size_t tokens, values;
    if (__builtin_mul_overflow(s.batch, s.tokens, &tokens) || __builtin_mul_overflow(tokens, s.head_dim, &values) ||
        __builtin_mul_overflow(values, s.heads, &values) || values > ((size_t)1 << 59) ||
        !resolve(s, &s.x_batch_stride, &s.x_token_stride, &s.x_head_stride) ||
        !resolve(s, &s.y_batch_stride, &s.y_token_stride, &s.y_head_stride) ||
        !apart(s, s.y_batch_stride, s.y_token_stride, s.y_head_stride))
        return GEO_B200_INVALID_ARGUMENT;
    const int64_t limit = (int64_t)1 << 31;
    if (device_positions == nullptr &&
        (s.first_position < -limit || s.first_position > limit || s.tokens > (size_t)limit ||
         s.first_position + (int64_t)(s.tokens - 1) > limit))
        return GEO_B200_INVALID_ARGUMENT;
    if (device_x == device_y && (s.x_batch_stride != s.y_batch_stride || s.x_token_stride != s.y_token_stride ||
                                 s.x_head_stride != s.y_head_stride))
        return GEO_B200_INVALID_ARGUMENT;
    if (!arrays_usable({{device_x, b}, {device_y, b}, {device_positions, s.position_type == GEO_B200_I32 ? 4u : 8u}}))
        return GEO_B200_INVALID_ARGUMENT;
    RotaryArgs a;
    a.x = device_x;
    a.positions = device_positions;
    a.y = device_y;
    a.batch = s.batch;
    a.tokens = s.tokens;
    a.heads = s.heads;
    a.head_dim = s.head_dim;
    a.xb = s.x_batch_stride;
    a.xt = s.x_token_stride;
    a.xh = s.x_head_stride;
    a.yb = s.y_batch_stride;
    a.yt = s.y_token_stride;
    a.yh = s.y_head_stride;
    a.pb = s.position_batch_stride;
    a.first_position = s.first_position;
    return status_of(by_type(s.type, [&](auto t) {
        using T = decltype(t);
        const size_t count = tokens * (s.head_dim - plan->rotary_dim / 2);
        const size_t blocks = (count + kThreads - 1) / kThreads, most = (size_t)geo::device_sm_count() * 32;
        const unsigned grid = (unsigned)(blocks < most ? blocks : most);
        if (s.position_type == GEO_B200_I32)
            rotary_kernel<T, int32_t><<<grid, kThreads, 0, stream>>>(a, *plan, backward);
        else
            rotary_kernel<T, int64_t><<<grid, kThreads, 0, stream>>>(a, *plan, backward);
        return cudaGetLastError();
    }));
}

}  // namespace

extern "C" geo_b200_status_t geo_b200_rotary(const geo_b200_rotary_plan_t *plan, const geo_b200_rotary_shape_t *shape,
                                             const void *device_x, const void *device_positions, void *device_y,
                                             cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.rotary");
    return rotary(plan, shape, device_x, device_positions, device_y, false, stream);
}

extern "C" geo_b200_status_t geo_b200_rotary_vjp(const geo_b200_rotary_plan_t *plan,
                                                 const geo_b200_rotary_shape_t *shape, const void *device_y_cotangent,
                                                 const void *device_positions, void *device_x_cotangent,
                                                 cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.rotary_vjp");
    return rotary(plan, shape, device_y_cotangent, device_positions, device_x_cotangent, true, stream);
}
