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
    size_t groups, share;  // heads are split into `groups` of `share`
    int narrow_positions;
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

// SPLIT: pair j is value j of p and of q; else pair j is values 2j, 2j + 1 of p.
template <typename T, int V, bool SPLIT, int C>
__device__ __forceinline__ void turn(Vec<T, V> &p, Vec<T, V> &q, const Pair<Wide<T>> (&c)[C],
                                     const Pair<Wide<T>> (&s)[C]) {
    using W = Wide<T>;
    if constexpr (V == 1) {
        const W a = p.one(), b = q.one();
        p.set_one(a * c[0].x - b * s[0].x);
        q.set_one(a * s[0].x + b * c[0].x);
    } else if constexpr (SPLIT) {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const Pair<W> a = p.pair(j), b = q.pair(j);
            p.set(j, fma(a, c[j], b * Pair<W>{-s[j].x, -s[j].y}));
            q.set(j, fma(a, s[j], b * c[j]));
        }
    } else {
#pragma unroll
        for (int j = 0; j < V / 2; ++j) {
            const Pair<W> a = p.pair(j);
            const W cosine = j & 1 ? c[j / 2].y : c[j / 2].x, sine = j & 1 ? s[j / 2].y : s[j / 2].x;
            p.set(j, {a.x * cosine - a.y * sine, a.x * sine + a.y * cosine});
        }
    }
}

// A thread takes the pairs that one vector (INTERLEAVED: V / 2 pairs) or two
// vectors half a head apart (HALF: V pairs) hold of one token, works their rotors
// out once, and turns them in `share` heads, kHeads loads ahead; the coordinates
// past rotary_dim go the same way as vectors that are only copied. Where nothing
// wider than a value is aligned, a pair is two values.
constexpr int kHeads = 4;
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kThreads)
    rotary_kernel(const RotaryArgs a, const __grid_constant__ geo_b200_rotary_plan_t plan, int backward) {
    using W = Wide<T>;
    constexpr bool SPLIT = HALF || V == 1;     // a pair's coordinates are in two vectors
    constexpr int N = SPLIT ? 2 : 1;           // vectors a head
    constexpr int PAIRS = SPLIT ? V : V / 2;   // pairs a thread
    const uint32_t half = plan.rotary_dim / 2, second = HALF ? half : 1;
    const uint32_t turned = plan.rotary_dim / (N * V);
    const uint32_t units = turned + ((uint32_t)a.head_dim - plan.rotary_dim) / V;
    const size_t count = a.batch * a.tokens * a.groups * units;
    for (size_t id = blockIdx.x * (size_t)kThreads + threadIdx.x; id < count; id += (size_t)gridDim.x * kThreads) {
        size_t rest = id / units;
        const uint32_t unit = (uint32_t)(id - rest * units);
        const size_t bt = rest / a.groups, group = rest - bt * a.groups;
        const size_t b = bt / a.tokens, t = bt - b * a.tokens;
        const size_t from = group * a.share, left = a.heads - from;
        const size_t heads = left < a.share ? left : a.share;
        const bool copied = unit >= turned;
        if (copied && a.x == a.y) continue;
        const size_t at = copied ? plan.rotary_dim + (size_t)(unit - turned) * V : (size_t)unit * (HALF ? V : N * V);
        const T *x = (const T *)a.x + b * a.xb + t * a.xt + from * a.xh + at;
        T *y = (T *)a.y + b * a.yb + t * a.yt + from * a.yh + at;
        Pair<W> c[(PAIRS + 1) / 2], s[(PAIRS + 1) / 2];
        if (!copied) {
            const size_t where = b * a.pb + t;
            const int64_t position = a.positions == nullptr ? a.first_position + (int64_t)t
                                     : a.narrow_positions   ? (int64_t)((const int32_t *)a.positions)[where]
                                                            : ((const int64_t *)a.positions)[where];
#pragma unroll
            for (int j = 0; j < PAIRS; ++j) {
                const uint32_t pair = unit * PAIRS + j;
                W cosine, sine;
                rotor<W>(position, plan.turns[pair], plan.turns_low[pair], (W)plan.amplitude, cosine, sine);
                if (backward) sine = -sine;
                (j & 1 ? c[j / 2].y : c[j / 2].x) = cosine;
                (j & 1 ? s[j / 2].y : s[j / 2].x) = sine;
            }
        }
        for (size_t h = 0; h < heads; h += kHeads) {
            Vec<T, V> v[kHeads][N];
#pragma unroll
            for (int k = 0; k < kHeads; ++k)
                if (h + k < heads) {
                    v[k][0] = load<T, V>(x + (h + k) * a.xh);
                    if (SPLIT && !copied) v[k][N - 1] = load<T, V>(x + (h + k) * a.xh + second);
                }
#pragma unroll
            for (int k = 0; k < kHeads; ++k)
                if (h + k < heads) {
                    if (!copied) turn<T, V, SPLIT>(v[k][0], v[k][N - 1], c, s);
                    store<T, V>(y + (h + k) * a.yh, v[k][0]);
                    if (SPLIT && !copied) store<T, V>(y + (h + k) * a.yh + second, v[k][N - 1]);
                }
        }
    }
}

// The widest vector, up to 16 bytes, that every head, half and row starts on.
int vector_width(const RotaryArgs &a, const geo_b200_rotary_plan_t &plan, size_t bytes) {
    const bool half = plan.layout == GEO_B200_ROTARY_HALF;
    size_t strides = a.head_dim | plan.rotary_dim;
    if (a.heads > 1) strides |= a.xh | a.yh;
    if (a.tokens > 1) strides |= a.xt | a.yt;
    if (a.batch > 1) strides |= a.xb | a.yb;
    if (half) strides |= plan.rotary_dim / 2;
    const uintptr_t low = (uintptr_t)a.x | (uintptr_t)a.y;
    int v = 16 / (int)bytes;
    while (v > 1 && (strides % v != 0 || low % (v * bytes) != 0)) v /= 2;
    return v;
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
    a.narrow_positions = s.position_type == GEO_B200_I32;
    // A rotor costs about as much as turning four heads: heads are shared out
    // only as far as it takes to give every multiprocessor 1024 threads.
    const int v = vector_width(a, *plan, b);
    const bool half = plan->layout == GEO_B200_ROTARY_HALF;
    const size_t units = plan->rotary_dim / (half || v == 1 ? 2 * v : v) + (s.head_dim - plan->rotary_dim) / v;
    const size_t wanted = (size_t)geo::device_sm_count() * 1024, threads = tokens * units;
    size_t groups = threads < wanted ? (wanted + threads - 1) / threads : 1;
    if (groups > s.heads) groups = s.heads;
    a.share = (s.heads + groups - 1) / groups;
    a.groups = (s.heads + a.share - 1) / a.share;
    const size_t blocks = (threads * a.groups + kThreads - 1) / kThreads;
    const unsigned grid = (unsigned)(blocks < 0x7fffffff ? blocks : 0x7fffffff);
    return status_of(by_type(s.type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto width) {
            constexpr int V = decltype(width)::value;
            if (half)
                rotary_kernel<T, V, true><<<grid, kThreads, 0, stream>>>(a, *plan, backward);
            else
                rotary_kernel<T, V, false><<<grid, kThreads, 0, stream>>>(a, *plan, backward);
        };
        if (v == 1) go(std::integral_constant<int, 1>{});
        if (v == 2) go(std::integral_constant<int, 2>{});
        if constexpr (sizeof(T) <= 4)
            if (v == 4) go(std::integral_constant<int, 4>{});
        if constexpr (sizeof(T) == 2)
            if (v == 8) go(std::integral_constant<int, 8>{});
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
