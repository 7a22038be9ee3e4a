// rotary.cu -- rotary positions and their VJP (geo/geo_b200.h section 5).
//
// Pair i of a head at position p is turned by t = p f_i. The angle is taken in
// quarter turns, p (hi + lo), in float64: adding 1.5 2^52 to p hi in a fused
// multiply-add rounds it to whole quarters, whose last two bits are the quadrant,
// and a second one leaves p hi - quarters with a single rounding. What is left is
// at most half a quarter turn and p lo, so its conversion to float32 costs 2^-26
// quarters and far positions lose nothing. Its sine and cosine are polynomials
// (interpolated at Chebyshev nodes, within 2^-28 up to half a quarter), two pairs at a
// time in packed float32 arithmetic. At positions of 2^31, p lo is at most 2^-21
// quarters for a pair of one turn a position; for one of 2^18, the most that a plan
// takes, it is 1/8 and the polynomials are within 2^-21, where the frequency's own
// last place is worth 2^-13.
// HBM bounds it where a token has heads enough: a rotor is worked out once for the
// heads that a thread turns, all of a token's where that leaves every multiprocessor
// 2048 threads, else a group of them (5777 tokens of nine: three groups, each rotor
// three times). Measured, calls in turn over three sets of arrays, host included: 16384
// tokens of 40 heads of 128 bfloat16 values 58 to 59 us (5.7 TB/s, 87% of the copy
// bandwidth); eight tokens of a decoding step 2.9 us on the device.
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
    size_t share;  // heads of a block: its row of the grid says which
    int narrow_positions;
};

// What is left of p (hi + lo) quarter turns after `quadrant` whole ones.
__device__ __forceinline__ double split_quarters(double p, double2 quarters, uint32_t &quadrant) {
    const double magic = 6755399441055744.0;  // 1.5 2^52: the sum's last bit is worth 1
    const double rounded = ::fma(p, quarters.x, magic);
    quadrant = (uint32_t)__double2loint(rounded);
    return ::fma(p, quarters.y, ::fma(p, quarters.x, -(rounded - magic)));
}

// Sine and cosine of x quarter turns, |x| <= 1/2.
__device__ __forceinline__ void sine_cosine(Pair<float> x, Pair<float> &sine, Pair<float> &cosine) {
    const Pair<float> u = x * x;
    Pair<float> p = fma(both(-0.00460214913748f), u, both(0.0796802176242f));
    p = fma(p, u, both(-0.645963477663f));
    p = fma(p, u, both(1.57079632195f));
    sine = x * p;
    Pair<float> c = fma(both(0.00090673988654f), u, both(-0.0208615283385f));
    c = fma(c, u, both(0.253669410357f));
    c = fma(c, u, both(-1.23370054937f));
    cosine = fma(c, u, both(1.0f));
}
__device__ __forceinline__ void sine_cosine(Pair<double> x, Pair<double> &sine, Pair<double> &cosine) {
    sincospi(0.5 * x.x, &sine.x, &cosine.x);
    sincospi(0.5 * x.y, &sine.y, &cosine.y);
}

__device__ __forceinline__ float signed_by(float v, uint32_t bit1) {
    return __uint_as_float(__float_as_uint(v) ^ (bit1 & 2u) << 30);
}
__device__ __forceinline__ double signed_by(double v, uint32_t bit1) { return bit1 & 2u ? -v : v; }

// amplitude times cosine and sine of p times two pairs' quarter turns per position.
template <typename W>
__device__ __forceinline__ void rotors(double p, double2 a, double2 b, W amplitude, Pair<W> &c, Pair<W> &s) {
    uint32_t qa, qb;
    const double xa = split_quarters(p, a, qa), xb = split_quarters(p, b, qb);
    Pair<W> sine, cosine;
    sine_cosine(Pair<W>{(W)xa, (W)xb}, sine, cosine);
    c = {signed_by(qa & 1 ? sine.x : cosine.x, qa + 1), signed_by(qb & 1 ? sine.y : cosine.y, qb + 1)};
    s = {signed_by(qa & 1 ? cosine.x : sine.x, qa), signed_by(qb & 1 ? cosine.y : sine.y, qb)};
    c = c * both(amplitude);
    s = s * both(amplitude);
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
// out once, and turns them in `share` heads; the coordinates past rotary_dim go
// the same way as vectors that are only copied. Heads come through slots of the
// thread's own in shared memory, kAhead asynchronous copies ahead, so that few
// registers keep the bytes in flight that HBM wants; the first ones are on their
// way while the rotors are worked out. Where nothing wider than a value is
// aligned, a pair is two values; vectors below 16 bytes are loaded directly.
constexpr int kAhead = 5;
template <typename T, int V, bool HALF>
constexpr int kSlots = V * sizeof(T) == 16 ? (kAhead + 1) * (HALF ? 2 : 1) : 0;  // vectors a thread
template <typename T, int V, bool HALF>
__global__ void __launch_bounds__(kThreads, 4)
    rotary_kernel(const RotaryArgs a, const __grid_constant__ geo_b200_rotary_plan_t plan, int backward) {
    using W = Wide<T>;
    constexpr bool SPLIT = HALF || V == 1;     // a pair's coordinates are in two vectors
    constexpr int N = SPLIT ? 2 : 1;           // vectors a head
    constexpr int PAIRS = SPLIT ? V : V / 2;   // pairs a thread
    constexpr bool RING = kSlots<T, V, HALF> > 0;
    const uint32_t half = plan.rotary_dim / 2, second = HALF ? half : 1;
    const uint32_t turned = plan.rotary_dim / (N * V);
    const uint32_t units = turned + ((uint32_t)a.head_dim - plan.rotary_dim) / V;
    const size_t count = a.tokens * units;
    const size_t from = blockIdx.y * a.share, left = a.heads - from;
    const uint32_t heads = (uint32_t)(left < a.share ? left : a.share);
    extern __shared__ __align__(128) unsigned char memory[];
    __shared__ double2 quarters[GEO_B200_ROTARY_MAX_DIM / 2];
    // Out of the parameters, where lanes that read different pairs wait for one another.
    for (uint32_t i = threadIdx.x; i < half; i += kThreads)
        quarters[i] = make_double2(4.0 * plan.turns[i], 4.0 * plan.turns_low[i]);
    __syncthreads();
    for (size_t id = blockIdx.x * (size_t)kThreads + threadIdx.x; id < a.batch * count;
         id += (size_t)gridDim.x * kThreads) {
        size_t b = 0, in_batch = id;
        if (a.batch > 1) {
            b = a.batch * count <= 0xFFFFFFFFu ? (uint32_t)id / (uint32_t)count : id / count;
            in_batch = id - b * count;
        }
        const size_t t = count <= 0xFFFFFFFFu ? (uint32_t)in_batch / units : in_batch / units;
        const uint32_t unit = (uint32_t)(in_batch - t * units);
        const bool copied = unit >= turned;
        if (copied && a.x == a.y) continue;
        const size_t at = copied ? plan.rotary_dim + (size_t)(unit - turned) * V : (size_t)unit * (HALF ? V : N * V);
        const T *x = (const T *)a.x + b * a.xb + t * a.xt + from * a.xh + at;
        T *y = (T *)a.y + b * a.yb + t * a.yt + from * a.yh + at;
        const uint32_t both_vectors = SPLIT && !copied;

        const unsigned char *slot = memory + threadIdx.x * 16;
        uint32_t write = 0, read = 0, fetched = 0;
        auto fetch = [&] {
            if (fetched < heads) {
                const uint32_t to = shared_address(slot) + write * (N * kThreads * 16);
                copy_async(to, x);
                if (both_vectors) copy_async(to + kThreads * 16, x + second);
                x += a.xh;
                ++fetched;
                write = write == kAhead ? 0 : write + 1;
            }
            commit_async();
        };
        if constexpr (RING)
            for (int k = 0; k < kAhead; ++k) fetch();

        Pair<W> c[(PAIRS + 1) / 2], s[(PAIRS + 1) / 2];
        if (!copied) {
            const size_t where = b * a.pb + t;
            const int64_t position = a.positions == nullptr ? a.first_position + (int64_t)t
                                     : a.narrow_positions   ? (int64_t)((const int32_t *)a.positions)[where]
                                                            : ((const int64_t *)a.positions)[where];
            const W amplitude = (W)plan.amplitude;
#pragma unroll
            for (int j = 0; j < PAIRS; j += 2) {
                const uint32_t pair = unit * PAIRS + j;
                rotors<W>((double)position, quarters[pair], quarters[PAIRS > 1 ? pair + 1 : pair], amplitude, c[j / 2],
                          s[j / 2]);
                if (backward) s[j / 2] = s[j / 2] * both(W(-1));
            }
        }
        for (uint32_t h = 0; h < heads; ++h) {
            Vec<T, V> v[N];
            if constexpr (RING) {
                fetch();
                wait_async<kAhead>();
                const unsigned char *got = slot + read * (N * kThreads * 16);
                v[0] = load<T, V>((const T *)got);
                if (both_vectors) v[N - 1] = load<T, V>((const T *)(got + kThreads * 16));
                read = read == kAhead ? 0 : read + 1;
            } else {
                v[0] = load<T, V>(x);
                if (both_vectors) v[N - 1] = load<T, V>(x + second);
                x += a.xh;
            }
            if (!copied) turn<T, V, SPLIT>(v[0], v[N - 1], c, s);
            store<T, V>(y, v[0]);
            if (both_vectors) store<T, V>(y + second, v[N - 1]);
            y += a.yh;
        }
        if constexpr (RING) wait_async<0>();
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
    // Heads are shared out, and rotors worked out more than once, as far as it takes to give every multiprocessor
    // 2048 threads (8192 tokens of 32 heads of 64 float16 values: 13.0 us, 13.9 with 1024).
    const int v = vector_width(a, *plan, b);
    const bool half = plan->layout == GEO_B200_ROTARY_HALF;
    const size_t units = plan->rotary_dim / (half || v == 1 ? 2 * v : v) + (s.head_dim - plan->rotary_dim) / v;
    const size_t wanted = (size_t)geo::device_sm_count() * 2048, threads = tokens * units;
    size_t groups = threads < wanted ? (wanted + threads - 1) / threads : 1;
    if (groups > s.heads) groups = s.heads;
    if (groups > 65535) groups = 65535;
    a.share = (s.heads + groups - 1) / groups;
    if (a.share > 0xFFFFFFFFu) return GEO_B200_INVALID_ARGUMENT;
    const size_t blocks = (threads + kThreads - 1) / kThreads;
    const dim3 grid((unsigned)(blocks < 0x7fffffff ? blocks : 0x7fffffff), (unsigned)((s.heads + a.share - 1) / a.share));
    return status_of(by_type(s.type, [&](auto t) {
        using T = decltype(t);
        auto go = [&](auto width) {
            constexpr int V = decltype(width)::value;
            const size_t ring = (size_t)(half ? kSlots<T, V, true> : kSlots<T, V, false>) * kThreads * 16;
            auto kernel = half ? rotary_kernel<T, V, true> : rotary_kernel<T, V, false>;
            if (ring > 40 * 1024) {
                const cudaError_t e =
                    cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)ring);
                if (e != cudaSuccess) return e;
            }
            kernel<<<grid, kThreads, ring, stream>>>(a, *plan, backward);
            return cudaGetLastError();
        };
        if constexpr (sizeof(T) == 2)
            if (v == 8) return go(std::integral_constant<int, 8>{});
        if constexpr (sizeof(T) <= 4)
            if (v == 4) return go(std::integral_constant<int, 4>{});
        return v == 2 ? go(std::integral_constant<int, 2>{}) : go(std::integral_constant<int, 1>{});
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
