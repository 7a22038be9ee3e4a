// feed_forward_scale.cu -- by what the VJP of a float16 feed-forward block multiplies
// its inner values (geo/geo_b200.h section 5).
//
// float16 ends at 65504 and has steps of 2^-24 below 2^-14, so that a second term adds
// nothing to a value of less than 2^-13 or so, and values under 2^-25 vanish: the
// cotangents of a mean over many values are of that size. The cotangents of gate and up
// are therefore multiplied by one power of two on their way to the workspace, h by
// another, and the sums that they enter by its inverse, in float32: exact both ways. The
// powers bring what the values can be at most, by their factors' largest,
//   |h_bar u act'| <= max_row(sum |y_bar|) max |down_weight| 1.2 max |u|, and so on,
// to between 2^14 and 2^15. That is some 2^13 of the values' usual size, whose own
// digits then are all there (8192 rows, y_bar of 1e-5: weights' float32 cotangents 2.5e-6
// off, 1.9e-3 without). Infinities and NaN are left out: they make what they enter so.
// Two launches; HBM bounds the first, which reads y_bar, gate, up and down_weight once
// more: 150 MB in 34 us, 14 MB in 9 (what a VJP takes more than bfloat16's, which has no
// need of it: 300 x 1000 x 4000 84 and 73 us, 200000 x 40 x 24 255 and 242, 8192 x 4096
// x 8192 within the boards' spread of a tenth).
#include "feed_forward.h"
#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

constexpr int kThreads = 256, kAhead = 4, V = 8;

// One array's part of the pass. A team (a part of a warp, as many neighbours as a row has
// vectors) looks at `segment` values of a row at a time, or at a vector each of kAhead
// rows where that is all of them; the warps' pieces of all arrays are counted one after
// another.
struct Scan {
    Matrix m;
    size_t rows, cols, parts, pieces_end;
    int lanes, segment;
    bool aligned, brief;  // brief: a row is a vector a lane
};
struct Scans {
    Scan of[4];  // y_bar (whose rows are summed up), down_weight, gate, up
    float4 *found;
};

// The largest size of the team's finite values, or (SUM) the largest sum of a row's, or of a segment's.
template <bool SUM>
__device__ __forceinline__ float look_at(const Scan &s, size_t piece) {
    using T = __half;
    const int lane = threadIdx.x % s.lanes, teams = 32 / s.lanes, team = threadIdx.x % 32 / s.lanes;
    float most = 0.0f, sum = 0.0f;
    auto take = [&](float v) {
        const float size = fabsf(v), finite = size < INFINITY ? size : 0.0f;
        if constexpr (SUM)
            sum += finite;
        else
            most = fmaxf(most, finite);
    };
    auto row_ends = [&] {
        if constexpr (SUM) {
            for (int o = s.lanes / 2; o > 0; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            most = fmaxf(most, sum);
            sum = 0.0f;
        }
    };
    auto take_vector = [&](const Vec<T, V> &v) {
#pragma unroll
        for (int q = 0; q < V / 2; ++q) take(v.pair(q).x), take(v.pair(q).y);
    };
    const T *const base = (const T *)s.m.p;
    if (s.brief) {
        const size_t row = piece * teams * kAhead + team;
        const int at = lane * V, held = (int)s.cols - at;  // values of the lane's vector, or more
        Vec<T, V> v[kAhead];
#pragma unroll
        for (int i = 0; i < kAhead; ++i) {
            const bool live = row + i * teams < s.rows;
            const T *p = base + (row + i * teams) * s.m.stride + at;
            v[i] = Vec<T, V>::zero();
            if (live && held >= V && s.aligned) {
                v[i] = load<T, V>(p);
            } else if (live) {
#pragma unroll
                for (int q = 0; q < V / 2; ++q)
                    v[i].set(q, {2 * q < held ? widen(p[2 * q]) : 0.0f, 2 * q + 1 < held ? widen(p[2 * q + 1]) : 0.0f});
            }
        }
#pragma unroll
        for (int i = 0; i < kAhead; ++i) take_vector(v[i]), row_ends();
        return most;
    }
    const size_t item = piece * teams + team, row = s.parts == 1 ? item : item / s.parts;
    const size_t first = (item - row * s.parts) * s.segment;
    const size_t last = row >= s.rows ? 0 : (first + s.segment < s.cols ? first + s.segment : s.cols);
    const T *p = base + row * s.m.stride;
    if (s.aligned) {
        const size_t gap = (size_t)s.lanes * V;
        for (size_t c = first + lane * V; c < last; c += kAhead * gap) {
            Vec<T, V> v[kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i)
                v[i] = c + i * gap + V <= last ? load<T, V>(p + c + i * gap) : Vec<T, V>::zero();
#pragma unroll
            for (int i = 0; i < kAhead; ++i) take_vector(v[i]);
        }
        // What is less than a vector at the end.
        for (size_t c = last / V * V + lane; c < last; c += s.lanes) take(widen(p[c]));
    } else {
        for (size_t c = first + lane; c < last; c += (size_t)s.lanes * 16) {
            T v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = c + (size_t)i * s.lanes < last ? p[c + (size_t)i * s.lanes] : T(0.0f);
#pragma unroll
            for (int i = 0; i < 16; ++i) take(widen(v[i]));
        }
    }
    row_ends();
    return most;
}

// The largest over the block's threads, on its first warp.
__device__ __forceinline__ void largest_of_block(float (&v)[4]) {
    __shared__ float found[32][4];
    auto of_warp = [&] {
#pragma unroll
        for (int o = 16; o > 0; o /= 2)
#pragma unroll
            for (int n = 0; n < 4; ++n) v[n] = fmaxf(v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
    };
    of_warp();
#pragma unroll
    for (int n = 0; n < 4; ++n)
        if ((threadIdx.x & 31) == 0) found[threadIdx.x / 32][n] = v[n];
    __syncthreads();
    if (threadIdx.x >= 32) return;
#pragma unroll
    for (int n = 0; n < 4; ++n) v[n] = threadIdx.x < blockDim.x / 32 ? found[threadIdx.x][n] : 0.0f;
    of_warp();
}

__global__ void __launch_bounds__(kThreads) largest_kernel(const __grid_constant__ Scans scans) {
    after_previous();
    let_next_start();
    float most[4] = {};
    const size_t warps = (size_t)gridDim.x * (kThreads / 32);
    for (size_t n = (size_t)blockIdx.x * (kThreads / 32) + threadIdx.x / 32; n < scans.of[3].pieces_end; n += warps) {
        size_t begin = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (n >= begin && n < scans.of[i].pieces_end)
                most[i] = fmaxf(most[i], i == 0 ? look_at<true>(scans.of[i], n - begin) : look_at<false>(scans.of[i], n - begin));
            begin = scans.of[i].pieces_end;
        }
    }
    largest_of_block(most);
    // A row's sum is at most the largest part's times the parts.
    if (threadIdx.x == 0)
        scans.found[1 + blockIdx.x] = make_float4(most[0] * (float)scans.of[0].parts, most[1], most[2], most[3]);
}

__global__ void __launch_bounds__(kScaleBlocks) scale_kernel(float4 *found, int activation, int blocks) {
    after_previous();
    let_next_start();
    const float4 mine = (int)threadIdx.x < blocks ? found[1 + threadIdx.x] : make_float4(0, 0, 0, 0);
    float most[4] = {mine.x, mine.y, mine.z, mine.w};
    largest_of_block(most);
    if (threadIdx.x != 0) return;
    const float dy = most[0], wd = most[1], gate = most[2], up = most[3];
    // |act'| <= 1.2; |act(a)| <= |a| but for the sigmoid.
    const float act = activation == GEO_B200_ACTIVATION_SIGMOID ? 1.0f : gate;
    auto power = [](float bound) { return bound > 0.0f ? 14 - ilogbf(bound) : 0; };
    const int inner = power(dy * wd * fmaxf(1.2f * up, act)), h = power(act * up);
    found[0] = make_float4(ldexpf(1.0f, inner), ldexpf(1.0f, -inner), ldexpf(1.0f, h), ldexpf(1.0f, -h));
}

}  // namespace

cudaError_t launch_scale(const InnerScale &s, cudaStream_t stream) {
    Scans scans = {};
    scans.found = s.found;
    const size_t values = s.cols * s.hidden + 2 * s.rows * s.hidden;
    size_t end = 0;
    auto add = [&](int i, const Matrix &m, size_t rows, size_t cols) {
        Scan &a = scans.of[i];
        const bool flat = i > 0 && m.stride == cols;  // packed rows are one long one
        a = {m, flat ? 1 : rows, flat ? rows * cols : cols};
        a.aligned = (uintptr_t)m.p % 16 == 0 && (a.rows == 1 || m.stride % V == 0);
        for (a.lanes = 1; a.lanes < 32 && (size_t)a.lanes * V < a.cols;) a.lanes *= 2;
        // Long pieces where there are enough for every warp.
        a.segment = i == 0 || values > (size_t)1 << 25 ? 4096 : 1024;
        a.parts = (a.cols + a.segment - 1) / a.segment;
        a.brief = a.cols <= (size_t)a.lanes * V;
        const size_t each = 32 / a.lanes * (a.brief ? kAhead : 1);  // items of a piece
        if (m.p != nullptr) end += (a.rows * a.parts + each - 1) / each;
        a.pieces_end = end;
    };
    add(0, s.dy, s.rows, s.cols);
    add(1, s.wd, s.cols, s.hidden);
    add(2, s.gate, s.rows, s.hidden);
    add(3, s.up, s.rows, s.hidden);
    const size_t wanted = (end + kThreads / 32 - 1) / (kThreads / 32);
    const unsigned blocks = (unsigned)(wanted < (size_t)kScaleBlocks ? wanted : kScaleBlocks);
    const cudaError_t e = launch_after(largest_kernel, blocks, kThreads, 0, 1, stream, scans);
    return e != cudaSuccess ? e : launch_after(scale_kernel, 1, kScaleBlocks, 0, 1, stream, s.found, s.activation, (int)blocks);
}

}  // namespace layers
}  // namespace geo
