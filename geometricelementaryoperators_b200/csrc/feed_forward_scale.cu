// feed_forward_scale.cu -- by what the VJP of a float16 feed-forward block multiplies
// its inner values (geo/geo_b200.h section 5).
//
// float16 ends at 65504 and has steps of 2^-24 below 2^-14, so that a second term adds
// nothing to a value of less than 2^-13 or so, and values under 2^-25 vanish: the
// cotangents of a mean over many values are of that size. The cotangents of gate and up
// are therefore multiplied by one power of two on their way to the workspace, h by
// another, and the sums that they enter by its inverse, in float32: exact both ways. The
// powers bring what the values can be at most, by their factors' largest in each row,
//   |h_bar u act'| <= sum |y_bar| max |down_weight| 1.2 max |u|, and so on,
// to between 2^14 and 2^15. That is some 2^13 of the values' usual size, whose own
// digits then are all there (8192 rows, y_bar of 1e-5: weights' float32 cotangents 9.0e-7
// off, 1.9e-3 without). Infinities and NaN are left out: they make what they enter so.
// Two launches; HBM bounds the first, which reads y_bar, gate, up and down_weight once
// more: 150 MB in 33 us, 14 MB in 8 (what a VJP takes more than bfloat16's, which has no
// need of it: 300 x 1000 x 4000 82 and 73 us, 200000 x 40 x 24 264 and 238, 8192 x 4096
// x 8192 within the boards' spread of a tenth). By rows, because one row's y_bar and
// another's projections may be far above all others and never meet: with the largest of
// all rows ordinary rows' values fell below float16's steps.
#include "feed_forward.h"
#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32, kAhead = 4, V = 8;
constexpr int kSegment = 1024;  // of down_weight, a warp's at a time

// `lanes` neighbouring threads of a block look at a row of y_bar, gate and up at a time
// (kThreads: the block), a warp at a segment of a row of down_weight; the blocks' rounds
// over rows and over segments are counted one after another.
struct Scans {
    Matrix dy, gate, up, wd;
    size_t rows, cols, hidden;
    size_t wd_rows, wd_cols, parts;  // down_weight, as one long row where it is packed
    size_t row_rounds, rounds;
    int lanes, activation;
    bool brief;  // rows are a vector a lane, or less
    float4 *found;
};

// Of this thread's part of n adjacent values, finite ones: their largest size, or (SUM)
// the sum of their sizes. AHEAD vectors are on their way at a time.
template <bool SUM, int AHEAD>
__device__ __forceinline__ float look_at(const __half *p, size_t n, int lane, int lanes) {
    using T = __half;
    float sum = 0.0f;
    __half2 most = __float2half2_rn(0.0f);
    auto take = [&](uint32_t two) {
        two &= 0x7FFF7FFFu;
        __half2 size = *reinterpret_cast<__half2 *>(&two);
        two &= __hlt2_mask(size, __half2(__ushort_as_half(0x7C00), __ushort_as_half(0x7C00)));
        size = *reinterpret_cast<__half2 *>(&two);
        if constexpr (SUM) {
            const float2 f = __half22float2(size);
            sum += f.x + f.y;
        } else {
            most = __hmax2(most, size);
        }
    };
    size_t head = (0 - (uintptr_t)p) % 16 / sizeof(T);  // before the first whole vector
    if (head > n) head = n;
    for (size_t e = lane; e < head; e += lanes) take(__half_as_ushort(p[e]));
    const size_t vectors = (n - head) / V;
    for (size_t i = lane; i < vectors; i += (size_t)lanes * AHEAD) {
        Vec<T, V> v[AHEAD];
#pragma unroll
        for (int k = 0; k < AHEAD; ++k) {
            const size_t at = i + (size_t)k * lanes;
            v[k] = at < vectors ? load<T, V>(p + head + at * V) : Vec<T, V>::zero();
        }
#pragma unroll
        for (int k = 0; k < AHEAD; ++k)
#pragma unroll
            for (int w = 0; w < 4; ++w) take(v[k].w[w]);
    }
    for (size_t e = head + vectors * V + lane; e < n; e += lanes) take(__half_as_ushort(p[e]));
    return SUM ? sum : fmaxf(__low2float(most), __high2float(most));
}

// f over neighbouring threads: of a team of up to a warp, or of the block, by way of `memory`.
template <int N, typename F>
__device__ __forceinline__ void over_team(float (&v)[N], int lanes, float (*memory)[N], F &&f) {
    for (int o = (lanes < 32 ? lanes : 32) / 2; o > 0; o /= 2)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = f(n, v[n], __shfl_xor_sync(0xffffffffu, v[n], o));
    if (lanes <= 32) return;
    __syncthreads();
    if (threadIdx.x % 32 == 0)
#pragma unroll
        for (int n = 0; n < N; ++n) memory[threadIdx.x / 32][n] = v[n];
    __syncthreads();
#pragma unroll
    for (int n = 0; n < N; ++n) v[n] = memory[0][n];
    for (int w = 1; w < lanes / 32; ++w)
#pragma unroll
        for (int n = 0; n < N; ++n) v[n] = f(n, v[n], memory[w][n]);
}

__global__ void __launch_bounds__(kThreads) largest_kernel(const __grid_constant__ Scans s) {
    __shared__ float memory[kWarps][3];
    after_previous();
    let_next_start();
    const int lane = threadIdx.x % s.lanes, team = threadIdx.x / s.lanes, teams = kThreads / s.lanes;
    float most[3] = {};  // of the rows' bounds of inner cotangents without down_weight, of h's, and of down_weight
    for (size_t round = blockIdx.x; round < s.rounds; round += gridDim.x) {
        if (round < s.row_rounds) {
            const size_t row = round * teams + team;
            float of_row[3] = {};
            auto look = [&](auto ahead) {
                constexpr int A = decltype(ahead)::value;
                const __half *dy = (const __half *)s.dy.p + row * s.dy.stride;
                const __half *gate = (const __half *)s.gate.p + row * s.gate.stride;
                const __half *up = (const __half *)s.up.p + row * s.up.stride;
                if (s.dy.p != nullptr) of_row[0] = look_at<true, A>(dy, s.cols, lane, s.lanes);
                of_row[1] = look_at<false, A>(gate, s.hidden, lane, s.lanes);
                of_row[2] = look_at<false, A>(up, s.hidden, lane, s.lanes);
            };
            if (row < s.rows) {
                if (s.brief)
                    look(std::integral_constant<int, 1>{});
                else
                    look(std::integral_constant<int, kAhead>{});
            }
            over_team(of_row, s.lanes, memory, [](int n, float a, float b) { return n == 0 ? a + b : fmaxf(a, b); });
            // |act'| <= 1.2; |act(a)| <= |a| but for the sigmoid.
            const float act = s.activation == GEO_B200_ACTIVATION_SIGMOID ? 1.0f : of_row[1];
            most[0] = fmaxf(most[0], of_row[0] * fmaxf(1.2f * of_row[2], act));
            most[1] = fmaxf(most[1], act * of_row[2]);
        } else {
            const size_t piece = (round - s.row_rounds) * kWarps + threadIdx.x / 32, row = piece / s.parts;
            const size_t first = (piece - row * s.parts) * kSegment, left = s.wd_cols - first;
            if (row < s.wd_rows)
                most[2] = fmaxf(most[2], look_at<false, kAhead>((const __half *)s.wd.p + row * s.wd.stride + first,
                                                        left < (size_t)kSegment ? left : kSegment, threadIdx.x % 32, 32));
        }
    }
    over_team(most, kThreads, memory, [](int, float a, float b) { return fmaxf(a, b); });
    if (threadIdx.x == 0) s.found[1 + blockIdx.x] = make_float4(most[0], most[1], most[2], 0);
}

__global__ void __launch_bounds__(kScaleBlocks) scale_kernel(float4 *found, int blocks) {
    __shared__ float memory[kScaleBlocks / 32][3];
    after_previous();
    let_next_start();
    const float4 mine = (int)threadIdx.x < blocks ? found[1 + threadIdx.x] : make_float4(0, 0, 0, 0);
    float most[3] = {mine.x, mine.y, mine.z};
    over_team(most, kScaleBlocks, memory, [](int, float a, float b) { return fmaxf(a, b); });
    if (threadIdx.x != 0) return;
    auto power = [](float bound) { return bound > 0.0f ? 14 - ilogbf(bound) : 0; };
    const int inner = power(most[0] * most[2]), h = power(most[1]);
    found[0] = make_float4(ldexpf(1.0f, inner), ldexpf(1.0f, -inner), ldexpf(1.0f, h), ldexpf(1.0f, -h));
}

}  // namespace

cudaError_t launch_scale(const InnerScale &i, cudaStream_t stream) {
    Scans s = {i.dy, i.gate, i.up, i.wd, i.rows, i.cols, i.hidden};
    s.activation = i.activation;
    s.found = i.found;
    // A vector each of a row, up to a warp a row; the block where there are no more rows than warps run at one time.
    const size_t widest = i.cols > i.hidden ? i.cols : i.hidden, warps = (size_t)geo::device_sm_count() * 32;
    for (s.lanes = 1; s.lanes < 32 && (size_t)s.lanes * V < widest;) s.lanes *= 2;
    if (widest > 2 * kSegment && i.rows * 2 <= warps) s.lanes = kThreads;
    s.brief = widest <= (size_t)s.lanes * V;
    const size_t teams = kThreads / s.lanes;
    s.row_rounds = (i.rows + teams - 1) / teams;
    const bool flat = i.wd.stride == i.hidden;
    s.wd_rows = flat ? 1 : i.cols;
    s.wd_cols = flat ? i.cols * i.hidden : i.hidden;
    s.parts = (s.wd_cols + kSegment - 1) / kSegment;
    s.rounds = s.row_rounds + (i.wd.p != nullptr ? (s.wd_rows * s.parts + kWarps - 1) / kWarps : 0);
    const unsigned blocks = (unsigned)(s.rounds < (size_t)kScaleBlocks ? s.rounds : kScaleBlocks);
    const cudaError_t e = launch_after(largest_kernel, blocks, kThreads, 0, 1, stream, s);
    return e != cudaSuccess ? e : launch_after(scale_kernel, 1, kScaleBlocks, 0, 1, stream, s.found, (int)blocks);
}

}  // namespace layers
}  // namespace geo
