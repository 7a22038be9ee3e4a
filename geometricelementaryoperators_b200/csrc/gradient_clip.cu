// gradient_clip.cu -- the norm over all gradients of a model, and clipping
// (geo/geo_b200.h section 6).
//
// norm = sqrt(sum g^2), clipped = min(1, max_norm / norm) g. Two passes over the
// gradients, nothing to compute: HBM bounds it, 2 bytes read and 1 written for each
// byte of gradients, less what the second pass still finds in L2: it goes backwards.
// A gradient is cut into pieces of 16 KB, whatever its type; the list travels in the
// kernel's parameters (nothing to copy or keep, graphs capture it), a block finds a
// piece's gradient by bisection. Sums are float64, in which no smaller type's square
// overflows or vanishes; float64's own are summed in three, of squares in the middle of
// its range and of those that would leave it, scaled (J. L. Blue, ACM TOMS 4, 1978).
// Each block leaves its partial sums; the second pass's blocks add them up in the same
// order each.
// 0.8 GB of bfloat16 gradients: 410 to 415 us. Cold, under the profiler, the first pass
// takes 125 of them (98% of the copy bandwidth) and the second 266 (92%); in calls one
// after another the first takes some 20 more, while what the call before left written in
// L2 goes out. 192 arrays of 64 float64 values 14 us, 6 of them on the device.
#include <cuda.h>
#include <cudaTypedefs.h>

#include "layers.h"

#include <algorithm>
#include <cmath>
#include <vector>

#include "geo_runtime.h"

namespace geo {
namespace layers {

namespace {

constexpr int kThreads = 256, kBlocks = 8;  // a multiprocessor
constexpr uint32_t kPieceBytes = 16384;

struct Entry {
    const void *gradient;
    void *clipped;
    size_t count;
    uint32_t first;  // piece
    uint32_t type;
};
// Entries of one launch, the fewest that hold the list: parameters take their time to
// be handed over (1 microsecond for each 10 KB of them), which short calls notice.
constexpr int kSmall = 62, kMiddle = 250, kLarge = 1000;
template <int CAPACITY>
struct Table {
    int count;
    uint32_t pieces;
    Entry entries[CAPACITY];
};

// Sums of squares: of values in the middle of float64's range, of those above 2^480 times
// 2^-600, and of those below 2^-480 times 2^600: 2^56 of any of them stay in it.
struct Squares {
    double middle, high, low;
};
__device__ __forceinline__ bool in_the_middle(double v) {
    const double size = fabs(v);
    return (size >= 0x1p-480 || size == 0.0) && size <= 0x1p480;
}
__device__ __forceinline__ void add_square(Squares &s, double v) {
    if (fabs(v) > 0x1p480)
        s.high = ::fma(v * 0x1p-600, v * 0x1p-600, s.high);
    else if (fabs(v) < 0x1p-480)
        s.low = ::fma(v * 0x1p600, v * 0x1p600, s.low);
    else
        s.middle = ::fma(v, v, s.middle);  // NaN too
}

// Squares of V adjacent values: exact but for the sums' own roundings (a float32's square has 48 bits).
template <typename T, int V>
__device__ __forceinline__ double squares(const Vec<T, V> &v) {
    double even = 0, odd = 0;
#pragma unroll
    for (int q = 0; q < V / 2; ++q) {
        const double a = v.pair(q).x, b = v.pair(q).y;
        even = ::fma(a, a, even);
        odd = ::fma(b, b, odd);
    }
    return even + odd;
}

// f(first value, last) of a piece of a gradient, in values.
template <typename T>
__device__ __forceinline__ void piece_range(const Entry &e, uint32_t piece, size_t &first, size_t &last) {
    constexpr size_t kValues = kPieceBytes / sizeof(T);
    first = (size_t)(piece - e.first) * kValues;
    last = first + kValues < e.count ? first + kValues : e.count;
}

template <typename T>
__device__ void add_squares(Squares &s, const Entry &e, uint32_t piece) {
    constexpr int V = 16 / (int)sizeof(T), kEach = kPieceBytes / 16 / kThreads;
    size_t first, last;
    piece_range<T>(e, piece, first, last);
    const T *g = (const T *)e.gradient;
    if ((uintptr_t)g % 16 == 0 && last - first == kPieceBytes / sizeof(T)) {
        Vec<T, V> v[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = load<T, V>(g + first + (size_t)(i * kThreads + threadIdx.x) * V);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            if constexpr (sizeof(T) == 8) {
                const double x = v[i].pair(0).x, y = v[i].pair(0).y;
                if (in_the_middle(x) && in_the_middle(y))
                    s.middle += squares<T, V>(v[i]);
                else
                    add_square(s, x), add_square(s, y);
            } else {
                s.middle += squares<T, V>(v[i]);
            }
        }
    } else {
        for (size_t i = first + threadIdx.x; i < last; i += kThreads) {
            const double v = (double)widen(g[i]);
            if constexpr (sizeof(T) == 8)
                add_square(s, v);
            else
                s.middle = ::fma(v, v, s.middle);
        }
    }
}

template <typename T>
__device__ void piece_clip(const Entry &e, uint32_t piece, double scale) {
    using W = Wide<T>;
    constexpr int V = 16 / (int)sizeof(T), kEach = kPieceBytes / 16 / kThreads;
    if (e.clipped == nullptr || (scale == 1.0 && e.clipped == e.gradient)) return;
    size_t first, last;
    piece_range<T>(e, piece, first, last);
    const T *g = (const T *)e.gradient;
    T *out = (T *)e.clipped;
    if (scale < 0x1p-126 && sizeof(W) == 4) {
        // In float32 a scale as small has lost digits, or all of them; the product need not be small.
        for (size_t i = first + threadIdx.x; i < last; i += kThreads)
            out[i] = narrow<T>((W)((double)widen(g[i]) * scale));
        return;
    }
    const W by = (W)scale;
    if (((uintptr_t)g | (uintptr_t)out) % 16 == 0 && last - first == kPieceBytes / sizeof(T)) {
        Vec<T, V> v[kEach];
#pragma unroll
        for (int i = 0; i < kEach; ++i) v[i] = load<T, V>(g + first + (size_t)(i * kThreads + threadIdx.x) * V);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
#pragma unroll
            for (int q = 0; q < V / 2; ++q) v[i].set(q, v[i].pair(q) * both(by));
            store<T, V>(out + first + (size_t)(i * kThreads + threadIdx.x) * V, v[i]);
        }
    } else {
        for (size_t i = first + threadIdx.x; i < last; i += kThreads) out[i] = narrow<T>(widen(g[i]) * by);
    }
}

template <int CAPACITY>
__device__ __forceinline__ const Entry &entry_of(const Table<CAPACITY> &table, uint32_t piece) {
    int low = 0, high = table.count - 1;  // the last entry whose first piece is not beyond
    while (low < high) {
        const int middle = (low + high + 1) / 2;
        if (table.entries[middle].first <= piece)
            low = middle;
        else
            high = middle - 1;
    }
    return table.entries[low];
}

// Sum over the block's threads, the same on every thread, in a fixed order.
__device__ __forceinline__ double sum_of_block(double v) {
    __shared__ double sums[kThreads / 32];
    __syncthreads();
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = v;
    __syncthreads();
    double sum = 0;
#pragma unroll
    for (int i = 0; i < kThreads / 32; ++i) sum += sums[i];
    return sum;
}

__device__ __forceinline__ Squares sum_of_block(Squares s) {
    const bool outside = __syncthreads_or(s.high != 0.0 || s.low != 0.0);
    s.middle = sum_of_block(s.middle);
    if (outside) s.high = sum_of_block(s.high), s.low = sum_of_block(s.low);
    return s;
}

template <int CAPACITY>
__global__ void __launch_bounds__(kThreads, kBlocks)
    squares_kernel(const __grid_constant__ Table<CAPACITY> table, Squares *partial) {
    Squares sum = {};
    for (uint32_t piece = blockIdx.x; piece < table.pieces; piece += gridDim.x) {
        const Entry &e = entry_of(table, piece);
        switch (e.type) {
            case GEO_B200_F64: add_squares<double>(sum, e, piece); break;
            case GEO_B200_F32: add_squares<float>(sum, e, piece); break;
            case GEO_B200_BF16: add_squares<__nv_bfloat16>(sum, e, piece); break;
            default: add_squares<__half>(sum, e, piece); break;
        }
    }
    sum = sum_of_block(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

struct Found {
    double norm, scale;
};
// Squares that are added with others 2^1200 as large count where they are not lost among
// those; a NaN is in the middle.
__device__ __forceinline__ Found found_of(const Squares *partial, int count, double max_norm) {
    Squares s = {};
    for (int i = threadIdx.x; i < count; i += kThreads) {
        s.middle += partial[i].middle;
        s.high += partial[i].high;
        s.low += partial[i].low;
    }
    s = sum_of_block(s);
    Found f;
    if (s.high != 0.0)
        f.norm = sqrt(s.high + s.middle * 0x1p-600 * 0x1p-600) * 0x1p600;
    else if (s.middle != 0.0)
        f.norm = sqrt(s.middle + s.low * 0x1p-600 * 0x1p-600);
    else
        f.norm = sqrt(s.low) * 0x1p-600;
    const double ratio = max_norm / f.norm;
    f.scale = !isfinite(f.norm) ? (double)NAN : (ratio < 1.0 ? ratio : 1.0);  // 0 / norm and norm 0 included
    return f;
}

// For lists of more than one launch: the partial sums of all of them.
__global__ void __launch_bounds__(kThreads)
    join_kernel(const Squares *partial, int count, double max_norm, Found *found, double *norm, double *scale) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Found f = found_of(partial, count, max_norm);
    if (threadIdx.x != 0) return;
    if (found != nullptr) *found = f;
    if (norm != nullptr) *norm = f.norm;
    if (scale != nullptr) *scale = f.scale;
}

// found: null, or what join_kernel left.
template <int CAPACITY>
__global__ void __launch_bounds__(kThreads, kBlocks)
    clip_kernel(const __grid_constant__ Table<CAPACITY> table, const Squares *partial, int count, double max_norm,
                const Found *found, double *norm, double *scale) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const Found f = found != nullptr ? *found : found_of(partial, count, max_norm);
    if (found == nullptr && blockIdx.x == 0 && threadIdx.x == 0) {
        if (norm != nullptr) *norm = f.norm;
        if (scale != nullptr) *scale = f.scale;
    }
    for (uint32_t n = blockIdx.x; n < table.pieces; n += gridDim.x) {
        const uint32_t piece = table.pieces - 1 - n;
        const Entry &e = entry_of(table, piece);
        switch (e.type) {
            case GEO_B200_F64: piece_clip<double>(e, piece, f.scale); break;
            case GEO_B200_F32: piece_clip<float>(e, piece, f.scale); break;
            case GEO_B200_BF16: piece_clip<__nv_bfloat16>(e, piece, f.scale); break;
            default: piece_clip<__half>(e, piece, f.scale); break;
        }
    }
}

// A kernel whose start-up overlaps the end of the one before.
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), unsigned grid, cudaStream_t stream, const A &...args) {
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(grid);
    config.blockDim = dim3(kThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute = {};
    attribute.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

unsigned blocks_of(uint32_t pieces) {
    const unsigned most = (unsigned)geo::device_sm_count() * kBlocks;
    return pieces < most ? pieces : most;
}

uint32_t pieces_of(const geo_b200_gradient_t &g) {
    const size_t bytes = g.count * type_bytes(g.type);
    return (uint32_t)((bytes + kPieceBytes - 1) / kPieceBytes);
}

// Parts of the list, one a launch: indices of its first entries, and of the end.
struct Part {
    size_t first, last;
    uint32_t pieces;
};
// False when a type, a count or the whole is out of range.
bool parts_of(const geo_b200_gradient_t *g, size_t count, std::vector<Part> &parts) {
    if (g == nullptr || count == 0 || count > GEO_B200_GRADIENT_MAX_TENSORS) return false;
    const size_t each = count <= (size_t)kLarge ? count : kLarge;
    for (size_t first = 0; first < count; first += each) {
        Part p = {first, first + each < count ? first + each : count, 0};
        size_t pieces = 0;
        for (size_t i = p.first; i < p.last; ++i) {
            if (type_bytes(g[i].type) == 0 || g[i].reserved != 0 || g[i].count > ((size_t)1 << 40)) return false;
            pieces += pieces_of(g[i]);
        }
        if (pieces > ((size_t)1 << 31)) return false;
        p.pieces = (uint32_t)pieces;
        parts.push_back(p);
    }
    return true;
}

size_t workspace_of(const std::vector<Part> &parts) {
    size_t blocks = 0;
    for (const Part &p : parts) blocks += blocks_of(p.pieces);
    return sizeof(Found) + (blocks + 1) / 2 * 2 * sizeof(Squares);
}

// The arrays of a call are usable (arrays_usable). A model's gradients are parts of few
// allocations: what lies in the one that was looked at last needs alignment alone, where
// looking at each costs half a microsecond on the host.
class UsableArrays {
public:
    bool operator()(const void *p, size_t value_bytes, size_t bytes) {
        if (p == nullptr) return true;
        const uintptr_t at = (uintptr_t)p;
        if (at % value_bytes != 0) return false;
        for (const Range &r : known_)
            if (at >= r.first && at < r.last && bytes <= r.last - at) return true;
        if (!arrays_usable({{p, value_bytes}})) return false;
        static const auto range_of = []() -> PFN_cuMemGetAddressRange_v3020 {
            void *f = nullptr;
            cudaDriverEntryPointQueryResult q;
            if (cudaGetDriverEntryPoint("cuMemGetAddressRange", &f, cudaEnableDefault, &q) != cudaSuccess ||
                q != cudaDriverEntryPointSuccess) {
                (void)cudaGetLastError();
                return nullptr;
            }
            return reinterpret_cast<PFN_cuMemGetAddressRange_v3020>(f);
        }();
        CUdeviceptr base = 0;
        size_t size = 0;
        if (range_of != nullptr && range_of(&base, &size, (CUdeviceptr)at) == CUDA_SUCCESS) {
            known_[next_] = {(uintptr_t)base, (uintptr_t)base + size};
            next_ = (next_ + 1) % 4;
        }
        return true;
    }

private:
    struct Range {
        uintptr_t first, last;
    };
    Range known_[4] = {};
    int next_ = 0;
};

// What is written overlaps nothing else of the call. Lists mostly lie in order, those
// read and those written each.
bool apart(const geo_b200_gradient_t *g, size_t count) {
    struct Range {
        uintptr_t first, last;
    };
    auto before = [](const Range &a, const Range &b) { return a.first < b.first; };
    std::vector<Range> read, written;
    read.reserve(count);
    written.reserve(count);
    for (size_t i = 0; i < count; ++i) {
        if (g[i].count == 0) continue;
        const size_t bytes = g[i].count * type_bytes(g[i].type);
        const uintptr_t in = (uintptr_t)g[i].gradient, out = (uintptr_t)g[i].clipped;
        if (out != 0) written.push_back({out, out + bytes});
        if (out != in) read.push_back({in, in + bytes});
    }
    for (std::vector<Range> *ranges : {&read, &written})
        if (!std::is_sorted(ranges->begin(), ranges->end(), before)) std::sort(ranges->begin(), ranges->end(), before);
    uintptr_t read_end = 0, written_end = 0;  // of what starts before
    auto r = read.begin();
    for (const Range &w : written) {
        for (; r != read.end() && r->first < w.first; ++r) {
            if (r->first < written_end) return false;
            read_end = std::max(read_end, r->last);
        }
        if (w.first < written_end || w.first < read_end) return false;
        written_end = std::max(written_end, w.last);
    }
    return r == read.end() || r->first >= written_end;
}

template <int CAPACITY>
void fill(Table<CAPACITY> &table, const geo_b200_gradient_t *g, const Part &part) {
    table.count = 0;
    table.pieces = 0;
    for (size_t i = part.first; i < part.last; ++i) {
        if (g[i].count == 0) continue;
        table.entries[table.count++] = {g[i].gradient, g[i].clipped, g[i].count, table.pieces, g[i].type};
        table.pieces += pieces_of(g[i]);
    }
}

template <int CAPACITY>
cudaError_t launch(const geo_b200_gradient_t *g, const std::vector<Part> &parts, double max_norm, double *norm,
                   double *scale, void *workspace, bool writes, cudaStream_t stream) {
    Found *found = (Found *)workspace;
    Squares *partial = (Squares *)(found + 1);
    Table<CAPACITY> table;
    int sums = 0;
    cudaError_t e = cudaSuccess;
    for (const Part &part : parts) {
        fill(table, g, part);
        const unsigned blocks = blocks_of(table.pieces);
        if (blocks == 0) continue;
        squares_kernel<CAPACITY><<<blocks, kThreads, 0, stream>>>(table, partial + sums);
        e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        sums += (int)blocks;
    }
    const bool join = !writes || parts.size() > 1 || sums == 0;
    if (join) {
        e = launch_after(join_kernel, 1, stream, partial, sums, max_norm, found, norm, scale);
        if (e != cudaSuccess) return e;
    }
    if (!writes) return e;
    for (size_t n = parts.size(); n > 0; --n) {
        if (parts.size() > 1) fill(table, g, parts[n - 1]);
        const unsigned blocks = blocks_of(table.pieces);
        if (blocks == 0) continue;
        // Only the kernel right behind the sums may start before they are there.
        e = launch_after(clip_kernel<CAPACITY>, blocks, stream, table, partial, sums, max_norm,
                         join ? found : (const Found *)nullptr, norm, scale);
        if (e != cudaSuccess) return e;
    }
    return e;
}

}  // namespace

}  // namespace layers
}  // namespace geo

using namespace geo::layers;

extern "C" size_t geo_b200_gradient_clip_workspace(const geo_b200_gradient_t *gradients, size_t count) {
    try {
        std::vector<Part> parts;
        return parts_of(gradients, count, parts) ? workspace_of(parts) : 0;
    } catch (...) {
        return 0;
    }
}

extern "C" geo_b200_status_t geo_b200_gradient_clip(const geo_b200_gradient_t *gradients, size_t count,
                                                    double max_norm, double *device_norm, double *device_scale,
                                                    void *device_workspace, size_t workspace_bytes,
                                                    cudaStream_t stream) try {
    geo::NvtxRange range("geo_b200.gradient_clip");
    std::vector<Part> parts;
    if (!(max_norm > 0.0) || !parts_of(gradients, count, parts) || device_workspace == nullptr ||
        workspace_bytes < workspace_of(parts))
        return GEO_B200_INVALID_ARGUMENT;
    bool writes = false;
    UsableArrays usable;
    for (size_t i = 0; i < count; ++i) {
        const geo_b200_gradient_t &g = gradients[i];
        if (g.count == 0) continue;
        const size_t b = type_bytes(g.type);
        if (g.gradient == nullptr || !usable(g.gradient, b, g.count * b) || !usable(g.clipped, b, g.count * b))
            return GEO_B200_INVALID_ARGUMENT;
        writes = writes || g.clipped != nullptr;
    }
    if (!apart(gradients, count) ||
        !arrays_usable({{device_norm, 8}, {device_scale, 8}, {device_workspace, 16}}))
        return GEO_B200_INVALID_ARGUMENT;
    auto run = [&](auto capacity) {
        return status_of(launch<decltype(capacity)::value>(gradients, parts, max_norm, device_norm, device_scale,
                                                           device_workspace, writes, stream));
    };
    if (count <= (size_t)kSmall) return run(std::integral_constant<int, kSmall>{});
    if (count <= (size_t)kMiddle) return run(std::integral_constant<int, kMiddle>{});
    return run(std::integral_constant<int, kLarge>{});
} catch (...) {
    return GEO_B200_RUNTIME_FAILURE;
}
