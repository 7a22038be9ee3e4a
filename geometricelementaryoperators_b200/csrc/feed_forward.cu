// feed_forward.cu -- the gated feed-forward block (geo/geo_b200.h section 5): entry
// points, which kernels a call takes, and its workspace.
//
// Forward, two products: gate and up with the activation and their product (h), then
// h down_weight^T. VJP, three: y_bar down_weight with the activation's derivative
// behind it, x_bar, and the weights' cotangents (one launch: with down_weight's turned,
// all three are [hidden][cols] sums over the rows).
// h and the cotangents of gate and up pass between them in the workspace, rounded to
// the arrays' type (the tensor cores' operands): a product of 16-bit values sums
// thousands of them in float32, so their roundings average out against the result's
// own. A float32 result has no rounding to hide them (2.3e-3 of its size off, where its
// sums are 2e-6): on their way to one, what was lost is kept as a second array of the
// type and multiplied as well. float16's inner values of the VJP are multiplied by powers
// of two while they are there (feed_forward_scale.cu).
#include "feed_forward.h"

#include <algorithm>

#include "geo_runtime.h"

namespace {

using namespace geo::layers;

constexpr size_t kAlign = 256;

// The config with its strides resolved; false for what the call would refuse.
bool resolve(const geo_b200_feed_forward_config_t *config, bool vjp, geo_b200_feed_forward_config_t *out) {
    if (config == nullptr || type_bytes(config->type) == 0 || config->reserved != 0) return false;
    geo_b200_feed_forward_config_t c = *config;
    if (c.gradient_type != c.type && !(type_bytes(c.type) == 2 && c.gradient_type == GEO_B200_F32)) return false;
    if (c.activation < GEO_B200_ACTIVATION_SILU || c.activation > GEO_B200_ACTIVATION_RELU) return false;
    if (c.rows == 0 || c.cols == 0 || c.hidden == 0 || c.rows > GEO_B200_FEED_FORWARD_MAX_ROWS ||
        c.cols > GEO_B200_FEED_FORWARD_MAX_WIDTH || c.hidden > GEO_B200_FEED_FORWARD_MAX_WIDTH)
        return false;
    if (!resolve_strides(c.hidden, c.cols, {&c.gate_weight_stride, &c.up_weight_stride}) ||
        !resolve_strides(c.cols, c.hidden, {&c.down_weight_stride}) ||
        !resolve_strides(c.rows, c.hidden, {&c.gate_stride, &c.up_stride}) ||
        !resolve_strides(c.rows, c.cols, {&c.x_stride}))
        return false;
    if (vjp ? !resolve_strides(c.rows, c.cols, {&c.y_cotangent_stride, &c.x_cotangent_stride})
            : !resolve_strides(c.rows, c.cols, {&c.y_stride}))
        return false;
    *out = c;
    return true;
}

size_t round8(size_t n) { return (n + 7) / 8 * 8; }
bool off16(size_t stride) { return stride % 8 != 0; }

// The most room that the parts of sums of these products take, by whichever kernels run.
struct Extent {
    ProductKind kind;
    size_t m, n, k;
};
size_t partial_bytes(const geo_b200_feed_forward_config_t &c, std::initializer_list<Extent> products) {
    const size_t wide = wide_bytes(c.type);
    size_t most = 0;
    for (const Extent &x : products) {
        if (type_bytes(c.type) == 2) {
            const bool twice = x.kind == kWeights && c.gradient_type != c.type;
            most = std::max(most, partial_values(x.kind, cut_tensor(x.kind, c.type, twice, x.m, x.n, x.k).splits, x.m, x.n));
            most = std::max(most, partial_values(x.kind, cut_plain(x.kind, x.m, x.n, x.k).splits, x.m, x.n));
        } else {
            most = std::max(most, partial_values(x.kind, cut_wide(x.kind, c.type, x.m, x.n, x.k).splits, x.m, x.n));
        }
    }
    return most * wide;
}

// Launches a product by the kernels that take it; `rest`: room for parts of its sums.
cudaError_t launch_product(const geo_b200_feed_forward_config_t &c, bool tensor, ProductKind kind, Product &p, void *rest,
                           cudaStream_t stream, PipelineStarve starve = {UINT32_MAX, kPipelinePolls}) {
    p.partial = rest;
    if (type_bytes(c.type) != 2) {
        p.splits = cut_wide(kind, c.type, p.m, p.n, p.k).splits;
        return launch_product_wide(kind, c.type, p, stream);
    }
    if (tensor) {
        p.splits = cut_tensor(kind, c.type, kind == kWeights && c.gradient_type != c.type, p.m, p.n, p.k).splits;
        return launch_product_tensor(kind, c.type, c.gradient_type, p, starve, stream);
    }
    p.splits = cut_plain(kind, p.m, p.n, p.k).splits;
    return launch_product_plain(kind, c.type, c.gradient_type, p, stream);
}

// Where things lie in the workspace. `take` returns the place of rows x stride values.
struct Space {
    unsigned char *base;
    size_t used = 0;
    void *take(size_t rows, size_t stride, size_t bytes) {
        void *p = base == nullptr ? nullptr : base + used;
        used += (rows * stride * bytes + kAlign - 1) / kAlign * kAlign;
        return p;
    }
};

// Few rows are the weights' way through memory: columns of the result by warps
// (feed_forward_plain.cu). Of 16-bit types the tensor cores' tiles take over early
// (4096 x 12288 bfloat16: 2 rows 70 us either way, 4 rows 95 and 70), later where the
// weights are small (1024 x 2048: 4 rows 14 us, 5 rows in tiles 22) or would have to be
// copied first; of float64 before 8 rows (2048 x 4096: 107 us, 9 rows in tiles 99), of
// float32 beyond (56 and 88 us).
bool few_rows(const geo_b200_feed_forward_config_t &c) {
    if (type_bytes(c.type) != 2) return c.rows <= (size_t)(c.type == GEO_B200_F64 ? kFewRows / 2 : kFewRows);
    const bool copied = c.gate_weight_stride % 8 != 0 || c.up_weight_stride % 8 != 0 || c.down_weight_stride % 8 != 0;
    return c.rows <= 2 || (c.rows <= 4 && (copied || c.cols * c.hidden <= (size_t)1 << 22));
}

// The arrays of a call that TMA would read, by rows of `stride` values; those off 16
// bytes by their stride are copied to the workspace.
struct Operand {
    Matrix m;
    size_t rows, cols;
};
size_t packed_bytes(const Operand &o) {
    return off16(o.m.stride) ? (o.rows * round8(o.cols) * 2 + kAlign - 1) / kAlign * kAlign : 0;
}
cudaError_t pack(std::initializer_list<Operand *> operands, Space &space, cudaStream_t stream) {
    Pack list = {};
    size_t end = 0;
    for (Operand *o : operands) {
        if (o->m.p == nullptr || !off16(o->m.stride)) continue;
        const size_t stride = round8(o->cols);
        void *to = space.take(o->rows, stride, 2);
        end += o->rows * (stride / 8);
        list.arrays[list.count++] = {o->m, o->rows, (int)o->cols, to, stride, end};
        o->m = {to, stride};
    }
    return launch_pack(list, stream);
}
// Whether the tensor-core kernels take these arrays, once those off 16 bytes by their stride are copied.
bool tensor_call(const geo_b200_feed_forward_config_t &c, std::initializer_list<const Operand *> arrays) {
    if (type_bytes(c.type) != 2 || !tensor_products_available()) return false;
    // A tensor map's strides end at 2^40 bytes.
    for (const Operand *o : arrays)
        if (!off16(o->m.stride) && ((uintptr_t)o->m.p % 16 != 0 || o->m.stride >= (size_t)1 << 39)) return false;
    return true;
}

// Outputs apart from the inputs and from each other, as far as their starts tell.
bool apart(std::initializer_list<const void *> outs, std::initializer_list<const void *> ins) {
    for (auto o = outs.begin(); o != outs.end(); ++o) {
        if (*o == nullptr) continue;
        for (const void *i : ins)
            if (*o == i) return false;
        for (auto other = o + 1; other != outs.end(); ++other)
            if (*o == *other) return false;
    }
    return true;
}

}  // namespace

extern "C" size_t geo_b200_feed_forward_workspace(const geo_b200_feed_forward_config_t *config) {
    geo_b200_feed_forward_config_t c;
    if (!resolve(config, false, &c)) return 0;
    Space space = {nullptr};
    const size_t b = type_bytes(c.type);
    space.take(c.rows, round8(c.hidden), b);
    if (b == 2 && !few_rows(c))
        for (const Operand &o : {Operand{{nullptr, c.x_stride}, c.rows, c.cols},
                                 Operand{{nullptr, c.gate_weight_stride}, c.hidden, c.cols},
                                 Operand{{nullptr, c.up_weight_stride}, c.hidden, c.cols},
                                 Operand{{nullptr, c.down_weight_stride}, c.cols, c.hidden}})
            space.used += packed_bytes(o);
    if (!few_rows(c)) space.used += partial_bytes(c, {{kGated, c.rows, c.hidden, c.cols}, {kDown, c.rows, c.cols, c.hidden}});
    return space.used;
}

extern "C" size_t geo_b200_feed_forward_vjp_workspace(const geo_b200_feed_forward_config_t *config) {
    geo_b200_feed_forward_config_t c;
    if (!resolve(config, true, &c)) return 0;
    Space space = {nullptr};
    const size_t b = type_bytes(c.type);
    for (int i = 0; i < (c.gradient_type != c.type ? 6 : 3); ++i) space.take(c.rows, round8(c.hidden), b);
    if (c.type == GEO_B200_F16) space.take(1 + kScaleBlocks, 1, sizeof(float4));
    if (b == 2)
        for (const Operand &o : {Operand{{nullptr, c.x_stride}, c.rows, c.cols},
                                 Operand{{nullptr, c.y_cotangent_stride}, c.rows, c.cols},
                                 Operand{{nullptr, c.gate_weight_stride}, c.hidden, c.cols},
                                 Operand{{nullptr, c.up_weight_stride}, c.hidden, c.cols},
                                 Operand{{nullptr, c.down_weight_stride}, c.cols, c.hidden}})
            space.used += packed_bytes(o);
    space.used += partial_bytes(c, {{kHidden, c.rows, c.hidden, c.cols},
                                    {kInput, c.rows, c.cols, c.hidden},
                                    {kWeights, c.hidden, c.cols, c.rows}});
    return space.used;
}

namespace {

// `starve`: null, or for the self-test of the tensor-core kernels' waits, which are then the only ones taken.
geo_b200_status_t forward(const geo_b200_feed_forward_config_t *config, const void *device_x,
                          const void *device_gate_weight, const void *device_up_weight, const void *device_down_weight,
                          void *device_gate, void *device_up, void *device_y, void *device_workspace,
                          size_t workspace_bytes, const PipelineStarve *starve, cudaStream_t stream) {
    geo_b200_feed_forward_config_t c;
    if (!resolve(config, false, &c) || device_x == nullptr || device_gate_weight == nullptr ||
        device_up_weight == nullptr || device_down_weight == nullptr || device_y == nullptr ||
        (device_gate == nullptr) != (device_up == nullptr) || device_workspace == nullptr ||
        workspace_bytes < geo_b200_feed_forward_workspace(config) ||
        !apart({device_gate, device_up, device_y, device_workspace},
               {device_x, device_gate_weight, device_up_weight, device_down_weight}))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type);
    if (!arrays_usable({{device_x, b}, {device_gate_weight, b}, {device_up_weight, b}, {device_down_weight, b},
                        {device_gate, b}, {device_up, b}, {device_y, b}, {device_workspace, kAlign}}))
        return GEO_B200_INVALID_ARGUMENT;
    Space space = {(unsigned char *)device_workspace};
    const size_t hidden_stride = round8(c.hidden);
    void *h = space.take(c.rows, hidden_stride, b);
    Operand x = {{device_x, c.x_stride}, c.rows, c.cols}, wg = {{device_gate_weight, c.gate_weight_stride}, c.hidden, c.cols},
            wu = {{device_up_weight, c.up_weight_stride}, c.hidden, c.cols},
            wd = {{device_down_weight, c.down_weight_stride}, c.cols, c.hidden};
    const bool few = few_rows(c), tensor = !few && tensor_call(c, {&x, &wg, &wu, &wd});
    if (tensor) {
        const cudaError_t e = pack({&x, &wg, &wu, &wd}, space, stream);
        if (e != cudaSuccess) return status_of(e);
    }
    Product gated = {};
    gated.m = (int)c.rows, gated.n = (int)c.hidden, gated.k = (int)c.cols, gated.problems = 1;
    gated.activation = (int)c.activation;
    gated.a[0] = x.m;
    gated.b[0] = wg.m;
    gated.b[1] = wu.m;
    gated.out[0] = {device_gate, c.gate_stride};
    gated.out[1] = {device_up, c.up_stride};
    gated.out[2] = {h, hidden_stride};
    Product down = {};
    down.m = (int)c.rows, down.n = (int)c.cols, down.k = (int)c.hidden, down.problems = 1;
    down.a[0] = {h, hidden_stride};
    down.b[0] = wd.m;
    down.out[0] = {device_y, c.y_stride};
    void *const rest = space.take(0, 0, 1);
    if (starve != nullptr) {
        if (!tensor) return GEO_B200_INVALID_ARGUMENT;
        const cudaError_t e = launch_product(c, tensor, kGated, gated, rest, stream, *starve);
        return status_of(e != cudaSuccess ? e : launch_product(c, tensor, kDown, down, rest, stream));
    }
    auto launch = [&](ProductKind kind, Product &p) {
        return few ? launch_product_few(kind, c.type, p, stream) : launch_product(c, tensor, kind, p, rest, stream);
    };
    const cudaError_t e = launch(kGated, gated);
    return status_of(e != cudaSuccess ? e : launch(kDown, down));
}

}  // namespace

extern "C" geo_b200_status_t geo_b200_feed_forward(const geo_b200_feed_forward_config_t *config, const void *device_x,
                                                   const void *device_gate_weight, const void *device_up_weight,
                                                   const void *device_down_weight, void *device_gate, void *device_up,
                                                   void *device_y, void *device_workspace, size_t workspace_bytes,
                                                   cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.feed_forward");
    return forward(config, device_x, device_gate_weight, device_up_weight, device_down_weight, device_gate, device_up,
                   device_y, device_workspace, workspace_bytes, nullptr, stream);
}

extern "C" geo_b200_status_t geo_b200_feed_forward_wait_selftest(
    const geo_b200_feed_forward_config_t *config, const void *device_x, const void *device_gate_weight,
    const void *device_up_weight, const void *device_down_weight, void *device_gate, void *device_up, void *device_y,
    void *device_workspace, size_t workspace_bytes, uint32_t block, uint32_t wait_limit, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.feed_forward_wait_selftest");
    if (wait_limit == 0 || wait_limit > kPipelinePolls) return GEO_B200_INVALID_ARGUMENT;
    const PipelineStarve starve = {block, wait_limit};
    return forward(config, device_x, device_gate_weight, device_up_weight, device_down_weight, device_gate, device_up,
                   device_y, device_workspace, workspace_bytes, &starve, stream);
}

extern "C" geo_b200_status_t geo_b200_feed_forward_vjp(
    const geo_b200_feed_forward_config_t *config, const void *device_x, const void *device_gate_weight,
    const void *device_up_weight, const void *device_down_weight, const void *device_gate, const void *device_up,
    const void *device_y_cotangent, void *device_x_cotangent, void *device_gate_weight_cotangent,
    void *device_up_weight_cotangent, void *device_down_weight_cotangent, void *device_workspace,
    size_t workspace_bytes, cudaStream_t stream) {
    geo::NvtxRange range("geo_b200.feed_forward_vjp");
    geo_b200_feed_forward_config_t c;
    const bool weights = device_gate_weight_cotangent != nullptr || device_up_weight_cotangent != nullptr;
    const bool inner = weights || device_x_cotangent != nullptr;  // needs the cotangents of gate and up
    if (!resolve(config, true, &c) || (!inner && device_down_weight_cotangent == nullptr) ||
        (weights && device_x == nullptr) ||
        (device_x_cotangent != nullptr && (device_gate_weight == nullptr || device_up_weight == nullptr)) ||
        device_down_weight == nullptr || device_gate == nullptr || device_up == nullptr ||
        device_y_cotangent == nullptr || device_workspace == nullptr ||
        workspace_bytes < geo_b200_feed_forward_vjp_workspace(config) ||
        !apart({device_x_cotangent, device_gate_weight_cotangent, device_up_weight_cotangent,
                device_down_weight_cotangent, device_workspace},
               {device_x, device_gate_weight, device_up_weight, device_down_weight, device_gate, device_up,
                device_y_cotangent}))
        return GEO_B200_INVALID_ARGUMENT;
    const size_t b = type_bytes(c.type), g = type_bytes(c.gradient_type);
    if (!arrays_usable({{device_x, b}, {device_gate_weight, b}, {device_up_weight, b}, {device_down_weight, b},
                        {device_gate, b}, {device_up, b}, {device_y_cotangent, b}, {device_x_cotangent, b},
                        {device_gate_weight_cotangent, g}, {device_up_weight_cotangent, g},
                        {device_down_weight_cotangent, g}, {device_workspace, kAlign}}))
        return GEO_B200_INVALID_ARGUMENT;
    Space space = {(unsigned char *)device_workspace};
    const size_t hidden_stride = round8(c.hidden);
    void *inside[3], *low[3] = {};  // cotangents of gate and up, h; what they lost to rounding
    for (void *&p : inside) p = space.take(c.rows, hidden_stride, b);
    if (c.gradient_type != c.type)
        for (void *&p : low) p = space.take(c.rows, hidden_stride, b);
    float *const scale = c.type == GEO_B200_F16 ? (float *)space.take(1 + kScaleBlocks, 1, sizeof(float4)) : nullptr;
    Operand x = {{device_x, c.x_stride}, c.rows, c.cols}, wg = {{device_gate_weight, c.gate_weight_stride}, c.hidden, c.cols},
            wu = {{device_up_weight, c.up_weight_stride}, c.hidden, c.cols},
            wd = {{device_down_weight, c.down_weight_stride}, c.cols, c.hidden},
            dy = {{device_y_cotangent, c.y_cotangent_stride}, c.rows, c.cols};
    const bool tensor = tensor_call(c, {&x, &wg, &wu, &wd, &dy});
    if (tensor) {
        const cudaError_t e = pack({&x, &wg, &wu, &wd, &dy}, space, stream);
        if (e != cudaSuccess) return status_of(e);
    }
    void *const rest = space.take(0, 0, 1);
    if (scale != nullptr) {
        InnerScale s = {dy.m, wd.m, {device_gate, c.gate_stride}, {device_up, c.up_stride}, c.rows, c.cols, c.hidden,
                        (int)c.activation, (float4 *)scale};
        if (!inner) s.dy.p = s.wd.p = nullptr;
        const cudaError_t e = launch_scale(s, stream);
        if (e != cudaSuccess) return status_of(e);
    }
    // Of the cotangents of gate and up (0, 1) and of h (2).
    auto times = [&](int i, bool inverse) { return scale == nullptr ? nullptr : scale + (i == 2 ? 2 : 0) + (inverse ? 1 : 0); };
    auto launch = [&](ProductKind kind, Product &p) { return launch_product(c, tensor, kind, p, rest, stream); };
    Product hidden = {};
    hidden.m = (int)c.rows, hidden.n = (int)c.hidden, hidden.k = (int)c.cols, hidden.problems = 1;
    hidden.activation = (int)c.activation;
    hidden.a[0] = dy.m;
    hidden.b[0] = wd.m;
    hidden.saved[0] = {device_gate, c.gate_stride};
    hidden.saved[1] = {device_up, c.up_stride};
    for (int i = 0; i < 3; ++i) {
        const bool wanted = i == 2 ? device_down_weight_cotangent != nullptr : inner;
        if (wanted) hidden.out[i] = {inside[i], hidden_stride};
        hidden.times[i] = times(i, false);
        if (wanted && (i == 2 || weights)) hidden.out_low[i] = {low[i], hidden_stride};
    }
    cudaError_t e = launch(kHidden, hidden);
    if (e == cudaSuccess && device_x_cotangent != nullptr) {
        Product input = {};
        input.m = (int)c.rows, input.n = (int)c.cols, input.k = (int)c.hidden, input.problems = 1;
        for (int i = 0; i < 2; ++i) input.a[i] = {inside[i], hidden_stride};
        input.b[0] = wg.m;
        input.b[1] = wu.m;
        input.out[0] = {device_x_cotangent, c.x_cotangent_stride};
        input.times[0] = times(0, true);
        e = launch(kInput, input);
    }
    Product w = {};
    w.m = (int)c.hidden, w.n = (int)c.cols, w.k = (int)c.rows;
    const OutMatrix outs[3] = {{device_gate_weight_cotangent, c.gate_weight_stride},
                               {device_up_weight_cotangent, c.up_weight_stride},
                               {device_down_weight_cotangent, c.down_weight_stride}};
    for (int i = 0; i < 3; ++i)
        if (outs[i].p != nullptr) {
            w.a[w.problems] = {inside[i], hidden_stride};
            w.low[w.problems] = {low[i], hidden_stride};
            w.b[w.problems] = i == 2 ? dy.m : x.m;
            w.transposed[w.problems] = i == 2;
            w.times[w.problems] = times(i, true);
            w.out[w.problems++] = outs[i];
        }
    if (e == cudaSuccess && w.problems > 0) e = launch(kWeights, w);
    return status_of(e);
}
