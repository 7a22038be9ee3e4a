"""The feed-forward half of a layer and what its training step needs: the gated feed-forward block, RMS norm, the norms
before and after a block fused with its gate and residual scale, each forward and VJP, and the norm and clipping of a
model's gradients.

`own = False` computes them in elementary torch operations; `own = True` calls the library's entry points
through ctypes, as a user's program does.
"""
import math

import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}
EPSILON = 1e-5
ALPHA, BETA = 1.0, 0.5  # of the residual, of the block
MOST_FLOPS = 3e12  # of a drawn feed-forward case (a tenth of it in float64); the largest listed one has more
MOST_BYTES = 512 << 20  # of another drawn case; the largest listed ones move more


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # One token of a served model: latency, and the weights' way through memory.
        dict(name="forward_one_token", op="forward", type="bf16", rows=1, cols=4096, hidden=12288, activation="silu",
             save=False, pad=0),
        # A decoding step of many sequences, a ragged hidden width.
        dict(name="forward_decode_batch", op="forward", type="f16", rows=96, cols=2048, hidden=5504, activation="gelu",
             save=False, pad=0),
        # Training forward of a long batch, the projections kept for the VJP.
        dict(name="forward_train", op="forward", type="bf16", rows=8192, cols=4096, hidden=12288, activation="silu",
             save=True, pad=0),
        # Its backward pass: the largest case.
        dict(name="vjp_train", op="vjp", type="bf16", gtype="f32", rows=8192, cols=4096, hidden=12288,
             activation="silu", pad=0),
        # The library's own rows: dense Cl(6,0) multivectors of 64 float64 coefficients through a small block.
        dict(name="vjp_multivectors", op="vjp", type="f64", gtype="f64", rows=16384, cols=64, hidden=256,
             activation="gelu", pad=0),
        # A prompt's activations before a product.
        dict(name="rms_prompt", op="rms", type="bf16", ptype="f32", rows=8192, cols=4096, pad=0),
        # A slice of a wider buffer, backward: odd row length, rows that start off a 16-byte boundary.
        dict(name="rms_vjp_odd", op="rms_vjp", type="f32", ptype="f32", rows=3001, cols=1003, pad=1),
        # One token of a served model between two blocks.
        dict(name="block_one_token", op="block", type="bf16", ptype="bf16", rows=1, cols=4096, gate="sigmoid", pad=0),
        # Training between two blocks, forward and backward, with a gate for every value.
        dict(name="block_train", op="block", type="bf16", ptype="f32", rows=16384, cols=4096, gate="sigmoid", pad=0),
        dict(name="block_vjp_train", op="block_vjp", type="bf16", ptype="f32", rows=16384, cols=4096, gate="sigmoid",
             pad=0),
        # The gradients of a layered model of geometric products: many parameters of 64 float64 coefficients.
        dict(name="clip_multivectors", op="clip", type="f64", layers=48, cols=64, hidden=0),
        # The gradients of feed-forward layers and their norms' weights.
        dict(name="clip_layers", op="clip", type="bf16", layers=4, cols=4096, hidden=8192),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(max(lo, hi))))))))


def _size(rng, lo, hi):
    """Over the logarithm of the range; half of them multiples of 8, the rest as they fall."""
    n = _log(rng, lo, hi)
    return max(8, n // 8 * 8) if rng.random() < 0.5 and n >= 8 else n


def draw(rng):
    op = rng.choice(["forward", "forward", "vjp", "vjp", "rms", "rms_vjp", "block", "block_vjp", "clip"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32", "f64"])
    if op in ("forward", "vjp"):
        cols, hidden = _size(rng, 16, 8192), _size(rng, 16, 16384)
        most = MOST_FLOPS / (10 if kind == "f64" else 1) / (6 if op == "forward" else 12) / cols / hidden
        case = dict(op=op, type=kind, rows=_log(rng, 1, int(max(1, min(16384, most)))), cols=cols, hidden=hidden,
                    activation=rng.choice(["silu", "silu", "gelu", "sigmoid", "relu"]), pad=rng.choice([0, 0, 0, 8, 1]))
        if op == "forward":
            case["save"] = rng.random() < 0.5
        else:
            case["gtype"] = rng.choice([kind, "f32" if kind != "f64" else "f64"])
        return case
    if op == "clip":
        cols = _size(rng, 16, 4096)
        hidden = rng.choice([0, _size(rng, 16, 8192)])
        most = MOST_BYTES // (2 * BYTES[kind] * max(1, 3 * hidden * cols))
        return dict(op=op, type=kind, layers=_log(rng, 1, max(1, min(64, most))), cols=cols, hidden=hidden)
    cols = _size(rng, 16, 16384)
    most = MOST_BYTES // (8 * BYTES[kind] * cols)
    case = dict(op=op, type=kind, ptype=rng.choice([kind, "f32" if kind != "f64" else "f64"]),
                rows=_log(rng, 1, max(1, min(65536, most))), cols=cols, pad=rng.choice([0, 0, 0, 8, 1]))
    if op.startswith("block"):
        case["gate"] = rng.choice(["none", "linear", "sigmoid", "sigmoid", "tanh"])
    return case


def _tensors(case):
    """Sizes and types of the gradients of a clip case: a layer's three products and two norms, or four multivectors'
    worth of parameters (hidden 0)."""
    norm = "f32" if BYTES[case["type"]] == 2 else case["type"]
    c, h = case["cols"], case["hidden"]
    layer = [(h * c, case["type"])] * 3 + [(c, norm)] * 2 if h else [(c, case["type"])] * 4
    return layer * case["layers"]


def _views(case, buffers):
    """The tensors of a clip case in the buffers of their types."""
    at, out = dict.fromkeys(buffers, 0), []
    for n, t in _tensors(case):
        out.append(buffers[t][at[t]:at[t] + n])
        at[t] += n
    return out


def work(case):
    op, b = case["op"], BYTES[case["type"]]
    if op == "clip":
        n = sum(count for count, _ in _tensors(case))
        return {"bytes": 2 * sum(count * BYTES[t] for count, t in _tensors(case)), "flops": 3 * n}
    rows, cols = case["rows"], case["cols"]
    if op in ("forward", "vjp"):
        weights, h = 3 * cols * case["hidden"], case["hidden"]
        if op == "forward":
            return {"bytes": b * (2 * rows * cols + weights + (2 * rows * h if case["save"] else 0)),
                    "flops": 2 * rows * weights}
        return {"bytes": b * (3 * rows * cols + weights + 2 * rows * h) + BYTES[case["gtype"]] * weights,
                "flops": 4 * rows * weights}
    n, par = rows * cols, cols * BYTES[case["ptype"]]
    stat = rows * (8 if case["type"] == "f64" else 4)
    gated = int(case.get("gate", "none") != "none")
    arrays, flops, extra = {
        "rms": (2, 4, stat + par),
        "rms_vjp": (3, 10, stat + 2 * par),
        "block": (4 + gated, 12, 2 * stat + 2 * par),
        "block_vjp": (6 + 2 * gated, 30, 2 * stat + 4 * par),
    }[op]
    return {"bytes": arrays * n * b + extra, "flops": flops * n}


# ---- inputs -----------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _normal(g, kind, *shape):
    t = TYPES[kind]
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float64 if t == torch.float64 else torch.float32)


def _rows(case, g, scale=1.0, outliers=False, offset=0.0):
    """A [rows][cols] array; `pad` > 0 makes it a slice of a wider buffer, starting `pad` values into it."""
    cols, pad = case["cols"], case["pad"]
    made = _normal(g, case["type"], case["rows"], cols + 2 * pad).mul_(scale).add_(offset)
    if outliers:  # activations: a few channels far larger than the rest
        made[:, ::97] *= 8.0
    return made.to(TYPES[case["type"]])[:, pad:pad + cols]


def _empty_rows(case):
    cols, pad = case["cols"], case["pad"]
    return torch.empty(case["rows"], cols + 2 * pad, device="cuda", dtype=TYPES[case["type"]])[:, pad:pad + cols]


def prepare(case, seed):
    g = _generator(seed)
    s, op = {"case": case}, case["op"]
    if op == "clip":
        # Small gradients with a spread of sizes from tensor to tensor; their norm is ten times what is allowed.
        # Those of one type lie one behind the other in one buffer, as a program keeps them.
        tensors, s["gradients"], s["buffers"] = _tensors(case), [], {}
        for t in sorted({t for _, t in tensors}):
            s["buffers"][t] = torch.empty(sum(n for n, k in tensors if k == t), device="cuda", dtype=TYPES[t])
        for i, v in enumerate(_views(case, s["buffers"])):
            v.copy_(_normal(g, tensors[i][1], v.numel()) * (1e-3 * (1 + i % 7)))
            s["gradients"].append(v)
        total = sum(n * (1e-3 * (1 + i % 7)) ** 2 for i, (n, _) in enumerate(_tensors(case)))
        s["most"] = 0.1 * math.sqrt(total)
    elif op in ("forward", "vjp"):
        t, cols, hidden = TYPES[case["type"]], case["cols"], case["hidden"]
        s["x"] = _rows(case, g)
        for name, rows, width in (("wg", hidden, cols), ("wu", hidden, cols), ("wd", cols, hidden)):
            s[name] = (_normal(g, case["type"], rows, width) / math.sqrt(width)).to(t)
        if op == "vjp":  # the forward's projections, as it keeps them
            x = _wide(s["x"])
            s["a"], s["u"] = (x @ _wide(s["wg"]).T).to(t), (x @ _wide(s["wu"]).T).to(t)
            s["dy"] = _rows(case, g, scale=0.1)
    else:
        p = TYPES[case["ptype"]]
        s["x"] = _rows(case, g, scale=2.0, outliers=True)
        s["w"] = (1 + 0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(p)
        keep = torch.float64 if case["type"] == "f64" else torch.float32
        root = lambda v: (v.double().square_().mean(1) + EPSILON).rsqrt().to(keep)  # noqa: E731
        if op.startswith("block"):
            s["pre"] = (1 + 0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(p)
            s["residual"] = _rows(case, g, outliers=True)
            s["gate"] = None if case["gate"] == "none" else _rows(case, g, offset=0.25)
        if op.endswith("vjp"):  # what the forward keeps
            s["dy"] = _rows(case, g, scale=0.1)
            s["rstd"] = root(s["x"])
            if op == "block_vjp":
                s["dz"] = _rows(case, g, scale=0.1)
                z = _join(s, _wide(s["x"]) * s["rstd"][:, None] * _wide(s["w"])).to(s["x"].dtype)
                s["z"] = _empty_rows(case)
                s["z"].copy_(z)
                s["z_rstd"] = root(s["z"])
                del s["residual"]
    if own:
        s["call"] = _bind(case, s)
    return s


# ---- plain forms ------------------------------------------------------------


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _activation(a, kind):
    """The activation and its derivative."""
    if kind == "relu":
        on = (a > 0).to(a.dtype)
        return a * on, on
    if kind == "gelu":
        below = torch.erfc(a * -math.sqrt(0.5)) * 0.5
        return a * below, below + a * torch.exp(-0.5 * a * a) * (1 / math.sqrt(2 * math.pi))
    s = 1 / (1 + torch.exp(-a))
    if kind == "sigmoid":
        return s, s * (1 - s)
    return a * s, s * (1 + a * (1 - s))


def _gate(s):
    """What the block is multiplied by, and its derivative."""
    kind = s["case"]["gate"]
    if kind == "none":
        return 1.0, None
    g = _wide(s["gate"])
    if kind == "linear":
        return g, torch.ones_like(g)
    if kind == "tanh":
        t = torch.tanh(g)
        return t, 1 - t * t
    v = 1 / (1 + torch.exp(-g))
    return v, v * (1 - v)


def _join(s, n):
    return ALPHA * _wide(s["residual"]) + BETA * _gate(s)[0] * n


def _rms(x, w):
    rstd = torch.rsqrt((x * x).sum(1, keepdim=True) / x.shape[1] + EPSILON)
    return x * rstd * _wide(w), rstd[:, 0]


def _rms_vjp(x, rstd, w, dy):
    """x_bar and what the weight's cotangent is the sum of."""
    xh, g = x * rstd[:, None], dy * _wide(w)
    return rstd[:, None] * (g - xh * ((g * xh).sum(1, keepdim=True) / x.shape[1])), dy * xh


def run(state):
    if own:
        return _call(state)
    s, case = state, state["case"]
    op = case["op"]
    if op == "clip":
        total = 0.0
        for v in s["gradients"]:
            w = v.double() if v.dtype == torch.float64 else v.float()
            total = total + (w * w).sum(dtype=torch.float64)
        norm = torch.sqrt(total)
        scale = torch.clamp(s["most"] / norm, max=1.0)
        return {"norm": norm, "scale": scale,
                **{t: (_wide(v) * scale.to(_wide(v).dtype)).to(v.dtype) for t, v in s["buffers"].items()}}
    t = s["x"].dtype
    if op == "forward":
        x = _wide(s["x"])
        a, u = x @ _wide(s["wg"]).T, x @ _wide(s["wu"]).T
        out = {"y": ((_activation(a, case["activation"])[0] * u) @ _wide(s["wd"]).T).to(t)}
        return {**out, "a": a.to(t), "u": u.to(t)} if case["save"] else out
    if op == "vjp":
        x, dy, a, u = (_wide(s[k]) for k in ("x", "dy", "a", "u"))
        f, slope = _activation(a, case["activation"])
        dh = dy @ _wide(s["wd"])
        da, du = dh * u * slope, dh * f
        p = TYPES[case["gtype"]]
        return {"dx": (da @ _wide(s["wg"]) + du @ _wide(s["wu"])).to(t), "dwg": (da.T @ x).to(p),
                "dwu": (du.T @ x).to(p), "dwd": (dy.T @ (f * u)).to(p)}
    if op == "rms":
        y, rstd = _rms(_wide(s["x"]), s["w"])
        return {"y": y.to(t), "rstd": rstd}
    if op == "rms_vjp":
        dx, dw = _rms_vjp(_wide(s["x"]), s["rstd"], s["w"], _wide(s["dy"]))
        return {"dx": dx.to(t), "dw": dw.sum(0).to(s["w"].dtype)}
    if op == "block":
        n, rstd = _rms(_wide(s["x"]), s["w"])
        z = _join(s, n)
        y, z_rstd = _rms(z, s["pre"])
        return {"z": z.to(t), "y": y.to(t), "rstd": rstd, "z_rstd": z_rstd}
    x, dy = _wide(s["x"]), _wide(s["dy"])
    dz, dpre = _rms_vjp(_wide(s["z"]), s["z_rstd"], s["pre"], dy)
    dz = dz + _wide(s["dz"])
    gate, slope = _gate(s)
    dx, dpost = _rms_vjp(x, s["rstd"], s["w"], BETA * gate * dz)
    out = {"dresidual": (ALPHA * dz).to(t), "dx": dx.to(t), "dpost": dpost.sum(0).to(s["w"].dtype),
           "dpre": dpre.sum(0).to(s["w"].dtype)}
    if slope is not None:
        out["dgate"] = (BETA * dz * x * s["rstd"][:, None] * _wide(s["w"]) * slope).to(t)
    return out


# ---- the library's entry points ---------------------------------------------


def _bind(case, s):
    """The configuration, output buffers and workspace that a program keeps from call to call."""
    import ctypes

    from geometricelementaryoperators_b200 import abi

    lib, op = abi.lib(), case["op"]
    kind = {"f64": abi.F64, "f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}
    ptr = lambda t: ctypes.c_void_p(t.data_ptr()) if t is not None else None  # noqa: E731
    ref = ctypes.byref
    space = lambda size: torch.empty(max(1, size), device="cuda", dtype=torch.uint8)  # noqa: E731
    if op == "clip":
        out = {t: torch.empty_like(v) for t, v in s["buffers"].items()}
        clipped = _views(case, out)
        found = torch.empty(2, device="cuda", dtype=torch.float64)
        table = (abi.Gradient * len(clipped))(*[
            abi.Gradient(type=kind[t], count=n, gradient=v.data_ptr(), clipped=c.data_ptr())
            for (n, t), v, c in zip(_tensors(case), s["gradients"], clipped)])
        size = lib.geo_b200_gradient_clip_workspace(table, len(clipped))
        work_space = space(size)
        return lib.geo_b200_gradient_clip, (table, len(clipped), s["most"], ptr(found[0]), ptr(found[1]),
                                            ptr(work_space), size), {
            "norm": found[0], "scale": found[1], **out}, (work_space,)
    rows, cols = case["rows"], case["cols"]
    stride = cols + 2 * case["pad"]
    new = lambda: _empty_rows(case)  # noqa: E731
    if op in ("forward", "vjp"):
        t, hidden = TYPES[case["type"]], case["hidden"]
        act = {"silu": abi.ACTIVATION_SILU, "gelu": abi.ACTIVATION_GELU, "sigmoid": abi.ACTIVATION_SIGMOID,
               "relu": abi.ACTIVATION_RELU}[case["activation"]]
        config = abi.FeedForwardConfig(type=kind[case["type"]], gradient_type=kind[case.get("gtype", case["type"])],
                                       activation=act, rows=rows, cols=cols, hidden=hidden, x_stride=stride,
                                       y_stride=stride, y_cotangent_stride=stride, x_cotangent_stride=stride)
        weights = (ptr(s["wg"]), ptr(s["wu"]), ptr(s["wd"]))
        if op == "forward":
            size = lib.geo_b200_feed_forward_workspace(ref(config))
            work_space = space(size)
            out = {"y": new()}
            if case["save"]:
                out["a"], out["u"] = (torch.empty(rows, hidden, device="cuda", dtype=t) for _ in range(2))
            return lib.geo_b200_feed_forward, (ref(config), ptr(s["x"]), *weights, ptr(out.get("a")), ptr(out.get("u")),
                                               ptr(out["y"]), ptr(work_space), size), out, (config, work_space)
        size = lib.geo_b200_feed_forward_vjp_workspace(ref(config))
        work_space, p = space(size), TYPES[case["gtype"]]
        out = {"dx": new(), "dwg": torch.empty(hidden, cols, device="cuda", dtype=p),
               "dwu": torch.empty(hidden, cols, device="cuda", dtype=p),
               "dwd": torch.empty(cols, hidden, device="cuda", dtype=p)}
        return lib.geo_b200_feed_forward_vjp, (
            ref(config), ptr(s["x"]), *weights, ptr(s["a"]), ptr(s["u"]), ptr(s["dy"]), ptr(out["dx"]),
            ptr(out["dwg"]), ptr(out["dwu"]), ptr(out["dwd"]), ptr(work_space), size), out, (config, work_space)
    keep = torch.float64 if case["type"] == "f64" else torch.float32
    if op in ("rms", "rms_vjp"):
        config = abi.LayerNormConfig(type=kind[case["type"]], parameter_type=kind[case["ptype"]], rows=rows, cols=cols,
                                     x_stride=stride, y_stride=stride, y_cotangent_stride=stride,
                                     x_cotangent_stride=stride, epsilon=EPSILON)
        if op == "rms":
            out = {"y": new(), "rstd": torch.empty(rows, device="cuda", dtype=keep)}
            return lib.geo_b200_rms_norm, (ref(config), ptr(s["x"]), ptr(s["w"]), ptr(out["y"]),
                                           ptr(out["rstd"])), out, (config,)
        size = lib.geo_b200_rms_norm_vjp_workspace(ref(config))
        work_space = space(size)
        out = {"dx": new(), "dw": torch.empty_like(s["w"])}
        return lib.geo_b200_rms_norm_vjp, (ref(config), ptr(s["x"]), ptr(s["w"]), ptr(s["rstd"]), ptr(s["dy"]),
                                           ptr(out["dx"]), ptr(out["dw"]), ptr(work_space), size), out, (
            config, work_space)
    gate = {"none": abi.GATE_NONE, "linear": abi.GATE_LINEAR, "sigmoid": abi.GATE_SIGMOID, "tanh": abi.GATE_TANH}
    config = abi.BlockNormConfig(type=kind[case["type"]], parameter_type=kind[case["ptype"]], gate=gate[case["gate"]],
                                 rows=rows, cols=cols, x_stride=stride, residual_stride=stride, gate_stride=stride,
                                 z_stride=stride, y_stride=stride, y_cotangent_stride=stride, z_cotangent_stride=stride,
                                 residual_cotangent_stride=stride, x_cotangent_stride=stride,
                                 gate_cotangent_stride=stride, epsilon=EPSILON, residual_scale=ALPHA, block_scale=BETA)
    if op == "block":
        stats = torch.empty(2, rows, device="cuda", dtype=keep)
        out = {"z": new(), "y": new(), "rstd": stats[0], "z_rstd": stats[1]}
        return lib.geo_b200_block_norm, (ref(config), ptr(s["x"]), ptr(s["residual"]), ptr(s["gate"]), ptr(s["w"]),
                                         ptr(s["pre"]), ptr(out["z"]), ptr(out["y"]), ptr(out["rstd"]),
                                         ptr(out["z_rstd"])), out, (config,)
    size = lib.geo_b200_block_norm_vjp_workspace(ref(config))
    work_space = space(size)
    out = {"dresidual": new(), "dx": new(), "dpost": torch.empty_like(s["w"]), "dpre": torch.empty_like(s["w"])}
    if case["gate"] != "none":
        out["dgate"] = new()
    return lib.geo_b200_block_norm_vjp, (
        ref(config), ptr(s["x"]), ptr(s["gate"]), ptr(s["z"]), ptr(s["w"]), ptr(s["pre"]), ptr(s["rstd"]),
        ptr(s["z_rstd"]), ptr(s["dy"]), ptr(s["dz"]), ptr(out["dresidual"]), ptr(out["dx"]), ptr(out.get("dgate")),
        ptr(out["dpost"]), ptr(out["dpre"]), ptr(work_space), size), out, (config, work_space)


def _call(s):
    call, args, out, _ = s["call"]
    status = call(*args, torch.cuda.current_stream().cuda_stream)
    if status:
        raise RuntimeError("status %d" % status)
    return out


# ---- 64-bit definitions -----------------------------------------------------


def _exact_activation(a, kind):
    """The activation and its slope by differentiation of the definition."""
    leaf = a.detach().clone().requires_grad_(True)
    with torch.enable_grad():
        if kind == "relu":
            f = torch.where(leaf > 0, leaf, torch.zeros_like(leaf))
        elif kind == "gelu":
            f = leaf * torch.special.ndtr(leaf)
        else:
            f = torch.sigmoid(leaf) * (leaf if kind == "silu" else 1.0)
        slope, = torch.autograd.grad(f.sum(), leaf)
    return f.detach(), slope


def exact(case, seed):
    s, op = prepare(case, seed), case["op"]
    if op == "clip":
        norm = torch.linalg.vector_norm(torch.stack([torch.linalg.vector_norm(v.double()) for v in s["gradients"]]))
        scale = torch.where(norm > s["most"], s["most"] / norm, torch.ones_like(norm))
        return {"norm": norm, "scale": scale, **{t: v.double() * scale for t, v in s["buffers"].items()}}
    x = s["x"].double()
    if op in ("forward", "vjp"):
        wg, wu, wd = (s[k].double() for k in ("wg", "wu", "wd"))
        if op == "forward":
            a, u = torch.einsum("rc,hc->rh", x, wg), torch.einsum("rc,hc->rh", x, wu)
            out = {"y": torch.einsum("rh,ch->rc", _exact_activation(a, case["activation"])[0] * u, wd)}
            return {**out, "a": a, "u": u} if case["save"] else out
        dy, u = s["dy"].double(), s["u"].double()
        f, slope = _exact_activation(s["a"].double(), case["activation"])
        dh = torch.einsum("rc,ch->rh", dy, wd)
        slope *= dh
        slope *= u
        dh *= f
        f *= u
        return {"dx": torch.einsum("rh,hc->rc", slope, wg) + torch.einsum("rh,hc->rc", dh, wu),
                "dwg": torch.einsum("rh,rc->hc", slope, x), "dwu": torch.einsum("rh,rc->hc", dh, x),
                "dwd": torch.einsum("rc,rh->ch", dy, f)}
    w = s["w"].double()
    if op == "rms":
        root = torch.sqrt(torch.mean(torch.square(x), 1) + EPSILON)
        return {"y": x / root[:, None] * w, "rstd": 1 / root}
    if op == "rms_vjp":
        r, dy = s["rstd"].double()[:, None], s["dy"].double()
        along = torch.einsum("rc,rc,c->r", dy, x * r, w)[:, None] / case["cols"]
        return {"dx": r * (dy * w - x * r * along), "dw": torch.einsum("rc,rc->c", dy, x * r)}
    kind = case["gate"]
    if kind == "none":
        value, slope = torch.ones((), dtype=torch.float64, device="cuda"), None
    else:
        g = s["gate"].double()
        value = {"linear": lambda v: v, "sigmoid": torch.sigmoid, "tanh": torch.tanh}[kind](g)
        slope = {"linear": lambda v: torch.ones_like(v), "sigmoid": lambda v: torch.sigmoid(v) * torch.sigmoid(-v),
                 "tanh": lambda v: 1 / torch.cosh(v).square()}[kind](g)
    pre = s["pre"].double()
    if op == "block":
        root = torch.sqrt(torch.mean(torch.square(x), 1) + EPSILON)
        z = s["residual"].double() * ALPHA + value * (x / root[:, None] * w) * BETA
        z_root = torch.sqrt(torch.mean(torch.square(z), 1) + EPSILON)
        return {"z": z, "y": z / z_root[:, None] * pre, "rstd": 1 / root, "z_rstd": 1 / z_root}
    r, zr, dy = s["rstd"].double()[:, None], s["z_rstd"].double()[:, None], s["dy"].double()
    zh, xh = s["z"].double() * zr, x * r
    dz = zr * (dy * pre - zh * (torch.einsum("rc,rc,c->r", dy, zh, pre)[:, None] / case["cols"])) + s["dz"].double()
    dn = dz * value * BETA
    dx = r * (dn * w - xh * (torch.einsum("rc,rc,c->r", dn, xh, w)[:, None] / case["cols"]))
    out = {"dresidual": dz * ALPHA, "dx": dx, "dpost": torch.einsum("rc,rc->c", dn, xh),
           "dpre": torch.einsum("rc,rc->c", dy, zh)}
    if slope is not None:
        out["dgate"] = dz * slope * (xh * w) * BETA
    return out
