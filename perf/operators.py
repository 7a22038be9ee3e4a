"""The layer operators that stand between the products of a model over rows of coefficients: layer norm,
dropout, the two fused with a residual, and rotary positions, each forward and VJP.

`own = False` computes them in elementary torch operations; `own = True` calls the library's entry points
through ctypes, as a user's program does.
"""
import math

import numpy as np
import torch

own = False

TYPES = {"f64": torch.float64, "f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BYTES = {"f64": 8, "f32": 4, "bf16": 2, "f16": 2}
EPSILON = 1e-5
LARGEST_BYTES = 640 << 20  # a drawn case moves no more than this; the largest listed one moves more


# ---- cases ------------------------------------------------------------------


def listed():
    return [
        # One token of a served model: latency alone.
        dict(name="norm_one_token", op="norm", type="bf16", ptype="bf16", rows=1, cols=1024, pad=0),
        # A prompt's activations, normalised before a product.
        dict(name="norm_prompt", op="norm", type="bf16", ptype="f32", rows=8192, cols=4096, pad=0),
        # Training on the library's own rows: one dense Cl(6,0) multivector of 64 float64 coefficients a row.
        dict(name="norm_vjp_multivectors", op="norm_vjp", type="f64", ptype="f64", rows=1 << 19, cols=64, pad=0),
        # A slice of a wider buffer: odd row length, rows that start off a 16-byte boundary.
        dict(name="norm_vjp_odd", op="norm_vjp", type="f32", ptype="f32", rows=3001, cols=1003, pad=1),
        # Dropout of a projection's output, added to the residual stream.
        dict(name="dropout_residual", op="dropout", type="bf16", rows=8192, cols=8192, pad=0, dimension=0,
             rate=0.1, residual=True),
        # Whole Cl(6,0) multivectors kept or dropped, backward.
        dict(name="dropout_vjp_multivectors", op="dropout_vjp", type="f64", rows=1 << 18, cols=64, pad=0, dimension=6,
             rate=0.25, residual=False),
        # A training step's residual + dropout + layer norm, forward and backward.
        dict(name="add_norm_train", op="add_norm", type="bf16", ptype="f32", rows=16384, cols=4096, pad=0,
             dimension=0, rate=0.1),
        dict(name="add_norm_vjp_train", op="add_norm_vjp", type="bf16", ptype="f32", rows=16384, cols=4096, pad=0,
             dimension=0, rate=0.1),
        # A short ragged batch in half precision, four-dimensional multivector units.
        dict(name="add_norm_vjp_short", op="add_norm_vjp", type="f16", ptype="f16", rows=77, cols=2000, pad=0,
             dimension=2, rate=0.2),
        # A decoding step: eight sequences, one token each, at positions of their own.
        dict(name="rotary_decode", op="rotary", type="bf16", batch=8, tokens=1, heads=40, head_dim=128,
             rotary_dim=128, layout="half", scaling="none", far=4096, headmajor=False),
        # Queries and keys of two prompts in one projection buffer.
        dict(name="rotary_prompt", op="rotary", type="bf16", batch=2, tokens=8192, heads=40, head_dim=128,
             rotary_dim=128, layout="half", scaling="linear", far=8192, headmajor=False),
        # Backward at far positions: part of the head, interleaved pairs, bands of frequencies scaled apart.
        dict(name="rotary_vjp_far", op="rotary_vjp", type="f32", batch=1, tokens=5777, heads=9, head_dim=96,
             rotary_dim=64, layout="interleaved", scaling="banded", far=1 << 20, headmajor=True),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _size(rng, lo, hi):
    """Over the logarithm of the range; half of them multiples of 8, the rest as they fall."""
    n = _log(rng, lo, hi)
    return max(8, n // 8 * 8) if rng.random() < 0.5 and n >= 8 else n


def draw(rng):
    op = rng.choice(["norm", "norm_vjp", "dropout", "dropout_vjp", "add_norm", "add_norm_vjp", "rotary", "rotary_vjp"])
    kind = rng.choice(["bf16", "bf16", "f16", "f32", "f64"])
    if op.startswith("rotary"):
        head_dim = rng.choice([16, 32, 64, 80, 96, 128, 192, 256])
        rotary_dim = rng.choice([head_dim, head_dim, head_dim // 2, 16])
        batch, heads = rng.choice([1, 1, 2, 5]), _log(rng, 1, 64)
        most = LARGEST_BYTES // (2 * BYTES[kind] * batch * heads * head_dim)
        return dict(op=op, type=kind, batch=batch, tokens=_log(rng, 1, min(32768, most)), heads=heads,
                    head_dim=head_dim, rotary_dim=rotary_dim, layout=rng.choice(["half", "interleaved"]),
                    scaling=rng.choice(["none", "linear", "base", "banded"]), far=1 << rng.randint(12, 20),
                    headmajor=rng.random() < 0.3)
    cols = _size(rng, 16, 16384)
    most = LARGEST_BYTES // (5 * BYTES[kind] * cols)
    case = dict(op=op, type=kind, rows=_log(rng, 1, min(65536, most)), cols=cols, pad=rng.choice([0, 0, 0, 8, 1]))
    if "norm" in op:
        case["ptype"] = rng.choice([kind, "f32" if kind != "f64" else "f64"])
    if op.startswith(("dropout", "add")):
        free = [n for n in range(7) if cols % (1 << n) == 0]
        case["dimension"] = rng.choice([0, rng.choice(free)])
        case["rate"] = rng.choice([0.0, 0.1, 0.2, 0.5])
    if op.startswith("dropout"):
        case["residual"] = op == "dropout" and rng.random() < 0.5
    return case


def work(case):
    op = case["op"]
    if op.startswith("rotary"):
        n = case["batch"] * case["tokens"] * case["heads"] * case["head_dim"]
        turned = n // case["head_dim"] * case["rotary_dim"]
        return {"bytes": 2 * n * BYTES[case["type"]] + 8 * case["batch"] * case["tokens"], "flops": 3 * turned}
    n, b = case["rows"] * case["cols"], BYTES[case["type"]]
    stat = case["rows"] * (8 if case["type"] == "f64" else 4)
    par = case["cols"] * BYTES[case.get("ptype", case["type"])]
    arrays, flops, extra = {
        "norm": (2, 8, 2 * stat + 2 * par),
        "norm_vjp": (3, 15, 2 * stat + 3 * par),
        "dropout": (2 + bool(case.get("residual")), 2, 0),
        "dropout_vjp": (2, 1, 0),
        "add_norm": (4, 10, 2 * stat + 2 * par),
        "add_norm_vjp": (5, 17, 2 * stat + 3 * par),
    }[op]
    return {"bytes": arrays * n * b + extra, "flops": flops * n}


# ---- inputs -----------------------------------------------------------------


def _generator(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _rows(case, g, scale=1.0, outliers=False):
    """A [rows][cols] array; `pad` > 0 makes it a slice of a wider buffer, starting `pad` values into it."""
    rows, cols, pad = case["rows"], case["cols"], case["pad"]
    t = TYPES[case["type"]]
    made = torch.randn(rows, cols + 2 * pad, generator=g, device="cuda", dtype=torch.float64 if t == torch.float64 else torch.float32)
    made.mul_(scale)
    if outliers:  # activations: an offset and a few channels far larger than the rest
        made.add_(0.25)
        made[:, ::97] *= 8.0
    return made.to(t)[:, pad:pad + cols]


def _empty_like(case):
    rows, cols, pad = case["rows"], case["cols"], case["pad"]
    return torch.empty(rows, cols + 2 * pad, device="cuda", dtype=TYPES[case["type"]])[:, pad:pad + cols]


def _threshold(rate):
    """The drop rate in steps of 2^-16."""
    return int(np.rint(rate * 65536.0))


def _turns(case):
    """Turns per position of each pair, in extended precision: high part of 30 fraction bits, low part the rest."""
    d = case["rotary_dim"]
    i = np.arange(d // 2, dtype=np.longdouble)
    base, factor = np.longdouble(_BASE), np.longdouble(_FACTOR)
    if case["scaling"] == "base" and d > 2:
        base = base * factor ** (np.longdouble(d) / np.longdouble(d - 2))
    f = base ** (-2 * i / np.longdouble(d))
    two_pi = 8 * np.arctan(np.longdouble(1))
    if case["scaling"] == "linear":
        f = f / factor
    if case["scaling"] == "banded":
        rotations = np.longdouble(_ORIGINAL) * f / two_pi
        keep = np.clip((rotations - _LOW) / (np.longdouble(_HIGH) - _LOW), 0, 1)
        f = f * keep + f / factor * (1 - keep)
    t = f / two_pi
    high = np.rint(t * 2.0 ** 30) / 2.0 ** 30
    return high.astype(np.float64), (t - high).astype(np.float64), t


_BASE, _FACTOR, _ORIGINAL, _LOW, _HIGH = 10000.0, 8.0, 4096.0, 1.0, 32.0


def _amplitude(case):
    return 0.1 * math.log(_FACTOR) + 1.0 if case["scaling"] == "banded" else 1.0


def prepare(case, seed):
    g = _generator(seed)
    s = {"case": case}
    op = case["op"]
    if op.startswith("rotary"):
        b, t, h, d = case["batch"], case["tokens"], case["heads"], case["head_dim"]
        shape = (b, h, t, d) if case["headmajor"] else (b, t, h, d)
        made = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(TYPES[case["type"]])
        s["x"] = made.transpose(1, 2) if case["headmajor"] else made  # [batch][tokens][heads][head_dim]
        first = torch.randint(0, max(1, case["far"] - t), (b, 1), generator=g, device="cuda")
        s["positions"] = first + torch.arange(t, device="cuda")  # each sequence from a position of its own
        high, low, _ = _turns(case)
        s["high"], s["low"] = torch.tensor(high, device="cuda"), torch.tensor(low, device="cuda")
    else:
        s["x"] = _rows(case, g, outliers=op in ("norm", "norm_vjp", "add_norm_vjp"))
        if case.get("residual") or op == "add_norm":
            s["residual"] = _rows(case, g, outliers=True)
        if op.endswith("vjp"):
            s["dy"] = _rows(case, g, scale=0.1)
        if op == "add_norm_vjp":
            s["dz"] = _rows(case, g, scale=0.1)
        if "rate" in case:
            s["threshold"] = _threshold(case["rate"])
            s["seed"], s["offset"] = (seed * 0x9E3779B97F4A7C15 + 0x632BE59BD9B4E019) % (1 << 64), seed % 1000
        if "ptype" in case:
            p = TYPES[case["ptype"]]
            s["weight"] = (1 + 0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(p)
            s["bias"] = (0.1 * torch.randn(case["cols"], generator=g, device="cuda")).to(p)
        if op in ("norm_vjp", "add_norm_vjp"):  # the forward's statistics
            x = s["x"].double()
            mean = x.mean(1)
            rstd = ((x - mean[:, None]).square_().mean(1) + EPSILON).rsqrt()
            keep = torch.float64 if case["type"] == "f64" else torch.float32
            s["mean"], s["rstd"] = mean.to(keep), rstd.to(keep)
    if own:
        s["call"] = _bind(case, s)
    return s


# ---- plain forms ------------------------------------------------------------


def _wide(t):
    return t if t.dtype == torch.float64 else t.float()


def _high_half(a, m):
    """(low, high) 32-bit words of the 64-bit product of a (32 bits in an int64) and the constant m."""
    p = a * m
    return p & 0xFFFFFFFF, (p >> 32) & 0xFFFFFFFF


def _draws(units, seed, offset):
    """One 16-bit draw a unit: Philox4x32-10 on the counter (unit // 8, offset), keyed by the seed."""
    block = torch.arange((units + 7) // 8, device="cuda")
    c0, c1 = block & 0xFFFFFFFF, block >> 32
    c2, c3 = torch.full_like(block, offset & 0xFFFFFFFF), torch.full_like(block, offset >> 32)
    k0, k1 = seed & 0xFFFFFFFF, seed >> 32
    for _ in range(10):
        lo0, hi0 = _high_half(c0, 0xD2511F53)
        lo1, hi1 = _high_half(c2, 0xCD9E8D57)
        c0, c1, c2, c3 = hi1 ^ c1 ^ k0, lo1, hi0 ^ c3 ^ k1, lo0
        k0, k1 = (k0 + 0x9E3779B9) & 0xFFFFFFFF, (k1 + 0xBB67AE85) & 0xFFFFFFFF
    words = torch.stack([c0, c1, c2, c3], 1)
    return torch.stack([words & 0xFFFF, words >> 16], 2).view(-1)[:units]


def _factors(s):
    """What each value is multiplied by: 0, or one over the rate of those kept."""
    c, t = s["case"], s["threshold"]
    unit = 1 << c["dimension"]
    kept = _draws(c["rows"] * c["cols"] // unit, s["seed"], s["offset"]) >= t
    f = kept.to(_wide(s["x"]).dtype) * (65536.0 / (65536 - t))
    return f.repeat_interleave(unit).view(c["rows"], c["cols"]) if unit > 1 else f.view(c["rows"], c["cols"])


def _norm(x, s):
    mean = x.sum(1, keepdim=True) / x.shape[1]
    d = x - mean
    rstd = torch.rsqrt((d * d).sum(1, keepdim=True) / x.shape[1] + EPSILON)
    y = d * rstd * _wide(s["weight"]) + _wide(s["bias"])
    return y.to(s["x"].dtype), mean[:, 0], rstd[:, 0]


def _norm_vjp(s):
    x, dy = _wide(s["x"]), _wide(s["dy"])
    xh = (x - s["mean"][:, None]) * s["rstd"][:, None]
    g = dy * _wide(s["weight"])
    cols = x.shape[1]
    dx = s["rstd"][:, None] * (g - g.sum(1, keepdim=True) / cols - xh * ((g * xh).sum(1, keepdim=True) / cols))
    p = s["weight"].dtype
    return dx, (dy * xh).sum(0).to(p), dy.sum(0).to(p)


def _rotate(s, backward):
    c, x = s["case"], s["x"]
    p = s["positions"].double()[:, :, None]
    turns = p * s["high"]
    angle = ((turns - torch.round(turns)) + p * s["low"]) * (2 * math.pi)
    wide = _wide(x)
    cos = (torch.cos(angle) * _amplitude(c)).to(wide.dtype)[:, :, None]
    sin = (torch.sin(angle) * (-_amplitude(c) if backward else _amplitude(c))).to(wide.dtype)[:, :, None]
    r = c["rotary_dim"]
    turned, rest = wide[..., :r], x[..., r:]
    if c["layout"] == "half":
        a, b = turned[..., :r // 2], turned[..., r // 2:]
        out = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        out = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(-2)
    return torch.cat([out.to(x.dtype), rest], -1)


def run(state):
    if own:
        return _call(state)
    s, op = state, state["case"]["op"]
    if op == "norm":
        y, mean, rstd = _norm(_wide(s["x"]), s)
        return {"y": y, "mean": mean, "rstd": rstd}
    if op == "norm_vjp":
        dx, dw, db = _norm_vjp(s)
        return {"dx": dx.to(s["x"].dtype), "dweight": dw, "dbias": db}
    if op == "dropout":
        z = _wide(s["x"]) * _factors(s)
        return {"y": (z + _wide(s["residual"]) if "residual" in s else z).to(s["x"].dtype)}
    if op == "dropout_vjp":
        return {"dx": (_wide(s["dy"]) * _factors(s)).to(s["x"].dtype)}
    if op == "add_norm":
        z = _wide(s["residual"]) + _wide(s["x"]) * _factors(s)
        y, mean, rstd = _norm(z, s)
        return {"z": z.to(s["x"].dtype), "y": y, "mean": mean, "rstd": rstd}
    if op == "add_norm_vjp":
        dx, dw, db = _norm_vjp(s)
        dz = dx + _wide(s["dz"])
        return {"dresidual": dz.to(s["x"].dtype), "dx": (dz * _factors(s)).to(s["x"].dtype), "dweight": dw, "dbias": db}
    return {"y" if op == "rotary" else "dx": _rotate(s, op == "rotary_vjp")}


# ---- the library's entry points ---------------------------------------------


def _bind(case, s):
    """The configuration, output buffers and workspace that a program keeps from call to call."""
    import ctypes

    from geometricelementaryoperators_b200 import abi

    lib, op = abi.lib(), case["op"]
    kind = {"f64": abi.F64, "f32": abi.F32, "bf16": abi.BF16, "f16": abi.F16}
    ptr = lambda t: ctypes.c_void_p(t.data_ptr()) if t is not None else None  # noqa: E731
    if op.startswith("rotary"):
        scaling = {"none": abi.ROTARY_SCALING_NONE, "linear": abi.ROTARY_SCALING_LINEAR,
                   "base": abi.ROTARY_SCALING_BASE, "banded": abi.ROTARY_SCALING_BANDED}
        layout = {"half": abi.ROTARY_HALF, "interleaved": abi.ROTARY_INTERLEAVED}
        config = abi.RotaryConfig(layout=layout[case["layout"]], rotary_dim=case["rotary_dim"], base=_BASE,
                                  scaling=scaling[case["scaling"]], factor=_FACTOR, original_length=_ORIGINAL,
                                  low_rotations=_LOW, high_rotations=_HIGH, amplitude=_amplitude(case))
        plan = abi.RotaryPlan()
        assert lib.geo_b200_rotary_plan_init(ctypes.byref(plan), ctypes.byref(config)) == 0
        x = s["x"]
        y = torch.empty_strided(x.shape, x.stride(), dtype=x.dtype, device="cuda")
        shape = abi.RotaryShape(type=kind[case["type"]], position_type=abi.I64, batch=case["batch"],
                                tokens=case["tokens"], heads=case["heads"], head_dim=case["head_dim"],
                                x_batch_stride=x.stride(0), x_token_stride=x.stride(1), x_head_stride=x.stride(2),
                                y_batch_stride=x.stride(0), y_token_stride=x.stride(1), y_head_stride=x.stride(2),
                                position_batch_stride=s["positions"].stride(0))
        call = lib.geo_b200_rotary if op == "rotary" else lib.geo_b200_rotary_vjp
        args = (ctypes.byref(plan), ctypes.byref(shape), ptr(x), ptr(s["positions"]), ptr(y))
        return call, args, {"y" if op == "rotary" else "dx": y}, (plan, shape)
    stride = case["cols"] + 2 * case["pad"]
    rows, cols = case["rows"], case["cols"]
    keep = torch.float64 if case["type"] == "f64" else torch.float32
    drop = norm = None
    if "rate" in case:
        drop = abi.DropoutConfig(type=kind[case["type"]], dimension=case["dimension"], rows=rows, cols=cols,
                                 x_stride=stride, residual_stride=stride, y_stride=stride,
                                 y_cotangent_stride=stride, x_cotangent_stride=stride, rate=case["rate"],
                                 seed=s["seed"], offset=s["offset"])
    if "ptype" in case:
        norm = abi.LayerNormConfig(type=kind[case["type"]], parameter_type=kind[case["ptype"]], rows=rows, cols=cols,
                                   x_stride=stride, y_stride=stride, y_cotangent_stride=stride,
                                   x_cotangent_stride=stride, epsilon=EPSILON)
    new = lambda: _empty_like(case)  # noqa: E731
    ref = ctypes.byref
    if op in ("norm", "add_norm"):
        stats = torch.empty(2, rows, device="cuda", dtype=keep)
        out = {"y": new(), "mean": stats[0], "rstd": stats[1]}
        tail = (ptr(s["weight"]), ptr(s["bias"]))
        if op == "norm":
            return lib.geo_b200_layer_norm, (ref(norm), ptr(s["x"]), *tail, ptr(out["y"]), ptr(out["mean"]),
                                             ptr(out["rstd"])), out, (norm,)
        out = {"z": new(), **out}
        return lib.geo_b200_residual_dropout_layer_norm, (
            ref(norm), ref(drop), ptr(s["x"]), ptr(s["residual"]), None, *tail, ptr(out["z"]), ptr(out["y"]),
            ptr(out["mean"]), ptr(out["rstd"])), out, (norm, drop)
    if op in ("norm_vjp", "add_norm_vjp"):
        size = lib.geo_b200_layer_norm_vjp_workspace(ref(norm))
        space = torch.empty(max(1, size), device="cuda", dtype=torch.uint8)
        grads = {"dweight": torch.empty_like(s["weight"]), "dbias": torch.empty_like(s["bias"])}
        tail = (ptr(grads["dweight"]), ptr(grads["dbias"]), ptr(space), size)
        if op == "norm_vjp":
            out = {"dx": new(), **grads}
            return lib.geo_b200_layer_norm_vjp, (ref(norm), ptr(s["x"]), ptr(s["weight"]), ptr(s["mean"]),
                                                 ptr(s["rstd"]), ptr(s["dy"]), ptr(out["dx"]), *tail), out, (norm, space)
        out = {"dresidual": new(), "dx": new(), **grads}
        return lib.geo_b200_residual_dropout_layer_norm_vjp, (
            ref(norm), ref(drop), None, ptr(s["x"]), ptr(s["weight"]), ptr(s["mean"]), ptr(s["rstd"]), ptr(s["dy"]),
            ptr(s["dz"]), ptr(out["dresidual"]), ptr(out["dx"]), *tail), out, (norm, drop, space)
    if op == "dropout":
        out = {"y": new()}
        return lib.geo_b200_dropout, (ref(drop), ptr(s["x"]), ptr(s.get("residual")), None, ptr(out["y"])), out, (drop,)
    out = {"dx": new()}
    return lib.geo_b200_dropout_vjp, (ref(drop), None, ptr(s["dy"]), ptr(out["dx"])), out, (drop,)


def _call(s):
    call, args, out, _ = s["call"]
    status = call(*args, torch.cuda.current_stream().cuda_stream)
    if status:
        raise RuntimeError("status %d" % status)
    return out


# ---- 64-bit definitions -----------------------------------------------------


def _exact_kept(case, s):
    """The kept units, by 64-bit unsigned arithmetic on the host."""
    units = case["rows"] * case["cols"] >> case["dimension"]
    m = np.uint64(0xFFFFFFFF)
    sh = np.uint64(32)
    b = np.arange((units + 7) // 8, dtype=np.uint64)
    x = [b & m, b >> sh, np.full_like(b, s["offset"] & 0xFFFFFFFF), np.full_like(b, s["offset"] >> 32)]
    key = [s["seed"] & 0xFFFFFFFF, s["seed"] >> 32]
    for r in range(10):
        k = [np.uint64((key[0] + r * 0x9E3779B9) % (1 << 32)), np.uint64((key[1] + r * 0xBB67AE85) % (1 << 32))]
        first, second = x[0] * np.uint64(0xD2511F53), x[2] * np.uint64(0xCD9E8D57)
        x = [(second >> sh) ^ x[1] ^ k[0], second & m, (first >> sh) ^ x[3] ^ k[1], first & m]
    draws = np.empty((len(b), 8), np.uint16)
    for w in range(4):
        draws[:, 2 * w], draws[:, 2 * w + 1] = x[w] & np.uint64(0xFFFF), x[w] >> np.uint64(16)
    kept = torch.from_numpy(draws.reshape(-1)[:units].astype(np.int32) >= s["threshold"]).cuda()
    return kept[:, None].expand(units, 1 << case["dimension"]).reshape(case["rows"], case["cols"])


def exact(case, seed):
    s = prepare(case, seed)
    op = case["op"]
    x = s["x"].double()
    if op.startswith("rotary"):
        p = s["positions"].cpu().numpy().astype(np.longdouble)[..., None]
        turns = p * _turns(case)[2]
        turns -= np.rint(turns)
        theta = torch.tensor((turns * (8 * np.arctan(np.longdouble(1)))).astype(np.float64), device="cuda")
        rotor = torch.polar(torch.full_like(theta, _amplitude(case)), theta if op == "rotary" else -theta)[:, :, None]
        r = case["rotary_dim"]
        if case["layout"] == "half":
            z = torch.complex(x[..., :r // 2].contiguous(), x[..., r // 2:r].contiguous()) * rotor
            x = torch.cat([z.real, z.imag, x[..., r:]], -1)
        else:
            z = torch.view_as_complex(x[..., :r].reshape(*x.shape[:-1], r // 2, 2).contiguous()) * rotor
            x = torch.cat([torch.view_as_real(z).flatten(-2), x[..., r:]], -1)
        return {"y" if op == "rotary" else "dx": x}
    gain = 65536.0 / (65536 - s["threshold"]) if "rate" in case else 1.0
    drop = lambda v: torch.where(_exact_kept(case, s), v * gain, torch.zeros_like(v))  # noqa: E731
    if op == "dropout":
        z = drop(x)
        return {"y": z + s["residual"].double() if "residual" in s else z}
    if op == "dropout_vjp":
        return {"dx": drop(s["dy"].double())}
    w = s["weight"].double()
    if op in ("norm", "add_norm"):
        z = s["residual"].double() + drop(x) if op == "add_norm" else x
        var, mean = torch.var_mean(z, 1, correction=0)
        y = torch.addcmul(s["bias"].double(), (z - mean[:, None]) / torch.sqrt(var + EPSILON)[:, None], w)
        out = {"y": y, "mean": mean, "rstd": 1 / torch.sqrt(var + EPSILON)}
        return {"z": z, **out} if op == "add_norm" else out
    dy, r = s["dy"].double(), s["rstd"].double()
    xh = x.sub_(s["mean"].double()[:, None]).mul_(r[:, None])
    dw, db = torch.einsum("rc,rc->c", dy, xh), dy.mean(0) * case["rows"]
    dy *= w
    along = torch.einsum("rc,rc->r", dy, xh) / case["cols"]
    dx = (dy - dy.mean(1, keepdim=True) - xh * along[:, None]) * r[:, None]
    if op == "norm_vjp":
        return {"dx": dx, "dweight": dw, "dbias": db}
    dx += s["dz"].double()
    return {"dresidual": dx, "dx": drop(dx), "dweight": dw, "dbias": db}
