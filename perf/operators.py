"""The operators of a block whose linears run in 8-bit floating point, as cases to measure.

A denoising block with e4m3 linears goes round: gated residual and norms -> quantised activations -> matrix product
with a scale for each block of 128 -> rotary positions on q and k -> attention -> the next product.  This file holds
the four operators of that round that are not attention: `quantize`, `block_norm`, `linear` and `rope`, each in its
plain form (elementary torch operations in 32 bits, in 64 where 32 lose what matters) and, where `own` is true, as the
calls of this repository's library.  Formulas:

quantize    blocks of 1 x 128 (activations) or 128 x 128 (weights): a = max |x| of the block's finite values, at least
            2^-100;  scale = a / 448,  q = e4m3(x * (448 / a));  q is NaN where x is not finite
linear      y[m, n] = sum_k xq[m, k] xs[m, k / 128] wq[n, k] ws[n / 128, k / 128], then bias, activation, and either
            a cast, residual + gate * y, or quantize() of the row for the product that follows
block_norm  t = post(x);  y = residual_scale * residual + gate * t;  z = pre(y) * (1 + scale) + shift, cast or quantized
rope        pair p of a head turns by position[axis(p)] * frequency(p), times the scaling's attention factor
"""
import importlib.util
import math
import os
import sys

import torch

own = False

F8 = torch.float8_e4m3fn
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16, "float8": F8}
FLOOR = 2.0 ** -100
EPS = 1e-6


def _edb():
    """The ctypes binding of the library (its directory's name is no Python identifier, so it is loaded by path)."""
    key = "edb200_pkg_edb200"
    if key not in sys.modules:
        root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
        spec = importlib.util.spec_from_file_location(key, os.path.join(root, "edge-dit.cpp_b200", "edb200.py"))
        mod = importlib.util.module_from_spec(spec)
        sys.modules[key] = mod
        spec.loader.exec_module(mod)
    return sys.modules[key]


# ------------------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # text-encoder rows on their way into a projection: a short call where the launch counts
        {"name": "quantize_text", "op": "quantize", "rows": 333, "k": 4096, "block_rows": 1, "dtype": "float16"},
        # an attention output of a whole video (21 x 30 x 52 tokens) before its out-projection
        {"name": "quantize_video", "op": "quantize", "rows": 32760, "k": 5120, "block_rows": 1, "dtype": "bfloat16"},
        # a feed-forward weight quantised while a checkpoint is loaded
        {"name": "quantize_weight", "op": "quantize", "rows": 13824, "k": 5120, "block_rows": 128, "dtype": "float32"},
        # one vector through a layer's norm: the smallest call
        {"name": "norm_one_row", "op": "block_norm", "rows": 1, "h": 5120, "post": "none", "pre": "layer", "x": "float16", "z": "float16", "rows_per_mod": 0},
        # context rows of a joint block, both passes of a guided step batched: a modulation vector for each 77 rows
        {"name": "norm_context", "op": "block_norm", "rows": 154, "h": 1536, "post": "none", "pre": "layer", "x": "bfloat16", "z": "float8", "rows_per_mod": 77},
        # a video's tokens between attention and feed-forward, normed on both sides, quantised for the next product
        {"name": "norm_video", "op": "block_norm", "rows": 32760, "h": 5120, "post": "rms", "pre": "rms", "x": "bfloat16", "z": "float8", "rows_per_mod": 0},
        # the conditional and unconditional timestep vectors through a modulation projection: weight streaming
        {"name": "linear_two_rows", "op": "linear", "m": 2, "k": 5120, "n": 30720, "act": "none", "bias": True, "out": "float32"},
        # context rows of a joint block through the first half of their feed-forward, handed on quantised
        {"name": "linear_context", "op": "linear", "m": 154, "k": 1536, "n": 6144, "act": "gelu_tanh", "bias": True, "out": "float8"},
        # an odd number of image tokens (83 x 83) into fused q, k, v
        {"name": "linear_qkv", "op": "linear", "m": 6889, "k": 3584, "n": 10752, "act": "none", "bias": True, "out": "float16"},
        # a video's tokens through the second half of their feed-forward, into the residual stream: the largest
        {"name": "linear_video", "op": "linear", "m": 32760, "k": 13824, "n": 5120, "act": "none", "bias": True, "out": "gated"},
        # a joint block's q and k at small size, one position axis, neighbouring channels
        {"name": "rope_context", "op": "rope", "tokens": 154, "q_heads": 24, "k_heads": 24, "d_head": 64, "axes": "64", "layout": "interleaved", "scaling": "none", "factor": 1.0, "dtype": "float16", "inverse": False},
        # a video's q and k over (t, h, w), stretched to a length beyond the trained one, channels in halves
        {"name": "rope_video", "op": "rope", "tokens": 32760, "q_heads": 40, "k_heads": 40, "d_head": 128, "axes": "44,42,42", "layout": "half", "scaling": "yarn", "factor": 4.0, "dtype": "bfloat16", "inverse": False},
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(("quantize", "block_norm", "linear", "linear", "rope"))
    if op == "quantize":
        br = rng.choice((1, 1, 128))
        k = _log(rng, 100, 16384)
        return {"op": op, "rows": _log(rng, 1, min(40000, 160_000_000 // k)), "k": k, "block_rows": br,
                "dtype": rng.choice(("float16", "bfloat16", "float32"))}
    if op == "block_norm":
        h = rng.choice((rng.randrange(40, 8200), 128 * rng.randrange(1, 64)))
        rows = _log(rng, 1, min(40000, 160_000_000 // h))
        return {"op": op, "rows": rows, "h": h, "post": rng.choice(("none", "rms", "layer")),
                "pre": rng.choice(("rms", "layer")), "x": rng.choice(("float16", "bfloat16", "float32")),
                "z": rng.choice(("float16", "bfloat16", "float32", "float8")),
                "rows_per_mod": rng.choice((0, 1, _log(rng, 1, 5000)))}
    if op == "linear":
        k, n = _log(rng, 64, 14000), _log(rng, 64, 14000)
        m = _log(rng, 1, max(2, min(40000, int(1.2e12 / (k * n)))))
        return {"op": op, "m": m, "k": k, "n": n, "act": rng.choice(("none", "gelu_tanh", "silu", "gelu_erf")),
                "bias": rng.random() < 0.7, "out": rng.choice(("float16", "bfloat16", "float32", "gated", "float8"))}
    d = rng.choice((64, 80, 128, 256))
    axes = rng.choice({64: ("64", "16,24,24", "32"), 80: ("80", "40"), 128: ("128", "44,42,42", "16,56,56", "64"),
                       256: ("256", "64")}[d])
    q = rng.choice((1, 8, 24, 40))
    return {"op": op, "tokens": _log(rng, 1, min(40000, 160_000_000 // (2 * q * d))), "q_heads": q,
            "k_heads": rng.choice((1, q)), "d_head": d, "axes": axes, "layout": rng.choice(("interleaved", "half")),
            "scaling": rng.choice(("none", "linear", "ntk", "yarn")), "factor": rng.choice((1.5, 2.0, 4.0, 8.0)),
            "dtype": rng.choice(("float16", "bfloat16", "float32")), "inverse": rng.random() < 0.3}


# ------------------------------------------------------------------------------------------------ what is in hand
def _up(a, b):
    return -(-a // b) * b


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)


def _rows(rows, cols, dtype):
    """[rows, cols] whose rows start on 16-byte boundaries, as an allocator of activations lays them."""
    return torch.empty(rows, _up(cols, 16), device="cuda", dtype=dtype)[:, :cols]


def _activations(g, rows, k):
    """Rows as a norm leaves them: unit size, a few channels far larger, rows of different strength."""
    x = _normal(g, rows, k)
    x *= torch.exp(0.5 * _normal(g, k)) * torch.where(torch.rand(k, generator=g, device="cuda") < 0.01, 20.0, 1.0)
    return x.mul_(torch.exp(0.3 * _normal(g, rows, 1)))


def _stored(x, dtype):
    out = _rows(x.shape[0], x.shape[1], dtype)
    out.copy_(x)
    return out


def _quantized(x, block_rows):
    q, scale = _quantize(x, block_rows, torch.float32)
    return _stored(q.float(), F8), scale


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    s = dict(case)
    if case["op"] == "quantize":
        rows, k = case["rows"], case["k"]
        x = _activations(g, rows, k) if case["block_rows"] == 1 else 0.02 * _normal(g, rows, k)
        s["x"] = _stored(x, TYPES[case["dtype"]])
        s["q"] = _rows(rows, k, F8)
        s["scale"] = torch.empty(-(-rows // case["block_rows"]), -(-k // 128), device="cuda")
    elif case["op"] == "block_norm":
        rows, h = case["rows"], case["h"]
        n_mod = -(-rows // case["rows_per_mod"]) if case["rows_per_mod"] else 1
        s["x_in"] = _stored(0.5 * _activations(g, rows, h), TYPES[case["x"]])
        s["residual"] = _stored(4.0 * _activations(g, rows, h), torch.float32)
        s["gate"] = 0.3 * _normal(g, n_mod, h)
        s["mod_scale"] = 0.2 * _normal(g, n_mod, h)
        s["mod_shift"] = 0.2 * _normal(g, n_mod, h)
        s["post_weight"] = 1.0 + 0.1 * _normal(g, h)
        s["pre_weight"] = 1.0 + 0.1 * _normal(g, h)
        s["residual_scale"] = 0.9
        s["y"] = _rows(rows, h, torch.float32)
        s["z_out"] = _rows(rows, h, TYPES[case["z"]])
        s["z_scale"] = torch.empty(rows, -(-h // 128), device="cuda") if case["z"] == "float8" else None
    elif case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        s["xq"], s["xs"] = _quantized(_activations(g, m, k), 1)
        s["wq"], s["ws"] = _quantized(0.02 * _normal(g, n, k), 128)
        s["b"] = 0.1 * _normal(g, n) if case["bias"] else None
        gated = case["out"] == "gated"
        s["residual"] = _stored(4.0 * _normal(g, m, n), torch.float32) if gated else None
        s["gate"] = 0.3 * _normal(g, n) if gated else None
        s["y"] = _rows(m, n, torch.float32 if gated else TYPES[case["out"]])
        s["y_scale"] = torch.empty(m, -(-n // 128), device="cuda") if case["out"] == "float8" else None
    else:
        t, d = case["tokens"], case["d_head"]
        axes = case["axes"].count(",") + 1
        # q and k lie beside one another in a projection's output
        both = _normal(g, t, (case["q_heads"] + case["k_heads"]) * d).to(TYPES[case["dtype"]])
        s["q"] = both[:, :case["q_heads"] * d].view(t, case["q_heads"], d)
        s["k"] = both[:, case["q_heads"] * d:].view(t, case["k_heads"], d)
        at = torch.arange(t, device="cuda")
        start = int(torch.randint(0, 1 << 20, (1,), generator=g, device="cuda"))   # far into a long sequence
        grid = torch.stack((at + start, at // 52 - 15, at % 52 - 26), 1)           # centred rows and columns
        s["positions"] = grid[:, :axes].to(torch.int32).contiguous()
        s["q_out"] = torch.empty(t, case["q_heads"], d, device="cuda", dtype=TYPES[case["dtype"]])
        s["k_out"] = torch.empty(t, case["k_heads"], d, device="cuda", dtype=TYPES[case["dtype"]])
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _quantize(x, block_rows, dtype):
    rows, k = x.shape
    r, c = _up(rows, block_rows), _up(k, 128)
    b = torch.nn.functional.pad(x.to(dtype), (0, c - k, 0, r - rows)).view(r // block_rows, block_rows, c // 128, 128)
    fine = torch.isfinite(b)
    a = torch.where(fine, b.abs(), 0.0).amax((1, 3)).clamp_min(FLOOR)
    top = torch.full_like(a, 448.0)
    q = torch.where(fine, b * (top / a)[:, None, :, None], float("nan"))
    return q.view(r, c)[:rows, :k].to(F8), (a / top).float()


def _wide(scale, block_rows, rows, k, dtype):
    s = scale.to(dtype).repeat_interleave(128, 1)[:, :k]
    return s.repeat_interleave(block_rows, 0)[:rows] if block_rows > 1 else s


def _activation(v, act):
    if act == "gelu_tanh":
        return 0.5 * v * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (v + 0.044715 * v * v * v)))
    if act == "gelu_erf":
        return 0.5 * v * (1.0 + torch.erf(v * math.sqrt(0.5)))
    return v / (1.0 + torch.exp(-v)) if act == "silu" else v


def _norm(v, kind, weight):
    if kind == "none":
        return v
    if kind == "layer":
        v = v - v.mean(1, keepdim=True)
    return v / torch.sqrt((v * v).mean(1, keepdim=True) + EPS) * weight


def _per_row(v, s):
    if v.shape[0] == 1:
        return v
    return v.repeat_interleave(s["rows_per_mod"], 0)[:s["rows"]]


def _frequencies(axes, scaling, factor):
    """(axis, angle of one step, share) of each pair, and what multiplies the rotated channels."""
    theta, original = 10000.0, 2048.0
    rows = []
    for axis, dim in enumerate(axes):
        base = theta * factor ** (dim / (dim - 2)) if scaling == "ntk" and dim > 2 else theta
        low = max(math.floor(dim * math.log(original / (32.0 * 2 * math.pi)) / (2 * math.log(theta))), 0)
        high = min(math.ceil(dim * math.log(original / (1.0 * 2 * math.pi)) / (2 * math.log(theta))), dim - 1)
        for j in range(dim // 2):
            f = base ** (-2.0 * j / dim)
            if scaling == "linear":
                f /= factor
            if scaling == "yarn":
                ramp = min(max((j - low) / max(high - low, 1e-3), 0.0), 1.0)
                f = f / factor * ramp + f * (1.0 - ramp)
            rows.append((axis, f))
    return rows, 0.1 * math.log(factor) + 1.0 if scaling == "yarn" else 1.0


def _rope(x, s, dtype):
    axes = [int(a) for a in s["axes"].split(",")]
    pairs, mul = _frequencies(axes, s["scaling"], s["factor"])
    half = len(pairs)
    axis = torch.tensor([a for a, _ in pairs], device=x.device)
    step = torch.tensor([f for _, f in pairs], device=x.device, dtype=torch.float64)
    angle = s["positions"].double()[:, axis] * step
    if s["inverse"]:
        angle = -angle
    c, n = (torch.cos(angle) * mul).to(dtype)[:, None], (torch.sin(angle) * mul).to(dtype)[:, None]
    v = x.to(dtype)
    turned = v[..., :2 * half]
    if s["layout"] == "half":
        a, b = turned[..., :half], turned[..., half:]
        y = torch.cat((a * c - b * n, a * n + b * c), -1)
    else:
        a, b = turned[..., 0::2], turned[..., 1::2]
        y = torch.stack((a * c - b * n, a * n + b * c), -1).flatten(-2)
    return torch.cat((y, v[..., 2 * half:]), -1)


def _plain(s):
    if s["op"] == "quantize":
        q, scale = _quantize(s["x"], s["block_rows"], torch.float32)
        return {"q": q, "scale": scale}
    if s["op"] == "block_norm":
        t = _norm(s["x_in"].float(), s["post"], s["post_weight"])
        y = s["residual_scale"] * s["residual"] + _per_row(s["gate"], s) * t
        z = _norm(y, s["pre"], s["pre_weight"]) * (1.0 + _per_row(s["mod_scale"], s)) + _per_row(s["mod_shift"], s)
        if s["z"] == "float8":
            q, scale = _quantize(z, 1, torch.float32)
            return {"y": y, "z": q, "z_scale": scale}
        return {"y": y, "z": z.to(TYPES[s["z"]])}
    if s["op"] == "linear":
        m, k, n = s["m"], s["k"], s["n"]
        x = s["xq"].float() * _wide(s["xs"], 1, m, k, torch.float32)
        w = s["wq"].float() * _wide(s["ws"], 128, n, k, torch.float32)
        y = x @ w.t()
        if s["b"] is not None:
            y = y + s["b"]
        y = _activation(y, s["act"])
        if s["out"] == "gated":
            return {"y": s["residual"] + s["gate"] * y}
        if s["out"] == "float8":
            q, scale = _quantize(y, 1, torch.float32)
            return {"y": q, "y_scale": scale}
        return {"y": y.to(TYPES[s["out"]])}
    return {"q": _rope(s["q"], s, torch.float32).to(s["q"].dtype), "k": _rope(s["k"], s, torch.float32).to(s["k"].dtype)}


# ------------------------------------------------------------------------------------------- the library's calls
def _own(s):
    edb = _edb()
    if s["op"] == "quantize":
        edb.quantize_fp8(s["x"], s["q"], s["scale"], block_rows=s["block_rows"])
        return {"q": s["q"], "scale": s["scale"]}
    if s["op"] == "block_norm":
        kinds = {"none": edb.NORM_NONE, "rms": edb.NORM_RMS, "layer": edb.NORM_LAYER}
        edb.block_norm(s["residual"], s["y"], s["z_out"], s["z_scale"], x=s["x_in"], gate=s["gate"],
                       residual_scale=s["residual_scale"], post_norm=kinds[s["post"]],
                       post_weight=s["post_weight"] if s["post"] != "none" else None, post_eps=EPS,
                       pre_norm=kinds[s["pre"]], pre_weight=s["pre_weight"], pre_eps=EPS, scale=s["mod_scale"],
                       shift=s["mod_shift"], rows_per_mod=s["rows_per_mod"])
        out = {"y": s["y"], "z": s["z_out"]}
        return {**out, "z_scale": s["z_scale"]} if s["z"] == "float8" else out
    if s["op"] == "linear":
        if "weight" not in s:   # kept with the weights, as a program keeps a layer
            acts = {"none": edb.ACT_NONE, "gelu_tanh": edb.ACT_GELU_TANH, "silu": edb.ACT_SILU, "gelu_erf": edb.ACT_GELU_ERF}
            s["weight"] = edb.Fp8Weight(s["wq"], s["ws"])
            s["epilogue"] = edb.make_epilogue(s["y"], bias=s["b"], act=acts[s["act"]], residual=s["residual"], gate=s["gate"])
        edb.mul_mat_fp8(s["weight"], s["xq"], s["xs"], s["epilogue"], s["y_scale"])
        return {"y": s["y"], "y_scale": s["y_scale"]} if s["out"] == "float8" else {"y": s["y"]}
    if "plan" not in s:         # kept with the model, as its table of positions is
        s["plan"] = edb.Rope([int(a) for a in s["axes"].split(",")], theta=10000.0,
                             layout=edb.ROPE_HALF if s["layout"] == "half" else edb.ROPE_INTERLEAVED,
                             scaling={"none": edb.ROPE_SCALE_NONE, "linear": edb.ROPE_SCALE_LINEAR, "ntk": edb.ROPE_SCALE_NTK, "yarn": edb.ROPE_SCALE_YARN}[s["scaling"]],
                             factor=s["factor"], original_length=2048)
    s["plan"].apply(s["positions"], s["q"], s["q_out"], s["k"], s["k_out"], inverse=s["inverse"])
    return {"q": s["q_out"], "k": s["k_out"]}


def run(s):
    return _own(s) if own else _plain(s)


# -------------------------------------------------------------------------------------------- what it cannot do without
def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2, "float8": 1}
    if case["op"] == "quantize":
        n = case["rows"] * case["k"]
        return {"bytes": n * (size[case["dtype"]] + 1) + 4 * -(-case["rows"] // case["block_rows"]) * -(-case["k"] // 128), "flops": 3 * n}
    if case["op"] == "block_norm":
        n = case["rows"] * case["h"]
        n_mod = -(-case["rows"] // case["rows_per_mod"]) if case["rows_per_mod"] else 1
        return {"bytes": n * (size[case["x"]] + 8 + size[case["z"]]) + 12 * n_mod * case["h"], "flops": 15 * n}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        out = {"gated": 8}.get(case["out"]) or size[case["out"]]
        return {"bytes": m * k + n * k + m * n * out, "flops": 2 * m * n * k}
    n = case["tokens"] * (case["q_heads"] + case["k_heads"]) * case["d_head"]
    return {"bytes": 2 * n * size[case["dtype"]] + 4 * case["tokens"] * (case["axes"].count(",") + 1), "flops": 3 * n}


# ------------------------------------------------------------------------------ from the definitions, in 64 bits
def _exact_quantize(v, block_rows):
    rows, k = v.shape
    padded = v.new_zeros(_up(rows, block_rows), _up(k, 128))
    padded[:rows, :k] = v
    tiles = padded.unflatten(1, (-1, 128)).unflatten(0, (-1, block_rows))     # [R, block_rows, K, 128]
    scale = tiles.abs().flatten(1, 1).amax(dim=(1, 3)).clamp(min=FLOOR) / 448.0
    q = padded / scale.repeat_interleave(128, 1).repeat_interleave(block_rows, 0)
    return q[:rows, :k].to(F8).double(), scale


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "quantize":
        q, scale = _exact_quantize(s["x"].double(), case["block_rows"])
        return {"q": q, "scale": scale}
    if case["op"] == "block_norm":
        def normed(v, kind, w):
            mean = v.mean(-1, keepdim=True) if kind == "layer" else 0.0
            var = torch.square(v - mean).sum(-1, keepdim=True) / case["h"]
            return v if kind == "none" else (v - mean) * w.double() * (var + EPS) ** -0.5

        which = torch.arange(case["rows"], device="cuda") // case["rows_per_mod"] if case["rows_per_mod"] else torch.zeros(case["rows"], dtype=torch.int64, device="cuda")
        y = normed(s["x_in"].double(), case["post"], s["post_weight"]) * s["gate"].double()[which]
        y += s["residual"].double() * s["residual_scale"]
        z = normed(y, case["pre"], s["pre_weight"])
        z = z + z * s["mod_scale"].double()[which] + s["mod_shift"].double()[which]
        if case["z"] == "float8":
            q, scale = _exact_quantize(z, 1)
            return {"y": y, "z": q, "z_scale": scale}
        return {"y": y, "z": z}
    if case["op"] == "linear":
        m, k, n = case["m"], case["k"], case["n"]
        kb = -(-k // 128)
        y = torch.zeros(m, n, device="cuda", dtype=torch.float64)
        for first in range(0, n, 128):         # one row of weight blocks at a time
            block = slice(first, min(first + 128, n))
            w = torch.zeros(block.stop - first, kb * 128, device="cuda", dtype=torch.float64)
            w[:, :k] = s["wq"][block].double()
            w = (w.view(-1, kb, 128) * s["ws"][first // 128].double()[:, None]).flatten(1)[:, :k]
            if first == 0:
                x = torch.zeros(m, kb * 128, device="cuda", dtype=torch.float64)
                x[:, :k] = s["xq"].double()
                x = (x.view(m, kb, 128) * s["xs"].double()[..., None]).flatten(1)[:, :k]
            y[:, block] = torch.matmul(x, w.t())
        if s["b"] is not None:
            y += s["b"].double()
        if case["act"] == "silu":
            y = y * torch.sigmoid(y)
        elif case["act"] == "gelu_erf":
            y = y * 0.5 * torch.erfc(-y / math.sqrt(2.0))
        elif case["act"] == "gelu_tanh":
            y = y * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (y + 0.044715 * y ** 3))
        if case["out"] == "gated":
            return {"y": s["residual"].double() + s["gate"].double() * y}
        if case["out"] == "float8":
            q, scale = _exact_quantize(y, 1)
            return {"y": q, "y_scale": scale}
        return {"y": y}
    # a pair of channels is a complex number and turning it is a product with e^(i angle)
    pairs, mul = _frequencies([int(a) for a in case["axes"].split(",")], case["scaling"], case["factor"])
    out = {}
    for name in ("q", "k"):
        v, half = s[name].double(), len(pairs)
        first = torch.arange(half, device="cuda") * (1 if case["layout"] == "half" else 2)
        second = first + (half if case["layout"] == "half" else 1)
        turned = v.clone()
        for p, (axis, f) in enumerate(pairs):
            angle = s["positions"][:, axis].double() * (-f if case["inverse"] else f)
            z = torch.complex(v[..., first[p]], v[..., second[p]]) * torch.polar(torch.full_like(angle, mul), angle)[:, None]
            turned[..., first[p]], turned[..., second[p]] = z.real, z.imag
        out[name] = turned
    return out
