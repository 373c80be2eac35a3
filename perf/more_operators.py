"""The operators of microscaled 4-bit floating point and of the norms around a block whose speed is tracked: rows
quantized to 4 bits, products of two such operands with bias, activation and residual (dense and by expert), and the
norms before and after a block with its gate and residual scale, forward and backward.

With ``own`` false ``run`` computes them in elementary torch operations in fp32, rounded once at the end; with ``own``
true it makes the calls of the framework.  Sizes are those of the two layer geometries of
``raon-npu_amd/geometry.py`` (H=2048, I=768, top-8 and H=2560, I=1088, top-6, 128 experts each), of the dense
matrices of a weights-d directory (gate/up [24064, 2560], head [260096, 2560]) and of the prompts of ``bench.py`` (445
and 6,700 tokens); ``draw`` spreads over the ranges around them, odd widths and other types included.

A block of 32 values shares a power of two 2^s, s = floor(log2(largest magnitude)) - 2; a value is held as one of 0,
0.5, 1, 1.5, 2, 3, 4, 6 times that with its sign.  Codes are two to a byte, the even column in the low half; a scale is
the byte s + 127.
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------ the cases --
def listed():
    return [
        # The hidden row of one generated token, to 4 bits and to the values these stand for: the smallest call.
        {"name": "quantize_token", "kind": "quantize", "T": 1, "K": 2048, "dtype": "bf16"},
        # A checkpoint's fp32 dense gate/up when it is loaded.
        {"name": "quantize_weights", "kind": "quantize", "T": 24064, "K": 2560, "dtype": "fp32"},
        # One generated token: its hidden row normalised, quantized and through the shared expert's gate/up.
        {"name": "linear_token", "kind": "linear", "T": 1, "M": 1536, "K": 2048, "act": "swiglu", "bias": False,
         "residual": False, "norm": True},
        # The head over four requests' tokens: 354 MB of weights.
        {"name": "linear_head_4", "kind": "linear", "T": 4, "M": 260096, "K": 2560, "act": "none", "bias": False,
         "residual": False, "norm": True},
        # A middling prompt through a down projection of odd depth (8.5 times 128) onto the residual stream.
        {"name": "linear_down_445", "kind": "linear", "T": 445, "M": 2560, "K": 1088, "act": "none", "bias": True,
         "residual": True, "norm": False},
        # A long prompt through the dense gate/up: the largest product.
        {"name": "linear_6700", "kind": "linear", "T": 6700, "M": 24064, "K": 2560, "act": "swiglu", "bias": False,
         "residual": False, "norm": True},
        # A decode step of four requests: the 32 rows of their experts through gate/up.
        {"name": "experts_decode_4", "kind": "experts", "T": 4, "k": 8, "E": 128, "M": 1536, "K": 2048,
         "act": "swiglu", "bias": False, "residual": False},
        # A long prompt's sorted rows through the gate/up of 128 experts.
        {"name": "experts_6700", "kind": "experts", "T": 6700, "k": 8, "E": 128, "M": 1536, "K": 2048,
         "act": "swiglu", "bias": False, "residual": False},
        # Between two blocks of one generated token: the norms after and before.
        {"name": "norm_token", "kind": "norm", "T": 1, "H": 2048, "dtype": "bf16", "post": True, "gate": "none",
         "scale": 1.0},
        # Between two blocks of a long prompt, the block's result gated by channel.
        {"name": "norm_6700", "kind": "norm", "T": 6700, "H": 2560, "dtype": "bf16", "post": True, "gate": "column",
         "scale": 0.5},
        # Training on a short prompt in fp32, a gate by row.
        {"name": "norm_backward_445", "kind": "norm_backward", "T": 445, "H": 2560, "dtype": "fp32", "post": True,
         "gate": "row", "scale": 1.0},
        # A training batch of odd length: gradients of both norms' weights and of the gate by channel.
        {"name": "norm_backward_4099", "kind": "norm_backward", "T": 4099, "H": 2048, "dtype": "bf16", "post": True,
         "gate": "column", "scale": 0.5},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["quantize", "linear", "linear", "experts", "norm", "norm_backward"])
    if kind == "quantize":
        K = rng.choice([2048, 2560, _log_int(rng, 1, 8192)])
        return {"kind": kind, "T": min(_log_int(rng, 1, 24064), 24064 * 2560 // K), "K": K,
                "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"])}
    act = rng.choice(["none", "silu", "gelu", "gelu_tanh", "swiglu"])
    if kind == "linear":
        T, K = _log_int(rng, 1, 6700), 32 * rng.randint(2, 128)
        M = min(_log_int(rng, 32, 24064), 6700 * 24064 * 2560 // (T * K))
        return {"kind": kind, "T": T, "M": M - M % 2 if act == "swiglu" else M, "K": K, "act": act,
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5, "norm": rng.random() < 0.5}
    if kind == "experts":
        E = _log_int(rng, 4, 128)
        M = rng.choice([1536, 2048, 2560, rng.randint(32, 2600)])
        return {"kind": kind, "T": _log_int(rng, 1, 4000), "k": rng.randint(1, min(8, E)), "E": E,
                "M": M - M % 2 if act == "swiglu" else M, "K": 32 * rng.randint(4, 80), "act": act,
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    H = rng.choice([2048, 2560, _log_int(rng, 8, 8192)])
    return {"kind": kind, "T": min(_log_int(rng, 1, 8192), 6700 * 2560 // H), "H": H,
            "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "post": rng.random() < 0.7,
            "gate": rng.choice(["none", "column", "row", "full"]), "scale": rng.choice([1.0, 0.5])}


# ------------------------------------------------------------ seeded values --
def _gen(seed, part):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + 7919 * part + 1) & 0x7FFFFFFFFFFF)


def _normal(shape, std, seed, part, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=_gen(seed, part)).mul_(std).to(dtype)


def _hidden(T, H, seed, part, dtype=torch.bfloat16):
    """Rows of a residual stream: normal values, one channel in 64 twenty times as large."""
    big = torch.rand(H, device="cuda", generator=_gen(seed, part + 50)) < 1 / 64
    x = torch.randn(T, H, device="cuda", generator=_gen(seed, part))
    return x.mul_(torch.where(big, 20.0, 1.0)).to(dtype)


def _weights(shape, seed, part):
    """(codes, scales) of a matrix as a checkpoint holds it: every code, scales of 2^-9 to 2^-7."""
    g = _gen(seed, part)
    lead, K = shape[:-1], shape[-1]
    codes = torch.randint(0, 256, (*lead, K // 2), device="cuda", generator=g, dtype=torch.uint8)
    scales = torch.randint(118, 121, (*lead, K // 32), device="cuda", generator=g, dtype=torch.uint8)
    return codes, scales


def _out_width(case):
    return case["M"] // 2 if case["act"] == "swiglu" else case["M"]


def _n_rows(case):
    return case["T"] * case["k"] if case["kind"] == "experts" else case["T"]


def _gate(case, seed):
    T, H, kind = case["T"], case["H"], case["gate"]
    if kind == "none":
        return None
    if kind == "full":
        return _normal((T, H), 0.5, seed, 15, _DT[case["dtype"]])
    return _normal((T, 1) if kind == "row" else (H,), 0.5, seed, 15, torch.float32)


def prepare(case, seed):
    """Inputs, weights and the buffers that a program keeps for the outputs; the same for both sides."""
    st, kind, cuda = {"case": case}, case["kind"], {"device": "cuda"}
    st["levels"] = torch.tensor(_LEVELS, **cuda)  # what a code stands for, and a byte's two codes
    signed = torch.cat([st["levels"], -st["levels"]])
    st["pairs"] = torch.stack([signed.repeat(16), signed.repeat_interleave(16)], 1)
    if kind == "quantize":
        T, K, dt = case["T"], case["K"], _DT[case["dtype"]]
        groups = -(-K // 32)
        st["x"] = _hidden(T, K, seed, 1, dt) if dt != torch.float32 else _normal((T, K), 0.02, seed, 1, dt)
        st["codes"] = torch.zeros(T, groups * 16, dtype=torch.uint8, **cuda)
        st["scales"] = torch.zeros(T, groups, dtype=torch.uint8, **cuda)
        st["values"] = torch.zeros_like(st["x"])
        return st
    if kind in ("linear", "experts"):
        n, K, M = _n_rows(case), case["K"], case["M"]
        st["x"] = _hidden(n, K, seed, 1)
        st["bias"] = st["residual"] = None
        lead = ()
        if kind == "experts":
            lead = (case["E"],)
            score = torch.rand(case["T"], case["E"], device="cuda", generator=_gen(seed, 2))
            counts = torch.bincount(score.topk(case["k"], dim=1).indices.reshape(-1), minlength=case["E"])
            st["offsets"] = torch.cat([counts.new_zeros(1), counts.cumsum(0)]).to(torch.int32)
            st["most"] = int(counts.max())
        elif case["norm"]:
            st["norm_weight"] = _normal((K,), 0.2, seed, 3, torch.float32).add_(1.0)
        st["w_codes"], st["w_scales"] = _weights((*lead, M, K), seed, 4)
        if case["bias"]:
            st["bias"] = _normal((*lead, M), 0.3, seed, 5, torch.float32)
        if case["residual"]:
            st["residual"] = _normal((n, _out_width(case)), 1.0, seed, 6)
        st["x_codes"] = torch.zeros(n, K // 2, dtype=torch.uint8, **cuda)
        st["x_scales"] = torch.zeros(n, K // 32, dtype=torch.uint8, **cuda)
        st["y"] = torch.zeros(n, _out_width(case), dtype=torch.bfloat16, **cuda)
        return st
    T, H, dt = case["T"], case["H"], _DT[case["dtype"]]
    st["block"], st["residual"] = _normal((T, H), 1.0, seed, 11, dt), _hidden(T, H, seed, 12, dt)
    st["post"] = _normal((H,), 0.2, seed, 13, torch.float32).add_(1.0) if case["post"] else None
    st["pre"] = _normal((H,), 0.2, seed, 14, torch.float32).add_(1.0)
    st["gate"] = _gate(case, seed)
    st["y"], st["h"] = torch.zeros(T, H, dtype=dt, **cuda), torch.zeros(T, H, dtype=dt, **cuda)
    if kind == "norm_backward":
        st["y"] = _plain_norm(st)["y"]
        st["dy"], st["dh"] = _normal((T, H), 1.0, seed, 16, dt), _normal((T, H), 1.0, seed, 17, dt)
        st["out"] = {"dblock": torch.zeros_like(st["y"]), "dresidual": torch.zeros_like(st["y"]),
                     "dpre": torch.zeros_like(st["pre"])}
        if case["post"]:
            st["out"]["dpost"] = torch.zeros_like(st["post"])
        if st["gate"] is not None:
            st["out"]["dgate"] = torch.zeros_like(st["gate"])
    return st


# ------------------------------------------------------------- the plain forms --
_LEVELS = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _power(e):
    """2^e in fp32, e an int32 tensor in -126..127."""
    return ((e + 127) << 23).view(torch.float32)


def _scaled(v, s):
    """v 2^s in fp32, s in -127..127: two factors, both normal."""
    half = s >> 1
    return v * _power(half) * _power(s - half)


def _plain_quantize(x):
    """(magnitude code and sign [T, P / 32, 32], scale exponent s [T, P / 32], block without NaN or infinity)."""
    T, K = x.shape
    v = torch.nn.functional.pad(x.float(), (0, -K % 32)).view(T, -1, 32)
    top = v.abs().amax(2)
    fine = torch.isfinite(top)
    top = torch.where(fine, top, 0.0)
    s = torch.where(top > 0, torch.frexp(top).exponent - 3, -127).clamp(-127, 127).int()
    a = _scaled(v.abs(), -s[..., None])
    code = (a > 0.25).int() + (a >= 0.75).int() + (a > 1.25).int() + (a >= 1.75).int()
    code = code + (a > 2.5).int() + (a >= 3.5).int() + (a > 5.0).int()
    return code, v.signbit(), s, fine


def _plain_values(x, levels):
    """What the 4-bit rows stand for, fp32 [T, K], and the scale bytes."""
    code, negative, s, fine = _plain_quantize(x)
    level = levels[code]
    v = _scaled(torch.where(negative, -level, level), s[..., None])
    v = torch.where(fine[..., None], v, math.nan).flatten(1)[:, :x.shape[1]]
    return v, torch.where(fine, s + 127, 255).to(torch.uint8)


def _plain_matrix(codes, scales, pairs):
    """The values of a matrix (or of a stack of them) held in 4 bits, fp32."""
    v = pairs[codes.int()].flatten(-2).unflatten(-1, (-1, 32))
    return (v * _power(scales.int() - 127)[..., None]).flatten(-2)


def _activate(act, z):
    if act == "swiglu":
        g, u = z.chunk(2, dim=-1)
        return g / (1.0 + torch.exp(-g)) * u
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_rms(x, weight):
    """x (mean x^2 + eps)^-1/2 weight in fp32."""
    return x * torch.rsqrt((x * x).mean(1, keepdim=True) + EPS) * weight


def _plain_product(st):
    case = st["case"]
    x = st["x"]
    if "norm_weight" in st:
        x = _plain_rms(x.float(), st["norm_weight"]).to(torch.bfloat16)
    x, w = _plain_values(x, st["levels"])[0], _plain_matrix(st["w_codes"], st["w_scales"], st["pairs"])
    if case["kind"] == "experts":  # each expert's rows padded to the most that one has
        off = st["offsets"].long()
        p = torch.arange(x.shape[0], device="cuda")
        e = (p[:, None] >= off[None, 1:]).sum(1)
        at = e * st["most"] + p - off[e]
        rows = x.new_zeros(case["E"] * st["most"], x.shape[1])
        rows[at] = x
        z = torch.bmm(rows.view(case["E"], st["most"], -1), w.transpose(1, 2).contiguous())
        if st["bias"] is not None:
            z = z + st["bias"][:, None]
        y = _activate(case["act"], z).flatten(0, 1)[at]
    else:
        z = x @ w.t()
        y = _activate(case["act"], z if st["bias"] is None else z + st["bias"])
    return (y if st["residual"] is None else y + st["residual"].float()).to(torch.bfloat16)


def _plain_norm(st):
    case, b = st["case"], st["block"].float()
    u = b if st["post"] is None else _plain_rms(b, st["post"])
    if st["gate"] is not None:
        u = u * st["gate"].float()
    y = (case["scale"] * st["residual"].float() + u).to(st["block"].dtype)
    return {"y": y, "h": _plain_rms(y.float(), st["pre"]).to(y.dtype)}


def _plain_rms_grad(x, weight, dh):
    """Gradients of _plain_rms to x and to weight."""
    n = torch.rsqrt((x * x).mean(1, keepdim=True) + EPS)
    a = dh * weight
    return n * a - x * n ** 3 * (a * x).mean(1, keepdim=True), (dh * x * n).sum(0)


def _plain_norm_backward(st):
    case, dt = st["case"], st["block"].dtype
    b, y, dh = st["block"].float(), st["y"].float(), st["dh"].float()
    dx, dpre = _plain_rms_grad(y, st["pre"], dh)
    d = st["dy"].float() + dx
    out = {"dresidual": (case["scale"] * d).to(dt), "dpre": dpre}
    du = d
    if st["gate"] is not None:
        dg = d * (b if st["post"] is None else _plain_rms(b, st["post"]))
        out["dgate"] = {"column": lambda: dg.sum(0), "row": lambda: dg.sum(1, keepdim=True),
                        "full": lambda: dg.to(dt)}[case["gate"]]()
        du = d * st["gate"].float()
    if st["post"] is None:
        out["dblock"] = du.to(dt)
    else:
        db, out["dpost"] = _plain_rms_grad(b, st["post"], du)
        out["dblock"] = db.to(dt)
    return out


def _plain(st):
    kind = st["case"]["kind"]
    if kind == "quantize":
        v, scales = _plain_values(st["x"], st["levels"])
        return {"values": v.to(st["x"].dtype), "scales": scales}
    if kind in ("linear", "experts"):
        return _plain_product(st)
    return _plain_norm(st) if kind == "norm" else _plain_norm_backward(st)


_contexts = {}


def _context():
    """The framework's context on the current GPU, one for the process."""
    device = torch.cuda.current_device()
    if device not in _contexts:
        _contexts[device] = importlib.import_module("raon-npu_amd.device").Context(device)
    return _contexts[device]


def run(st):
    """One pass."""
    if not own:
        return _plain(st)
    ctx, case, stream = _context(), st["case"], torch.cuda.current_stream()
    kind = case["kind"]
    if kind == "quantize":
        ctx.mx_quantize_dev(st["x"], st["codes"], st["scales"], values_dev=st["values"], stream=stream)
        return {"values": st["values"], "scales": st["scales"]}
    if kind in ("linear", "experts"):
        if "norm_weight" in st:
            ctx.norm_dev(st["x"], st["norm_weight"], codes_dev=st["x_codes"], scales_dev=st["x_scales"], eps=EPS,
                         stream=stream)
        else:
            ctx.mx_quantize_dev(st["x"], st["x_codes"], st["x_scales"], stream=stream)
        args = (st["x_codes"], st["x_scales"], st["w_codes"], st["w_scales"])
        if kind == "linear":
            ctx.mx_linear_dev(*args, st["y"], bias_dev=st["bias"], act=case["act"], residual_dev=st["residual"],
                              stream=stream)
        else:
            ctx.mx_experts_linear_dev(*args, st["offsets"], st["y"], bias_dev=st["bias"], act=case["act"],
                                      residual_dev=st["residual"], stream=stream)
        return st["y"]
    if kind == "norm":
        ctx.residual_norm_dev(st["block"], st["residual"], st["y"], post_weight_dev=st["post"], gate_dev=st["gate"],
                              scale=case["scale"], pre_weight_dev=st["pre"], h_dev=st["h"], eps=EPS, stream=stream)
        return {"y": st["y"], "h": st["h"]}
    out = st["out"]
    if "work" not in st:
        st["work"] = torch.empty(ctx.norm_backward_work(case["T"], case["H"]), device="cuda")
    ctx.residual_norm_backward_dev(st["dy"], st["dh"], st["block"], st["y"], out["dblock"], out["dresidual"],
                                   st["work"], post_weight_dev=st["post"], dpost_weight_dev=out.get("dpost"),
                                   gate_dev=st["gate"], dgate_dev=out.get("dgate"), scale=case["scale"],
                                   pre_weight_dev=st["pre"], dpre_weight_dev=out["dpre"], eps=EPS, stream=stream)
    return dict(out)


# ------------------------------------------------------------------------ work --
def work(case):
    """Bytes (each operand once; of the experts' weights those that expect a row) and operations of a pass."""
    kind = case["kind"]
    if kind == "quantize":
        size = 4 if case["dtype"] == "fp32" else 2
        n = case["T"] * case["K"]
        return {"bytes": 2 * n * size + case["T"] * -(-case["K"] // 32) * 17, "flops": 2 * n}
    if kind in ("linear", "experts"):
        n, M, K, out = _n_rows(case), case["M"], case["K"], _out_width(case)
        weights = M * (17 * K // 32 + (4 if case["bias"] else 0))
        if kind == "experts":
            weights = int(weights * case["E"] * (1.0 - (1.0 - case["k"] / case["E"]) ** case["T"]))
        nbytes = weights + n * (2 * K + 2 * out * (2 if case["residual"] else 1))
        return {"bytes": nbytes, "flops": 2 * n * M * K}
    size = 4 if case["dtype"] == "fp32" else 2
    row, full = case["T"] * case["H"] * size, case["gate"] == "full"
    if kind == "norm":
        return {"bytes": row * (5 if full else 4) + 8 * case["H"], "flops": 10 * case["T"] * case["H"]}
    return {"bytes": row * (8 if full else 6) + 16 * case["H"], "flops": 24 * case["T"] * case["H"]}


# ---------------------------------------------------------- the results in fp64 --
def _exact_codes(x):
    """The values the 4-bit rows of x stand for, fp64 [T, K], and the scale bytes: the nearest of the signed levels
    by distance, of two as near the one with an even place."""
    x = x.double()
    T, K = x.shape
    v = torch.zeros(T, -(-K // 32) * 32, dtype=torch.float64, device=x.device)
    v[:, :K] = x
    v = v.view(T, -1, 32)
    top = v.abs().max(2).values
    bad = ~torch.isfinite(top)
    s = torch.floor(torch.log2(torch.where(bad | (top == 0), 1.0, top)))
    s = s + (torch.exp2(s + 1) <= top).double() - (torch.exp2(s) > top).double()  # where the logarithm was rounded
    s = torch.where(top == 0, -127.0, (s - 2).clamp(-127, 127))
    a = (v.abs() * torch.exp2(-s)[..., None]).clamp(max=6.0)
    best, far = torch.zeros_like(a), a.clone()
    for i, level in enumerate(_LEVELS[1:], 1):
        d = (a - level).abs()
        nearer = (d < far) | ((d == far) & (i % 2 == 0))
        best, far = torch.where(nearer, level, best), torch.where(nearer, d, far)
    out = torch.copysign(best, v) * torch.exp2(s)[..., None]
    out = torch.where(bad[..., None], math.nan, out).flatten(1)[:, :K]
    return out, torch.where(bad, 255.0, s + 127).to(torch.uint8)


def _exact_matrix(codes, scales):
    n = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    e, m = ((n >> 1) & 3).double(), (n & 1).double()
    v = torch.where(e == 0, 0.5 * m, (1.0 + 0.5 * m) * torch.exp2(e - 1)) * torch.where(n >= 8, -1.0, 1.0)
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def _exact_rms(x, weight):
    return x / torch.sqrt(x.square().mean(1, keepdim=True) + EPS) * weight.double()


def _exact_act(act, z):
    half = z.shape[1] // 2
    if act == "swiglu":
        return z[:, :half] * torch.sigmoid(z[:, :half]) * z[:, half:]
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    if act == "gelu_tanh":
        return z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    return z


def exact(case, seed):
    """The outputs in 64 bits from the definitions, laid out as ``run``'s."""
    st = prepare(case, seed)
    kind = case["kind"]
    if kind == "quantize":
        v, scales = _exact_codes(st["x"])
        return {"values": v, "scales": scales}
    if kind in ("linear", "experts"):
        x = st["x"].double()
        if "norm_weight" in st:  # what is quantized are the normalised rows in their own type
            x = _exact_rms(x, st["norm_weight"]).to(torch.bfloat16)
        x = _exact_codes(x)[0]
        bounds = st["offsets"].tolist() if kind == "experts" else [0, x.shape[0]]
        y = torch.zeros(x.shape[0], _out_width(case), dtype=torch.float64, device="cuda")
        for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
            if a == b:
                continue
            wc, ws, bias = st["w_codes"], st["w_scales"], st["bias"]
            if kind == "experts":
                wc, ws, bias = wc[e], ws[e], None if bias is None else bias[e]
            z = x[a:b] @ _exact_matrix(wc, ws).t()
            y[a:b] = _exact_act(case["act"], z if bias is None else z + bias.double())
        return y if st["residual"] is None else y + st["residual"].double()
    b, r, g = st["block"].double(), st["residual"].double(), st["gate"]
    g = torch.ones(1, dtype=torch.float64, device="cuda") if g is None else g.double()
    if kind == "norm":
        u = b if st["post"] is None else _exact_rms(b, st["post"])
        y = case["scale"] * r + g * u
        return {"y": y, "h": _exact_rms(y.to(st["block"].dtype).double(), st["pre"])}  # of y as it is stored
    y, dy, dh = st["y"].double(), st["dy"].double(), st["dh"].double()

    def grad(x, weight, d):
        """Through x_i / q weight_i, q = sqrt(mean x^2 + eps): the Jacobian is (diag(weight) - h x^T / (H q^2)) / q."""
        q = torch.sqrt(x.square().mean(1, keepdim=True) + EPS)
        along = (d * weight * x).sum(1, keepdim=True) / (x.shape[1] * q.square())
        return (d * weight - along * x) / q, (d * x / q).sum(0)

    dx, dpre = grad(y, st["pre"].double(), dh)
    d = dy + dx
    out = {"dresidual": case["scale"] * d, "dpre": dpre}
    u = b
    if st["post"] is None:
        out["dblock"] = g * d
    else:
        u = _exact_rms(b, st["post"])
        out["dblock"], out["dpost"] = grad(b, st["post"].double(), g * d)
    if st["gate"] is not None:
        out["dgate"] = (d * u) if case["gate"] == "full" else (d * u).sum(0) if case["gate"] == "column" \
            else (d * u).sum(1, keepdim=True)
    return out
