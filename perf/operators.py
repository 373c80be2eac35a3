"""The operators around the experts' products whose speed is tracked: tokens sorted by expert and back with
their gradients, and products of quantized weights with bias, activation and residual, dense or by expert.

With ``own`` false ``run`` computes them in elementary torch operations in fp32, rounded once at the end; with
``own`` true it makes the calls of the framework.  Sizes are those of the two layer geometries of
``raon-npu_amd/geometry.py`` (H=2048, I=768, top-8 and H=2560, I=1088, top-6, 128 experts each), of the dense
matrices of a weights-d directory and of the prompts of ``bench.py`` (445 and 6,700 tokens); ``draw`` spreads
over the ranges around them, odd widths and other types included.
"""

from __future__ import annotations

import importlib
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
SITU = (4.0, 25.0)
GATED = ("swiglu", "situ")


# ------------------------------------------------------------------ the cases --
def listed():
    return [
        # A decode step of four requests: the rows of their experts, the smallest call.
        {"name": "sort_decode", "kind": "sort", "T": 4, "k": 8, "E": 128, "H": 2048, "dtype": "bf16", "pad": 0.0,
         "zipf": False},
        # A long prompt with skewed routing, 3 % of the batch padding that no expert takes.
        {"name": "sort_prefill", "kind": "sort", "T": 6700, "k": 8, "E": 128, "H": 2048, "dtype": "bf16", "pad": 0.03,
         "zipf": True},
        # Training a router and adapters around the experts: the rows' gradients, in fp32, back to the tokens.
        {"name": "sort_backward_fp32", "kind": "sort_backward", "T": 445, "k": 6, "E": 128, "H": 2560, "dtype": "fp32",
         "pad": 0.0, "zipf": False},
        # One generated token: its experts' outputs weighted and added.
        {"name": "combine_decode", "kind": "combine", "T": 1, "k": 6, "E": 128, "H": 2560, "dtype": "bf16", "pad": 0.0,
         "zipf": False},
        # The long prompt's expert outputs back in token order.
        {"name": "combine_prefill", "kind": "combine", "T": 6700, "k": 8, "E": 128, "H": 2048, "dtype": "bf16",
         "pad": 0.03, "zipf": True},
        # A training batch of odd length: gradients of the expert outputs and of the router's weights.
        {"name": "combine_backward", "kind": "combine_backward", "T": 4099, "k": 8, "E": 128, "H": 2048,
         "dtype": "bf16", "pad": 0.0, "zipf": False},
        # The shared expert's down projection of one token onto the residual stream.
        {"name": "linear_decode", "kind": "linear", "fmt": "q4nx", "T": 1, "M": 2048, "K": 768, "act": "none",
         "bias": False, "residual": True},
        # The shared expert's gate/up with its activation for a middling prompt.
        {"name": "linear_swiglu_445", "kind": "linear", "fmt": "q4nx", "T": 445, "M": 1536, "K": 2048, "act": "swiglu",
         "bias": False, "residual": False},
        # shared_gu of a weights-d layer, biased, for a long prefill chunk.
        {"name": "linear_situ_4096", "kind": "linear", "fmt": "bfp16", "T": 4096, "M": 2176, "K": 2560, "act": "situ",
         "bias": True, "residual": False},
        # One token's sorted rows through the gate/up of its eight experts.
        {"name": "experts_decode", "kind": "experts", "part": "gate_up", "T": 1, "k": 8, "E": 128, "H": 2048, "I": 768,
         "act": "swiglu", "bias": False, "residual": False, "zipf": False},
        # A middling prompt's activations through the bfp16 down projections of a weights-d layer.
        {"name": "experts_down_445", "kind": "experts", "part": "down", "T": 445, "k": 6, "E": 128, "H": 2560,
         "I": 1088, "act": "none", "bias": False, "residual": False, "zipf": False},
        # The long prompt's sorted rows through gate/up: the largest call.
        {"name": "experts_gate_up_6700", "kind": "experts", "part": "gate_up", "T": 6700, "k": 8, "E": 128, "H": 2048,
         "I": 768, "act": "swiglu", "bias": False, "residual": False, "zipf": True},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.5)))))))


def draw(rng):
    kind = rng.choice(["sort", "sort_backward", "combine", "combine_backward", "linear", "linear", "experts"])
    if kind == "linear":
        return {"kind": kind, "fmt": rng.choice(["q4nx", "bfp16"]), "T": _log_int(rng, 1, 4096),
                "M": 128 * rng.randint(2, 17), "K": 256 * rng.randint(2, 10),
                "act": rng.choice(["none", "silu", "gelu", "gelu_tanh", "swiglu", "situ"]),
                "bias": rng.random() < 0.5, "residual": rng.random() < 0.5}
    E = _log_int(rng, 8, 256)
    k = rng.randint(1, min(16, E))
    if kind == "experts":
        E, k = min(E, 128), min(k, 8)
        part = rng.choice(["gate_up", "down"])
        return {"kind": kind, "part": part, "T": _log_int(rng, 1, 4000), "k": k, "E": E, "H": 256 * rng.randint(2, 8),
                "I": 64 * rng.randint(4, 12), "act": rng.choice(["swiglu", "situ"]) if part == "gate_up" else "none",
                "bias": rng.random() < 0.5, "residual": part == "down" and rng.random() < 0.5,
                "zipf": rng.random() < 0.5}
    H = rng.choice([2048, 2560, rng.randint(1, 2600)])
    return {"kind": kind, "T": max(1, min(_log_int(rng, 1, 6700), 6700 * 8 * 2048 // (k * H * 2))), "k": k, "E": E,
            "H": H, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "pad": rng.choice([0.0, 0.0, 0.1]),
            "zipf": rng.random() < 0.5}


# ------------------------------------------------------------ seeded values --
def _gen(seed, part):
    return torch.Generator(device="cuda").manual_seed((int(seed) * 1000003 + 7919 * part + 1) & 0x7FFFFFFFFFFF)


def _normal(shape, std, seed, part, dtype=torch.bfloat16):
    return torch.randn(*shape, device="cuda", generator=_gen(seed, part)).mul_(std).to(dtype)


def _n_padding(case):
    return int(case["T"] * case.get("pad", 0.0))


def _routing(case, seed):
    """int32 ids [T, k], distinct for each token; a padding token has -1 in every route."""
    T, E, k = case["T"], case["E"], case["k"]
    score = torch.rand(T, E, device="cuda", generator=_gen(seed, 1)).clamp_(min=1e-9).log_()
    if case["zipf"]:  # popularity rank^-1.1, ranks dealt by the seed
        rank = torch.rand(E, device="cuda", generator=_gen(seed, 2)).argsort().float() + 1
        score = score / rank.pow(-1.1)
    ids = score.topk(k, dim=1).indices.to(torch.int32)
    n = _n_padding(case)
    if n:
        ids[torch.rand(T, device="cuda", generator=_gen(seed, 3)).argsort()[:n]] = -1
    return ids.contiguous()


def _sorted(ids, E):
    """(order [A], inv [T, k], offsets [E + 1]) int32: the assignments t * k + r by expert, in their order within
    one; inv -1 and order 0 where there is none."""
    flat = ids.reshape(-1).long()
    live = flat >= 0
    perm = torch.where(live, flat, E).sort(stable=True).indices
    pos = torch.empty_like(perm)
    pos[perm] = torch.arange(perm.numel(), device=perm.device)
    inv = torch.where(live, pos, -1)
    bounds = torch.arange(E + 1, device=ids.device)
    offsets = (flat[None, :].clamp(min=-1) < bounds[:, None]).sum(1) - (~live).sum()
    behind = torch.arange(perm.numel(), device=perm.device) >= live.sum()
    order = torch.where(behind, 0, perm)
    return order.int(), inv.view_as(ids).int().contiguous(), offsets.int()


def _route_weights(case, seed):
    w = torch.rand(case["T"], case["k"], device="cuda", generator=_gen(seed, 4)).add_(0.1)
    return (w / w.sum(1, keepdim=True)).contiguous()


def _q4nx(M, K, seed, part):
    """A q4nx matrix as a checkpoint holds it, by groups of 32 columns: codes 0..15 (both ends taken), scales and
    mins that bf16 holds, about N(0, 0.02)'s spread.  Its values m + s * code are exact in fp32."""
    g = _gen(seed, part)
    code = torch.randint(0, 16, (M, K // 32, 32), device="cuda", generator=g, dtype=torch.int32)
    code[..., 5], code[..., 17] = 0, 15
    s = (torch.rand(M, K // 32, device="cuda", generator=g) * 0.004 + 0.004).to(torch.bfloat16).float()
    m = ((torch.rand(M, K // 32, device="cuda", generator=g) * -2.0 - 6.5) * s).to(torch.bfloat16).float()
    return code, s, m


def _bfp16(M, K, seed, part, live=None):
    """A bfp16 matrix: int8 mantissas and one exponent byte e per 8 columns, values m * 2^(e - 133); zero mantissas
    from column ``live`` on."""
    g = _gen(seed, part)
    mant = torch.randint(-128, 128, (M, K // 8, 8), device="cuda", generator=g, dtype=torch.int32)
    e = torch.randint(119, 122, (M, K // 8), device="cuda", generator=g, dtype=torch.int32)
    if live is not None:
        mant.view(M, K)[:, live:] = 0
    return mant, e


def _values(w, dtype):
    """[M, K] in ``dtype`` of (codes, scales, mins) or (mantissas, exponents)."""
    if len(w) == 3:
        code, s, m = w
        return (code.to(dtype) * s.to(dtype)[..., None] + m.to(dtype)[..., None]).flatten(1)
    mant, e = w
    return (mant.to(dtype) * torch.exp2((e - 133).to(dtype))[..., None]).flatten(1)


def _bfp16_bytes(w):
    """The GEMV bytes of a bfp16 matrix: blocks of 32 rows by 256 columns (four down a slice of 128 rows), in each
    half of 16 rows and group of 8 columns 16 exponents, then the mantissas column by column."""
    mant, e = w
    M, kb = e.shape[0], e.shape[1] // 32
    ee = e.to(torch.uint8).view(M // 128, 4, 2, 16, kb, 32).permute(0, 4, 1, 2, 5, 3)
    mm = mant.to(torch.int8).view(torch.uint8).view(M // 128, 4, 2, 16, kb, 32, 8).permute(0, 4, 1, 2, 5, 6, 3)
    return torch.cat([ee, mm.flatten(-2)], -1).contiguous().view(-1).cpu().numpy()


def _pad256(n):
    return -(-n // 256) * 256


def _bias(case, M, seed):
    if not case["bias"]:
        return None
    lead = (case["E"], M) if case["kind"] == "experts" else (M,)
    return _normal(lead, 0.3, seed, 6, torch.float32)


def _out_width(case):
    if case["kind"] == "experts":
        return case["I"] if case["part"] == "gate_up" else case["H"]
    return case["M"] // 2 if case["act"] in GATED else case["M"]


def _expert_weight(case, seed, e):
    if case["part"] == "gate_up":
        return _q4nx(2 * case["I"], case["H"], seed, 1000 + e)
    return _bfp16(case["H"], _pad256(case["I"]), seed, 1000 + e, live=case["I"])


def _inputs(case, seed):
    """The operands of a case without its weights."""
    kind, T = case["kind"], case["T"]
    s = {}
    if kind == "linear":
        s["x"] = _normal((T, case["K"]), 1.0, seed, 5)
        s["bias"] = _bias(case, case["M"], seed)
        s["residual"] = _normal((T, _out_width(case)), 1.0, seed, 7) if case["residual"] else None
        return s
    ids = _routing(case, seed)
    order, inv, offsets = _sorted(ids, case["E"])
    A = ids.numel()
    if kind == "experts":
        wide = case["H"] if case["part"] == "gate_up" else case["I"]
        s["rows"] = _normal((A, wide), 1.0, seed, 5)
        s["offsets"] = offsets
        s["bias"] = _bias(case, 2 * case["I"] if case["part"] == "gate_up" else case["H"], seed)
        s["residual"] = _normal((A, _out_width(case)), 1.0, seed, 7) if case["residual"] else None
        return s
    dt = _DT[case["dtype"]]
    if kind == "sort":
        s["x"], s["ids"] = _normal((T, case["H"]), 1.0, seed, 5, dt), ids
        return s
    s["inv"] = inv
    if kind == "sort_backward":
        s["drows"] = _normal((A, case["H"]), 1.0, seed, 5, dt)
        return s
    s["rows"], s["wts"] = _normal((A, case["H"]), 1.0, seed, 5, dt), _route_weights(case, seed)
    if kind == "combine_backward":
        s["dout"] = _normal((T, case["H"]), 1.0, seed, 7, dt)
    return s


# --------------------------------------------------------------------- prepare --
def prepare(case, seed):
    """Inputs, and what a program keeps: weights (own: uploaded to a context; else fp32 values), output buffers."""
    st = _inputs(case, seed)
    st["case"] = case
    kind = case["kind"]
    if not own:
        if kind == "linear":
            q = _q4nx(case["M"], case["K"], seed, 8) if case["fmt"] == "q4nx" else _bfp16(case["M"], case["K"], seed, 8)
            st["w"] = _values(q, torch.float32)
        elif kind == "experts":
            st["bounds"] = st["offsets"].tolist()
            wide = st["rows"].shape[1]
            st["w"] = [_values(_expert_weight(case, seed, e), torch.float32)[:, :wide].contiguous()
                       for e in range(case["E"])]
        return st
    device = importlib.import_module("raon-npu_amd.device")
    geometry = importlib.import_module("raon-npu_amd.geometry")
    ctx = st["ctx"] = device.Context(torch.cuda.current_device())
    T, cuda = case["T"], {"device": "cuda"}
    if kind == "linear":
        if case["fmt"] == "q4nx":
            w = _values(_q4nx(case["M"], case["K"], seed, 8), torch.float32)
            st["matrix"] = ctx.quantize_matrix(w, case["M"], case["K"])
        else:
            w = _bfp16_bytes(_bfp16(case["M"], case["K"], seed, 8))
            st["matrix"] = ctx.upload_matrix(w, case["M"], case["K"], fmt="bfp16")
        st["matrix"].reserve_act(T)
        st["y"] = torch.zeros(T, _out_width(case), dtype=torch.bfloat16, **cuda)
    elif kind == "experts":
        g = geometry.MoeGeometry(hidden=case["H"], inter=case["I"], n_routed=case["E"], n_shared=1,
                                 top_k=min(16, case["E"]))
        if case["part"] == "gate_up":
            layer = ctx.create_layer(0, g)
            down = torch.zeros(case["H"], case["I"], **cuda)
            for e in range(case["E"]):
                layer.quantize_expert(e, _values(_expert_weight(case, seed, e), torch.float32), down)
        else:
            layer = ctx.create_layer_d(0, g)
            for e in range(case["E"]):
                layer.upload_d(2, e, _bfp16_bytes(_expert_weight(case, seed, e)))
        st["layer"] = layer
        A = st["rows"].shape[0]
        layer.reserve_experts_linear(A)
        st["y"] = torch.zeros(A, _out_width(case), dtype=torch.bfloat16, **cuda)
    else:
        A, H, dt = T * case["k"], case["H"], _DT[case["dtype"]]
        if kind == "sort":
            st["rows"] = torch.zeros(A, H, dtype=dt, **cuda)
            st["order"] = torch.zeros(A, dtype=torch.int32, **cuda)
            st["inv"] = torch.zeros(T, case["k"], dtype=torch.int32, **cuda)
            st["offsets"] = torch.zeros(case["E"] + 1, dtype=torch.int32, **cuda)
        elif kind == "combine_backward":
            st["drows"] = torch.zeros(A, H, dtype=dt, **cuda)
            st["dwts"] = torch.zeros(T, case["k"], **cuda)
        else:
            st["out"] = torch.zeros(T, H, dtype=dt, **cuda)
    torch.cuda.synchronize()
    return st


# ------------------------------------------------------------- the plain forms --
def _activate(act, z):
    if act in GATED:
        g, u = z.chunk(2, dim=1)
        if act == "swiglu":
            return g / (1.0 + torch.exp(-g)) * u
        gb, vb = SITU
        return gb * torch.tanh(g / gb) / (1.0 + torch.exp(-g)) * (vb * torch.tanh(u / vb))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    if act == "gelu":
        return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(math.sqrt(2.0 / math.pi) * (z + 0.044715 * z * z * z)))
    return z


def _plain_linear(x, w, bias, act, residual):
    z = x.float() @ w.t()
    if bias is not None:
        z = z + bias
    y = _activate(act, z)
    return (y if residual is None else y + residual.float()).to(torch.bfloat16)


def _plain(st):
    case = st["case"]
    kind = case["kind"]
    if kind == "linear":
        return _plain_linear(st["x"], st["w"], st["bias"], case["act"], st["residual"])
    if kind == "experts":
        y = torch.zeros(st["rows"].shape[0], _out_width(case), dtype=torch.bfloat16, device="cuda")
        for e in range(case["E"]):
            a, b = st["bounds"][e], st["bounds"][e + 1]
            if a < b:
                y[a:b] = _plain_linear(st["rows"][a:b], st["w"][e], None if st["bias"] is None else st["bias"][e],
                                       case["act"], None if st["residual"] is None else st["residual"][a:b])
        return y
    k = case["k"]
    if kind == "sort":
        order, inv, offsets = _sorted(st["ids"], case["E"])
        live = torch.arange(order.numel(), device="cuda") < offsets[-1]
        rows = torch.where(live[:, None], st["x"][(order // k).long()], st["x"].new_zeros(()))
        return {"rows": rows, "order": order, "inv": inv, "offsets": offsets}
    inv, live = st["inv"].clamp(min=0).long(), st["inv"] >= 0
    if kind in ("sort_backward", "combine"):
        src = st["drows"] if kind == "sort_backward" else st["rows"]
        out = torch.zeros(case["T"], case["H"], device="cuda")
        for r in range(k):
            v = src[inv[:, r]].float()
            if kind == "combine":
                v = v * st["wts"][:, r, None]
            out += torch.where(live[:, r, None], v, 0.0)
        return out.to(src.dtype)
    dout, A = st["dout"].float(), st["rows"].shape[0]
    drows = torch.zeros(A + 1, case["H"], dtype=st["rows"].dtype, device="cuda")  # routes without a row end in the last
    dwts = torch.zeros_like(st["wts"])
    for r in range(k):
        drows[torch.where(live[:, r], inv[:, r], A)] = (st["wts"][:, r, None] * dout).to(drows.dtype)
        dwts[:, r] = torch.where(live[:, r], (dout * st["rows"][inv[:, r]].float()).sum(1), 0.0)
    return {"drows": drows[:A], "dwts": dwts}


def run(st):
    """One pass.  Rows behind the last sorted one keep the zeros their buffers began with."""
    if not own:
        return _plain(st)
    case, stream = st["case"], torch.cuda.current_stream()
    kind = case["kind"]
    betas = SITU if case.get("act") == "situ" else (None, None)
    if kind == "linear":
        st["matrix"].linear_act_dev(st["x"], case["T"], st["y"], bias_dev=st["bias"], act=case["act"],
                                    residual_dev=st["residual"], gate_beta=betas[0], value_beta=betas[1], stream=stream)
        return st["y"]
    if kind == "experts":
        st["layer"].experts_linear_dev(case["part"], st["rows"], st["offsets"], st["y"], bias_dev=st["bias"],
                                       act=case["act"], residual_dev=st["residual"], gate_beta=betas[0],
                                       value_beta=betas[1], stream=stream)
        return st["y"]
    ctx = st["ctx"]
    if kind == "sort":
        ctx.sort_tokens_dev(st["x"], st["ids"], case["E"], st["rows"], st["order"], st["inv"], st["offsets"],
                            stream=stream)
        return {n: st[n] for n in ("rows", "order", "inv", "offsets")}
    if kind == "sort_backward":
        ctx.sort_tokens_backward_dev(st["drows"], st["inv"], st["out"], stream=stream)
        return st["out"]
    if kind == "combine":
        ctx.combine_tokens_dev(st["rows"], st["inv"], st["wts"], st["out"], stream=stream)
        return st["out"]
    ctx.combine_tokens_backward_dev(st["dout"], st["rows"], st["inv"], st["wts"], st["drows"], st["dwts"],
                                    stream=stream)
    return {"drows": st["drows"], "dwts": st["dwts"]}


# ------------------------------------------------------------------------ work --
def work(case):
    """Bytes (each operand once; of the experts' weights those that expect a row) and operations of a pass."""
    T, kind = case["T"], case["kind"]
    out = _out_width(case) if kind in ("linear", "experts") else 0
    if kind == "linear":
        bits = 5 if case["fmt"] == "q4nx" else 9
        nbytes = case["M"] * case["K"] * bits // 8 + T * (2 * case["K"] + 2 * out * (2 if case["residual"] else 1))
        return {"bytes": nbytes + (4 * case["M"] if case["bias"] else 0), "flops": 2 * T * case["M"] * case["K"]}
    k, E, H = case["k"], case["E"], case["H"]
    A = (T - _n_padding(case)) * k
    if kind == "experts":
        up = case["part"] == "gate_up"
        M, K = (2 * case["I"], H) if up else (H, case["I"])
        taken = E * (1.0 - (1.0 - k / E) ** T)
        weights = int(taken * M * (K * 5 // 8 if up else _pad256(K) * 9 // 8))
        bias = int(taken) * M * 4 if case["bias"] else 0
        return {"bytes": weights + bias + A * (2 * K + 2 * out * (2 if case["residual"] else 1)) + 4 * (E + 1),
                "flops": 2 * A * M * K}
    size = 4 if case["dtype"] == "fp32" else 2
    token, row, index = T * H * size, A * H * size, 4 * T * k
    if kind == "sort":
        return {"bytes": (T - _n_padding(case)) * H * size + row + 3 * index + 4 * (E + 1), "flops": 0}
    if kind == "sort_backward":
        return {"bytes": row + token + index, "flops": A * H}
    if kind == "combine":
        return {"bytes": row + token + 2 * index, "flops": 2 * A * H}
    return {"bytes": 2 * row + token + 3 * index, "flops": 3 * A * H}


# ---------------------------------------------------------- the results in fp64 --
def _exact_product(x, w, bias, act, residual):
    z = torch.mm(x.double(), w.t().contiguous())
    if bias is not None:
        z += bias.double()
    half = z.shape[1] // 2
    if act == "swiglu":
        z = z[:, :half] * torch.sigmoid(z[:, :half]) * z[:, half:]
    elif act == "situ":
        g, u = z[:, :half], z[:, half:]
        z = SITU[0] * torch.tanh(g / SITU[0]) * torch.sigmoid(g) * SITU[1] * torch.tanh(u / SITU[1])
    elif act == "silu":
        z = z * torch.sigmoid(z)
    elif act == "gelu":
        z = z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0))
    elif act == "gelu_tanh":
        z = z * torch.sigmoid(2.0 * math.sqrt(2.0 / math.pi) * (z + 0.044715 * z ** 3))
    return z if residual is None else z + residual.double()


def exact(case, seed):
    """The outputs in 64 bits from the definitions, laid out as ``run``'s."""
    st = _inputs(case, seed)
    kind = case["kind"]
    if kind == "linear":
        w = _q4nx(case["M"], case["K"], seed, 8) if case["fmt"] == "q4nx" else _bfp16(case["M"], case["K"], seed, 8)
        return _exact_product(st["x"], _values(w, torch.float64), st["bias"], case["act"], st["residual"])
    if kind == "experts":
        y = torch.zeros(st["rows"].shape[0], _out_width(case), dtype=torch.float64, device="cuda")
        bounds = st["offsets"].tolist()
        for e, (a, b) in enumerate(zip(bounds, bounds[1:])):
            if a == b:
                continue
            w = _values(_expert_weight(case, seed, e), torch.float64)[:, :st["rows"].shape[1]]
            y[a:b] = _exact_product(st["rows"][a:b], w, None if st["bias"] is None else st["bias"][e], case["act"],
                                    None if st["residual"] is None else st["residual"][a:b])
        return y
    k, H, dev = case["k"], case["H"], torch.device("cuda")
    if kind == "sort":
        # By counting: an assignment's place is the number with a smaller expert, plus those of its own before it.
        flat = st["ids"].reshape(-1).cpu().tolist()
        places = [[] for _ in range(case["E"])]
        for a, e in enumerate(flat):
            if e >= 0:
                places[e].append(a)
        seq = [a for p in places for a in p]
        offsets, inv = [0], [-1] * len(flat)
        for p in places:
            offsets.append(offsets[-1] + len(p))
        for i, a in enumerate(seq):
            inv[a] = i
        rows = torch.zeros(len(flat), H, dtype=torch.float64, device=dev)
        if seq:
            rows[:len(seq)] = st["x"].double()[torch.tensor(seq, device=dev) // k]
        i32 = {"dtype": torch.int32, "device": dev}
        return {"rows": rows, "order": torch.tensor(seq + [0] * (len(flat) - len(seq)), **i32),
                "inv": torch.tensor(inv, **i32).view(-1, k), "offsets": torch.tensor(offsets, **i32)}
    live = st["inv"].reshape(-1) >= 0
    a = live.nonzero()[:, 0]  # assignments, and the sorted row and token of each
    p, t = st["inv"].reshape(-1)[a].long(), a // k
    if kind == "combine_backward":
        drows = torch.zeros(live.numel(), H, dtype=torch.float64, device=dev)
        dwts = torch.zeros(live.numel(), dtype=torch.float64, device=dev)
        for i in range(0, a.numel(), 16384):
            s = slice(i, i + 16384)
            d = st["dout"].double()[t[s]]
            drows[p[s]] = d * st["wts"].reshape(-1)[a[s]].double()[:, None]
            dwts[a[s]] = (d * st["rows"][p[s]].double()).sum(1)
        return {"drows": drows, "dwts": dwts.view(-1, k)}
    out = torch.zeros(case["T"], H, dtype=torch.float64, device=dev)
    for i in range(0, a.numel(), 16384):
        s = slice(i, i + 16384)
        if kind == "combine":
            out.index_add_(0, t[s], st["rows"][p[s]].double() * st["wts"].reshape(-1)[a[s]].double()[:, None])
        else:
            out.index_add_(0, t[s], st["drows"][p[s]].double())
    return out
