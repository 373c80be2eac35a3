"""CPU: calls that the microscaled 4-bit operators and the norms around a block refuse, in the wrappers and in the C entry
points.  A refused call reaches neither the device nor the context (a buffer stands in for it)."""

from __future__ import annotations

import ctypes as C

import pytest

from raon_npu_amd import _lib
from test_operator_refusals import Tensor, ctx, f32, i32, raw  # noqa: F401  (fixtures)

T, K, M, E, H = 4, 64, 48, 3, 72


def u8(*shape, **kw):
    return Tensor(*shape, dtype="uint8", **kw)


@pytest.mark.parametrize("kw", [
    {"x": Tensor(T, K, dtype="float64")}, {"x": Tensor(T * K)}, {"x": Tensor(T, K, contiguous=False)},
    {"x": Tensor(T, K, device=1)}, {"codes": u8(T, K)}, {"codes": Tensor(T, K // 2)}, {"scales": u8(T, K // 16)},
    {"scales": u8(T, K // 32, device=1)}, {"values": Tensor(T, K, dtype="float32")}, {"values": Tensor(T, K + 1)},
    {"x": Tensor(T, 33), "codes": u8(T, 17), "scales": u8(T, 2)}])
def test_quantize_wrapper(ctx, kw):  # noqa: F811
    a = {"x": Tensor(T, K), "codes": u8(T, K // 2), "scales": u8(T, K // 32), "values": None, **kw}
    with pytest.raises(ValueError):
        ctx.mx_quantize_dev(a["x"], a["codes"], a["scales"], values_dev=a["values"])


def test_wrappers_take_the_calls(ctx):  # noqa: F811
    for dt in ("bfloat16", "int16", "float16", "float32"):
        with pytest.raises(AssertionError, match="rmoe_mx_quantize_dev"):
            ctx.mx_quantize_dev(Tensor(T, 33, dtype=dt), Tensor(T, 32, dtype="float4_e2m1fn_x2"),
                                Tensor(T, 2, dtype="float8_e8m0fnu"), values_dev=Tensor(T, 33, dtype=dt))
    with pytest.raises(AssertionError, match="rmoe_mx_linear_dev"):
        _linear(ctx)
    with pytest.raises(AssertionError, match="rmoe_mx_experts_linear_dev"):
        _experts(ctx)
    with pytest.raises(AssertionError, match="rmoe_residual_norm_dev"):
        _norm(ctx)
    for gate in (f32(H), f32(T, 1), Tensor(T, H)):
        with pytest.raises(AssertionError, match="rmoe_residual_norm_dev"):
            _norm(ctx, gate_dev=gate)


def _linear(ctx, **kw):  # noqa: F811
    a = {"x": u8(T, K // 2), "xs": u8(T, K // 32), "w": u8(M, K // 2), "ws": u8(M, K // 32), "y": Tensor(T, M), **kw}
    args = [a.pop(n) for n in ("x", "xs", "w", "ws", "y")]
    ctx.mx_linear_dev(*args, **a)


@pytest.mark.parametrize("kw", [
    {"x": u8(T * K)}, {"x": Tensor(T, K // 2)}, {"x": u8(T, K // 4)}, {"xs": u8(T, K // 16)}, {"w": u8(M, K)},
    {"ws": u8(M, K // 32, contiguous=False)}, {"ws": u8(M + 1, K // 32)}, {"w": u8(M, K // 2, device=1)},
    {"y": Tensor(T, M // 2)}, {"y": Tensor(T, M, dtype="float16")}, {"act": "swiglu"}, {"act": "relu"}, {"act": "situ"},
    {"act": "silu", "gate_beta": 4.0, "value_beta": 25.0}, {"bias_dev": f32(M + 1)}, {"bias_dev": Tensor(M)},
    {"residual_dev": Tensor(T, M + 1)}, {"residual_dev": Tensor(T, M, dtype="float32")}])
def test_linear_wrapper(ctx, kw):  # noqa: F811
    with pytest.raises(ValueError):
        _linear(ctx, **kw)


def _experts(ctx, **kw):  # noqa: F811
    a = {"x": u8(T, K // 2), "xs": u8(T, K // 32), "w": u8(E, M, K // 2), "ws": u8(E, M, K // 32), "off": i32(E + 1),
         "y": Tensor(T, M), **kw}
    args = [a.pop(n) for n in ("x", "xs", "w", "ws", "off", "y")]
    ctx.mx_experts_linear_dev(*args, **a)


@pytest.mark.parametrize("kw", [
    {"w": u8(M, K // 2)}, {"ws": u8(E, M, K)}, {"off": i32(E)}, {"off": Tensor(E + 1, dtype="int64")}, {"y": Tensor(T, M + 1)},
    {"bias_dev": f32(M)}, {"bias_dev": f32(E, M + 1)}, {"residual_dev": Tensor(T + 1, M)}, {"act": "swiglu"}])
def test_experts_wrapper(ctx, kw):  # noqa: F811
    with pytest.raises(ValueError):
        _experts(ctx, **kw)


def _norm(ctx, **kw):  # noqa: F811
    a = {"block": Tensor(T, H), "residual": Tensor(T, H), "y": Tensor(T, H), "pre_weight_dev": f32(H), "h_dev": Tensor(T, H), **kw}
    args = [a.pop(n) for n in ("block", "residual", "y")]
    ctx.residual_norm_dev(*args, **a)


@pytest.mark.parametrize("kw", [
    {"block": None}, {"y": None}, {"block": Tensor(T, H + 1)}, {"block": Tensor(T, H, dtype="float16")},
    {"residual": Tensor(T * H)}, {"y": Tensor(T, H, contiguous=False)}, {"h_dev": Tensor(T, H, device=1)},
    {"post_weight_dev": Tensor(H)}, {"pre_weight_dev": f32(H + 1)}, {"gate_dev": Tensor(H)}, {"gate_dev": f32(T)},
    {"gate_dev": f32(T, H)}, {"codes_dev": u8(T, 48)}, {"scales_dev": u8(T, 3)}, {"codes_dev": u8(T, 36), "scales_dev": u8(T, 3)}])
def test_norm_wrapper(ctx, kw):  # noqa: F811
    with pytest.raises(ValueError):
        _norm(ctx, **kw)


@pytest.mark.parametrize("kw", [
    {"dblock": None}, {"block": None}, {"dy": Tensor(T, H + 1)}, {"dh": f32(T, H)}, {"dgate_dev": f32(H)},
    {"gate_dev": f32(H), "dgate_dev": f32(T, 1)}, {"gate_dev": Tensor(T, H), "dgate_dev": f32(T, H)},
    {"dpre_weight_dev": f32(H + 1)}, {"post_weight_dev": f32(H), "dpost_weight_dev": Tensor(H)}, {"work": f32(10)},
    {"work": f32(2, 10000)}, {"work": Tensor(10000)}])
def test_backward_wrapper(ctx, monkeypatch, kw):  # noqa: F811
    monkeypatch.setattr("raon_npu_amd.device.Context.norm_backward_work", lambda *a: 3 * T * H)
    a = {"dy": Tensor(T, H), "dh": Tensor(T, H), "block": Tensor(T, H), "y": Tensor(T, H), "dblock": Tensor(T, H),
         "dresidual": Tensor(T, H), "work": f32(10000), "pre_weight_dev": f32(H), **kw}
    args = [a.pop(n) for n in ("dy", "dh", "block", "y", "dblock", "dresidual", "work")]
    with pytest.raises(ValueError):
        ctx.residual_norm_backward_dev(*args, **a)


# ------------------------------------------------------------ the C entry points --
P = [0x10000000 * (i + 1) for i in range(16)]  # addresses far apart; never followed
BF16, F32 = _lib.DT_BF16, _lib.DT_F32


@pytest.mark.parametrize("args,what", [
    ((P[0], 7, T, K, P[1], P[2], None), "element type"), ((P[0], BF16, 0, K, P[1], P[2], None), "T"),
    ((P[0], BF16, T, 0, P[1], P[2], None), "H"), ((P[0], BF16, 1, (1 << 30) + 1, P[1], P[2], None), "H"),
    ((None, BF16, T, K, P[1], P[2], None), "null"), ((P[0], BF16, T, K, None, P[2], None), "null"),
    ((P[0], BF16, T, K, P[1], None, None), "null"), ((P[0] + 1, BF16, T, K, P[1], P[2], None), "aligned"),
    ((P[0], F32, T, K, P[1], P[2], P[3] + 2), "aligned"), ((P[0], BF16, T, K, P[1] + 8, P[2], None), "16-byte"),
    ((P[0], BF16, T, K, P[0] + 32, P[2], None), "overlaps"), ((P[0], BF16, T, K, P[1], P[2], P[0] + 2), "overlaps"),
    ((P[0], BF16, T, K, P[1], P[1] + 16, None), "outputs overlap"), ((P[0], BF16, T, K, P[1], P[2], P[1]), "outputs overlap")])
def test_quantize_entry_point(raw, args, what):  # noqa: F811
    with pytest.raises(ValueError, match=what):
        raw("rmoe_mx_quantize_dev", *args, None)


def _linear_args(x=P[0], xs=P[1], n=T, k=K, w=P[2], ws=P[3], m=M, bias=P[4], act=_lib.ACT_NONE, gb=0.0, vb=0.0, residual=P[5],
                 y=P[6]):
    return x, xs, n, k, w, ws, m, bias, act, gb, vb, residual, y


@pytest.mark.parametrize("kw,what", [
    ({"x": None}, "null"), ({"ws": None}, "null"), ({"y": None}, "null"), ({"n": 0}, "rows"), ({"k": 0}, "K"), ({"k": 48}, "K"),
    ({"k": -32}, "K"), ({"m": 0}, "M"), ({"m": 47, "act": _lib.ACT_SWIGLU}, "M"), ({"act": 6}, "activation"), ({"act": -1}, "activation"),
    ({"act": _lib.ACT_SITU}, "betas"), ({"act": _lib.ACT_SITU, "gb": 4.0, "vb": float("nan")}, "betas"), ({"x": P[0] + 8}, "16-byte"),
    ({"w": P[2] + 1}, "16-byte"), ({"y": P[6] + 1}, "aligned"), ({"residual": P[5] + 1}, "aligned"), ({"bias": P[4] + 2}, "aligned"),
    ({"y": P[0] + 16}, "overlaps"), ({"y": P[3]}, "overlaps"), ({"y": P[4] + 4}, "overlaps"), ({"residual": P[6] + 2}, "overlaps")])
def test_linear_entry_point(raw, kw, what):  # noqa: F811
    a = _linear_args(**kw)
    with pytest.raises(ValueError, match=what):
        raw("rmoe_mx_linear_dev", *a, None)
    with pytest.raises(ValueError, match=what):
        raw("rmoe_mx_experts_linear_dev", *a[:7], P[7], E, *a[7:], None)


@pytest.mark.parametrize("off,e,what", [(None, E, "null"), (P[7], 0, "n_experts"), (P[7], 257, "n_experts"),
                                        (P[7] + 2, E, "aligned"), (P[6] + 8, E, "overlaps")])
def test_experts_entry_point(raw, off, e, what):  # noqa: F811
    a = _linear_args()
    with pytest.raises(ValueError, match=what):
        raw("rmoe_mx_experts_linear_dev", *a[:7], off, e, *a[7:], None)


def _norm_args(block=P[0], residual=P[1], dtype=BF16, t=T, h=H, post=P[2], gate=P[3], kind=_lib.GATE_COLUMN, scale=1.0, pre=P[4],
               eps=1e-6, y=P[5], out=P[6], codes=P[7], scales=P[8]):
    return block, residual, dtype, t, h, post, gate, kind, scale, pre, eps, y, out, codes, scales


@pytest.mark.parametrize("kw,what", [
    ({"dtype": 3}, "element type"), ({"t": 0}, "T"), ({"h": 0}, "H"), ({"h": 8193}, "H"), ({"eps": 0.0}, "eps"),
    ({"eps": float("nan")}, "eps"), ({"eps": float("inf")}, "eps"), ({"kind": 4}, "gate"), ({"kind": -1}, "gate"),
    ({"kind": _lib.GATE_NONE}, "gate"), ({"gate": None}, "gate"), ({"block": None, "y": None}, "with a block"),
    ({"residual": None}, "null"), ({"y": None}, "null"), ({"codes": None}, "together"), ({"scales": None}, "together"),
    ({"pre": None}, "pre_weight"), ({"out": None, "codes": None, "scales": None}, "pre_weight"),
    ({"block": None, "y": None, "gate": None, "kind": 0, "post": None, "pre": None, "out": None, "codes": None, "scales": None}, "neither"),
    ({"codes": P[7] + 4}, "16-byte"), ({"block": P[0] + 1}, "aligned"), ({"post": P[2] + 2}, "aligned to 4"),
    ({"gate": P[3] + 2}, "aligned to 4"), ({"gate": P[3] + 1, "kind": _lib.GATE_FULL}, "aligned"), ({"y": P[1] + 2}, "overlaps"),
    ({"out": P[1]}, "overlaps"), ({"out": P[0] + 2}, "overlaps"), ({"y": P[2]}, "overlaps"), ({"codes": P[0]}, "overlaps"),
    ({"out": P[5]}, "outputs overlap"), ({"y": P[0], "out": P[0]}, "outputs overlap"), ({"y": P[3], "kind": _lib.GATE_FULL}, "overlaps"),
    ({"scales": P[6] + 4}, "outputs overlap")])
def test_norm_entry_point(raw, kw, what):  # noqa: F811
    with pytest.raises(ValueError, match=what):
        raw("rmoe_residual_norm_dev", *_norm_args(**kw), None)


def _grad_args(dy=P[0], dh=P[1], block=P[2], y=P[3], dtype=BF16, t=T, h=H, post=P[4], gate=P[5], kind=_lib.GATE_ROW, scale=1.0,
               pre=P[6], eps=1e-6, dblock=P[7], dresidual=P[8], dpost=P[9], dgate=P[10], dpre=P[11], work=P[12]):
    return dy, dh, block, y, dtype, t, h, post, gate, kind, scale, pre, eps, dblock, dresidual, dpost, dgate, dpre, work


@pytest.mark.parametrize("kw,what", [
    ({"dtype": 5}, "element type"), ({"t": 0}, "T"), ({"h": 8193}, "H"), ({"eps": -1.0}, "eps"), ({"kind": 9}, "gate"),
    ({"y": None}, "null"), ({"dresidual": None}, "null"), ({"work": None}, "null"), ({"dblock": None}, "null"),
    ({"block": None}, "with a block"), ({"dy": None, "dh": None}, "neither"), ({"dh": None}, "pre_weight"), ({"pre": None}, "pre_weight"),
    ({"gate": None, "kind": 0}, "gradient goes"), ({"post": None}, "gradient goes"), ({"work": P[12] + 2}, "aligned to 4"),
    ({"dgate": P[10] + 1}, "aligned"), ({"dy": P[0] + 1}, "aligned"), ({"dblock": P[2]}, "overlaps"), ({"dresidual": P[3] + 2}, "overlaps"),
    ({"dresidual": P[7] + 2}, "outputs overlap"), ({"work": P[11] - 64}, "outputs overlap"), ({"dblock": P[0]}, "overlaps"),
    ({"dpre": P[5]}, "overlaps")])
def test_backward_entry_point(raw, kw, what):  # noqa: F811
    with pytest.raises(ValueError, match=what):
        raw("rmoe_residual_norm_backward_dev", *_grad_args(**kw), None)


def test_work_size():
    n = C.c_size_t()
    for bad in ((0, 8), (8, 0), (8, 8193)):
        with pytest.raises(ValueError):
            _lib.call("rmoe_norm_backward_work", *bad, C.byref(n))
    with pytest.raises(ValueError):
        _lib.call("rmoe_norm_backward_work", 1, 1, None)
    _lib.call("rmoe_norm_backward_work", 3, 10, C.byref(n))
    assert n.value >= 3 * 3 * 10


def test_null_context():
    lib = _lib.load()
    for name, n in (("rmoe_mx_quantize_dev", 8), ("rmoe_mx_linear_dev", 14), ("rmoe_mx_experts_linear_dev", 16),
                    ("rmoe_residual_norm_dev", 16), ("rmoe_residual_norm_backward_dev", 20)):
        with pytest.raises(ValueError, match="null context"):
            _lib.check(getattr(lib, name)(None, *([0] * n)))


@pytest.mark.parametrize("n,m,e", [((1 << 31) - 1, 1 << 16, None), (1 << 23, 1 << 18, None), (1000, 1 << 30, 256),
                                   ((1 << 31) - 1, 1 << 12, 256)])
@pytest.mark.parametrize("act", [_lib.ACT_NONE, _lib.ACT_SWIGLU])
def test_more_tiles_than_a_launch_takes(raw, n, m, e, act):  # noqa: F811
    """Refused before the device is looked at."""
    far = [1 << (48 + i) for i in range(8)]
    a = (far[0], far[1], n, 32, far[2], far[3], m, None), (act, 0.0, 0.0, None, far[5])
    with pytest.raises(ValueError, match="too many"):
        if e is None:
            raw("rmoe_mx_linear_dev", *a[0], *a[1], None)
        else:
            raw("rmoe_mx_experts_linear_dev", *a[0][:7], far[6], e, None, *a[1], None)
