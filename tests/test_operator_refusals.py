"""CPU: calls that the operators around the experts' products refuse, in the wrappers and in the C entry points.

A refused call reaches neither the device nor the context (a buffer stands in for it)."""

from __future__ import annotations

import ctypes as C
import types

import pytest

from raon_npu_amd import _lib
from raon_npu_amd.device import Context, Matrix, MoeLayer
from raon_npu_amd.geometry import MoeGeometry


class Tensor:
    """What the wrappers look at of a GPU tensor."""

    def __init__(self, *shape, dtype="bfloat16", device=0, contiguous=True, ptr=1 << 20):
        self.shape, self.dtype, self.is_cuda = shape, f"torch.{dtype}", True
        self.device = types.SimpleNamespace(index=device)
        self._c, self._p = contiguous, ptr

    def is_contiguous(self):
        return self._c

    def get_device(self):
        return self.device.index

    def data_ptr(self):
        return self._p


def i32(*shape, **kw):
    return Tensor(*shape, dtype="int32", **kw)


def f32(*shape, **kw):
    return Tensor(*shape, dtype="float32", **kw)


@pytest.fixture
def ctx(monkeypatch):
    """A context without a device; a call that passes the wrapper's checks is a test's failure."""
    class Library:
        def __getattr__(self, name):
            def entry(*a):
                raise AssertionError(f"{name} was called")

            return entry

    monkeypatch.setattr("raon_npu_amd._lib.load", Library)
    c = Context.__new__(Context)
    c._h, c.device = None, 0
    return c


T, k, E, H = 4, 2, 8, 64


def _sort(ctx, **kw):
    a = {"x": Tensor(T, H), "ids": i32(T, k), "rows": Tensor(T * k, H), "order": i32(T * k), "inv": i32(T, k),
         "offsets": i32(E + 1), **kw}
    ctx.sort_tokens_dev(a["x"], a["ids"], E, a["rows"], a["order"], a["inv"], a["offsets"])


@pytest.mark.parametrize("kw", [
    {"x": Tensor(T, H, dtype="float64")}, {"x": Tensor(T, H, contiguous=False)}, {"x": Tensor(T * H)},
    {"ids": Tensor(T, k, dtype="int64")}, {"ids": i32(T + 1, k)}, {"ids": i32(T * k)},
    {"rows": Tensor(T * k, H, dtype="float32")}, {"rows": Tensor(T * k - 1, H)}, {"rows": Tensor(T * k, H, device=1)},
    {"order": i32(T, k)}, {"inv": i32(T * k)}, {"offsets": i32(E)}, {"inv": i32(T, k, contiguous=False)}])
def test_sort_wrapper(ctx, kw):
    with pytest.raises(ValueError):
        _sort(ctx, **kw)


def test_sort_wrapper_takes_the_call(ctx):
    for dt in ("bfloat16", "int16", "float16", "float32"):
        with pytest.raises(AssertionError, match="rmoe_sort_tokens_dev"):
            _sort(ctx, x=Tensor(T, H, dtype=dt), rows=Tensor(T * k, H, dtype=dt))


@pytest.mark.parametrize("kw", [{"rows": Tensor(T * k + 1, H)}, {"inv": i32(T, k + 1)}, {"wts": f32(T, k + 1)},
                                {"wts": Tensor(T, k)}, {"out": Tensor(T, H, dtype="float16")}, {"out": Tensor(T, H + 1)},
                                {"out": Tensor(T, H, device=1)}])
def test_combine_wrappers(ctx, kw):
    a = {"rows": Tensor(T * k, H), "inv": i32(T, k), "wts": f32(T, k), "out": Tensor(T, H), **kw}
    with pytest.raises(ValueError):
        ctx.combine_tokens_dev(a["rows"], a["inv"], a["wts"], a["out"])
    with pytest.raises(ValueError):
        ctx.combine_tokens_backward_dev(a["out"], a["rows"], a["inv"], a["wts"], Tensor(T * k, H), f32(T, k))
    if "wts" not in kw:
        with pytest.raises(ValueError):
            ctx.sort_tokens_backward_dev(a["rows"], a["inv"], a["out"])


@pytest.mark.parametrize("kw", [
    {"act": "relu"}, {"act": "situ"}, {"act": "silu", "gate_beta": 4.0, "value_beta": 25.0},
    {"act": "situ", "gate_beta": 4.0}, {"act": "swiglu"}, {"bias_dev": f32(127)}, {"bias_dev": Tensor(128)},
    {"residual_dev": Tensor(3, 64)}, {"residual_dev": Tensor(3, 128, device=1)}, {"x": Tensor(2, 256)},
    {"x": Tensor(3, 256, dtype="float16")}, {"y": Tensor(3, 128, contiguous=False)}])
def test_linear_act_wrapper(ctx, kw):
    a = {"x": Tensor(3, 256), "y": Tensor(3, 128), **kw}
    x, y = a.pop("x"), a.pop("y")
    with pytest.raises(ValueError):
        Matrix(ctx, 1, 128, 256).linear_act_dev(x, 3, y, **a)


@pytest.mark.parametrize("kw", [
    {"part": "up"}, {"act": "swiglu"}, {"offsets": i32(8)}, {"offsets": Tensor(9, dtype="int64")}, {"y": Tensor(5, 256)},
    {"bias_dev": f32(512)}, {"bias_dev": f32(9, 512)}, {"residual_dev": Tensor(4, 512)}, {"rows": Tensor(5 * 256)}])
def test_experts_linear_wrapper(ctx, kw):
    lyr = MoeLayer(ctx, 0, MoeGeometry(hidden=256, inter=256, n_routed=8, top_k=2))
    a = {"part": "gate_up", "rows": Tensor(5, 256), "offsets": i32(9), "y": Tensor(5, 512), **kw}
    part, rows, off, y = (a.pop(n) for n in ("part", "rows", "offsets", "y"))
    with pytest.raises(ValueError):
        lyr.experts_linear_dev(part, rows, off, y, **a)


# ------------------------------------------------------------ the C entry points --
@pytest.fixture
def raw():
    """(a stand-in for a context, call(name, *args) -> raises what the status maps to)."""
    held = C.create_string_buffer(4096)
    lib = _lib.load()
    return lambda name, *a: _lib.check(getattr(lib, name)(C.addressof(held), *a))


P = [0x10000000 * (i + 1) for i in range(8)]  # addresses far apart; never followed
BF16, F32 = _lib.DT_BF16, _lib.DT_F32


@pytest.mark.parametrize("args,what", [
    ((P[0], 3, T, H, P[1], k, E, P[2], P[3], P[4], P[5]), "element type"),
    ((P[0], BF16, 0, H, P[1], k, E, P[2], P[3], P[4], P[5]), "T"),
    ((P[0], BF16, T, 0, P[1], k, E, P[2], P[3], P[4], P[5]), "H"),
    ((P[0], BF16, 1, (1 << 30) + 1, P[1], k, E, P[2], P[3], P[4], P[5]), "H"),
    ((P[0], BF16, T, H, P[1], 0, E, P[2], P[3], P[4], P[5]), "k"),
    ((P[0], BF16, T, H, P[1], 17, E, P[2], P[3], P[4], P[5]), "k"),
    ((P[0], BF16, 1 << 30, H, P[1], 2, E, P[2], P[3], P[4], P[5]), "too many"),
    ((P[0] + 1, BF16, T, H, P[1], k, E, P[2], P[3], P[4], P[5]), "aligned"),
    ((P[0] + 2, F32, T, H, P[1], k, E, P[2], P[3], P[4], P[5]), "aligned"),
    ((P[0], BF16, T, H, P[1] + 2, k, E, P[2], P[3], P[4], P[5]), "aligned to 4"),
    ((P[0], BF16, T, H, P[1], k, E, P[2], P[3] + 1, P[4], P[5]), "aligned to 4"),
    ((P[0], BF16, T, H, P[1], k, E, P[2], P[3], P[4], P[5] + 2), "aligned to 4"),
    ((P[0], BF16, T, H, P[1], k, 0, P[2], P[3], P[4], P[5]), "n_experts"),
    ((P[0], BF16, T, H, P[1], k, 257, P[2], P[3], P[4], P[5]), "n_experts"),
    ((None, BF16, T, H, P[1], k, E, P[2], P[3], P[4], P[5]), "null"),
    ((P[0], BF16, T, H, P[1], k, E, P[2], P[3], P[4], None), "null"),
    ((P[0], BF16, T, H, P[1], k, E, P[0] + 2 * H, P[3], P[4], P[5]), "overlaps"),
    ((P[0], BF16, T, H, P[1], k, E, P[2], P[3], P[1], P[5]), "overlaps"),
    ((P[0], BF16, T, H, P[1], k, E, P[2], P[3], P[3] + 4, P[5]), "outputs overlap")])
def test_sort_entry_point(raw, args, what):
    with pytest.raises(ValueError, match=what):
        raw("rmoe_sort_tokens_dev", *args, None)


@pytest.mark.parametrize("name,args,what", [
    ("rmoe_sort_tokens_backward_dev", (P[0], 9, T, H, P[1], k, P[2]), "element type"),
    ("rmoe_sort_tokens_backward_dev", (P[0], BF16, T, H, P[1], k, P[0]), "overlaps"),
    ("rmoe_sort_tokens_backward_dev", (P[0], BF16, T, H, None, k, P[2]), "null"),
    ("rmoe_combine_tokens_dev", (P[0], BF16, T, H, P[1], None, k, P[2]), "null"),
    ("rmoe_sort_tokens_backward_dev", (P[0], BF16, T, H, P[1] + 2, k, P[2]), "aligned to 4"),
    ("rmoe_combine_tokens_dev", (P[0], BF16, T, H, P[1], P[3] + 2, k, P[2]), "aligned to 4"),
    ("rmoe_combine_tokens_backward_dev", (P[0], P[1], BF16, T, H, P[2], P[3], k, P[4], P[5] + 2), "aligned to 4"),
    ("rmoe_combine_tokens_dev", (P[0], BF16, T, H, P[1], P[3], 17, P[2]), "k"),
    ("rmoe_combine_tokens_dev", (P[0], BF16, T, H, P[1], P[3], k, P[0] + 64), "overlaps"),
    ("rmoe_combine_tokens_backward_dev", (P[0], P[1], BF16, T, H, P[2], P[3], k, P[1], P[5]), "overlaps"),
    ("rmoe_combine_tokens_backward_dev", (P[0], P[1], BF16, T, H, P[2], P[3], k, P[4], P[4]), "outputs overlap"),
    ("rmoe_combine_tokens_backward_dev", (P[0], P[1], BF16, T, H, P[2], P[3], k, P[4], None), "null"),
    ("rmoe_combine_tokens_backward_dev", (P[0], P[1], F32, T, H, P[2], P[3], k, P[4] + 2, P[5]), "aligned")])
def test_sum_entry_points(raw, name, args, what):
    with pytest.raises(ValueError, match=what):
        raw(name, *args, None)


def test_null_context():
    lib = _lib.load()
    for name, n in (("rmoe_sort_tokens_dev", 12), ("rmoe_combine_tokens_dev", 9), ("rmoe_linear_act_dev", 11),
                    ("rmoe_experts_linear_dev", 13), ("rmoe_reserve_linear_act", 2), ("rmoe_reserve_experts_linear", 2)):
        with pytest.raises(ValueError, match="null context"):
            _lib.check(getattr(lib, name)(None, *([0] * n)))
