"""GPU: the norms before and after a block with gate and residual scale (csrc/block_norm.hip) against the formulas in 64
bits, and their gradients also against differences.

Bounds, with u = 2^-24.  A row's sum of H squares: each thread adds up to 16 of them, then 6 + 8 additions join the lanes
and waves, so it is off by at most 32 u of itself; (.)^-1/2 halves that and adds a division, a root and a division: n and m
are off by 20 u of themselves.  y is off by 24 u (|g u| + |scale r|), then one rounding (finfo.eps / 2 of the result and half
the type's least subnormal); h likewise by 24 u |h| and one rounding.  In the gradient D = dy + m a - y m^3 S / H, S = sum a
y: 128 u of the sum A of its terms' magnitudes (m^3: 60; S: 32 of sum |a y|; products and sums: the rest); dblock by twice
that bound carried through its own two terms.  Columns' sums over T rows add up to T / 512 + 40 more values: (T / 512 + 168)
2 u of the sum of the magnitudes."""

from __future__ import annotations

import numpy as np
import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = [torch.bfloat16, torch.float16, torch.float32]
U = 2.0 ** -24
EPS = 1e-5
GATES = ["none", "column", "row", "full"]


def _stream():
    return torch.cuda.current_stream()


def _half_step(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def _case(T, H, dtype, post, gate, seed):
    g = torch.Generator().manual_seed(seed)
    s = {"block": torch.randn(T, H, generator=g).to(dtype), "residual": (3 * torch.randn(T, H, generator=g)).to(dtype),
         "post": 1 + 0.3 * torch.randn(H, generator=g) if post else None, "pre": 1 + 0.3 * torch.randn(H, generator=g),
         "dy": torch.randn(T, H, generator=g).to(dtype), "dh": torch.randn(T, H, generator=g).to(dtype)}
    s["gate"] = {"none": None, "column": 0.5 * torch.randn(H, generator=g), "row": 0.5 * torch.randn(T, 1, generator=g),
                 "full": (0.5 * torch.randn(T, H, generator=g)).to(dtype)}[gate]
    return s


def _dev(s):
    return {k: None if v is None else v.cuda() for k, v in s.items()}


def _n(x):
    return (x.square().mean(1, keepdim=True) + EPS).rsqrt()


def _forward64(s, scale):
    """(y, magnitude of its terms) in 64 bits."""
    b, r = s["block"].double(), s["residual"].double()
    u = b if s["post"] is None else b * _n(b) * s["post"].double()
    if s["gate"] is not None:
        u = u * s["gate"].double()
    return scale * r + u, u.abs() + (scale * r).abs()


def _run(ctx, d, scale, y=None, h=None, codes=None, scales=None, stream=None):
    y = torch.full_like(d["block"], 7) if y is None else y
    ctx.residual_norm_dev(d["block"], d["residual"], y, post_weight_dev=d["post"], gate_dev=d["gate"], scale=scale,
                          pre_weight_dev=None if h is None and codes is None else d["pre"], h_dev=h, codes_dev=codes, scales_dev=scales, eps=EPS,
                          stream=stream or _stream())
    return y


def _check_h(h, y, pre, dtype):
    want = y.double() * _n(y.double()) * pre.double()
    rel, least = _half_step(dtype)
    off, bound = (h.double() - want).abs(), want.abs() * (24 * U + rel * (1 + 2.0 ** -10)) + least
    assert bool((off <= bound).all()), float((off / bound).max())


SHAPES = [(1, 1), (1, 7), (3, 8), (2, 33), (5, 64), (1, 2048), (17, 511), (9, 520), (445, 2560), (4, 4096), (3, 4097), (2, 8192),
          (6, 5001), (2, 8191), (64, 4104), (33, 7000), (40, 2568)]


@pytest.mark.parametrize("T,H", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("post,gate", [(True, "column"), (False, "none"), (True, "row"), (False, "full"), (True, "none")])
def test_forward(gpu_ctx, T, H, dtype, post, gate):
    s = _case(T, H, dtype, post, gate, T + H)
    d, scale = _dev(s), 0.75
    P = -(-H // 32) * 32
    h = torch.full_like(d["block"], 7)
    codes = torch.full((T, P // 2), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((T, P // 32), 0xEE, dtype=torch.uint8, device="cuda")
    y = _run(gpu_ctx, d, scale, h=h, codes=codes, scales=scales)
    want, size = _forward64(s, scale)
    rel, least = _half_step(dtype)
    off, bound = (y.cpu().double() - want).abs(), 24 * U * size + want.abs() * rel * (1 + 2.0 ** -10) + least
    assert bool((off <= bound).all()), float((off / bound).max())
    _check_h(h.cpu(), y.cpu(), s["pre"], dtype)
    # The codes are those of the stored rows; by themselves, and without h, the same.
    c2, s2 = torch.zeros_like(codes), torch.zeros_like(scales)
    gpu_ctx.mx_quantize_dev(h, c2, s2, stream=_stream())
    assert torch.equal(codes, c2) and torch.equal(scales, s2)
    codes.fill_(0xEE), scales.fill_(0xEE)
    assert torch.equal(_run(gpu_ctx, d, scale, codes=codes, scales=scales), y)
    assert torch.equal(codes, c2) and torch.equal(scales, s2)
    # Without a norm before; the norm of the stored rows alone.
    assert torch.equal(_run(gpu_ctx, d, scale), y)
    h2 = torch.full_like(h, 7)
    gpu_ctx.norm_dev(y, d["pre"], h2, eps=EPS, stream=_stream())
    assert torch.equal(h, h2)
    codes.fill_(0xEE), scales.fill_(0xEE)
    gpu_ctx.norm_dev(y, d["pre"], codes_dev=codes, scales_dev=scales, eps=EPS, stream=_stream())
    assert torch.equal(codes, c2) and torch.equal(scales, s2)
    # In place: y over the residual and h over the block, y over the block.
    e = _dev(s)
    _run(gpu_ctx, e, scale, y=e["residual"], h=e["block"])
    assert torch.equal(e["residual"], y) and torch.equal(e["block"], h)
    e = _dev(s)
    _run(gpu_ctx, e, scale, y=e["block"], h=h2)
    assert torch.equal(e["block"], y) and torch.equal(h2, h)


def test_rows_of_zeros_infinities_and_nan(gpu_ctx):
    """A row of zeros has the norm 0; NaN and infinities stay in their rows."""
    for dtype in TYPES:
        s = _case(6, 96, dtype, True, "none", 1)
        s["block"][1] = 0.0
        s["residual"][1] = 0.0
        s["block"][2, 5], s["block"][3, 7], s["residual"][4, 0] = float("nan"), float("inf"), float("inf")
        h = torch.empty(6, 96, dtype=dtype, device="cuda")
        y = _run(gpu_ctx, _dev(s), 1.0, h=h)
        assert not y[1].any() and not h[1].any()
        assert bool(torch.isfinite(h[[0, 1, 5]]).all()) and bool(torch.isfinite(y[[0, 1, 5]]).all())
        assert bool(torch.isnan(y[2]).all()) and bool(torch.isnan(h[2]).all())
        assert bool(torch.isnan(y[3, 7])) and bool(torch.isnan(h[3]).all())
        assert bool(torch.isinf(y[4, 0])) and bool(torch.isnan(h[4, 0])) and not h[4, 1:].any()


def test_rows_at_any_address(gpu_ctx):
    """Rows that start inside 16 bytes give the bits of aligned ones; vectors that do, too."""
    T, H = 5, 136
    for dtype in TYPES:
        s = _case(T, H, dtype, True, "full", 3)
        d = _dev(s)
        h = torch.empty_like(d["block"])
        y = _run(gpu_ctx, d, 0.5, h=h)

        def shifted(t):
            buf = torch.zeros(t.numel() + 9, dtype=t.dtype, device="cuda")
            v = buf[3:3 + t.numel()].view(t.shape)
            v.copy_(t)
            return v

        e = {k: None if v is None else shifted(v) for k, v in d.items()}
        h2 = shifted(torch.zeros_like(h))
        assert torch.equal(_run(gpu_ctx, e, 0.5, y=shifted(torch.zeros_like(y)), h=h2), y) and torch.equal(h, h2)
        a, b = _backward(gpu_ctx, d, y, "full", 0.5), _backward(gpu_ctx, e, shifted(y), "full", 0.5)
        for k in a:
            assert torch.equal(a[k], b[k]), k


# -------------------------------------------------------------------- gradients --
def _backward(ctx, d, y, gate, scale, dy=True, dh=True, out=None, stream=None, work=None):
    T, H = y.shape
    o = {"dblock": torch.full_like(y, 7), "dresidual": torch.full_like(y, 7)} if out is None else out
    if dh:
        o["dpre"] = torch.full((H,), 7.0, device="cuda")
    if d["post"] is not None:
        o["dpost"] = torch.full((H,), 7.0, device="cuda")
    if gate != "none":
        o["dgate"] = torch.full_like(d["gate"], 7)
    work = torch.full((ctx.norm_backward_work(T, H),), float("nan"), device="cuda") if work is None else work
    ctx.residual_norm_backward_dev(d["dy"] if dy else None, d["dh"] if dh else None, d["block"], y, o["dblock"],
                                   o["dresidual"], work, post_weight_dev=d["post"], dpost_weight_dev=o.get("dpost"),
                                   gate_dev=d["gate"], dgate_dev=o.get("dgate"), scale=scale,
                                   pre_weight_dev=d["pre"] if dh else None, dpre_weight_dev=o.get("dpre"), eps=EPS,
                                   stream=stream or _stream())
    return o


def _backward64(s, y, gate, scale, dy=True, dh=True):
    """{name: (gradient, magnitude of its terms)} in 64 bits."""
    b, y = s["block"].double(), y.double()
    T, H = b.shape
    zero = torch.zeros_like(b)
    dyv, dhv = s["dy"].double() if dy else zero, s["dh"].double() if dh else zero
    out, D, A = {}, dyv, dyv.abs()
    if dh:
        m, a = _n(y), dhv * s["pre"].double()
        D = D + m * a - y * m ** 3 * (a * y).mean(1, keepdim=True)
        A = A + (m * a).abs() + y.abs() * m ** 3 * (a * y).abs().mean(1, keepdim=True)
        out["dpre"] = ((dhv * y * m).sum(0), (dhv * y * m).abs().sum(0))
    out["dresidual"] = (scale * D, scale * A)
    g = 1.0 if s["gate"] is None else s["gate"].double()
    ga = 1.0 if s["gate"] is None else g.abs()
    n, w = (_n(b), s["post"].double()) if s["post"] is not None else (1.0, 1.0)
    wa = w.abs() if s["post"] is not None else 1.0
    u = b * n * w
    if gate != "none":
        dims = {"column": 0, "row": 1, "full": None}[gate]
        out["dgate"] = (D * u, A * u.abs()) if dims is None else ((D * u).sum(dims, keepdim=gate == "row"),
                                                                  (A * u.abs()).sum(dims, keepdim=gate == "row"))
    du, dA = g * D, ga * A
    if s["post"] is None:
        out["dblock"] = (du, dA)
    else:
        v, vA = du * w, dA * wa
        out["dblock"] = (n * v - b * n ** 3 * (v * b).mean(1, keepdim=True),
                         n * vA + b.abs() * n ** 3 * (vA * b.abs()).mean(1, keepdim=True))
        out["dpost"] = ((du * b * n).sum(0), (dA * (b * n).abs()).sum(0))
    return out


def _check_gradients(got, want, T, dtype):
    rel, least = _half_step(dtype)
    for k, (v, size) in want.items():
        g = got[k].cpu()
        if k in ("dpre", "dpost") or g.dtype == torch.float32 and k == "dgate" and dtype != torch.float32:
            bound = (T / 512 + 168 + (64 if k == "dgate" else 0)) * 2 * U * size + 1e-40
        else:
            bound = 512 * U * size + v.abs() * rel * (1 + 2.0 ** -10) + least
            if k == "dgate":  # fp32 rows: full gates, or sums of them
                bound = bound + (T / 512 + 232) * 2 * U * size
        off = (g.double() - v).abs()
        assert bool((off <= bound).all()), (k, float((off / bound).max()))


@pytest.mark.parametrize("T,H", [(1, 1), (1, 7), (2, 33), (5, 64), (1, 2048), (17, 511), (445, 520), (1030, 96), (9, 2560), (3, 4097),
                                 (2, 8192), (600, 5001), (64, 4104), (300, 7000), (40, 2568)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("post,gate", [(True, "column"), (False, "none"), (True, "row"), (False, "full"), (True, "none"),
                                       (False, "column"), (True, "full")])
def test_backward(gpu_ctx, T, H, dtype, post, gate):
    s = _case(T, H, dtype, post, gate, T + H + 1)
    d, scale = _dev(s), 0.75
    y = _run(gpu_ctx, d, scale)
    got = _backward(gpu_ctx, d, y, gate, scale)
    _check_gradients(got, _backward64(s, y.cpu(), gate, scale), T, dtype)
    again = _backward(gpu_ctx, d, y, gate, scale)
    for k in got:
        assert torch.equal(got[k], again[k]), k
    if T * H < 10000:
        for dy, dh in ((True, False), (False, True)):
            part = _backward(gpu_ctx, d, y, gate, scale, dy=dy, dh=dh)
            _check_gradients(part, _backward64(s, y.cpu(), gate, scale, dy=dy, dh=dh), T, dtype)
    # In place: dresidual over dy, dblock over dh.
    e = _dev(s)
    _backward(gpu_ctx, e, y, gate, scale, out={"dresidual": e["dy"], "dblock": e["dh"]})
    assert torch.equal(e["dy"], got["dresidual"]) and torch.equal(e["dh"], got["dblock"])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,H", [(1, 5), (70, 264)])
def test_norm_backward(gpu_ctx, T, H, dtype):
    s = _case(T, H, dtype, False, "none", 5)
    d = _dev(s)
    x, work = d["residual"], torch.empty(gpu_ctx.norm_backward_work(T, H), device="cuda")
    dx, dw = torch.empty_like(x), torch.empty(H, device="cuda")
    for dy in (False, True):
        gpu_ctx.norm_backward_dev(d["dh"], x, d["pre"], dx, work, dweight_dev=dw, dy_dev=d["dy"] if dy else None, eps=EPS,
                                  stream=_stream())
        want = _backward64(s, s["residual"], "none", 1.0, dy=dy)
        _check_gradients({"dresidual": dx, "dpre": dw}, {k: want[k] for k in ("dresidual", "dpre")}, T, dtype)


@pytest.mark.parametrize("post,gate", [(True, "column"), (True, "row"), (False, "full"), (True, "none")])
def test_gradients_against_differences(gpu_ctx, post, gate):
    """Along random directions: (L(x + t d) - L(x - t d)) / 2 t in 64 bits, L = <dy, y> + <dh, h>, with fp32 gradients.  The
    difference is off by O(t^2) (t = 1e-4: under 1e-6 of the terms) and its cancellation (1e-12); the gradients by 2^-14."""
    T, H, scale, t = 6, 72, 0.75, 1e-4
    s = _case(T, H, torch.float32, post, gate, 11)
    d = _dev(s)
    y64 = _forward64(s, scale)[0]
    y = y64.float()
    got = _backward(gpu_ctx, d, y.cuda(), gate, scale)

    def loss(p):
        y = _forward64(p, scale)[0]
        return float((s["dy"].double() * y).sum() + (s["dh"].double() * (y * _n(y) * p["pre"].double())).sum())

    g = torch.Generator().manual_seed(2)
    for name, grad in (("block", "dblock"), ("residual", "dresidual"), ("post", "dpost"), ("pre", "dpre"), ("gate", "dgate")):
        if s[name] is None:
            continue
        direction = torch.randn(s[name].shape, generator=g, dtype=torch.float64)
        up, down = dict(s), dict(s)
        up[name], down[name] = s[name].double() + t * direction, s[name].double() - t * direction
        want = (loss(up) - loss(down)) / (2 * t)
        along = got[grad].cpu().double() * direction
        assert abs(float(along.sum()) - want) <= 2.0 ** -14 * float(along.abs().sum()) + 1e-6, name


def test_on_other_streams_and_captured(gpu_ctx):
    """Forward and backward in a graph of another stream, replayed between eager calls with new inputs."""
    T, H = 37, 320
    d = _dev(_case(T, H, torch.bfloat16, True, "column", 1))
    y, h = torch.zeros_like(d["block"]), torch.zeros_like(d["block"])
    work = torch.empty(gpu_ctx.norm_backward_work(T, H), device="cuda")
    out = {"dblock": torch.zeros_like(y), "dresidual": torch.zeros_like(y)}
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph, stream=st):
        _run(gpu_ctx, d, 0.5, y=y, h=h, stream=torch.cuda.current_stream())
        out = _backward(gpu_ctx, d, y, "column", 0.5, out=out, stream=torch.cuda.current_stream(), work=work)
    for turn in range(3):
        new = _case(T, H, torch.bfloat16, True, "column", 100 + turn)
        for k, v in new.items():
            d[k].copy_(v)
        torch.cuda.synchronize()
        with torch.cuda.stream(st):
            graph.replay()
        torch.cuda.synchronize()
        h2 = torch.empty_like(h)
        y2 = _run(gpu_ctx, d, 0.5, h=h2)
        assert torch.equal(y, y2) and torch.equal(h, h2)
        for k, v in _backward(gpu_ctx, d, y2, "column", 0.5).items():
            assert torch.equal(out[k], v), k


def test_past_32_bits(gpu_ctx):
    """Rows past 2^32 bytes and 2^31 elements: the last ones are normalised, and have the gradients, that they have alone."""
    T, H, n = 530_000, 4096, 300
    d = {k: torch.zeros(T, H, dtype=torch.bfloat16, device="cuda") for k in ("block", "residual", "dy", "dh")}
    few = _dev(_case(n, H, torch.bfloat16, True, "column", 5))
    for k in d:
        d[k][-n:] = few[k]
    d.update({k: few[k] for k in ("post", "pre", "gate")})
    y, h = torch.zeros_like(d["block"]), torch.zeros_like(d["block"])
    _run(gpu_ctx, d, 0.75, y=y, h=h)
    h2 = torch.zeros_like(few["block"])
    y2 = _run(gpu_ctx, few, 0.75, h=h2)
    assert torch.equal(y[-n:], y2) and torch.equal(h[-n:], h2) and not y[:-n].any() and not h[:-n].any()
    del h
    a, b = _backward(gpu_ctx, d, y, "column", 0.75), _backward(gpu_ctx, few, y2, "column", 0.75)
    for k in ("dblock", "dresidual"):
        assert torch.equal(a[k][-n:], b[k]) and not a[k][:-n].any()
    for k in ("dpre", "dpost", "dgate"):  # the rows are dealt to other groups: another order of the sums
        size = _backward64({k: None if v is None else v.cpu() for k, v in few.items()}, y2.cpu(), "column", 0.75)[k][1]
        assert bool(((a[k] - b[k]).abs().cpu().double() <= (T / 512 + 168) * 4 * U * size).all()), k


@pytest.mark.parametrize("H", [40, 1000, 1536, 2048, 2560, 2568, 4104, 5000, 5128, 8192, 2559])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("post,gate", [(True, "column"), (True, "row"), (False, "none"), (True, "full")])
def test_many_rows(gpu_ctx, H, dtype, post, gate):
    """Rows of many are held by fewer waves: the same bits as of few, in place too, and right."""
    T = 3009
    s = _case(T, H, dtype, post, gate, H)
    d = _dev(s)
    h = torch.full_like(d["block"], 7)
    codes = torch.full((T, -(-H // 32) * 16), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((T, -(-H // 32)), 0xEE, dtype=torch.uint8, device="cuda")
    y = _run(gpu_ctx, d, 0.75, h=h, codes=codes, scales=scales)
    some = slice(0, T, 100)
    part = {k: v[some] if v is not None and v.shape[0] == T else v for k, v in s.items()}
    want, size = _forward64(part, 0.75)
    rel, least = _half_step(dtype)
    off, bound = (y[some].cpu().double() - want).abs(), 24 * U * size + want.abs() * rel * (1 + 2.0 ** -10) + least
    assert bool((off <= bound).all()), float((off / bound).max())
    _check_h(h[some].cpu(), y[some].cpu(), s["pre"], dtype)
    for a in range(0, T, 1003):
        few = {k: v[a:a + 1003].contiguous() if v is not None and v.shape[0] == T else v for k, v in d.items()}
        h1 = torch.full_like(few["block"], 7)
        c1, s1 = torch.zeros_like(codes[:1003]), torch.zeros_like(scales[:1003])
        assert torch.equal(_run(gpu_ctx, few, 0.75, h=h1, codes=c1, scales=s1), y[a:a + 1003])
        assert torch.equal(h1, h[a:a + 1003]) and torch.equal(c1, codes[a:a + 1003]) and torch.equal(s1, scales[a:a + 1003])
    h2, c2, s2 = torch.full_like(h, 7), torch.zeros_like(codes), torch.zeros_like(scales)
    gpu_ctx.norm_dev(y, d["pre"], h2, c2, s2, eps=EPS, stream=_stream())
    assert torch.equal(h, h2) and torch.equal(codes, c2) and torch.equal(scales, s2)
    gpu_ctx.norm_dev(y, d["pre"], codes_dev=c2.zero_(), scales_dev=s2.zero_(), eps=EPS, stream=_stream())
    assert torch.equal(codes, c2) and torch.equal(scales, s2)
    e = _dev(s)
    _run(gpu_ctx, e, 0.75, y=e["residual"], h=e["block"])
    assert torch.equal(e["residual"], y) and torch.equal(e["block"], h)
    e = _dev(s)
    _run(gpu_ctx, e, 0.75, y=e["block"], h=h2)
    assert torch.equal(e["block"], y) and torch.equal(h2, h)


def test_vectors_at_any_address_beside_aligned_rows(gpu_ctx):
    for T in (9, 3001):
        for dtype in TYPES:
            d = _dev(_case(T, 264, dtype, True, "column", 7))
            h = torch.empty_like(d["block"])
            y = _run(gpu_ctx, d, 0.5, h=h)
            e = dict(d)
            for k in ("post", "gate", "pre"):
                buf = torch.full((264 + 9,), float("nan"), device="cuda")
                e[k] = buf[3:3 + 264]
                e[k].copy_(d[k])
            h2 = torch.empty_like(h)
            assert torch.equal(_run(gpu_ctx, e, 0.5, h=h2), y) and torch.equal(h, h2)
            a, b = _backward(gpu_ctx, d, y, "column", 0.5), _backward(gpu_ctx, e, y, "column", 0.5)
            for k in a:
                assert torch.equal(a[k], b[k]), k


def test_more_rows_than_a_launch_takes(gpu_ctx):
    T, H, n = (1 << 26) + 70, 8, 200
    g = torch.Generator().manual_seed(2)
    few, w = torch.randn(n, H, generator=g).to(torch.bfloat16).cuda(), torch.randn(H, generator=g).cuda()
    x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
    x[:n], x[-n:] = few, few
    h, h2 = torch.full_like(x, 7), torch.full_like(few, 7)
    gpu_ctx.norm_dev(few, w, h2, eps=EPS, stream=_stream())
    gpu_ctx.norm_dev(x, w, h, eps=EPS, stream=_stream())
    assert torch.equal(h[:n], h2) and torch.equal(h[-n:], h2) and not h[n:-n].any()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32], ids=str)
@pytest.mark.parametrize("H", [72, 2560, 4104])
@pytest.mark.parametrize("row,grad,eps", [(55, 10, 1e-5), (54, -10, 1e-5), (-63, -10, 2.0 ** -126), (-55, -20, 2.0 ** -110)])
def test_gradients_of_rows_far_from_one(gpu_ctx, dtype, H, row, grad, eps):
    """Rows of 2^55, and of 2^-63 with an eps as small: the cube of their inverse root, times the row's sum, leaves fp32, the
    gradients do not.  Rows of 2^row through both norms, dh of 2^grad: dresidual is about 2^(grad - row), dblock 2^(grad - 2 row).
    Bounds as above: 512 u of the terms' magnitudes and one rounding."""
    T = 9
    s = _case(T, H, dtype, True, "none", H)
    for k, e in (("block", row), ("residual", row), ("dh", grad)):
        s[k] = (s[k].double() * 2.0 ** e).to(dtype)
    d = _dev(s)
    y = s["residual"]
    dblock, dresidual = torch.full_like(d["block"], 7), torch.full_like(d["block"], 7)
    dpre, dpost = torch.empty(H, device="cuda"), torch.empty(H, device="cuda")
    gpu_ctx.residual_norm_backward_dev(None, d["dh"], d["block"], d["residual"], dblock, dresidual,
                                       torch.empty(gpu_ctx.norm_backward_work(T, H), device="cuda"), post_weight_dev=d["post"],
                                       dpost_weight_dev=dpost, pre_weight_dev=d["pre"], dpre_weight_dev=dpre, eps=eps,
                                       stream=_stream())
    e32 = float(np.float32(eps))
    b, y, dh, pre, post = (t.double() for t in (s["block"], y, s["dh"], s["pre"], s["post"]))
    m, n = (y.square().mean(1, keepdim=True) + e32).rsqrt(), (b.square().mean(1, keepdim=True) + e32).rsqrt()
    a = dh * pre
    D = m * (a - y * m * (m * (a * y).mean(1, keepdim=True)))
    A = m * (a.abs() + (y * m).abs() * (m * (a * y).abs().mean(1, keepdim=True)))
    v, vA = D * post, A * post.abs()
    db = n * (v - b * n * (n * (v * b).mean(1, keepdim=True)))
    dbA = n * (vA + (b * n).abs() * (n * (vA * b.abs()).mean(1, keepdim=True)))
    want = {"dresidual": (D, A), "dblock": (db, dbA), "dpre": ((dh * y * m).sum(0), (dh * y * m).abs().sum(0)),
            "dpost": ((D * b * n).sum(0), (A * (b * n).abs()).sum(0))}
    _check_gradients({"dresidual": dresidual, "dblock": dblock, "dpre": dpre, "dpost": dpost}, want, T, dtype)


@pytest.mark.parametrize("T,H", [(445, 2560), (4099, 2048), (2500, 264), (2500, 259), (700, 1536), (600, 4096), (600, 4095)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("post,gate", [(True, "column"), (True, "row"), (True, "full"), (False, "none")])
def test_backward_of_more_rows_than_a_pass_takes(gpu_ctx, T, H, dtype, post, gate):
    """Workgroups that go on to further rows, the next one requested while a row is worked on: of one to eight waves a row,
    the last pass with rows for some of the workgroups and some of a workgroup's waves; in place too, where the next row's
    gradients have been read when a row's are written."""
    s = _case(T, H, dtype, post, gate, T + H + 2)
    d, scale = _dev(s), 0.75
    y = _run(gpu_ctx, d, scale)
    got = _backward(gpu_ctx, d, y, gate, scale)
    _check_gradients(got, _backward64(s, y.cpu(), gate, scale), T, dtype)
    e = _dev(s)
    _backward(gpu_ctx, e, y, gate, scale, out={"dresidual": e["dy"], "dblock": e["dh"]})
    assert torch.equal(e["dy"], got["dresidual"]) and torch.equal(e["dh"], got["dblock"])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("T,H", [(300, 2560), (2500, 264), (300, 5000), (40, 8191)])
def test_norm_backward_of_many_rows(gpu_ctx, T, H, dtype):
    """Without a block, dx over dy too."""
    s = _case(T, H, dtype, False, "none", 6)
    d = _dev(s)
    x, work = d["residual"], torch.empty(gpu_ctx.norm_backward_work(T, H), device="cuda")
    dx, dw = torch.empty_like(x), torch.empty(H, device="cuda")
    for dy in (False, True):
        gpu_ctx.norm_backward_dev(d["dh"], x, d["pre"], dx, work, dweight_dev=dw, dy_dev=d["dy"] if dy else None, eps=EPS,
                                  stream=_stream())
        want = _backward64(s, s["residual"], "none", 1.0, dy=dy)
        _check_gradients({"dresidual": dx, "dpre": dw}, {k: want[k] for k in ("dresidual", "dpre")}, T, dtype)
    dw2 = torch.empty_like(dw)
    gpu_ctx.norm_backward_dev(d["dh"], x, d["pre"], d["dy"], work, dweight_dev=dw2, dy_dev=d["dy"], eps=EPS, stream=_stream())
    assert torch.equal(d["dy"], dx) and torch.equal(dw2, dw)


@pytest.mark.parametrize("T,H", [(5, 96), (300, 2560), (300, 5001)])
@pytest.mark.parametrize("gate", ["column", "row", "full"])
def test_gradients_that_are_not_wanted(gpu_ctx, T, H, gate):
    """Any of the weights' and the gate's gradients left out: the others keep their bits."""
    d = _dev(_case(T, H, torch.bfloat16, True, gate, 3))
    y = _run(gpu_ctx, d, 0.75)
    want = _backward(gpu_ctx, d, y, gate, 0.75)
    work = torch.empty(gpu_ctx.norm_backward_work(T, H), device="cuda")
    for some in range(8):
        o = {k: torch.full_like(v, 7) for k, v in want.items()}
        wanted = {k: some >> i & 1 for i, k in enumerate(("dpre", "dpost", "dgate"))}
        gpu_ctx.residual_norm_backward_dev(
            d["dy"], d["dh"], d["block"], y, o["dblock"], o["dresidual"], work.fill_(float("nan")), post_weight_dev=d["post"],
            dpost_weight_dev=o["dpost"] if wanted["dpost"] else None, gate_dev=d["gate"],
            dgate_dev=o["dgate"] if wanted["dgate"] else None, scale=0.75, pre_weight_dev=d["pre"],
            dpre_weight_dev=o["dpre"] if wanted["dpre"] else None, eps=EPS, stream=_stream())
        for k in want:
            assert torch.equal(o[k], want[k] if wanted.get(k, True) else torch.full_like(o[k], 7)), (k, some)


@pytest.mark.parametrize("T,H", [(4, 96), (300, 2560), (3009, 1000)])
def test_one_tensor_as_block_and_residual(gpu_ctx, T, H):
    """Inputs may be the same: y = scale x + gate N(x) post, over x too."""
    for dtype in TYPES:
        s = _case(T, H, dtype, True, "column", 4)
        s["residual"] = s["block"]
        d = _dev(s)
        d["residual"] = d["block"]
        h = torch.empty_like(d["block"])
        y = _run(gpu_ctx, d, 0.75, h=h)
        want, size = _forward64(s, 0.75)
        rel, least = _half_step(dtype)
        off, bound = (y.cpu().double() - want).abs(), 24 * U * size + want.abs() * rel * (1 + 2.0 ** -10) + least
        assert bool((off <= bound).all()), float((off / bound).max())
        h2 = torch.empty_like(h)
        _run(gpu_ctx, d, 0.75, y=d["block"], h=h2)
        assert torch.equal(d["block"], y) and torch.equal(h2, h)
