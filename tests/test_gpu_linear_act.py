"""GPU: products of quantized weights with bias, activation and residual (csrc/linear_act.hip), dense and by
expert, against the dequantized weights in 64 bits.

Bounds.  A sum over K products in fp32 is off by at most (K + 64) 2^-23 sum |x w|; the weights' rounding to fp16 in
the kernel of many rows adds at most 2^-11 sum |x w| (and K times 2^-30 of the largest |x| and |w| for values at the
end of fp16's range: x is off by 2^-38 of its row's largest there, a q4nx weight by 2^-31).  z = that + bias carries d; an activation with |f'| <= L passes L d on and adds 32 steps of
fp32; the sum with the residual and the rounding to bf16 add 2^-8 of the result."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle import bfp16 as B
from oracle import q4nx as Q

from raon_npu_amd.geometry import MoeGeometry

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

ACTS = ["none", "silu", "gelu", "gelu_tanh", "swiglu", "situ"]
SITU = (4.0, 25.0)
MANY = 32  # rows of one matrix from which the kernel of many rows may run; by expert: one an expert in the mean


def _weights(fmt, M, K, seed, live=None, std=0.02):
    rng = np.random.default_rng(seed)
    w = rng.normal(0.0, std, (M, K)).astype(np.float32)
    if live is not None:
        w[:, live:] = 0
    if fmt == "q4nx":
        c, s, m = Q.quantize(w)
        return Q.pack_gemv(c, s, m), torch.from_numpy(Q.dequantize_simple(c, s, m)).double()
    blob = B.pack_gemv(w)
    return blob, torch.from_numpy(B.dequantize_packed(blob, K, M)).double()


def _reference(x, w, bias, act, residual, many):
    """(y, bound) of y in float64."""
    x = x.double()
    K = x.shape[1]
    absum = x.abs() @ w.abs().t()
    z = x @ w.t()
    d = (K + 64) * 2.0 ** -23 * absum
    if many:
        d += 2.0 ** -11 * absum + K * 2.0 ** -30 * x.abs().amax(1, keepdim=True) * w.abs().amax(1)[None]
    if bias is not None:
        z = z + bias.double()
        d = d + 2.0 ** -24 * z.abs()
    half = z.shape[1] // 2
    if act in ("swiglu", "situ"):
        g, u, dg, du = z[:, :half], z[:, half:], d[:, :half], d[:, half:]
        if act == "swiglu":
            f, L, h = g * torch.sigmoid(g), 1.1, u
        else:
            f, L, h = SITU[0] * torch.tanh(g / SITU[0]) * torch.sigmoid(g), 1.0 + SITU[0] / 4, SITU[1] * torch.tanh(u / SITU[1])
        y = f * h
        e = L * dg * (h.abs() + du) + f.abs() * du
    else:
        y = {"none": lambda: z, "silu": lambda: z * torch.sigmoid(z),
             "gelu": lambda: z * 0.5 * torch.special.erfc(-z / math.sqrt(2.0)),
             "gelu_tanh": lambda: z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))}[act]()
        e = 1.2 * d
    e = e + 32 * 2.0 ** -24 * y.abs()
    if residual is not None:
        y = y + residual.double()
        e = e + 2.0 ** -24 * y.abs()
    return y, e


def _check(got, ref, e, what=""):
    got = got.cpu().double()
    bound = 2.0 ** -8 * (ref.abs() + e) + e + 2.0 ** -133
    bad = ~((got - ref).abs() <= bound)
    assert not bad.any(), (what, bad.nonzero()[:4].tolist(), got[bad][:4].tolist(), ref[bad][:4].tolist())


def _betas(act):
    return {"gate_beta": SITU[0], "value_beta": SITU[1]} if act == "situ" else {}


def _operands(T, M, K, act, bias, residual, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g).to(torch.bfloat16)
    b = torch.randn(M, generator=g) * 0.3 if bias else None
    width = M // 2 if act in ("swiglu", "situ") else M
    r = torch.randn(T, width, generator=g).to(torch.bfloat16) if residual else None
    return x, b, r, width


def _cuda(t):
    return None if t is None else t.cuda()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,K", [(128, 256), (384, 768), (1536, 2048)])
def test_dense(gpu_ctx, fmt, act, M, K):
    blob, w = _weights(fmt, M, K, M + K)
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(700)
    for T, bias, residual in ((1, True, True), (4, False, False), (5, False, True), (33, True, False), (130, True, True),
                              (700, True, True)):
        x, b, r, width = _operands(T, M, K, act, bias, residual, 7 * T + M)
        buf = torch.full((T + 1, width), 9.0, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(_cuda(x), T, buf[:T], bias_dev=_cuda(b), act=act, residual_dev=_cuda(r),
                           stream=torch.cuda.current_stream(), **_betas(act))
        ref, e = _reference(x, w, b, act, r, T >= MANY)
        _check(buf[:T], ref, e, T)
        assert bool((buf[T] == 9).all())
    mat.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("T", [1, 3, 40, 300])
def test_input_narrower_than_the_matrix(gpu_ctx, fmt, T):
    """K_in < K, also ending inside a tile of 128 columns; what lies behind a row is the next row."""
    M, K = 256, 1280
    blob, w = _weights(fmt, M, K, 3)
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    for K_in in (8, 120, 136, 1024, 1088, 1272, 1280):
        x, b, r, width = _operands(T, M, K_in, "silu", True, True, K_in)
        y = torch.zeros(T, width, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(_cuda(x), T, y, bias_dev=_cuda(b), act="silu", residual_dev=_cuda(r),
                           stream=torch.cuda.current_stream())
        _check(y, *_reference(x, w[:, :K_in], b, "silu", r, T >= MANY), K_in)
    mat.free()


@pytest.mark.parametrize("T", [1, 40, 300])
def test_residual_in_place_int16_and_odd_addresses(gpu_ctx, T):
    """y is the residual; int16 bits are bfloat16 values; y at an address its 16-byte stores cannot take."""
    M, K = 256, 512
    blob, w = _weights("q4nx", M, K, 5)
    mat = gpu_ctx.upload_matrix(blob, M, K)
    mat.reserve_act(T)
    x, b, r, _ = _operands(T, M, K, "gelu", True, True, 6)
    st = torch.cuda.current_stream()
    want = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
    mat.linear_act_dev(x.cuda(), T, want, bias_dev=b.cuda(), act="gelu", residual_dev=r.cuda(), stream=st)
    _check(want, *_reference(x, w, b, "gelu", r, T >= MANY))
    for shift in (0, 1, 4):
        buf = torch.zeros(T * M + 16, dtype=torch.int16, device="cuda")
        y = buf[shift:shift + T * M].view(T, M)
        y.copy_(r.view(torch.int16))
        mat.linear_act_dev(x.cuda().view(torch.int16), T, y, bias_dev=b.cuda(), act="gelu", residual_dev=y, stream=st)
        assert torch.equal(y.view(torch.bfloat16), want)
        assert not buf[:shift].any() and not buf[shift + T * M:].any()
    mat.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("T", [2, 64, 300])
def test_ranges_of_values(gpu_ctx, fmt, T):
    """Rows of x and weights of very different sizes, as no type of 16 bits with a short exponent holds them:
    2^-60 to 2^60, rows of zeros, and rows with one large value."""
    M, K = 128, 512
    for ws in (2.0 ** -40, 1.0, 2.0 ** 30):
        blob, w = _weights(fmt, M, K, 9, std=ws)
        mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
        mat.reserve_act(T)
        g = torch.Generator().manual_seed(T)
        x = torch.randn(T, K, generator=g) * 2.0 ** torch.linspace(-60, 60, T)[:, None].round()
        x[T // 2] = 0
        x[0, 5] = x[0, 5] * 2.0 ** 20
        x = x.to(torch.bfloat16)
        y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(x.cuda(), T, y, stream=torch.cuda.current_stream())
        _check(y, *_reference(x, w, None, "none", None, T >= MANY), ws)
        assert not y[T // 2].any()
        mat.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("T", [18, 200])
def test_non_finite_rows_stay_in_their_row(gpu_ctx, fmt, T):
    M, K = 128, 512
    blob, w = _weights(fmt, M, K, 9)
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    x, _, _, _ = _operands(T, M, K, "none", False, False, 2)
    st = torch.cuda.current_stream()
    want, y = (torch.zeros(T, M, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    mat.linear_act_dev(x.cuda(), T, want, stream=st)
    bad = x.clone()
    bad[3, 7], bad[17, 300] = float("inf"), float("nan")
    mat.linear_act_dev(bad.cuda(), T, y, stream=st)
    keep = [t for t in range(T) if t not in (3, 17)]
    assert torch.equal(y[keep], want[keep])
    assert not y[[3, 17]].isfinite().any()
    mat.free()


def _layer(gpu_ctx, H, I, E, d_layout, seed):
    """A layer and its float64 (gate_up [E, 2I, H], down [E, H, I]); weights-d layers have a bfp16 down."""
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=min(4, E))
    Ip = g.inter_pad
    gu = [_weights("q4nx", 2 * I, H, seed + 2 * e) for e in range(E + 1)]
    dn = [_weights("bfp16" if d_layout else "q4nx", H, Ip, seed + 2 * e + 1, live=I) for e in range(E + 1)]
    if d_layout:
        lyr = gpu_ctx.create_layer_d(7300, g)
        lyr.upload_d(1, 0, b"".join(b for b, _ in gu[:E]))
        lyr.upload_d(2, 0, b"".join(b for b, _ in dn))
    else:
        lyr = gpu_ctx.create_layer(7300, g)
        lyr.upload_experts(b"".join(b for b, _ in gu), b"".join(b for b, _ in dn))
    return lyr, [w for _, w in gu[:E]], [w[:, :I] for _, w in dn[:E]]


COUNTS = [[1, 0, 0, 0, 0], [0, 0, 0, 0, 3], [1, 1, 1, 1, 1], [0, 17, 0, 5, 1], [4, 5, 16, 33, 0], [129, 0, 64, 65, 200],
          [0, 700, 0, 0, 1], [0, 0, 0, 0, 0]]


@pytest.mark.parametrize("d_layout", [False, True])
@pytest.mark.parametrize("part", ["gate_up", "down"])
def test_experts(gpu_ctx, d_layout, part):
    """Each row with its expert's matrix; experts without rows, rows behind the last left as they were."""
    H, I, E = 512, 320, 5
    lyr, gu, dn = _layer(gpu_ctx, H, I, E, d_layout, 40)
    ws, M, K = (gu, 2 * I, H) if part == "gate_up" else (dn, H, I)
    lyr.reserve_experts_linear(1000)
    for i, counts in enumerate(COUNTS):
        live = sum(counts)
        n = live + (3 if i % 2 else 0) or 2
        offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
        act = ACTS[i % 6] if part == "gate_up" else ["none", "gelu"][i % 2]
        x, _, r, width = _operands(n, M, K, act, False, i % 3 == 0, 60 + i)
        x[live:] = float("nan")
        b = torch.randn(E, M, generator=torch.Generator().manual_seed(i)) * 0.3 if i % 2 else None
        y = torch.full((n, width), 9.0, dtype=torch.bfloat16, device="cuda")
        lyr.experts_linear_dev(part, x.cuda(), offsets.cuda(), y, bias_dev=_cuda(b), act=act, residual_dev=_cuda(r),
                               stream=torch.cuda.current_stream(), **_betas(act))
        for e in range(E):
            a, z = int(offsets[e]), int(offsets[e + 1])
            if a < z:
                ref, err = _reference(x[a:z], ws[e], None if b is None else b[e], act, None if r is None else r[a:z],
                                      n >= E)
                _check(y[a:z], ref, err, (counts, e))
        assert bool((y[live:] == 9).all())
    lyr.free()


def test_experts_with_offsets_outside_the_rows(gpu_ctx):
    """Offsets are device data: whatever they hold, nothing outside the rows is read or written."""
    H, I, E = 256, 128, 5
    lyr, gu, _ = _layer(gpu_ctx, H, I, E, False, 70)
    n = 40
    lyr.reserve_experts_linear(n)
    x, _, _, width = _operands(n, 2 * I, H, "none", False, False, 3)
    buf = torch.full((n + 64, width), 9.0, dtype=torch.bfloat16, device="cuda")
    for offsets in ([-5, 3, 3, 900, 7, 2 ** 31 - 1], [50, 40, 30, 20, 10, 0], [2 ** 31 - 1] * 6, [-2 ** 31] * 6):
        buf.fill_(9.0)
        lyr.experts_linear_dev("gate_up", x.cuda(), torch.tensor(offsets, dtype=torch.int32, device="cuda"), buf[:n],
                               stream=torch.cuda.current_stream())
        assert bool((buf[n:] == 9).all())
    torch.cuda.synchronize()
    lyr.free()


def test_one_token_sorted_through_its_experts(gpu_ctx):
    """The operators in a row against the framework's closed call: route, sort, gate/up with SwiGLU, down, combine,
    for one token and for batches; the closed call rounds gate and up to bf16 first, so both are compared with 64
    bits at the parity bar (max-abs 1e-2, rel-L2 3e-3, of which roundings of h and of the result take
    2^-8 / sqrt(3) each)."""
    H, I, E, k = 512, 320, 8, 3
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=k)
    for d_layout in (False, True):
        lyr, gu, dn = _layer(gpu_ctx, H, I, E, d_layout, 90)
        for T in (1, 5, 77, 600):
            gen = torch.Generator().manual_seed(T)
            x = torch.randn(T, H, generator=gen).to(torch.bfloat16)
            ids = torch.rand(T, E, generator=gen).argsort(1)[:, :k].to(torch.int32).contiguous()
            if T > 5:
                ids[3] = -1  # a padding token
                ids[4, 1] = -1
            w = torch.rand(T, k, generator=gen)
            st = torch.cuda.Stream()
            A = T * k
            lyr.reserve_experts_linear(A)
            dev = {"device": "cuda"}
            rows = torch.zeros(A, H, dtype=torch.bfloat16, **dev)
            order, off = torch.zeros(A, dtype=torch.int32, **dev), torch.zeros(E + 1, dtype=torch.int32, **dev)
            inv = torch.zeros(T, k, dtype=torch.int32, **dev)
            h = torch.zeros(A, I, dtype=torch.bfloat16, **dev)
            d = torch.zeros(A, H, dtype=torch.bfloat16, **dev)
            out = torch.zeros(T, H, dtype=torch.bfloat16, **dev)
            xd, idd, wd = x.cuda(), ids.cuda(), w.cuda()
            torch.cuda.synchronize()

            def run():
                gpu_ctx.sort_tokens_dev(xd, idd, E, rows, order, inv, off, stream=st)
                lyr.experts_linear_dev("gate_up", rows, off, h, act="swiglu", stream=st)
                lyr.experts_linear_dev("down", h, off, d, stream=st)
                gpu_ctx.combine_tokens_dev(d, inv, wd, out, stream=st)

            run()
            torch.cuda.synchronize()
            ref = torch.zeros(T, H, dtype=torch.float64)
            for t in range(T):
                for r in range(k):
                    e = int(ids[t, r])
                    if e >= 0:
                        z = gu[e] @ x[t].double()
                        hh = (z[:I] * torch.sigmoid(z[:I]) * z[I:]).to(torch.bfloat16).double()
                        ref[t] += float(w[t, r]) * (dn[e] @ hh)
            got = out.cpu().double()
            assert float((got - ref).abs().max()) <= 1e-2
            assert float((got - ref).norm()) <= 3e-3 * float(ref.norm())
            if T > 5:
                assert not out[3].any()
            # captured and replayed, with new tokens
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph, stream=st):
                run()
            for i in range(3):
                xd.copy_(x.roll(i, 0))
                torch.cuda.synchronize()
                graph.replay()
                torch.cuda.synchronize()
                replayed = out.clone()
                run()
                torch.cuda.synchronize()
                assert torch.equal(out, replayed)
        lyr.free()


def test_refused_operands(gpu_ctx):
    """What the entry points themselves refuse; nothing is launched."""
    M, K, T = 128, 512, 4
    blob, _ = _weights("q4nx", M, K, 1)
    mat = gpu_ctx.upload_matrix(blob, M, K)
    mat.reserve_act(T)
    x = torch.zeros(T * K + 8, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
    buf = torch.zeros(2 * T * M, dtype=torch.bfloat16, device="cuda")
    with pytest.raises(ValueError, match="16-byte"):
        mat.linear_act_dev(x[1:1 + T * K].view(T, K), T, y)
    with pytest.raises(ValueError, match="multiple of 8"):
        mat.linear_act_dev(x[:T * 100].view(T, 100), T, y)
    with pytest.raises(ValueError, match="at most K"):
        mat.linear_act_dev(x.new_zeros(T, K + 8), T, y)
    with pytest.raises(ValueError, match="overlaps"):
        mat.linear_act_dev(x[:T * K].view(T, K), T, x[T * M:2 * T * M].view(T, M))
    with pytest.raises(ValueError, match="overlaps"):
        mat.linear_act_dev(x[:T * K].view(T, K), T, buf[:T * M].view(T, M), residual_dev=buf[M:M + T * M].view(T, M))
    with pytest.raises(ValueError, match="betas"):
        mat.linear_act_dev(x[:T * K].view(T, K), T, y[:, :64].contiguous(), act="situ", gate_beta=0.0, value_beta=25.0)
    with pytest.raises(ValueError):
        mat.reserve_act(0)
    mat.free()
    with pytest.raises(KeyError):
        mat.linear_act_dev(x[:T * K].view(T, K), T, y)


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("M", [128, 14336, 28672])
@pytest.mark.parametrize("K,widths", [(256, (256, 136)), (1280, (1280, 1088, 520))])
def test_every_tile_of_few_rows(gpu_ctx, fmt, M, K, widths):
    """The tile shapes that the rule picks by rows and weight rows (16 x 16 to 32 x 64, up to four rows or more,
    gated or not, narrower rows or not), with K splits of one to three K tiles a wave."""
    parts = [_weights(fmt, 128, K, s) for s in (1, 2, 3)]
    order = [0, 1, 2, 1] * (M // 512) + [2] * (M // 128 % 4)
    mat = gpu_ctx.upload_matrix(b"".join(parts[i][0] for i in order), M, K, fmt=fmt)
    w = torch.cat([p[1] for p in parts]).cuda()
    rows = torch.cat([torch.arange(128) + 128 * i for i in order]).cuda()  # weight row -> row of w
    st = torch.cuda.current_stream()
    for T in (3, 9, 17, 40, 100):
        mat.reserve_act(T)
        for K_in in widths:
            x = torch.randn(T, K_in, generator=torch.Generator().manual_seed(T + K_in)).to(torch.bfloat16).cuda()
            absum = (x.double().abs() @ w[:, :K_in].abs().t())[:, rows]
            z = (x.double() @ w[:, :K_in].t())[:, rows]
            many = 2.0 ** -11 * absum if T >= MANY else 0.0
            d = (K_in + 64) * 2.0 ** -23 * absum + many
            y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
            mat.linear_act_dev(x, T, y, stream=st)
            assert bool(((y.double() - z).abs() <= 2.0 ** -8 * (z.abs() + d) + d).all()), (T, K_in)
            g, u, dg, du = z[:, :M // 2], z[:, M // 2:], d[:, :M // 2], d[:, M // 2:]
            f = g * torch.sigmoid(g)
            e = 1.1 * dg * (u.abs() + du) + f.abs() * du + 32 * 2.0 ** -24 * (f * u).abs()
            h = torch.zeros(T, M // 2, dtype=torch.bfloat16, device="cuda")
            mat.linear_act_dev(x, T, h, act="swiglu", stream=st)
            assert bool(((h.double() - f * u).abs() <= 2.0 ** -8 * ((f * u).abs() + e) + e).all()), (T, K_in)
    mat.free()


@pytest.mark.parametrize("part,act", [("gate_up", "swiglu"), ("down", "none")])
@pytest.mark.parametrize("d_layout", [False, True])
def test_experts_by_rows_an_expert(gpu_ctx, part, act, d_layout):
    """Row counts on both sides of every change of kernel and tile: fewer rows than experts, then 24 and 64 an expert
    in the mean, spread evenly and all on two experts."""
    H, I, E = 256, 192, 6
    lyr, gu, dn = _layer(gpu_ctx, H, I, E, d_layout, 120)
    ws, M, K = (gu, 2 * I, H) if part == "gate_up" else (dn, H, I)
    for n in (1, 4, 5, 6, 7, 149, 150, 389, 390, 391, 1200):
        lyr.reserve_experts_linear(n)
        x, _, _, width = _operands(n, M, K, act, False, False, n)
        for counts in ([n // E + (e < n % E) for e in range(E)], [0, n // 3, 0, 0, n - n // 3, 0]):
            offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
            y = torch.full((n, width), 9.0, dtype=torch.bfloat16, device="cuda")
            lyr.experts_linear_dev(part, x.cuda(), offsets.cuda(), y, act=act, stream=torch.cuda.current_stream())
            for e in range(E):
                a, z = int(offsets[e]), int(offsets[e + 1])
                if a < z:
                    ref, err = _reference(x[a:z], ws[e], None, act, None, True)
                    _check(y[a:z], ref, err, (n, counts, e))
    lyr.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
def test_dense_of_many_rows(gpu_ctx, fmt):
    """Enough rows for the kernel of many rows, whole and ragged tiles, widths that end inside a tile of 256 weight
    rows, every epilogue; a token's neighbours do not matter."""
    K = 512
    for M, T, act in ((256, 128 * 144, "none"), (384, 128 * 72 + 5, "gelu"), (1280, 128 * 29 + 77, "situ"),
                      (2176, 128 * 16 + 1, "swiglu")):
        blob, w = _weights(fmt, M, K, M)
        mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
        mat.reserve_act(T)
        x, b, r, width = _operands(T, M, K, act, True, True, T)
        y = torch.zeros(T, width, dtype=torch.bfloat16, device="cuda")
        st = torch.cuda.current_stream()
        mat.linear_act_dev(x.cuda(), T, y, bias_dev=b.cuda(), act=act, residual_dev=r.cuda(), stream=st, **_betas(act))
        pick = torch.cat([torch.arange(300), torch.arange(T - 300, T)])
        _check(y[pick], *_reference(x[pick], w, b, act, r[pick], True), (M, T))
        in_place = r.cuda()
        mat.linear_act_dev(x.cuda(), T, in_place, bias_dev=b.cuda(), act=act, residual_dev=in_place, stream=st, **_betas(act))
        assert torch.equal(in_place, y)
        odd = torch.zeros(T * width + 9, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(x.cuda(), T, odd[1:1 + T * width].view(T, width), bias_dev=b.cuda(), act=act,
                           residual_dev=r.cuda(), stream=st, **_betas(act))
        assert torch.equal(odd[1:1 + T * width].view(T, width), y) and not odd[0] and not odd[1 + T * width:].any()
        mat.free()


def test_exponents_follow_the_weights(gpu_ctx):
    """Weights written anew under the same layer (another size by 2^12) are served with their own exponents."""
    H, I, E, n = 256, 128, 2, 64
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=1)
    lyr = gpu_ctx.create_layer(7301, g)
    lyr.reserve_experts_linear(n)
    x = torch.randn(n, H, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16)
    offsets = torch.tensor([0, n // 2, n], dtype=torch.int32, device="cuda")
    y = torch.zeros(n, 2 * I, dtype=torch.bfloat16, device="cuda")
    for std in (0.02, 0.02 * 2.0 ** 12, 0.02 * 2.0 ** -20):
        parts = [_weights("q4nx", 2 * I, H, e, std=std) for e in range(E + 1)]
        dn = [_weights("q4nx", H, 256, 9, live=I)[0]] * (E + 1)
        lyr.upload_experts(b"".join(p[0] for p in parts), b"".join(dn))
        lyr.experts_linear_dev("gate_up", x.cuda(), offsets, y, stream=torch.cuda.current_stream())
        for e in range(E):
            s = slice(e * n // 2, (e + 1) * n // 2)
            _check(y[s], *_reference(x[s], parts[e][1], None, "none", None, True), std)
        w = torch.randn(2 * I, H, generator=torch.Generator().manual_seed(5)) * std * 2.0 ** 5
        lyr.quantize_expert(1, w.cuda(), torch.zeros(H, I, device="cuda"))
        c, s, m = Q.quantize(w.numpy())
        lyr.experts_linear_dev("gate_up", x.cuda(), offsets, y, stream=torch.cuda.current_stream())
        _check(y[n // 2:], *_reference(x[n // 2:], torch.from_numpy(Q.dequantize_simple(c, s, m)).double(), None, "none",
                                       None, True), std)
    lyr.free()


@pytest.mark.parametrize("act", ACTS)
def test_activations_over_their_range(gpu_ctx, act):
    """y = act(bias) for z from -300 to 300, where exp(z) ends fp32's range and the results bf16's: x is zero, so z
    is the bias itself.  Relative to the result exp(z) is off by (2 + |z|) 2^-23 and the rest by 32 steps of fp32,
    then half a step of bf16; a probability below fp32's normal numbers is off by one subnormal step, 2^-149, more
    (times |z|, and SiTU's or the gate's other factor), a bf16 subnormal by 2^-134."""
    M, K, E = 4096, 256, 2
    blob, _ = _weights("q4nx", M, K, 1)
    mat = gpu_ctx.upload_matrix(blob, M, K)
    gated = act in ("swiglu", "situ")
    half = M // 2 if gated else M
    z = torch.cat([torch.linspace(-300, 300, half // 2), torch.linspace(-3, 3, half - half // 2)])
    z[5], z[6], z[half // 2], z[half // 2 + 1] = 0.0, -0.0, 1e-30, -1e-30
    u = torch.linspace(-40, 40, half).roll(half // 3)
    b = torch.cat([z, u]) if gated else z
    x = torch.zeros(2, K, dtype=torch.bfloat16, device="cuda")
    y = torch.zeros(2, half, dtype=torch.bfloat16, device="cuda")
    mat.reserve_act(2)
    mat.linear_act_dev(x, 2, y, bias_dev=b.cuda(), act=act, stream=torch.cuda.current_stream(), **_betas(act))
    zd, ud = z.double(), u.double()
    p = torch.sigmoid(zd)
    ref = {"none": lambda: zd, "silu": lambda: zd * p, "gelu": lambda: zd * 0.5 * torch.special.erfc(-zd / math.sqrt(2.0)),
           "gelu_tanh": lambda: zd * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (zd + 0.044715 * zd ** 3)),
           "swiglu": lambda: zd * p * ud,
           "situ": lambda: SITU[0] * torch.tanh(zd / SITU[0]) * p * SITU[1] * torch.tanh(ud / SITU[1])}[act]()
    # gelu's exponent is z^2 / 2, gelu_tanh's 1.6 (z + 0.045 z^3)
    arg = {"gelu": zd * zd, "gelu_tanh": 2 * (zd.abs() + 0.05 * zd.abs() ** 3)}.get(act, zd.abs())
    e = ref.abs() * (34 + arg.clamp(max=200.0)) * 2.0 ** -23 + 2.0 ** -149 * 1000.0 * zd.abs().clamp(min=1.0)
    got = y.cpu().double()
    bound = 2.0 ** -8 * (ref.abs() + e) + e + 2.0 ** -134
    for row in got:
        bad = ~((row - ref).abs() <= bound)
        assert not bad.any(), (z[bad][:4].tolist(), row[bad][:4].tolist(), ref[bad][:4].tolist())
    mat.free()


def test_graph_captured_before_a_larger_reserve(gpu_ctx):
    """A captured product of many rows replays as before after the scratch has grown, and other rows have gone
    through the new one.  (The same rows in a larger batch may be summed in another order.)"""
    M, K, T = 1024, 512, 2100
    blob, _ = _weights("q4nx", M, K, 3)
    mat = gpu_ctx.upload_matrix(blob, M, K)
    mat.reserve_act(T)
    st = torch.cuda.Stream()
    x = torch.randn(3 * T, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    y, big = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda"), torch.zeros(3 * T, M, dtype=torch.bfloat16, device="cuda")
    torch.cuda.synchronize()
    mat.linear_act_dev(x[:T], T, y, act="silu", stream=st)
    torch.cuda.synchronize()
    want = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        mat.linear_act_dev(x[:T], T, y, act="silu", stream=st)
    for grown in (T, 2 * T, 3 * T):
        mat.reserve_act(grown)
        mat.linear_act_dev(x[:grown], grown, big[:grown], act="silu", stream=st)
        junk = torch.full((grown, 4 * K), float("nan"), dtype=torch.bfloat16, device="cuda")
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
        del junk
    mat.free()


def test_two_contexts_on_two_streams(gpu_ctx):
    """Products of many rows that overlap, a context each: the same bits as one after the other."""
    from raon_npu_amd import Context

    M, K, T = 1024, 1024, 3000
    blob, _ = _weights("bfp16", M, K, 3)
    runs = []
    for seed, c in ((1, gpu_ctx), (2, Context(0))):
        mat = c.upload_matrix(blob, M, K, fmt="bfp16")
        mat.reserve_act(T)
        x = torch.randn(T, K, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).cuda()
        y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
        runs.append((c, mat, x, y, torch.cuda.Stream()))
    torch.cuda.synchronize()
    want = []
    for c, mat, x, y, st in runs:
        mat.linear_act_dev(x, T, y, act="gelu", stream=st)
        torch.cuda.synchronize()
        want.append(y.clone())
        y.zero_()
    torch.cuda.synchronize()
    for _ in range(8):
        for c, mat, x, y, st in runs:
            mat.linear_act_dev(x, T, y, act="gelu", stream=st)
    torch.cuda.synchronize()
    for w, (c, mat, x, y, st) in zip(want, runs):
        assert torch.equal(y, w)
        mat.free()
    runs[1][0].close()


@pytest.mark.parametrize("M,K,T", [
    (256, 512, 128 * 211 + 5),   # 212 tiles of 128 x 256, no whole round of 256
    (256, 512, 128 * 256 + 3),   # one tile past a round, ragged, of a K too short to cut
    (256, 2048, 128 * 256 + 100),  # the same, in four slices of four K tiles
    (1280, 1280, 128 * 54 - 60),  # 270 tiles: 14 past a round, four slices of two and three K tiles
    (2176, 1280, 128 * 40),      # 360: 104 past a round, too many to cut
    (768, 2560, 128 * 113 + 1),  # 342: 86, the same
    (1280, 768, 128 * 68),       # 340: 84, in three slices of two
    (512, 1792, 128 * 161),      # 322: 66, in three slices of four and five
    (2560, 1024, 128 * 55),      # 550: 38 past two rounds, in four
    (512, 512, 128 * 193)])      # 386: 130 past a round
@pytest.mark.parametrize("act", ["none", "swiglu"])
def test_dense_around_whole_rounds_of_tiles(gpu_ctx, M, K, T, act):
    """Tile counts on both sides of multiples of the CUs, where the last tiles' sums are cut along K: every row against
    64 bits, rows behind the last as they were, and the same bits each time."""
    for fmt in ("q4nx", "bfp16"):
        blob, w = _weights(fmt, M, K, M + K)
        mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
        mat.reserve_act(T)
        gated = act == "swiglu"
        width = M // 2 if gated else M
        x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)).to(torch.bfloat16).cuda()
        b = torch.randn(M, generator=torch.Generator().manual_seed(1)).cuda()
        y = torch.full((T + 1, width), 9.0, dtype=torch.bfloat16, device="cuda")
        st = torch.cuda.current_stream()
        mat.linear_act_dev(x, T, y[:T], bias_dev=b, act=act, stream=st)
        w = w.cuda()
        for t0 in range(0, T, 4096):
            ref, e = _reference(x[t0:t0 + 4096], w, b, act, None, True)
            _check(y[t0:min(t0 + 4096, T)], ref.cpu(), e.cpu(), (fmt, t0))
        assert bool((y[T] == 9).all())
        first = y.clone()
        for _ in range(5):
            y[:T].zero_()
            mat.linear_act_dev(x, T, y[:T], bias_dev=b, act=act, stream=st)
            assert torch.equal(y, first)
        mat.free()


def test_split_tiles_in_a_graph(gpu_ctx):
    """The cut tiles' counters are cleared by each call, captured or not, also after a call of other rows."""
    M, K, T = 2176, 1280, 128 * 32
    blob, _ = _weights("q4nx", M, K, 3)
    mat = gpu_ctx.upload_matrix(blob, M, K)
    mat.reserve_act(T)
    st = torch.cuda.Stream()
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    y, other = (torch.zeros(T, M, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    torch.cuda.synchronize()
    mat.linear_act_dev(x, T, y, stream=st)
    torch.cuda.synchronize()
    want = y.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        mat.linear_act_dev(x, T, y, stream=st)
    for n in (T, 128 * 30, 128 * 31, 7):
        mat.linear_act_dev(x[:n], n, other[:n], stream=st)
        torch.cuda.synchronize()
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    mat.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("T", [128 * 64 + 1, 128 * 256 + 3])
def test_many_rows_narrower_than_the_matrix(gpu_ctx, fmt, T):
    """K_in < K with tiles by two groups of K, which may get unequal shares, and with the last tiles cut along K."""
    M, K = 256, 1280
    blob, w = _weights(fmt, M, K, 3)
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    w = w.cuda()
    for K_in in (8, 128, 136, 640, 1024, 1088, 1152, 1272):
        x = torch.randn(T, K_in, generator=torch.Generator().manual_seed(K_in)).to(torch.bfloat16).cuda()
        y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(x, T, y, act="silu", stream=torch.cuda.current_stream())
        ref, e = _reference(x, w[:, :K_in], None, "silu", None, True)
        _check(y, ref.cpu(), e.cpu(), K_in)
    mat.free()


def test_layer_of_one_expert(gpu_ctx):
    """One expert with all rows, some of them, or none: the tiles of one matrix, found from its offsets."""
    H, I = 256, 192
    g = MoeGeometry(hidden=H, inter=I, n_routed=1, n_shared=1, top_k=1)
    lyr = gpu_ctx.create_layer(7302, g)
    gu = [_weights("q4nx", 2 * I, H, s) for s in (1, 2)]
    dn = [_weights("q4nx", H, 256, s, live=I)[0] for s in (3, 4)]
    lyr.upload_experts(b"".join(b for b, _ in gu), b"".join(dn))
    w = gu[0][1]
    n = 128 * 64 + 77
    lyr.reserve_experts_linear(n)
    x = torch.randn(n, H, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    for rows, first, last in ((n, 0, n), (n, 100, n - 900), (n, 5, 5), (9, 0, 9), (9, 3, 4)):
        y = torch.full((rows, I), 9.0, dtype=torch.bfloat16, device="cuda")
        lyr.experts_linear_dev("gate_up", x[:rows].cuda(), torch.tensor([first, last], dtype=torch.int32, device="cuda"), y,
                               act="swiglu", stream=torch.cuda.current_stream())
        if first < last:
            _check(y[first:last], *_reference(x[first:last], w, None, "swiglu", None, rows > 9), (rows, first, last))
        assert bool((y[:first] == 9).all()) and bool((y[last:] == 9).all())
    lyr.free()


def _agree(a, b):
    """Two bf16 roundings of sums that differ by the weights' rounding to fp16: each rounding is uniform in half a step,
    2^-8 / sqrt(3) of a value at most, the sums differ by 2^-11 / sqrt(3) of the terms' rms."""
    a, b = a.double(), b.double()
    return float((a - b).norm()) <= (2 ** 0.5 * 2.0 ** -8 + 2.0 ** -11) / 3 ** 0.5 * float(b.norm())


def test_every_way_to_write_weights(gpu_ctx):
    """Many rows, which use the exponents kept with the weights, against a few rows of the same weights, which do not:
    layers synthesized, quantized on the device or from Q4_K, and matrices of every kind, views of experts included."""
    st = torch.cuda.current_stream()
    H, I, E, n = 512, 256, 3, 96
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=1)
    lyr = gpu_ctx.create_layer(7303, g)
    lyr.reserve_experts_linear(n)
    offsets = torch.tensor([0, 32, 64, 96], dtype=torch.int32, device="cuda")

    def check_layer(what):
        for part, M, K in (("gate_up", 2 * I, H), ("down", H, I)):
            x = torch.randn(n, K, generator=torch.Generator().manual_seed(K)).to(torch.bfloat16).cuda()
            y, few = (torch.zeros(n, M, dtype=torch.bfloat16, device="cuda") for _ in range(2))
            lyr.experts_linear_dev(part, x, offsets, y, stream=st)
            for e in range(E):
                view = lyr.expert_matrix(e, part)
                view.reserve_act(32)
                view.linear_act_dev(x[32 * e:32 * e + 32], 32, few[32 * e:32 * e + 32], stream=st)
                big_n = 64 * (256 * 128 // M + 1)
                view.reserve_act(big_n)
                big = torch.zeros(big_n, M, dtype=torch.bfloat16, device="cuda")
                view.linear_act_dev(x[32 * e:32 * e + 32].repeat(big_n // 32, 1).contiguous(), big_n, big, stream=st)
                assert _agree(big[:32], few[32 * e:32 * e + 32]) and torch.equal(big[-32:], big[:32]), (what, part, e)
                view.free()
            assert bool(y.any()) and _agree(y, few), (what, part)

    lyr.synthesize(3, std=0.5, stream=st)
    check_layer("synthesized")
    lyr.synthesize(4, std=2.0 ** -12)
    check_layer("synthesized smaller")
    for e in range(E):
        lyr.quantize_expert(e, torch.randn(2 * I, H, device="cuda") * 2.0 ** (3 * e), torch.randn(H, I, device="cuda"))
    check_layer("quantized")
    rng = np.random.default_rng(5)

    def q4k(rows, cols, d):  # random 144-byte super-blocks with sane scales
        b = rng.integers(0, 256, (rows * cols // 256, 144), dtype=np.uint8)
        b[:, :4] = np.frombuffer(np.array([d, d / 2], dtype=np.float16).tobytes(), dtype=np.uint8)
        return b.tobytes()

    for e in range(E):
        lyr.upload_expert_q4k(e, "gate", q4k(I, H, 0.01 * 4 ** e))
        lyr.upload_expert_q4k(e, "up", q4k(I, H, 0.3))
        lyr.upload_expert_q4k(e, "down", q4k(H, I, 0.002))
    check_layer("Q4_K")
    lyr.free()
    M, K = 512, 768
    T = 64 * 65
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    for mat in (gpu_ctx.quantize_matrix(torch.randn(M, K, device="cuda") * 300, M, K),
                gpu_ctx.upload_matrix(_weights("q4nx", M, K, 1)[0], M, K),
                gpu_ctx.upload_matrix(_weights("bfp16", M, K, 1, std=2.0 ** -30)[0], M, K, fmt="bfp16"),
                gpu_ctx.upload_matrix(q4k(M, K, 0.02), M, K, fmt="q4k")):
        mat.reserve_act(T)
        y, few = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda"), torch.zeros(32, M, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(x, T, y, stream=st)
        mat.linear_act_dev(x[:32], 32, few, stream=st)
        assert bool(few.any()) and _agree(y[:32], few), mat.fmt
        mat.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
def test_groups_of_very_different_sizes(gpu_ctx, fmt):
    """Rows whose groups' weights differ by 2^20, met by tokens that are zero where the large ones are: the small ones
    keep their precision, so that the bound is 2^-11 of the terms alone."""
    M, K, T = 512, 512, 64 * 65
    rng = np.random.default_rng(3)
    w = rng.normal(0.0, 0.5, (M, K)).astype(np.float32)
    scale = 2.0 ** -rng.integers(0, 21, (M, K // 32))
    scale[:, 0] = 1.0
    scale[:, 1:9] = 2.0 ** -20
    w *= np.repeat(scale, 32, 1).astype(np.float32)
    if fmt == "q4nx":
        c, s, m = Q.quantize(w)
        blob, wd = Q.pack_gemv(c, s, m), torch.from_numpy(Q.dequantize_simple(c, s, m)).double()
    else:
        blob = B.pack_gemv(w)
        wd = torch.from_numpy(B.dequantize_packed(blob, K, M)).double()
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    x[::2, :32] = 0
    x[::2, 288:] = 0
    y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
    mat.linear_act_dev(x.cuda(), T, y, stream=torch.cuda.current_stream())
    xd = x.double()
    z, absum = xd @ wd.t(), xd.abs() @ wd.abs().t()
    d = ((K + 64) * 2.0 ** -23 + 2.0 ** -11) * absum
    _check(y, z, d, fmt)
    mat.free()


@pytest.mark.parametrize("E", [255, 256])
def test_the_most_experts(gpu_ctx, E):
    """As many experts as the wave that finds a row's expert holds, the last with and without rows, few and many."""
    H, I = 256, 64
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=8)
    lyr = gpu_ctx.create_layer(7304, g)
    gu = [_weights("q4nx", 2 * I, H, s) for s in range(5)]
    dn = [_weights("q4nx", H, 256, s, live=I) for s in range(5)]
    lyr.upload_experts(b"".join(gu[e % 5][0] for e in range(E + 1)), b"".join(dn[e % 5][0] for e in range(E + 1)))
    st = torch.cuda.current_stream()
    rng = np.random.default_rng(E)
    for counts in (np.eye(E, dtype=int)[E - 1], rng.integers(0, 2, E), rng.integers(0, 90, E), np.eye(E, dtype=int)[0] * 700,
                   np.eye(E, dtype=int)[E - 1] * 700):
        n = int(counts.sum())
        lyr.reserve_experts_linear(n)
        offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
        expert = torch.repeat_interleave(torch.arange(E), torch.from_numpy(counts))
        for part, ws, M, K in (("gate_up", gu, 2 * I, H), ("down", dn, H, I)):
            x = torch.randn(n, K, generator=torch.Generator().manual_seed(n + K)).to(torch.bfloat16)
            y = torch.zeros(n, M, dtype=torch.bfloat16, device="cuda")
            lyr.experts_linear_dev(part, x.cuda(), offsets.cuda(), y, stream=st)
            for s in range(5):
                rows = (expert % 5 == s).nonzero()[:, 0]
                if len(rows):
                    _check(y.cpu()[rows], *_reference(x[rows], ws[s][1][:, :K], None, "none", None, n >= E), (E, n, part, s))
    lyr.free()


def test_rows_past_4_gib(gpu_ctx):
    """x, its fp16 form and (by expert) y of more than 4 GiB: rows on both sides of that offset, the first and the
    last, against 64 bits."""
    st = torch.cuda.current_stream()
    K, T = 8192, 262144 + 77
    blob, w = _weights("q4nx", 128, K, 13)
    mat = gpu_ctx.upload_matrix(blob, 128, K)
    mat.reserve_act(T)
    x = torch.empty(T, K, dtype=torch.bfloat16, device="cuda")
    g = torch.Generator(device="cuda").manual_seed(14)
    for t0 in range(0, T, 65536):
        rows = x[t0:t0 + 65536]
        rows.copy_(torch.randn(rows.shape, device="cuda", generator=g))
    y = torch.zeros(T, 128, dtype=torch.bfloat16, device="cuda")
    mat.linear_act_dev(x, T, y, stream=st)
    for s in (slice(0, 64), slice(262144 - 64, 262144 + 77)):
        _check(y[s], *[t.cpu() for t in _reference(x[s], w.cuda(), None, "none", None, True)], s)
    assert bool((y != 0).any(1).all())
    mat.free()
    del x, y
    H, I, E, n = 256, 2048, 2, 2 ** 19 + 300  # y [n, 4096]
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=1)
    lyr = gpu_ctx.create_layer(7305, g)
    lyr.synthesize(3)
    lyr.reserve_experts_linear(n)
    x = torch.empty(n, H, dtype=torch.bfloat16, device="cuda")
    x.copy_(torch.randn(4096, H, generator=torch.Generator().manual_seed(1)).repeat(n // 4096 + 1, 1)[:n])
    y = torch.zeros(n, 2 * I, dtype=torch.bfloat16, device="cuda")
    # expert 1 begins before the 4 GiB of y and ends behind them
    lyr.experts_linear_dev("gate_up", x, torch.tensor([0, n - 4096, n], dtype=torch.int32, device="cuda"), y, stream=st)
    for e, rows in ((0, slice(2 ** 19 - 8192, 2 ** 19 - 8192 + 64)), (1, slice(n - 4096, n - 4000)), (1, slice(n - 64, n))):
        view = lyr.expert_matrix(e, "gate_up")
        few = torch.zeros(rows.stop - rows.start, 2 * I, dtype=torch.bfloat16, device="cuda")
        view.linear_act_dev(x[rows], len(few), few, stream=st)
        assert _agree(y[rows], few)
        view.free()
    lyr.free()
