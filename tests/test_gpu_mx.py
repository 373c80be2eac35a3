"""GPU: microscaled 4-bit rows and their products (csrc/mx_quantize.hip, mx_linear.hip) against plain forms in 64 bits.

Bounds.  Codes, scales and values: equality.  A product's terms are exact in fp32 (two 2-bit significands and a power of
two); each of the K additions is off by at most 2^-23 of S = sum |x w| (half of that if it rounds to nearest; the matrix
pipes may truncate), as is the bias: (K + 2) 2^-23 (S + |bias|) for z.  An activation passes that on with its largest slope
(silu, gelu and its tanh form: at most 1.13; a product of two factors: each one's bound times the other) and adds 2^-18 of
itself for its own exp, erf and divisions; then one rounding to bf16 of half a step (2^-8 of the result, finfo.eps / 2)."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import mx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = [torch.bfloat16, torch.float16, torch.float32]
SITU = (4.0, 25.0)


def _stream():
    return torch.cuda.current_stream()


def _rows(T, K, seed, dtype=torch.float32):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, K, generator=g) * torch.exp2(torch.randint(-6, 7, (T, 1), generator=g).float())
    x[torch.rand(T, K, generator=g) < 0.05] = 0.0
    return x.to(dtype)


def _quantize(ctx, x, **kw):
    T, K = x.shape
    P = -(-K // 32) * 32
    codes = torch.full((T, P // 2), 0xEE, dtype=torch.uint8, device="cuda")
    scales = torch.full((T, P // 32), 0xEE, dtype=torch.uint8, device="cuda")
    ctx.mx_quantize_dev(x, codes, scales, stream=_stream(), **kw)
    return codes, scales


def _check_quantized(ctx, x):
    """x on the host, of a row type: codes, scales and values against the oracle, by every way to call."""
    codes, scales = mx.quantize(x.double().numpy())
    values = torch.from_numpy(mx.dequantize(codes, scales, x.shape[1])).to(x.dtype)
    d = x.cuda()
    got = torch.full_like(d, 3)
    c, s = _quantize(ctx, d, values_dev=got)
    assert np.array_equal(s.cpu().numpy(), scales)
    assert np.array_equal(c.cpu().numpy(), codes)
    assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=777.0), torch.nan_to_num(values.float(), nan=777.0))
    c2, s2 = _quantize(ctx, d)
    assert torch.equal(c, c2) and torch.equal(s, s2)
    c2, s2 = _quantize(ctx, d, values_dev=d)  # in place
    assert torch.equal(c, c2) and torch.equal(s, s2)
    assert torch.equal(torch.nan_to_num(got, nan=777.0), torch.nan_to_num(d, nan=777.0))


@pytest.mark.parametrize("T,K", [(1, 1), (1, 31), (1, 32), (3, 33), (1, 2048), (445, 1088), (5, 2047), (257, 96), (2, 8192),
                                 (1000, 7), (33, 2560)])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantize(gpu_ctx, T, K, dtype):
    _check_quantized(gpu_ctx, _rows(T, K, T + K, dtype))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_quantize_special_values(gpu_ctx, dtype):
    f = torch.finfo(dtype)
    g = torch.Generator().manual_seed(3)
    x = torch.randn(24, 64, generator=g, dtype=torch.float64)
    x[0, 5], x[1, 40], x[2, 3], x[2, 4] = float("nan"), float("inf"), -float("inf"), float("nan")
    x[3] = 0.0
    x[4] = -0.0
    x[5] *= f.smallest_normal  # subnormal values and scales below the format's least
    x[6] = f.smallest_normal * f.eps
    x[7] *= f.max / x[7].abs().max()
    x[8] *= 4 * f.smallest_normal / x[8].abs().max()
    # Every tie and its neighbours, at three scales.
    ties = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0, 7.9]
    for r, e in ((9, 0), (10, 5), (11, -7)):
        v = torch.tensor(ties, dtype=dtype)
        near = torch.cat([v, v * (1 - f.eps), v * (1 + f.eps)]).double()
        x[r] = 0.0
        x[r, :27] = near * 2.0 ** e
        x[r, 32:59] = -near * 2.0 ** e
    _check_quantized(gpu_ctx, x.to(dtype))


def test_quantize_rows_at_any_address_and_bits(gpu_ctx):
    """Rows that start inside 16 bytes, and bf16 as int16 bits."""
    for dtype in TYPES:
        for K in (64, 70):
            buf = _rows(1, 9 * K + 5, K, dtype).cuda().view(-1)
            x = buf[3:3 + 9 * K].view(9, K)
            codes, scales = mx.quantize(x.double().cpu().numpy())
            c, s = _quantize(gpu_ctx, x)
            assert np.array_equal(c.cpu().numpy(), codes) and np.array_equal(s.cpu().numpy(), scales)
    x = _rows(4, 64, 1, torch.bfloat16).cuda()
    a, b = _quantize(gpu_ctx, x), _quantize(gpu_ctx, x.view(torch.int16))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    codes = torch.empty(4, 32, dtype=torch.uint8, device="cuda").view(torch.float4_e2m1fn_x2)
    scales = torch.empty(4, 2, dtype=torch.uint8, device="cuda").view(torch.float8_e8m0fnu)
    gpu_ctx.mx_quantize_dev(x, codes, scales, stream=_stream())
    assert torch.equal(codes.view(torch.uint8), a[0]) and torch.equal(scales.view(torch.uint8), a[1])


def test_quantize_past_32_bits(gpu_ctx):
    """More than 2^32 bytes and more than 2^31 values: the last rows are quantized as they are alone."""
    T, K = 70001, 32768
    x = torch.zeros(T, K, dtype=torch.bfloat16, device="cuda")
    x[-5:] = _rows(5, K, 9, torch.bfloat16).cuda()
    c, s = _quantize(gpu_ctx, x)
    c5, s5 = _quantize(gpu_ctx, x[-5:].contiguous())
    assert torch.equal(c[-5:], c5) and torch.equal(s[-5:], s5) and not c[:-5].any() and not s[:-5].any()


# -------------------------------------------------------------------- products --
def _act(act, z):
    half = z.shape[-1] // 2
    if act == "swiglu":
        return z[..., :half] * torch.sigmoid(z[..., :half]) * z[..., half:]
    if act == "situ":
        g, u = z[..., :half], z[..., half:]
        return SITU[0] * torch.tanh(g / SITU[0]) * torch.sigmoid(g) * SITU[1] * torch.tanh(u / SITU[1])
    if act == "silu":
        return z * torch.sigmoid(z)
    if act == "gelu":
        return z * 0.5 * torch.special.erfc(-z / 2 ** 0.5)
    if act == "gelu_tanh":
        return z * torch.sigmoid(2.0 * (2 / np.pi) ** 0.5 * (z + 0.044715 * z ** 3))
    return z


def _plain(x, w, bias, act, residual):
    """(y, bound) in 64 bits of the values x [T, K] and w [M, K]."""
    K = x.shape[1]
    z, S = x @ w.t(), x.abs() @ w.abs().t()
    if bias is not None:
        z, S = z + bias, S + bias.abs()
    e = (K + 2) * 2.0 ** -23 * S
    y = _act(act, z)
    half = z.shape[-1] // 2
    if act in ("swiglu", "situ"):
        one = torch.sigmoid if act == "swiglu" else None
        g, u, eg, eu = z[..., :half], z[..., half:], e[..., :half], e[..., half:]
        fg = g * one(g) if one else SITU[0] * torch.tanh(g / SITU[0]) * torch.sigmoid(g)
        fu = u if one else SITU[1] * torch.tanh(u / SITU[1])
        e = 1.13 * eg * (fu.abs() + eu) + fg.abs() * eu
    elif act != "none":
        e = 1.13 * e
    e = e + 2.0 ** -18 * y.abs()
    if residual is not None:
        y = y + residual
        e = e + 2.0 ** -23 * (y.abs() + residual.abs())
    return y, e + (y.abs() + e) * 2.0 ** -8 + 2.0 ** -133


def _weights(lead, K, seed, lo=110, hi=125):
    g = torch.Generator().manual_seed(seed)
    return (torch.randint(0, 256, (*lead, K // 2), generator=g, dtype=torch.uint8),
            torch.randint(lo, hi, (*lead, K // 32), generator=g, dtype=torch.uint8))


def _values(codes, scales):
    return torch.from_numpy(mx.dequantize(codes.cpu().numpy(), scales.cpu().numpy()))


def _product(ctx, x, w, act="none", bias=None, residual=None, y=None, offsets=None, stream=None):
    betas = SITU if act == "situ" else (None, None)
    M = w[0].shape[-2]
    if y is None:
        y = torch.full((x[0].shape[0], M // 2 if act in ("swiglu", "situ") else M), 7, dtype=torch.bfloat16, device="cuda")
    kw = {"bias_dev": bias, "act": act, "residual_dev": residual, "gate_beta": betas[0], "value_beta": betas[1],
          "stream": stream or _stream()}
    if offsets is None:
        ctx.mx_linear_dev(*x, *w, y, **kw)
    else:
        ctx.mx_experts_linear_dev(*x, *w, offsets, y, **kw)
    return y


def _cuda(pair):
    return tuple(t.cuda() for t in pair)


def _check_product(ctx, T, M, K, act, bias, residual, seed=0):
    x, w = _weights((T,), K, seed + 1, 120, 130), _weights((M,), K, seed + 2)
    width = M // 2 if act in ("swiglu", "situ") else M
    g = torch.Generator().manual_seed(seed)
    b = torch.randn(M, generator=g) if bias else None
    r = torch.randn(T, width, generator=g).to(torch.bfloat16) if residual else None
    y, bound = _plain(_values(*x), _values(*w), None if b is None else b.double(), act, None if r is None else r.double())
    got = _product(ctx, _cuda(x), _cuda(w), act, None if b is None else b.cuda(), None if r is None else r.cuda())
    off = (got.cpu().double() - y).abs()
    assert bool((off <= bound).all()), (float((off / bound).max()), act)
    if r is not None:  # in place
        at = r.cuda()
        _product(ctx, _cuda(x), _cuda(w), act, None if b is None else b.cuda(), at, at)
        assert torch.equal(at, got)


@pytest.mark.parametrize("T", [1, 2, 15, 16, 17, 31, 33, 64, 65, 129, 300])
@pytest.mark.parametrize("M,K", [(1, 32), (2, 64), (31, 96), (48, 128), (130, 160), (256, 256), (514, 1088)])
def test_product(gpu_ctx, T, M, K):
    _check_product(gpu_ctx, T, M, K, "none", bias=T % 2 == 0, residual=M % 2 == 0, seed=T + M)


@pytest.mark.parametrize("act", ["silu", "gelu", "gelu_tanh", "swiglu", "situ"])
@pytest.mark.parametrize("T,M,K", [(1, 2, 32), (3, 1536, 2048), (16, 62, 96), (40, 66, 544), (445, 384, 288), (130, 1032, 512)])
def test_product_with_activation(gpu_ctx, act, T, M, K):
    _check_product(gpu_ctx, T, M, K, act, bias=True, residual=True, seed=T)
    _check_product(gpu_ctx, T, M, K, act, bias=False, residual=False, seed=T + 1)


@pytest.mark.parametrize("T,M,K,act", [(1, 1536, 2048, "swiglu"), (4, 20001, 2560, "none"), (445, 2560, 1088, "none"),
                                       (1030, 4096, 2048, "swiglu"), (2100, 4100, 992, "none"), (700, 8200, 352, "silu"),
                                       (1100, 9300, 512, "none"), (1100, 9300, 1056, "swiglu"), (1030, 12000, 1024, "swiglu"),
                                       (1030, 12001, 1024, "gelu_tanh"), (600, 16000, 96, "none"), (300, 1200, 544, "situ"),
                                       (300, 1200, 1536, "situ")])
def test_product_of_size(gpu_ctx, T, M, K, act):
    _check_product(gpu_ctx, T, M, K, act, bias=True, residual=True, seed=5)


def test_unaligned_outputs(gpu_ctx):
    """y and residual that start inside 16 bytes."""
    for T, M, K in ((5, 64, 64), (200, 320, 160), (600, 512, 256)):
        x, w = _cuda(_weights((T,), K, 1, 120, 130)), _cuda(_weights((M,), K, 2))
        r = torch.randn(T, M, device="cuda").to(torch.bfloat16)
        want = _product(gpu_ctx, x, w, "none", residual=r)
        for shift in (1, 2, 4):
            buf = torch.full((T * M + 16,), 7, dtype=torch.bfloat16, device="cuda")
            rbuf = torch.zeros(T * M + 16, dtype=torch.bfloat16, device="cuda")
            y, rr = buf[shift:shift + T * M].view(T, M), rbuf[shift:shift + T * M].view(T, M)
            rr.copy_(r)
            _product(gpu_ctx, x, w, "none", residual=rr, y=y)
            assert torch.equal(y, want)
            assert bool((buf[:shift] == 7).all()) and bool((buf[shift + T * M:] == 7).all())


@pytest.mark.parametrize("T", [2, 70, 300])
def test_bad_blocks_stay_in_their_rows(gpu_ctx, T):
    """A scale byte of 255 makes NaN of its row of results (weights: its column) and of nothing else, in the last, odd
    block of K too."""
    M, K = 96, 160
    x, w = _weights((T,), K, 1, 120, 130), _weights((M,), K, 2)
    clean = _product(gpu_ctx, _cuda(x), _cuda(w))
    for block in (0, 2, 4):
        xs, ws = x[1].clone(), w[1].clone()
        xs[1, block], ws[33, block] = 255, 255
        y = _product(gpu_ctx, (x[0].cuda(), xs.cuda()), (w[0].cuda(), ws.cuda()))
        nan = torch.zeros(T, M, dtype=torch.bool)
        nan[1], nan[:, 33] = True, True
        assert torch.equal(torch.isnan(y).cpu(), nan)
        assert torch.equal(y.cpu()[~nan], clean.cpu()[~nan])


def test_scales_at_their_ends(gpu_ctx):
    """2^-127 and 2^127 on either side; past fp32 the results are infinite, below it zero."""
    K = 96
    for a, b, want in ((0, 254, 1.0), (254, 0, 1.0), (0, 127, 2.0 ** -127), (254, 254, float("inf")), (0, 0, 0.0)):
        for T in (1, 100):
            x = torch.full((T, K // 2), 0x22, dtype=torch.uint8), torch.full((T, K // 32), a, dtype=torch.uint8)
            w = torch.full((40, K // 2), 0x22, dtype=torch.uint8), torch.full((40, K // 32), b, dtype=torch.uint8)
            y = _product(gpu_ctx, _cuda(x), _cuda(w)).cpu().double()
            assert bool((y == (want * K if want < 2 else want)).all()), (a, b, float(y[0, 0]))


def test_rows_alone_and_in_a_batch(gpu_ctx):
    """The same rows in calls of every size agree to the bound of the sums' order."""
    M, K = 544, 1056
    w, x = _weights((M,), K, 3), _weights((600,), K, 4, 120, 130)
    y, bound = _plain(_values(*x), _values(*w), None, "none", None)
    for T in (1, 7, 16, 17, 40, 64, 100, 128, 256, 300, 512, 600):
        got = _product(gpu_ctx, (x[0][:T].cuda(), x[1][:T].cuda()), _cuda(w)).cpu().double()
        assert bool(((got - y[:T]).abs() <= bound[:T]).all())


def test_weights_past_32_bits(gpu_ctx):
    """Weights of more than 2^32 bytes of codes: the last rows."""
    M, K, T = 2_100_000, 4128, 3
    w = torch.zeros(M, K // 2, dtype=torch.uint8, device="cuda"), torch.full((M, K // 32), 127, dtype=torch.uint8, device="cuda")
    few, x = _cuda(_weights((50,), K, 3)), _cuda(_weights((T,), K, 4, 120, 130))
    w[0][-50:], w[1][-50:] = few
    y = _product(gpu_ctx, x, w)
    y50 = _product(gpu_ctx, x, few)
    bound = _plain(_values(*x), _values(*few), None, "none", None)[1]
    assert bool(((y[:, -50:].double() - y50.double()).abs().cpu() <= 2 * bound).all()) and not y[:, :-50].any()


# ------------------------------------------------------------------- by expert --
def _check_experts(ctx, counts, M, K, act="none", bias=True, residual=True, behind=0, seed=0):
    E, n = len(counts), sum(counts) + behind
    width = M // 2 if act in ("swiglu", "situ") else M
    x, w = _weights((n,), K, seed + 1, 120, 130), _weights((E, M), K, seed + 2)
    g = torch.Generator().manual_seed(seed)
    b = torch.randn(E, M, generator=g) if bias else None
    r = torch.randn(n, width, generator=g).to(torch.bfloat16) if residual else None
    offsets = torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32).cuda()
    got = _product(ctx, _cuda(x), _cuda(w), act, None if b is None else b.cuda(), None if r is None else r.cuda(),
                   offsets=offsets)
    a = 0
    for e, c in enumerate(counts):
        if c:
            y, bound = _plain(_values(x[0][a:a + c], x[1][a:a + c]), _values(w[0][e], w[1][e]),
                              None if b is None else b[e].double(), act, None if r is None else r[a:a + c].double())
            off = (got[a:a + c].cpu().double() - y).abs()
            assert bool((off <= bound).all()), (e, float((off / bound).max()))
        a += c
    assert bool((got[a:] == 7).all())  # rows behind the last stay as they were


@pytest.mark.parametrize("counts", [[1], [0, 0, 3], [5, 0, 1, 16, 17, 0], [0, 130, 0, 0, 300, 1, 64], [33] * 9, [0] * 255 + [2],
                                    [1] * 256, [2, 0] * 64])
@pytest.mark.parametrize("M,K,act", [(96, 160, "swiglu"), (130, 256, "none")])
def test_experts(gpu_ctx, counts, M, K, act):
    _check_experts(gpu_ctx, counts, M, K, act, behind=3, seed=len(counts))
    _check_experts(gpu_ctx, counts, M, K, act, bias=False, residual=False, seed=len(counts) + 1)


@pytest.mark.parametrize("act", ["situ", "gelu", "silu", "gelu_tanh"])
def test_experts_with_activation(gpu_ctx, act):
    _check_experts(gpu_ctx, [3, 0, 40, 1], 64, 96, act, behind=1)


@pytest.mark.parametrize("counts,M,K", [([500, 3, 0, 700, 260, 0, 40, 90] * 2, 520, 544), ([130] * 20, 1536, 256),
                                        ([700, 900], 1030, 288), ([40] * 64, 768, 1088),
                                        ([30, 0, 70] * 3, 520, 1024), ([1, 2] * 12, 2000, 512),
                                        ([1500, 3, 2100, 500], 3200, 512), ([1000, 1500, 0, 1600], 3200, 352)])
def test_experts_of_size(gpu_ctx, counts, M, K):
    _check_experts(gpu_ctx, counts, M, K, "swiglu", behind=2)


def test_no_rows_and_offsets_past_them(gpu_ctx):
    """Experts without rows write nothing; offsets past the rows (a caller's mistake) are cut to them."""
    x, w = _cuda(_weights((40,), 64, 1, 120, 130)), _cuda(_weights((3, 64), 64, 2))
    none = _product(gpu_ctx, x, w, offsets=torch.zeros(4, dtype=torch.int32, device="cuda"))
    assert bool((none == 7).all())
    wild = _product(gpu_ctx, x, w, offsets=torch.tensor([-5, 10, 1 << 30, 1 << 30], dtype=torch.int32, device="cuda"))
    tame = _product(gpu_ctx, x, w, offsets=torch.tensor([0, 10, 40, 40], dtype=torch.int32, device="cuda"))
    assert torch.equal(wild, tame)


# ------------------------------------------------- streams, graphs and contexts --
def test_on_other_streams_and_captured(gpu_ctx):
    """Quantizing and products captured into two graphs that replay at once on two streams, between eager calls."""
    T, M, K = 33, 256, 288
    xs = [_rows(T, K, i, torch.bfloat16).cuda() for i in range(2)]
    w = _cuda(_weights((M,), K, 7))
    sides = []
    for i in range(2):
        c, s = torch.zeros(T, K // 2, dtype=torch.uint8, device="cuda"), torch.zeros(T, K // 32, dtype=torch.uint8, device="cuda")
        y, st, gr = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda"), torch.cuda.Stream(), torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(gr, stream=st):
            gpu_ctx.mx_quantize_dev(xs[i], c, s, stream=torch.cuda.current_stream())
            gpu_ctx.mx_linear_dev(c, s, *w, y, act="silu", stream=torch.cuda.current_stream())
        sides.append((gr, st, y))
    for turn in range(3):
        for i in range(2):
            xs[i].copy_(_rows(T, K, 10 * turn + i, torch.bfloat16))
        torch.cuda.synchronize()
        for gr, st, _ in sides:
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(sides[i][2], _product(gpu_ctx, _quantize(gpu_ctx, xs[i]), w, "silu"))


def test_two_contexts_and_the_contexts_own_stream(gpu_ctx):
    from raon_npu_amd.device import Context

    x, w = _rows(20, 96, 1, torch.bfloat16).cuda(), _cuda(_weights((64,), 96, 2))
    want = _product(gpu_ctx, _quantize(gpu_ctx, x), w)
    other = Context(0)
    try:
        c = torch.empty(20, 48, dtype=torch.uint8, device="cuda")
        s = torch.empty(20, 3, dtype=torch.uint8, device="cuda")
        y = torch.empty(20, 64, dtype=torch.bfloat16, device="cuda")
        torch.cuda.synchronize()
        other.mx_quantize_dev(x, c, s)
        other.mx_linear_dev(c, s, *w, y)
        other.synchronize()
        assert torch.equal(y, want)
    finally:
        other.close()


# ------------------------------------------------------------ calls at the limits --
@pytest.mark.parametrize("T,M,K", [(3, 40, 96), (3, 200, 1024), (90, 200, 1024), (90, 200, 96), (1100, 9300, 512)])
def test_scales_at_any_address(gpu_ctx, T, M, K):
    x, w = _cuda(_weights((T,), K, 1, 120, 130)), _cuda(_weights((M,), K, 2))
    want = _product(gpu_ctx, x, w)
    bound = None
    for shift in (1, 2, 3, 4, 8):
        moved = []
        for s in (x[1], w[1]):
            buf = torch.zeros(s.numel() + 16, dtype=torch.uint8, device="cuda")
            moved.append(buf[shift:shift + s.numel()].view(s.shape))
            moved[-1].copy_(s)
        got = _product(gpu_ctx, (x[0], moved[0]), (w[0], moved[1]))
        if bound is None:  # scales that are not aligned take another kernel: the sums' order may be another
            bound = _plain(_values(*x), _values(*w), None, "none", None)[1]
        assert bool(((got.cpu().double() - want.cpu().double()).abs() <= 2 * bound).all()), shift


@pytest.mark.parametrize("T", [1, 100, 1100])
def test_swiglu_where_the_exponential_is_subnormal(gpu_ctx, T):
    """Gates of -80 to -104 give results down to bf16's subnormal ones, 0 only below; gates past 88 give gate times up; -0 and
    NaN as they come.  g sigmoid(g) u: exp(g) is off by (4 + |g|) 2^-23 of it (its argument's rounding, twice, for it is
    squared), the rest by 2^-21."""
    M = 9300
    sums = torch.tensor([0.0, 0.5, 4.5, 5.0, 5.5, 6.0, 6.5, 7.0, 7.5, 10.0, 12.0])
    g = torch.Generator().manual_seed(1)
    pick = torch.randint(0, len(sums), (M // 2,), generator=g)
    sign = torch.where(torch.rand(M // 2, generator=g) < 0.8, -1.0, 1.0)
    w = torch.zeros(M, 64)
    first = sums[pick].clamp(max=6.0)
    first = torch.where((first == 4.5) | (first == 5.0) | (first == 5.5), 4.0, first)
    w[:M // 2, 0], w[:M // 2, 1] = sign * first, sign * (sums[pick] - first)
    w[M // 2:, 32], w[:, 5], w[:, 37] = 1.0, 6.0, 6.0  # the blocks' scales are 2^0; columns 5 and 37 meet zeros
    x = torch.zeros(T, 64)
    x[:, :2], x[:, 32] = 16.0, 1.0
    codes = [tuple(torch.from_numpy(c).cuda() for c in mx.quantize(v.numpy())) for v in (x, w)]
    assert torch.equal(_values(*codes[1]), w.double()) and torch.equal(_values(*codes[0]), x.double())
    z = (16 * sign * sums[pick]).double()
    want = z * torch.sigmoid(z)
    got = _product(gpu_ctx, *codes, "swiglu").cpu().double()
    bound = want.abs() * (2.0 ** -8 + (6 + 2 * z.abs()) * 2.0 ** -23 + 2.0 ** -21) + 2.0 ** -133
    assert bool(((got - want).abs() <= bound).all()), float(((got - want).abs() / bound).max())
    assert bool((got[:, (z < -70) & (z > -90)] != 0).all())


def test_rows_in_front_of_the_first_expert(gpu_ctx):
    """Offsets that begin past 0 leave the rows in front as they were."""
    for n, M in ((40, 64), (3000, 4096)):
        x, w = _cuda(_weights((n,), 64, 1, 120, 130)), _cuda(_weights((2, M), 64, 2))
        off = torch.tensor([7, n // 2, n - 3], dtype=torch.int32, device="cuda")
        y = _product(gpu_ctx, x, w, offsets=off)
        assert bool((y[:7] == 7).all()) and bool((y[n - 3:] == 7).all())
        for e, (a, b) in enumerate(((7, n // 2), (n // 2, n - 3))):
            rows = slice(a, b, max(1, (b - a) // 50))
            want, bound = _plain(_values(x[0][rows], x[1][rows]), _values(w[0][e], w[1][e]), None, "none", None)
            assert bool(((y[rows].cpu().double() - want).abs() <= bound).all())


def test_very_wide_rows_and_many_scales(gpu_ctx):
    """More columns than the tiles' 32-bit offsets serve, and scales of a matrix past 2^32 bytes: the last weight rows."""
    for T, M, K in ((20, 8200, (1 << 20) + 32), (20, 4_300_000, 32 * 1024)):
        w = torch.zeros(M, K // 2, dtype=torch.uint8, device="cuda"), torch.full((M, K // 32), 127, dtype=torch.uint8, device="cuda")
        few, x = _cuda(_weights((30,), K, 3)), _cuda(_weights((T,), K, 4, 120, 130))
        w[0][-30:], w[1][-30:] = few
        y = _product(gpu_ctx, x, w)
        want, bound = _plain(_values(*x), _values(*few), None, "none", None)
        assert bool(((y[:, -30:].cpu().double() - want).abs() <= bound).all()) and not y[:, :-30].any()
        del w, y
        torch.cuda.empty_cache()


def test_the_largest_call_is_refused_or_served(gpu_ctx):
    """Grids past 2^32 threads are refused; nothing is launched."""
    held = torch.zeros(64, dtype=torch.uint8, device="cuda")
    from raon_npu_amd import _lib

    with pytest.raises(ValueError, match="too many"):
        _lib.call("rmoe_mx_linear_dev", gpu_ctx.handle, 1 << 40, 1 << 50, (1 << 31) - 1, 32, 1 << 45, 1 << 46, 1 << 16, None,
                  _lib.ACT_NONE, 0.0, 0.0, None, 1 << 52, None)
    assert not held.any()


@pytest.mark.parametrize("T,M,K,act", [(2100, 9300, 1024, "swiglu"), (4100, 5001, 512, "gelu"), (5200, 4096, 1536, "none"),
                                       (2304, 8192, 512, "situ")])
def test_more_tiles_than_workgroups(gpu_ctx, T, M, K, act):
    """Workgroups that go on to further tiles, their first stage requested while the one before is finished."""
    _check_product(gpu_ctx, T, M, K, act, True, True)


@pytest.mark.parametrize("counts,M,K,act", [([3000, 1, 0, 5000, 257, 2700], 2056, 512, "swiglu"),
                                            ([300] * 20 + [0, 4000, 1, 255, 256], 1536, 1024, "none"),
                                            ([130] * 63 + [0, 256], 1536, 512, "swiglu"),
                                            ([125] * 70, 1540, 544, "swiglu")])
def test_more_experts_tiles_than_workgroups(gpu_ctx, counts, M, K, act):
    _check_experts(gpu_ctx, counts, M, K, act, True, True, behind=700)


def test_further_tiles_are_the_same_each_time(gpu_ctx):
    """The same rows in one call and in calls of at most as many tiles as workgroups, again and again."""
    x, w = _cuda(_weights((6144,), 2048, 1, 120, 130)), _cuda(_weights((4096,), 2048, 2))
    parts = [_product(gpu_ctx, tuple(t[i:i + 2048] for t in x), w, "swiglu") for i in range(0, 6144, 2048)]
    for _ in range(20):
        assert torch.equal(_product(gpu_ctx, x, w, "swiglu"), torch.cat(parts))


def test_many_tiles_captured_with_new_offsets(gpu_ctx):
    """Products of more tiles than workgroups in a graph: replayed with other rows and other offsets, eager work between."""
    n, E, M, K = 6000, 4, 4096, 512
    x, w = _cuda(_weights((n,), K, 1, 120, 130)), _cuda(_weights((E, M), K, 2))
    off = torch.tensor([0, 1500, 3000, 4500, 6000], dtype=torch.int32, device="cuda")
    y = torch.zeros(n, M, dtype=torch.bfloat16, device="cuda")
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        _product(gpu_ctx, x, w, y=y, offsets=off, stream=torch.cuda.current_stream())
    for turn, counts in enumerate(([1500] * 4, [6000, 0, 0, 0], [1, 0, 0, 5999], [0, 0, 0, 0], [257, 2000, 3, 600])):
        for t, s in zip(x, _weights((n,), K, 10 + turn, 120, 130)):
            t.copy_(s)
        off.copy_(torch.tensor([0, *np.cumsum(counts)], dtype=torch.int32))
        y.fill_(7)
        graph.replay()
        torch.cuda.synchronize()
        want = _product(gpu_ctx, x, w, y=torch.full_like(y, 7), offsets=off)
        assert bool((want[sum(counts):] == 7).all()) and (not counts[0] or not bool((want[0] == 7).all()))
        assert torch.equal(y, want), counts


@pytest.mark.parametrize("T,M,K,act", [(1, 64010, 96, "swiglu"), (2, 64003, 512, "none"), (3, 64010, 160, "situ"),
                                       (40, 64010, 512, "swiglu"), (96, 33001, 288, "silu"), (97, 33001, 96, "none")])
def test_few_rows_of_many_weights(gpu_ctx, T, M, K, act):
    _check_product(gpu_ctx, T, M, K, act, True, True)


def test_quantize_the_widest_rows(gpu_ctx):
    """Rows of 2^30 columns and of a few fewer (a last block that is filled up): their last and first columns."""
    few = _rows(4, 4096, 3, torch.bfloat16).cuda()
    for K in (1 << 30, (1 << 30) - 37):
        x = torch.zeros(2, K, dtype=torch.bfloat16, device="cuda")
        P, width = -(-K // 32) * 32, 4096 - (-K % 32)
        x[:, :4096], x[:, -width:] = few[:2], few[2:, :width]
        c = torch.full((2, P // 2), 0xEE, dtype=torch.uint8, device="cuda")
        s = torch.full((2, P // 32), 0xEE, dtype=torch.uint8, device="cuda")
        gpu_ctx.mx_quantize_dev(x, c, s, stream=_stream())
        for rows, part, got in ((few[:2], slice(0, 2048), slice(0, 128)),
                                (few[2:, :width].contiguous(), slice(P // 2 - 2048, None), slice(P // 32 - 128, None))):
            c1, s1 = _quantize(gpu_ctx, rows)
            assert torch.equal(c[:, part], c1) and torch.equal(s[:, got], s1)
        assert not c[:, 2048:-2048].any() and not s[:, 128:-128].any()
        del x, c, s
        torch.cuda.empty_cache()
