"""GPU: products with an epilogue whose weights hold arbitrary bytes behind the columns that count: the padding of
an expert's down projection past I, and what a narrower input does not reach of a dense matrix.

Each result equals, bit for bit, that of the same weights with zeros there, at row counts on both sides of every
change of kernel and tile, and meets the bounds against 64 bits."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import bfp16 as B
from oracle import q4nx as Q
from raon_npu_amd.geometry import MoeGeometry
from test_gpu_linear_act import _check, _reference

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

H, I, E = 512, 832, 6  # down [512, 832 of 1024]: six and a half K tiles of 128
KINDS = {"q4nx": ["inf", "nan", "1e30", "overflow"], "bfp16": ["1e30", "bytes", "e255"]}


def _blobs(fmt, M, K, live, kind, seed):
    """(bytes with ``kind`` from column ``live`` on, bytes with zeros there, the live weights in float64)."""
    rng = np.random.default_rng(seed)
    w = rng.normal(0.0, 0.02, (M, K)).astype(np.float32)
    if fmt == "q4nx":
        c, s, m = Q.quantize(w)
        wd = torch.from_numpy(Q.dequantize_simple(c, s, m)[:, :live]).double()
        g = -(-live // 32)
        s0, m0 = s.copy(), m.copy()
        s0[:, g:] = 0
        m0[:, g:] = 0
        fill = {"inf": (np.inf, -np.inf), "nan": (np.nan, np.nan), "1e30": (1e30, -3e30), "overflow": (3e38, 3e38)}[kind]
        s[:, g:], m[:, g:] = fill
        return Q.pack_gemv(c, s, m), Q.pack_gemv(c, s0, m0), wd
    w[:, live:] = 0
    zero = B.pack_gemv(w)
    wd = torch.from_numpy(B.dequantize_packed(zero, K, M)[:, :live]).double()
    if kind == "1e30":
        w[:, live:] = rng.normal(0, 1e30, (M, K - live))
        return B.pack_gemv(w), zero, wd
    buf = np.frombuffer(zero, np.uint8).reshape(M // 128, K // 256, 4, 2, 32, 144).copy()
    junk = rng.integers(0, 256, buf.shape, dtype=np.uint8)
    if kind == "e255":
        junk[..., :16] = 255
        junk[..., 16:] = 0x80  # mantissas of -128
    block = np.arange(K // 256)[:, None] * 32 + np.arange(32)[None]
    behind = np.broadcast_to((block >= live // 8)[None, :, None, None, :, None], buf.shape)
    buf[behind] = junk[behind]
    return buf.tobytes(), zero, wd


def _layers(gpu_ctx, fmt, kind, I=I):
    """Two layers that differ in the padding of down alone, and down's live weights."""
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=2)
    dn = [_blobs(fmt, H, g.inter_pad, I, kind, 10 + e) for e in range(E + 1)]
    out = []
    for which in (0, 1):
        blob = b"".join(b[which] for b in dn)
        if fmt == "bfp16":
            lyr = gpu_ctx.create_layer_d(7400 + which, g)
            lyr.upload_d(2, 0, blob)
        else:
            lyr = gpu_ctx.create_layer(7400 + which, g)
            c, s, m = Q.quantize(np.zeros((2 * I, H), np.float32))
            lyr.upload_experts(Q.pack_gemv(c, s, m) * (E + 1), blob)
        out.append(lyr)
    return out, [b[2] for b in dn]


def _rows(n, width, live, seed, tail):
    """Rows of ``width`` columns, from ``live`` on zero or (``tail``) of any value."""
    x = torch.randn(n, width, generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16)
    if not tail:
        x[:, live:] = 0
    return x


@pytest.mark.parametrize("fmt,kind", [(f, k) for f in KINDS for k in KINDS[f]])
def test_down_by_expert(gpu_ctx, fmt, kind):
    """Fewer rows than experts, then up to 24, 64 and more an expert; rows of I columns and of Ipad."""
    (got, want), w = _layers(gpu_ctx, fmt, kind)
    st = torch.cuda.current_stream()
    for n in (1, 5, 6, 150, 390, 1200):
        counts = [0, n // 2, 0, n - n // 2 - n // 5, n // 5, 0]
        offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
        for lyr in (got, want):
            lyr.reserve_experts_linear(n)
        for width, tail in ((I, False), (1024, False), (1024, True)):
            x = _rows(n, width, I, n, tail)
            ys = []
            for lyr in (got, want):
                y = torch.full((n, H), 9.0, dtype=torch.bfloat16, device="cuda")
                lyr.experts_linear_dev("down", x.cuda(), offsets.cuda(), y, stream=st)
                ys.append(y)
            assert torch.equal(*ys), (n, width, tail)
            for e in range(E):
                a, z = int(offsets[e]), int(offsets[e + 1])
                if a < z:
                    _check(ys[0][a:z], *_reference(x[a:z, :I], w[e], None, "none", None, n >= E), (n, width, e))
    got.free()
    want.free()


@pytest.mark.parametrize("fmt,kind", [(f, k) for f in KINDS for k in KINDS[f]])
def test_down_that_ends_with_a_tile(gpu_ctx, fmt, kind):
    """I = 384 of 512: three whole K tiles, the fourth is padding alone."""
    (got, want), w = _layers(gpu_ctx, fmt, kind, 384)
    st = torch.cuda.current_stream()
    for n in (5, 60, 700):
        offsets = torch.tensor([0, 0, n // 3, n // 3, n, n, n], dtype=torch.int32)
        for width in (384, 512):
            x = _rows(n, width, 384, n, True)
            ys = []
            for lyr in (got, want):
                lyr.reserve_experts_linear(n)
                y = torch.full((n, H), 9.0, dtype=torch.bfloat16, device="cuda")
                lyr.experts_linear_dev("down", x.cuda(), offsets.cuda(), y, stream=st)
                ys.append(y)
            assert torch.equal(*ys), (n, width)
            for e in (1, 3):
                a, z = int(offsets[e]), int(offsets[e + 1])
                _check(ys[0][a:z], *_reference(x[a:z, :384], w[e], None, "none", None, n >= E), (n, width, e))
    got.free()
    want.free()


# Rows of a dense [512, .] matrix: tiles of few rows up to 4,032 (q4nx 5,056), 64 x 128 tiles by two groups of K up to
# 12,672, 128 x 256 tiles, and (258 tiles) the last two of them cut along K.
ROWS = (1, 4, 5, 40, 64 * 63, 64 * 63 + 1, 64 * 79, 64 * 79 + 1, 128 * 100, 128 * 129)


def _many(M, T):
    return -(-T // 64) * (M // 128) >= 256


def _compare(mats, w, width, live, tail=False):
    M = mats[0].M
    st = torch.cuda.current_stream()
    wd = w.cuda()
    for T in ROWS:
        x = _rows(T, width, live, T + width, tail).cuda()
        ys = []
        for mat in mats:
            mat.reserve_act(T)
            y = torch.full((T, M), 9.0, dtype=torch.bfloat16, device="cuda")
            mat.linear_act_dev(x, T, y, act="silu", stream=st)
            ys.append(y)
        assert torch.equal(*ys), (T, width)
        pick = torch.cat([torch.arange(min(T, 130)), torch.arange(max(0, T - 130), T)]).cuda()
        ref, e = _reference(x[pick, :live], wd, None, "silu", None, _many(M, T))
        _check(ys[0][pick], ref.cpu(), e.cpu(), (T, width))


@pytest.mark.parametrize("fmt,kind", [(f, k) for f in KINDS for k in KINDS[f]])
def test_views_of_down(gpu_ctx, fmt, kind):
    layers, w = _layers(gpu_ctx, fmt, kind)
    views = [lyr.expert_matrix(3, "down") for lyr in layers]
    _compare(views, w[3], I, I)
    _compare(views, w[3], 1024, I, tail=True)
    for v in views:
        v.free()
    for lyr in layers:
        lyr.free()


@pytest.mark.parametrize("fmt,kind", [(f, k) for f in KINDS for k in KINDS[f]])
@pytest.mark.parametrize("K_in", [8, 136, 832, 1000, 1088])
def test_dense_narrower_than_the_matrix(gpu_ctx, fmt, kind, K_in):
    """A narrower input meets the leading columns alone, whatever stands behind them (q4nx: from the next group on)."""
    M, K = 512, 1280
    got, want, w = _blobs(fmt, M, K, K_in, kind, 30)
    mats = [gpu_ctx.upload_matrix(b, M, K, fmt=fmt) for b in (got, want)]
    _compare(mats, w, K_in, K_in)
    for m in mats:
        m.free()
