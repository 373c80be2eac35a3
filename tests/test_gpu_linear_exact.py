"""GPU: products with an epilogue use the weights as they are, whichever kernel a number of rows selects: each weight
is seen alone, to fp32's precision, and rows of any size, of zeros, of infinities and NaN go through the kernel of
many rows as through the one of few.

Bounds.  A q4nx product adds s (n - 8) x, 8 s X and m X (X: a group's sum of x) or 16 s n / 16 x and m X in fp32: with
T = |s (n - 8)| + 8 |s| + |m| (bfp16: |w|) a sum over K columns is off by at most (K + 64) 2^-23 sum |x| T.  The kernel
of many rows cuts values of x below 2^-30 of their row's largest by up to 2^-37 of it and is off by up to 2^-35 of a
row's largest weight in groups far below it, by 2^-28 in bfp16 blocks more than 2^27 below (there are none here):
K 2^-34 max |x| max |w| together."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import bfp16 as B
from oracle import q4nx as Q
from raon_npu_amd.geometry import MoeGeometry
from test_gpu_linear_act import _check

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _weights(fmt, M, K, seed, std=0.02, live=None):
    """(bytes, w, T of the bounds) in float64."""
    rng = np.random.default_rng(seed)
    w = rng.normal(0.0, std, (M, K)).astype(np.float32)
    if live is not None:
        w[:, live:] = 0
    if fmt == "bfp16":
        blob = B.pack_gemv(w)
        wd = torch.from_numpy(B.dequantize_packed(blob, K, M)).double()
        return blob, wd, wd.abs()
    c, s, m = Q.quantize(w)
    c, s, m = (torch.from_numpy(a) for a in (c, s, m))
    cd, sd, md = c.double(), s.double().repeat_interleave(32, 1), m.double().repeat_interleave(32, 1)
    return Q.pack_gemv(c.numpy(), s.numpy(), m.numpy()), md + sd * cd, sd.abs() * (cd - 8).abs() + 8 * sd.abs() + md.abs()


def _bound(x, w, t):
    """How far the sums x w^T may be off."""
    K = x.shape[1]
    far = K * 2.0 ** -34 * x.abs().amax(1, keepdim=True) * w.abs().amax(1)[None]
    return (K + 64) * 2.0 ** -23 * (x.abs() @ t.t().contiguous()) + far


def _one_by_one(T, K, seed):
    """Row t holds one power of two, at a column that differs from its neighbours'."""
    col = (torch.arange(T) * 37 + seed) % K
    x = torch.zeros(T, K, dtype=torch.bfloat16)
    x[torch.arange(T), col] = (2.0 ** (torch.arange(T) % 7 - 3)).to(torch.bfloat16)
    return x, col


def _weight_left(x, col, w, t, run):
    """``run(residual)`` of y = x w^T + residual with the bf16 rounding of each product taken away: what is left of
    the weight itself comes back.  One column a row: the sum has three nonzero terms (and the kernel's own zeros),
    off by 4 steps of fp32 of them."""
    v = x[torch.arange(len(col)), col].double()[:, None]
    z = (v * w[:, col].t()).contiguous()
    r = -z.to(torch.bfloat16)
    y = run(r).cpu().double()
    ref, terms = z + r.double(), v.abs() * 2 * t[:, col].t()
    e = 2.0 ** -22 * terms
    bad = ~((y - ref).abs() <= 2.0 ** -8 * (ref.abs() + e) + e)
    assert not bad.any(), (bad.nonzero()[:4].tolist(), y[bad][:4].tolist(), ref[bad][:4].tolist(), float(bad.float().mean()))


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("T", [1, 4, 40, 130, 700, 64 * 64 + 1, 64 * 80 + 1, 128 * 100, 128 * 129])
def test_each_weight_of_a_matrix(gpu_ctx, fmt, T):
    """Tiles of few rows up to 700 (q4nx 4,097), 64 x 128 tiles by two groups of K, 128 x 256 tiles, and the last of them
    cut."""
    M, K = 512, 1024
    blob, w, t = _weights(fmt, M, K, 3)
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    x, col = _one_by_one(T, K, T)
    y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")

    def run(r):
        mat.linear_act_dev(x.cuda(), T, y, residual_dev=r.cuda(), stream=torch.cuda.current_stream())
        return y

    _weight_left(x, col, w, t, run)
    mat.free()


@pytest.mark.parametrize("d_layout", [False, True])
@pytest.mark.parametrize("part", ["gate_up", "down"])
def test_each_weight_of_the_experts(gpu_ctx, d_layout, part):
    """Fewer rows than experts, then 24, 64 and more an expert in the mean."""
    H, I, E = 512, 320, 5
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=2)
    gu = [_weights("q4nx", 2 * I, H, e) for e in range(E + 1)]
    dn = [_weights("bfp16" if d_layout else "q4nx", H, g.inter_pad, 50 + e, live=I) for e in range(E + 1)]
    if d_layout:
        lyr = gpu_ctx.create_layer_d(7500, g)
        lyr.upload_d(1, 0, b"".join(b for b, _, _ in gu[:E]))
        lyr.upload_d(2, 0, b"".join(b for b, _, _ in dn))
    else:
        lyr = gpu_ctx.create_layer(7500, g)
        lyr.upload_experts(b"".join(b for b, _, _ in gu), b"".join(b for b, _, _ in dn))
    ws, M, K = (gu, 2 * I, H) if part == "gate_up" else (dn, H, I)
    for n in (4, 5, 120, 320, 900):
        lyr.reserve_experts_linear(n)
        counts = [n // E + (e < n % E) for e in range(E)]
        offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32)
        x, col = _one_by_one(n, K, n)
        y = torch.zeros(n, M, dtype=torch.bfloat16, device="cuda")
        for e in range(E):
            a, z = int(offsets[e]), int(offsets[e + 1])
            if a == z:
                continue
            _, w, t = ws[e]

            def run(r):
                res = torch.zeros(n, M, dtype=torch.bfloat16)
                res[a:z] = r
                lyr.experts_linear_dev(part, x.cuda(), offsets.cuda(), y, residual_dev=res.cuda(),
                                       stream=torch.cuda.current_stream())
                return y[a:z]

            _weight_left(x[a:z], col[a:z], w[:, :K], t[:, :K], run)
    lyr.free()


MANY = [(512, 64 * 81), (256, 128 * 200)]  # 64 x 128 and 128 x 256 tiles


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("M,T", MANY)
def test_ranges_of_values_in_many_rows(gpu_ctx, fmt, M, T):
    """Rows of 2^-60 to 2^60, of zeros, and with one value far above the others, under weights of 2^-40 to 2^30."""
    K = 512
    st = torch.cuda.current_stream()
    for std in (2.0 ** -40, 1.0, 2.0 ** 30):
        blob, w, t = _weights(fmt, M, K, 9, std=std)
        mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
        mat.reserve_act(T)
        x = torch.randn(T, K, generator=torch.Generator().manual_seed(T)) * 2.0 ** torch.linspace(-60, 60, T)[:, None].round()
        x[T // 2] = 0
        x[5::64, 5] *= 2.0 ** 20
        x[6::64, 7] *= 2.0 ** 34  # the others end below fp16's range
        x = x.to(torch.bfloat16)
        y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(x.cuda(), T, y, stream=st)
        xd, wd = x.cuda().double(), w.cuda()
        _check(y, (xd @ wd.t().contiguous()).cpu(), _bound(xd, wd, t.cuda()).cpu(), std)
        assert not y[T // 2].any()
        mat.free()


@pytest.mark.parametrize("T", [40, 64 * 81])
def test_weights_at_the_end_of_the_range(gpu_ctx, T):
    """Groups whose largest possible weight, m + 15 s, is past fp32's range, and whose weights are not."""
    M, K = 512, 256
    rng = np.random.default_rng(4)
    c = rng.integers(0, 3, (M, K)).astype(np.uint8)
    s, m = np.full((M, K // 32), 1.2e37, np.float32), rng.choice([3e38, -3e38, 1e37], (M, K // 32)).astype(np.float32)
    blob = Q.pack_gemv(c, s, m)
    _, s, m = (torch.from_numpy(np.asarray(a)).double() for a in Q.parse_gemv(blob, K, M))
    cd, sd, md = torch.from_numpy(c).double(), s.repeat_interleave(32, 1), m.repeat_interleave(32, 1)
    w, t = md + sd * cd, sd * (cd - 8).abs() + 8 * sd + md.abs()
    assert bool((md + 15 * sd > 3.4028235e38).any()) and float(w.abs().max()) < 3.4028235e38
    mat = gpu_ctx.upload_matrix(blob, M, K)
    mat.reserve_act(T)
    x = (torch.randn(T, K, generator=torch.Generator().manual_seed(1)) * 2.0 ** -118).to(torch.bfloat16)
    y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
    mat.linear_act_dev(x.cuda(), T, y, stream=torch.cuda.current_stream())
    _check(y, x.double() @ w.t(), _bound(x.double(), w, t))
    mat.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
@pytest.mark.parametrize("M,T", MANY)
def test_non_finite_rows_among_many_stay_in_their_row(gpu_ctx, fmt, M, T):
    K = 512
    blob, _, _ = _weights(fmt, M, K, 9)
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    st = torch.cuda.current_stream()
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(2)).to(torch.bfloat16)
    want, y = (torch.zeros(T, M, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    mat.linear_act_dev(x.cuda(), T, want, stream=st)
    bad = [3, 17, 70, T - 1]
    x[3, 7], x[17, 300], x[70, 0], x[T - 1, K - 1] = (float(v) for v in ("inf", "nan", "-inf", "nan"))
    x[17, 301] = float("inf")
    mat.linear_act_dev(x.cuda(), T, y, stream=st)
    keep = torch.ones(T, dtype=torch.bool)
    keep[bad] = False
    assert torch.equal(y[keep.cuda()], want[keep.cuda()])
    assert not y[bad].isfinite().any()
    mat.free()


@pytest.mark.parametrize("d_layout", [False, True])
def test_ranges_and_non_finite_rows_by_expert(gpu_ctx, d_layout):
    """The same by expert, in tiles of 32, 64 and 128 rows."""
    H, I, E = 512, 320, 3
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=1)
    fmt = "bfp16" if d_layout else "q4nx"
    dn = [_weights(fmt, H, g.inter_pad, 60 + e, live=I) for e in range(E + 1)]
    blob = b"".join(b for b, _, _ in dn)
    if d_layout:
        lyr = gpu_ctx.create_layer_d(7501, g)
        lyr.upload_d(2, 0, blob)
    else:
        lyr = gpu_ctx.create_layer(7501, g)
        c, s, m = Q.quantize(np.zeros((2 * I, H), np.float32))
        lyr.upload_experts(Q.pack_gemv(c, s, m) * (E + 1), blob)
    st = torch.cuda.current_stream()
    for n in (3, 60, 180, 700):
        lyr.reserve_experts_linear(n)
        offsets = torch.tensor([0, n // 3, n // 3, n], dtype=torch.int32)
        x = torch.randn(n, I, generator=torch.Generator().manual_seed(n)) * 2.0 ** torch.linspace(-60, 60, n)[:, None].round()
        x[n // 2] = 0
        x[n - 1, 5] *= 2.0 ** 20
        x = x.to(torch.bfloat16)
        y, other = (torch.zeros(n, H, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        lyr.experts_linear_dev("down", x.cuda(), offsets.cuda(), y, stream=st)
        for e in (0, 2):
            a, z = int(offsets[e]), int(offsets[e + 1])
            xd, w, t = x[a:z].double(), dn[e][1][:, :I], dn[e][2][:, :I]
            _check(y[a:z], xd @ w.t(), _bound(xd, w, t), (n, e))
        x[0, 7], x[n - 1, 300] = float("inf"), float("nan")
        lyr.experts_linear_dev("down", x.cuda(), offsets.cuda(), other, stream=st)
        assert torch.equal(other[1:n - 1], y[1:n - 1])
        assert not other[[0, n - 1]].isfinite().any()
    lyr.free()


def _same(a, b):
    """Two bf16 roundings of sums that differ by their order alone."""
    a, b = a.double(), b.double()
    return float((a - b).norm()) <= (2 / 3) ** 0.5 * 2.0 ** -8 * float(b.norm())


def test_many_rows_of_weights_of_every_origin(gpu_ctx):
    """The exponents that many rows use are kept with the weights by every call that writes them: against few rows,
    which use none, for layers synthesized, quantized and from Q4_K through views of their experts, and for matrices."""
    st = torch.cuda.current_stream()
    H, I, E = 512, 256, 2
    g = MoeGeometry(hidden=H, inter=I, n_routed=E, n_shared=1, top_k=1)
    T = 64 * 81
    rng = np.random.default_rng(5)

    def check(mat, K, what):
        x = torch.randn(T, K, generator=torch.Generator().manual_seed(K)).to(torch.bfloat16).cuda()
        mat.reserve_act(T)
        y, few = (torch.zeros(n, mat.M, dtype=torch.bfloat16, device="cuda") for n in (T, 32))
        mat.linear_act_dev(x, T, y, stream=st)
        mat.linear_act_dev(x[:32], 32, few, stream=st)
        assert bool(few.any()) and _same(y[:32], few), what
        mat.free()

    def q4k(rows, cols, d):  # random 144-byte super-blocks with sane scales
        b = rng.integers(0, 256, (rows * cols // 256, 144), dtype=np.uint8)
        b[:, :4] = np.frombuffer(np.array([d, d / 2], dtype=np.float16).tobytes(), dtype=np.uint8)
        return b.tobytes()

    lyr = gpu_ctx.create_layer(7502, g)

    def check_layer(what):
        for e in range(E):
            check(lyr.expert_matrix(e, "gate_up"), H, (what, e, "gate_up"))
            check(lyr.expert_matrix(e, "down"), I, (what, e, "down"))

    lyr.synthesize(3, std=0.5, stream=st)
    check_layer("synthesized")
    for e in range(E):
        lyr.quantize_expert(e, torch.randn(2 * I, H, device="cuda") * 2.0 ** (13 * e), torch.randn(H, I, device="cuda"))
    check_layer("quantized")
    for e in range(E):
        lyr.upload_expert_q4k(e, "gate", q4k(I, H, 0.01 * 4 ** e))
        lyr.upload_expert_q4k(e, "up", q4k(I, H, 0.3))
        lyr.upload_expert_q4k(e, "down", q4k(H, I, 0.002))
    check_layer("Q4_K")
    lyr.free()
    M, K = 512, 768
    for mat in (gpu_ctx.quantize_matrix(torch.randn(M, K, device="cuda") * 300, M, K),
                gpu_ctx.upload_matrix(_weights("q4nx", M, K, 1)[0], M, K),
                gpu_ctx.upload_matrix(_weights("bfp16", M, K, 1, std=2.0 ** -30)[0], M, K, fmt="bfp16"),
                gpu_ctx.upload_matrix(q4k(M, K, 0.02), M, K, fmt="q4k")):
        check(mat, K, mat.fmt)


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
def test_groups_of_very_different_sizes_in_many_rows(gpu_ctx, fmt):
    """Rows whose groups' weights differ by 2^20, met by tokens that are zero where the large ones are."""
    M, K, T = 512, 512, 64 * 81
    rng = np.random.default_rng(3)
    scale = 2.0 ** -rng.integers(0, 21, (M, K // 32))
    scale[:, 0] = 1.0
    scale[:, 1:9] = 2.0 ** -20
    w = (rng.normal(0.0, 0.5, (M, K)) * np.repeat(scale, 32, 1)).astype(np.float32)
    if fmt == "q4nx":
        c, s, m = Q.quantize(w)
        blob = Q.pack_gemv(c, s, m)
        cd, sd, md = torch.from_numpy(c).double(), *(torch.from_numpy(a).double().repeat_interleave(32, 1) for a in (s, m))
        wd, t = md + sd * cd, sd.abs() * (cd - 8).abs() + 8 * sd.abs() + md.abs()
    else:
        blob = B.pack_gemv(w)
        wd = torch.from_numpy(B.dequantize_packed(blob, K, M)).double()
        t = wd.abs()
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(4)).to(torch.bfloat16)
    x[::2, :32] = 0
    x[::2, 288:] = 0
    y = torch.zeros(T, M, dtype=torch.bfloat16, device="cuda")
    mat.linear_act_dev(x.cuda(), T, y, stream=torch.cuda.current_stream())
    xd = x.double()
    _check(y, xd @ wd.t(), (K + 64) * 2.0 ** -23 * (xd.abs() @ t.t()), fmt)
    mat.free()


@pytest.mark.parametrize("fmt", ["q4nx", "bfp16"])
def test_many_rows_captured_before_a_larger_reserve(gpu_ctx, fmt):
    """A captured call with its group sums and, for a narrower input, its own exponents in the context's scratch
    replays as before after calls of other rows and after the scratch has grown."""
    M, K, K_in, T = 1024, 768, 520, 64 * 41
    blob, _, _ = _weights(fmt, M, K, 3)
    mat = gpu_ctx.upload_matrix(blob, M, K, fmt=fmt)
    mat.reserve_act(T)
    st = torch.cuda.Stream()
    x = torch.randn(3 * T, K_in, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    y, big = (torch.zeros(n, M, dtype=torch.bfloat16, device="cuda") for n in (T, 3 * T))
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
        y.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    mat.free()
