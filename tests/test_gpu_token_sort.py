"""GPU: tokens sorted by expert and back (csrc/token_sort.hip) against plain forms in 64 bits.

Bounds.  The sort moves bits: equality.  Sums over k routes take k products and k - 1 additions in fp32, each off by
at most 2^-24 of a value no larger than S = sum |w v|, then one rounding of half a step of the type (eps / 2, and half
its smallest subnormal).  A dot product over H columns takes H products and additions: H 2^-23 sum |a b|."""

from __future__ import annotations

import pytest

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

TYPES = [torch.bfloat16, torch.float16, torch.float32]


def _half_step(dtype):
    f = torch.finfo(dtype)
    return f.eps / 2, f.smallest_normal * f.eps / 2


def _ids(T, k, E, seed, drop=0.2):
    """Distinct experts per token; some routes dropped, one token (of several) left without any."""
    g = torch.Generator().manual_seed(seed)
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :k].to(torch.int32)
    ids[torch.rand(T, k, generator=g) < drop] = -1
    if T > 2:
        ids[T // 2] = -1
    return ids


def _plain_sort(ids, E):
    """By listing: (order, inv, offsets) of host ids."""
    seq = [[] for _ in range(E)]
    flat = ids.reshape(-1).tolist()
    for a, e in enumerate(flat):
        if 0 <= e < E:
            seq[e].append(a)
    order = [a for s in seq for a in s]
    inv = [-1] * len(flat)
    for p, a in enumerate(order):
        inv[a] = p
    offsets = [0]
    for s in seq:
        offsets.append(offsets[-1] + len(s))
    return order, torch.tensor(inv, dtype=torch.int32).view(ids.shape), torch.tensor(offsets, dtype=torch.int32)


def _buffers(T, k, E, H, dtype, fill=7):
    return (torch.full((T * k, H), fill, dtype=dtype, device="cuda"),
            torch.full((T * k,), -9, dtype=torch.int32, device="cuda"),
            torch.full((T, k), -9, dtype=torch.int32, device="cuda"),
            torch.full((E + 1,), -9, dtype=torch.int32, device="cuda"))


# Both sides of one launch and two (1,024 assignments), of two and four (65,536) and of a chunk of 1,024; a last
# chunk shorter than the experts.
SHAPES = [(1, 1, 1, 1), (1, 8, 128, 2048), (4, 8, 128, 2048), (3, 16, 256, 33), (128, 8, 128, 64), (129, 8, 128, 64),
          (1024, 1, 256, 8), (1025, 1, 256, 8), (64, 16, 128, 8), (65, 16, 128, 8),
          (256, 8, 128, 8), (257, 8, 128, 8), (2048, 1, 200, 8), (2049, 1, 200, 8), (445, 6, 128, 2560), (300, 7, 9, 1027), (2049, 3, 64, 136),
          (4096, 16, 255, 24),
          (4100, 16, 255, 24), (65537, 1, 256, 8), (9400, 7, 9, 24)]


@pytest.mark.parametrize("T,k,E,H", SHAPES)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_sort(gpu_ctx, T, k, E, H, dtype):
    x = torch.randn(T, H, generator=torch.Generator().manual_seed(T + H)).to(dtype)
    ids = _ids(T, k, E, T * 7 + k)
    order, inv, offsets = _plain_sort(ids, E)
    rows_d, order_d, inv_d, off_d = _buffers(T, k, E, H, dtype)
    gpu_ctx.sort_tokens_dev(x.cuda(), ids.cuda(), E, rows_d, order_d, inv_d, off_d, stream=torch.cuda.current_stream())
    assert torch.equal(inv_d.cpu(), inv) and torch.equal(off_d.cpu(), offsets)
    n = len(order)
    assert order_d.cpu().tolist() == order + [-9] * (T * k - n)
    assert torch.equal(rows_d[:n].cpu(), x[torch.tensor(order, dtype=torch.long) // k])
    assert bool((rows_d[n:] == 7).all())  # rows behind the last stay as they were


def test_sort_without_any_route_and_all_on_one_expert(gpu_ctx):
    for T, k, E, H in ((5, 2, 4, 16), (3000, 2, 4, 16), (33000, 2, 4, 16)):
        x = torch.randn(T, H, device="cuda").to(torch.bfloat16)
        st = torch.cuda.current_stream()
        for ids in (torch.full((T, k), -1, dtype=torch.int32), torch.full((T, k), 2, dtype=torch.int32),
                    torch.full((T, k), -(1 << 31), dtype=torch.int32)):
            order, inv, offsets = _plain_sort(ids, E)
            rows_d, order_d, inv_d, off_d = _buffers(T, k, E, H, torch.bfloat16)
            gpu_ctx.sort_tokens_dev(x, ids.cuda(), E, rows_d, order_d, inv_d, off_d, stream=st)
            assert torch.equal(inv_d.cpu(), inv) and torch.equal(off_d.cpu(), offsets)
            n = len(order)
            assert torch.equal(rows_d[:n].cpu(), x.cpu()[torch.tensor(order, dtype=torch.long) // k])
            dx = torch.full_like(x, 3)
            gpu_ctx.sort_tokens_backward_dev(rows_d, inv_d, dx, stream=st)
            if n == 0:
                assert not dx.any()
            else:
                assert torch.equal(dx, (x.float() * k).to(torch.bfloat16))


def test_expert_past_the_last_is_reported(gpu_ctx):
    """Its route has no row; the next synchronous call raises, once."""
    for T in (4, 2000, 40000):
        x = torch.randn(T, 32, device="cuda").to(torch.bfloat16)
        ids = _ids(T, 2, 8, 5, drop=0.0)
        ids[1, 1] = 8
        rows_d, order_d, inv_d, off_d = _buffers(T, 2, 8, 32, torch.bfloat16)
        gpu_ctx.sort_tokens_dev(x, ids.cuda(), 8, rows_d, order_d, inv_d, off_d, stream=torch.cuda.current_stream())
        order, inv, offsets = _plain_sort(ids, 8)
        assert torch.equal(inv_d.cpu(), inv) and torch.equal(off_d.cpu(), offsets)
        with pytest.raises(ValueError, match="expert id out of range"):
            gpu_ctx.synchronize()
        gpu_ctx.synchronize()


def test_position_past_the_rows_is_reported(gpu_ctx):
    inv = torch.tensor([[0, 4]], dtype=torch.int32, device="cuda")
    rows = torch.ones(2, 16, device="cuda")
    out = torch.zeros(1, 16, device="cuda")
    w = torch.ones(1, 2, device="cuda")
    st = torch.cuda.current_stream()
    gpu_ctx.combine_tokens_dev(rows, inv, w, out, stream=st)
    torch.cuda.synchronize()
    assert bool((out == 1).all())
    with pytest.raises(ValueError, match="sorted position out of range"):
        gpu_ctx.synchronize()
    drows, dw = torch.zeros_like(rows), torch.ones_like(w)
    gpu_ctx.combine_tokens_backward_dev(out, rows, inv, w, drows, dw, stream=st)
    with pytest.raises(ValueError, match="sorted position out of range"):
        gpu_ctx.synchronize()
    assert dw.tolist() == [[16.0, 0.0]] and bool((drows[0] == 1).all()) and not drows[1].any()


def _case(T, k, E, H, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    ids = _ids(T, k, E, seed)
    _, inv, offsets = _plain_sort(ids, E)
    rows = torch.randn(T * k, H, generator=g).to(dtype)
    w = torch.rand(T, k, generator=g) - 0.2
    dout = torch.randn(T, H, generator=g).to(dtype)
    return inv, int(offsets[-1]), rows, w, dout


def _gather(rows, inv):
    live = (inv >= 0)[..., None]
    return torch.where(live, rows.double()[inv.clamp(min=0).long()], 0.0)  # [T, k, H]


SUMS = [(1, 1, 1, 1), (1, 6, 128, 2560), (3, 16, 256, 33), (445, 6, 128, 2560), (300, 7, 9, 1027), (5, 8, 64, 520),
        (257, 2, 4, 8)]


@pytest.mark.parametrize("T,k,E,H", SUMS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_combine_and_sort_backward(gpu_ctx, T, k, E, H, dtype):
    inv, n, rows, w, _ = _case(T, k, E, H, dtype, 11 * T + H)
    rows[n:] = float("nan")  # behind the last row: never read
    wn = torch.where(inv < 0, torch.full_like(w, float("nan")), w)  # a weight without a row takes no part
    st = torch.cuda.current_stream()
    u, sub = _half_step(dtype)
    for weights in (wn, None):
        out = torch.full((T, H), 5.0, dtype=dtype, device="cuda")
        if weights is None:
            gpu_ctx.sort_tokens_backward_dev(rows.cuda(), inv.cuda(), out, stream=st)
            terms = _gather(rows, inv)
        else:
            gpu_ctx.combine_tokens_dev(rows.cuda(), inv.cuda(), wn.cuda(), out, stream=st)
            terms = _gather(rows, inv) * w.double()[..., None]
        ref, S = terms.sum(1), terms.abs().sum(1)
        slack = 2 * k * 2.0 ** -24 * S
        assert bool(((out.cpu().double() - ref).abs() <= u * (ref.abs() + slack) + slack + sub).all())


@pytest.mark.parametrize("T,k,E,H", SUMS)
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_combine_backward(gpu_ctx, T, k, E, H, dtype):
    inv, n, rows, w, dout = _case(T, k, E, H, dtype, 13 * T + H)
    rows[n:] = float("nan")
    drows = torch.full((T * k, H), 7.0, dtype=dtype, device="cuda")
    dw = torch.full((T, k), 5.0, device="cuda")
    gpu_ctx.combine_tokens_backward_dev(dout.cuda(), rows.cuda(), inv.cuda(), w.cuda(), drows, dw,
                                        stream=torch.cuda.current_stream())
    drows, dw = drows.cpu().double(), dw.cpu().double()
    u, sub = _half_step(dtype)
    terms = _gather(rows, inv) * dout.double()[:, None]
    assert bool(((dw - terms.sum(2)).abs() <= H * 2.0 ** -23 * terms.abs().sum(2)).all())
    assert bool((dw[inv < 0] == 0).all())
    t, r = (inv >= 0).nonzero(as_tuple=True)
    ref = w.double()[t, r, None] * dout.double()[t]
    got = drows[inv[t, r].long()]
    assert bool(((got - ref).abs() <= (u + 2.0 ** -24 * (1 + u)) * ref.abs() + sub).all())
    assert bool((drows[n:] == 7).all())


def test_gradients_against_differences(gpu_ctx):
    """L = <c, combine(sort(x), w)> in fp32: dx and dw against central differences of the calls themselves.  L is
    linear in x and in w, so the difference is exact but for roundings: values of size about 1 summed over H = 24
    columns and k = 3 routes carry at most (3 k + H) 2^-24 of sum |terms| each, divided by the step 2^-2."""
    T, k, E, H = 5, 3, 6, 24
    g = torch.Generator().manual_seed(3)
    x, c = torch.randn(T, H, generator=g).cuda(), torch.randn(T, H, generator=g).cuda()
    ids = _ids(T, k, E, 8).cuda()
    w = torch.rand(T, k, generator=g).cuda()
    st = torch.cuda.current_stream()

    def forward(x, w):
        rows, order, inv, off = _buffers(T, k, E, H, torch.float32, fill=0)
        out = torch.zeros(T, H, device="cuda")
        gpu_ctx.sort_tokens_dev(x, ids, E, rows, order, inv, off, stream=st)
        gpu_ctx.combine_tokens_dev(rows, inv, w, out, stream=st)
        return (out.double() * c.double()).sum().item(), rows, inv

    _, rows, inv = forward(x, w)
    drows, dw, dx = torch.zeros_like(rows), torch.zeros_like(w), torch.zeros_like(x)
    gpu_ctx.combine_tokens_backward_dev(c, rows, inv, w, drows, dw, stream=st)
    gpu_ctx.sort_tokens_backward_dev(drows, inv, dx, stream=st)
    size = float((x.abs() * c.abs()).sum(1).max()) * k + 1.0
    tol = 2 * (3 * k + H) * 2.0 ** -24 * size * T / 2.0 ** -2
    h = 2.0 ** -3
    for v, grad in ((x, dx), (w, dw)):
        for i in range(0, v.numel(), 7):
            p, m = v.clone(), v.clone()
            p.view(-1)[i] += h
            m.view(-1)[i] -= h
            args = ((p, w), (m, w)) if v is x else ((x, p), (x, m))
            step = float(p.view(-1)[i].double() - m.view(-1)[i].double())
            diff = (forward(*args[0])[0] - forward(*args[1])[0]) / step
            assert abs(diff - float(grad.view(-1)[i])) <= tol


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("shift", [1, 3, 8])
def test_rows_at_odd_addresses(gpu_ctx, dtype, shift):
    """Operands that 16-byte (or 4-byte) accesses cannot take: the same bytes, and nothing around them."""
    T, k, E, H = 9, 4, 8, 64

    def at(v):
        b = torch.zeros(v.numel() + shift + 8, dtype=v.dtype, device="cuda")
        w = b[shift:shift + v.numel()].view(v.shape)
        w.copy_(v)
        return b, w

    x = torch.randn(T, H, device="cuda").to(dtype)
    ids = _ids(T, k, E, 4).cuda()
    w = torch.rand(T, k, device="cuda")
    st = torch.cuda.current_stream()
    want = _buffers(T, k, E, H, dtype)
    gpu_ctx.sort_tokens_dev(x, ids, E, *want, stream=st)
    rows_b, rows = at(torch.full((T * k, H), 7, dtype=dtype, device="cuda"))
    _, order, inv, off = _buffers(T, k, E, H, dtype)
    gpu_ctx.sort_tokens_dev(at(x)[1], ids, E, rows, order, inv, off, stream=st)
    assert torch.equal(rows, want[0]) and torch.equal(inv, want[2])
    assert not rows_b[:shift].any() and not rows_b[shift + rows.numel():].any()
    outs = []
    for aligned in (True, False):
        src = want[0] if aligned else rows
        d = torch.zeros_like(x) if aligned else at(torch.zeros_like(x))[1]
        dr = torch.zeros_like(want[0]) if aligned else at(torch.zeros_like(want[0]))[1]
        dw = torch.zeros_like(w)
        gpu_ctx.combine_tokens_dev(src, inv, w, d, stream=st)
        gpu_ctx.combine_tokens_backward_dev(x if aligned else at(x)[1], src, inv, w, dr, dw, stream=st)
        outs.append((d.clone(), dr.clone(), dw))
    assert torch.equal(outs[0][0], outs[1][0]) and torch.equal(outs[0][1], outs[1][1])
    # another order of the dot product's sum
    S = (_gather(want[0].cpu(), inv.cpu()) * x.cpu().double()[:, None]).abs().sum(2)
    assert bool(((outs[0][2] - outs[1][2]).cpu().double().abs() <= 2 * H * 2.0 ** -23 * S).all())


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_same_bits_at_every_address(gpu_ctx, dtype):
    """Sums and products round alike whether 16-byte accesses take them or single elements: 100,000 products, of
    which, with 13 bits between fp32 and fp16, some 2^-14 round otherwise once than twice."""
    T, k, E, H = 64, 4, 8, 512
    g = torch.Generator().manual_seed(21)
    rows, dout = torch.randn(T * k, H, generator=g).to(dtype).cuda(), torch.randn(T, H, generator=g).to(dtype).cuda()
    w = (torch.rand(T, k, generator=g) - 0.3).cuda()
    inv = _plain_sort(_ids(T, k, E, 4), E)[1].cuda()
    st = torch.cuda.current_stream()

    def odd(v):
        b = torch.zeros(v.numel() + 1, dtype=v.dtype, device="cuda")
        b[1:].copy_(v.reshape(-1))
        return b[1:].view(v.shape)

    got = []
    for f in (lambda v: v, odd):
        out, dx, dr, dw = f(torch.zeros_like(dout)), f(torch.zeros_like(dout)), f(torch.zeros_like(rows)), torch.zeros_like(w)
        gpu_ctx.combine_tokens_dev(f(rows), inv, w, out, stream=st)
        gpu_ctx.sort_tokens_backward_dev(f(rows), inv, dx, stream=st)
        gpu_ctx.combine_tokens_backward_dev(f(dout), f(rows), inv, w, dr, dw, stream=st)
        got.append((out.clone(), dx.clone(), dr.clone()))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_non_finite_values(gpu_ctx):
    """Infinities and NaN come back where their rows go, and nowhere else; NaN bits are moved unchanged."""
    x = torch.randn(4, 16, device="cuda").to(torch.bfloat16)
    x[1, 3], x[2, 5] = float("inf"), float("nan")
    x.view(torch.int16)[2, 6] = 0x7F81
    ids = torch.tensor([[0, 1], [1, 2], [0, 2], [1, 0]], dtype=torch.int32, device="cuda")
    st = torch.cuda.current_stream()
    rows, order, inv, off = _buffers(4, 2, 3, 16, torch.bfloat16)
    gpu_ctx.sort_tokens_dev(x, ids, 3, rows, order, inv, off, stream=st)
    assert torch.equal(rows.view(torch.int16), x.view(torch.int16)[order.long() // 2])
    out = torch.zeros_like(x)
    w = torch.ones(4, 2, device="cuda")
    gpu_ctx.combine_tokens_dev(rows, inv, w, out, stream=st)
    assert torch.equal(out.isnan(), x.isnan()) and torch.equal(out.isinf(), x.isinf())


def test_graph_replays_and_streams(gpu_ctx):
    """Captured forward and backward, replayed with new inputs and eager work between; two graphs on two streams at
    once share nothing."""
    T, k, E, H = 700, 4, 32, 96
    graphs = []
    for seed in (1, 2):
        st = torch.cuda.Stream()
        x = torch.zeros(T, H, dtype=torch.bfloat16, device="cuda")
        ids = torch.zeros(T, k, dtype=torch.int32, device="cuda")
        w = torch.rand(T, k, device="cuda")
        bufs = _buffers(T, k, E, H, torch.bfloat16)
        out, dr, dw, dx = torch.zeros_like(x), torch.zeros_like(bufs[0]), torch.zeros_like(w), torch.zeros_like(x)

        def run(x=x, ids=ids, w=w, bufs=bufs, out=out, dr=dr, dw=dw, dx=dx, st=st):
            gpu_ctx.sort_tokens_dev(x, ids, E, *bufs, stream=st)
            gpu_ctx.combine_tokens_dev(bufs[0], bufs[2], w, out, stream=st)
            gpu_ctx.combine_tokens_backward_dev(x, bufs[0], bufs[2], w, dr, dw, stream=st)
            gpu_ctx.sort_tokens_backward_dev(dr, bufs[2], dx, stream=st)

        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=st):
            run()
        graphs.append((graph, st, x, ids, (*bufs, out, dr, dw, dx), run))
    for rnd in range(4):
        for s, (_, _, x, ids, _, _) in enumerate(graphs):
            x.copy_(torch.randn(T, H, generator=torch.Generator().manual_seed(10 * rnd + s)).to(torch.bfloat16))
            ids.copy_(_ids(T, k, E, 100 * rnd + s))
        torch.cuda.synchronize()
        for graph, st, *_ in graphs:
            with torch.cuda.stream(st):
                graph.replay()
        torch.cuda.synchronize()
        got = [[t.clone() for t in g[4]] for g in graphs]
        for g in graphs:
            g[5]()
        torch.cuda.synchronize()
        for a, g in zip(got, graphs):
            n = int(g[4][3][-1])
            for i, (p, q) in enumerate(zip(a, g[4])):
                if i == 0 or i == 5:  # behind the last row: what an earlier round left
                    p, q = p[:n], q[:n]
                if i == 1:
                    p, q = p[:n], q[:n]
                assert torch.equal(p, q), (rnd, i)


def test_rows_past_4_gib(gpu_ctx):
    """Byte offsets past 32 bits into the rows: the first and last tokens of a large sort and combine."""
    T, k, E, H = 300_000, 4, 8, 2048  # 4.9 GB of rows
    x = torch.empty(T, H, dtype=torch.bfloat16, device="cuda")
    x.copy_((torch.arange(T, device="cuda") % 251).to(torch.bfloat16)[:, None].expand(T, H))
    ids = ((torch.arange(T, device="cuda")[:, None] + torch.arange(k, device="cuda") * 2) % E).to(torch.int32).contiguous()
    rows, order, inv, off = _buffers(T, k, E, H, torch.bfloat16)
    st = torch.cuda.current_stream()
    gpu_ctx.sort_tokens_dev(x, ids, E, rows, order, inv, off, stream=st)
    perm = ids.reshape(-1).long().sort(stable=True).indices
    assert torch.equal(order.long(), perm)
    assert torch.equal(rows[:, ::511], x[perm // k, ::511])
    out = torch.zeros_like(x)
    gpu_ctx.combine_tokens_dev(rows, inv, torch.full((T, k), 0.25, device="cuda"), out, stream=st)
    assert torch.equal(out, x)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_larger_than_the_caches(gpu_ctx, dtype):
    """Rows of 64 MB and more are read with another hint: the same bits as in pieces that are not."""
    T, k, E, H = 2200, 8, 32, 2056
    g = torch.Generator().manual_seed(6)
    ids = _ids(T, k, E, 6).cuda()
    x = torch.randn(T, H, generator=g).to(dtype).cuda()
    w = torch.rand(T, k, generator=g).cuda()
    rows, order, inv, off = _buffers(T, k, E, H, dtype)
    st = torch.cuda.current_stream()
    gpu_ctx.sort_tokens_dev(x, ids, E, rows, order, inv, off, stream=st)
    out, dx, dr, dw = torch.zeros_like(x), torch.zeros_like(x), torch.zeros_like(rows), torch.zeros_like(w)
    gpu_ctx.combine_tokens_dev(rows, inv, w, out, stream=st)
    gpu_ctx.sort_tokens_backward_dev(rows, inv, dx, stream=st)
    gpu_ctx.combine_tokens_backward_dev(x, rows, inv, w, dr, dw, stream=st)
    for t0 in (0, 1000, 2100):
        n = 100
        s = slice(t0, t0 + n)
        part = _buffers(n, k, E, H, dtype)
        gpu_ctx.sort_tokens_dev(x[s], ids[s], E, *part, stream=st)
        o, d, r, q = torch.zeros_like(x[s]), torch.zeros_like(x[s]), torch.zeros_like(part[0]), torch.zeros_like(w[s])
        gpu_ctx.combine_tokens_dev(part[0], part[2], w[s], o, stream=st)
        gpu_ctx.sort_tokens_backward_dev(part[0], part[2], d, stream=st)
        gpu_ctx.combine_tokens_backward_dev(x[s], part[0], part[2], w[s], r, q, stream=st)
        assert torch.equal(o, out[s]) and torch.equal(d, dx[s]) and torch.equal(q, dw[s])
        live = part[2] >= 0
        assert torch.equal(r[part[2][live].long()], dr[inv[s][live].long()])
