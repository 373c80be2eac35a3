"""GPU: the microscaled 4-bit operators, the norms and the sort and combine together, as a decoder's blocks use them: a dense
block and one of experts on a residual stream, eager and replayed from a graph, and the gradients through the dense block
of what trains there (the norms' weights and the gate, with the values of the quantized rows and weights).

Each step is compared with the oracle's on what the step before left on the GPU, so that a bound is one step's: codes and
scales equal; products of K terms within K 2^-22 of the sum of the terms' magnitudes (twice, for the activation's slope and
the other factor's error) and 2^-7 of the result (two roundings: the products' and the oracle's order of an epilogue);
norms within 2^-7 of the result and 2^-16 of the terms.  Eager and replayed results are the same bits."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import mx

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")

EPS = 1e-6
BF16 = torch.bfloat16


def _mx(rows, K):
    return (torch.zeros(*rows, K // 2, dtype=torch.uint8, device="cuda"),
            torch.zeros(*rows, K // 32, dtype=torch.uint8, device="cuda"))


def _zeros(*shape, dtype=BF16):
    return torch.zeros(*shape, dtype=dtype, device="cuda")


def _values(pair):
    return torch.from_numpy(mx.dequantize(pair[0].cpu().numpy(), pair[1].cpu().numpy()))


def _same_codes(pair, rows):
    codes, scales = mx.quantize(rows.double().cpu().numpy())
    assert np.array_equal(pair[0].cpu().numpy(), codes) and np.array_equal(pair[1].cpu().numpy(), scales)


def _near(got, want, size):
    off = (got.cpu().double() - want).abs()
    bound = 2.0 ** -7 * want.abs() + size + 2.0 ** -126
    assert bool((off <= bound).all()), float((off / bound).max())


def _swiglu(z):
    g, u = z.chunk(2, dim=-1)
    return g * torch.sigmoid(g) * u


def _check_gate_up(y, x, w):
    z, size = x @ w.t(), x.shape[1] * 2.0 ** -22 * (x.abs() @ w.abs().t())
    (g, u), (eg, eu) = z.chunk(2, dim=-1), size.chunk(2, dim=-1)
    _near(y, _swiglu(z), 2 * (eg * (u.abs() + eu) + eu * g.abs()))


def _rms(v):
    return v * (v.square().mean(1, keepdim=True) + EPS).rsqrt()


def _weights(ctx, shape, seed):
    w = (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * 0.05).cuda()
    pair = _mx(shape[:-1], shape[-1])
    flat = w.view(-1, shape[-1])
    ctx.mx_quantize_dev(flat, pair[0].view(flat.shape[0], -1), pair[1].view(flat.shape[0], -1), stream=torch.cuda.current_stream())
    return pair


def _replayed(run, outputs):
    """run() eagerly and from a graph: the same bits, three replays with eager work between."""
    run()
    torch.cuda.synchronize()
    want = [t.clone() for t in outputs]
    st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=st):
        run()
    for _ in range(3):
        for t in outputs:
            t.zero_()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        for t, w in zip(outputs, want):
            assert torch.equal(t, w)


@pytest.mark.parametrize("T,H,I", [(1, 256, 192), (19, 256, 192), (300, 512, 1024), (1100, 1024, 5120)])
def test_dense_block(gpu_ctx, T, H, I):
    g = torch.Generator().manual_seed(T)
    stream0, block0 = torch.randn(T, H, generator=g).to(BF16).cuda(), torch.randn(T, H, generator=g).to(BF16).cuda()
    post, pre, gate = (1 + 0.2 * torch.randn(H, generator=g)).cuda(), (1 + 0.2 * torch.randn(H, generator=g)).cuda(), \
        (0.5 * torch.randn(H, generator=g)).cuda()
    gate_up, down = _weights(gpu_ctx, (2 * I, H), 1), _weights(gpu_ctx, (H, I), 2)
    y, h, x4, a, a4, d, y2, h2 = (_zeros(T, H), _zeros(T, H), _mx((T,), H), _zeros(T, I), _mx((T,), I), _zeros(T, H),
                                  _zeros(T, H), _zeros(T, H))

    def run():
        st = torch.cuda.current_stream()
        gpu_ctx.residual_norm_dev(block0, stream0, y, pre_weight_dev=pre, h_dev=h, codes_dev=x4[0], scales_dev=x4[1],
                                  eps=EPS, stream=st)
        gpu_ctx.mx_linear_dev(*x4, *gate_up, a, act="swiglu", stream=st)
        gpu_ctx.mx_quantize_dev(a, *a4, stream=st)
        gpu_ctx.mx_linear_dev(*a4, *down, d, stream=st)
        gpu_ctx.residual_norm_dev(d, y, y2, post_weight_dev=post, gate_dev=gate, scale=0.5, pre_weight_dev=pre, h_dev=h2,
                                  eps=EPS, stream=st)

    _replayed(run, [y, h, *x4, a, *a4, d, y2, h2])
    b, r = block0.cpu().double(), stream0.cpu().double()
    _near(y, b + r, 2.0 ** -16 * (b.abs() + r.abs()))
    yv = y.cpu().double()
    _near(h, _rms(yv) * pre.cpu().double(), 0)
    _same_codes(x4, h)
    _check_gate_up(a, _values(x4), _values(gate_up))
    _same_codes(a4, a)
    x, w = _values(a4), _values(down)
    _near(d, x @ w.t(), I * 2.0 ** -22 * (x.abs() @ w.abs().t()))
    u = _rms(d.cpu().double()) * post.cpu().double() * gate.cpu().double()
    _near(y2, 0.5 * yv + u, 2.0 ** -16 * (yv.abs() + u.abs()))
    _near(h2, _rms(y2.cpu().double()) * pre.cpu().double(), 0)


@pytest.mark.parametrize("T,H,I,E,k", [(1, 256, 128, 8, 2), (5, 512, 96, 16, 4), (200, 256, 160, 8, 2), (900, 512, 3200, 3, 2)])
def test_block_of_experts(gpu_ctx, T, H, I, E, k):
    g = torch.Generator().manual_seed(T + 1)
    stream0, pre = torch.randn(T, H, generator=g).to(BF16).cuda(), (1 + 0.2 * torch.randn(H, generator=g)).cuda()
    ids = torch.rand(T, E, generator=g).argsort(1)[:, :k].to(torch.int32)
    ids[T // 2, 0] = -1  # a dropped route
    ids, wts = ids.cuda(), torch.rand(T, k, generator=g).cuda()
    gate_up, down = _weights(gpu_ctx, (E, 2 * I, H), 3), _weights(gpu_ctx, (E, H, I), 4)
    n = T * k
    h, rows, order = _zeros(T, H), _zeros(n, H), torch.zeros(n, dtype=torch.int32, device="cuda")
    inv, off = torch.zeros(T, k, dtype=torch.int32, device="cuda"), torch.zeros(E + 1, dtype=torch.int32, device="cuda")
    x4, a, a4, d, out, y = _mx((n,), H), _zeros(n, I), _mx((n,), I), _zeros(n, H), _zeros(T, H), _zeros(T, H)

    def run():
        st = torch.cuda.current_stream()
        gpu_ctx.norm_dev(stream0, pre, h, eps=EPS, stream=st)
        gpu_ctx.sort_tokens_dev(h, ids, E, rows, order, inv, off, stream=st)
        gpu_ctx.mx_quantize_dev(rows, *x4, stream=st)
        gpu_ctx.mx_experts_linear_dev(*x4, *gate_up, off, a, act="swiglu", stream=st)
        gpu_ctx.mx_quantize_dev(a, *a4, stream=st)
        gpu_ctx.mx_experts_linear_dev(*a4, *down, off, d, stream=st)
        gpu_ctx.combine_tokens_dev(d, inv, wts, out, stream=st)
        gpu_ctx.residual_norm_dev(out, stream0, y, stream=st)

    _replayed(run, [h, rows, *x4, a, *a4, d, out, y])
    _same_codes(x4, rows)
    _same_codes(a4, a)
    x, xa, gu, dn = _values(x4), _values(a4), _values(gate_up), _values(down)
    bounds = off.tolist()
    assert bounds[-1] == n - 1
    for e, (p, q) in enumerate(zip(bounds, bounds[1:])):
        if p < q:
            _check_gate_up(a[p:q], x[p:q], gu[e])
            _near(d[p:q], xa[p:q] @ dn[e].t(), I * 2.0 ** -22 * (xa[p:q].abs() @ dn[e].abs().t()))
    assert not a[bounds[-1]:].any() and not d[bounds[-1]:].any()
    o, r = out.cpu().double(), stream0.cpu().double()
    _near(y, o + r, 2.0 ** -16 * (o.abs() + r.abs()))


def test_training_through_the_block(gpu_ctx):
    """Forward with the values of the quantized rows and weights; backward by the framework's norms and torch's products, in
    fp32, against autograd of the same function in 64 bits with the quantizing passed straight through."""
    T, H, I = 37, 256, 160
    g = torch.Generator().manual_seed(7)
    p = {"stream": torch.randn(T, H, generator=g), "block": torch.randn(T, H, generator=g), "post": 1 + 0.2 * torch.randn(H, generator=g),
         "pre": 1 + 0.2 * torch.randn(H, generator=g), "gate": 0.5 * torch.randn(H, generator=g)}
    dev = {k: v.cuda() for k, v in p.items()}
    W = torch.randn(I, H, generator=g).cuda() * 0.05
    dout, dgo = torch.randn(T, I, generator=g).cuda(), torch.randn(T, H, generator=g).cuda()
    st = torch.cuda.current_stream()
    Wv, hv, y, h = torch.empty_like(W), _zeros(T, H, dtype=torch.float32), _zeros(T, H, dtype=torch.float32), \
        _zeros(T, H, dtype=torch.float32)
    gpu_ctx.mx_quantize_dev(W, *_mx((I,), H), values_dev=Wv, stream=st)
    gpu_ctx.residual_norm_dev(dev["block"], dev["stream"], y, post_weight_dev=dev["post"], gate_dev=dev["gate"], scale=0.75,
                              pre_weight_dev=dev["pre"], h_dev=h, eps=EPS, stream=st)
    gpu_ctx.mx_quantize_dev(h, *_mx((T,), H), values_dev=hv, stream=st)
    # out = hv Wv^T; the loss is <dout, out> + <dgo, y>.
    dh = dout @ Wv
    o = {k: torch.empty_like(v) for k, v in dev.items()}
    gpu_ctx.residual_norm_backward_dev(dgo, dh, dev["block"], y, o["block"], o["stream"],
                                       torch.empty(gpu_ctx.norm_backward_work(T, H), device="cuda"), post_weight_dev=dev["post"],
                                       dpost_weight_dev=o["post"], gate_dev=dev["gate"], dgate_dev=o["gate"], scale=0.75,
                                       pre_weight_dev=dev["pre"], dpre_weight_dev=o["pre"], eps=EPS, stream=st)
    q = {k: v.double().requires_grad_() for k, v in p.items()}
    yy = 0.75 * q["stream"] + q["gate"] * _rms(q["block"]) * q["post"]
    hh = _rms(yy) * q["pre"]
    ((hh @ Wv.cpu().double().t()) * dout.cpu().double()).sum().add((yy * dgo.cpu().double()).sum()).backward()
    # fp32 throughout: torch's product of 160 terms and the gradients' own sums, each within 2^-14 of their largest value.
    for k in p:
        want = q[k].grad
        assert bool(((o[k].cpu().double() - want).abs() <= 2.0 ** -14 * (want.abs() + want.abs().max())).all()), k
    # The wgrad of the quantized product is the caller's: its operand is what the forward pass multiplied.
    codes, scales = mx.quantize(h.double().cpu().numpy())
    assert np.array_equal(hv.cpu().double().numpy(), mx.dequantize(codes, scales))
