"""GPU: microscaled products at shapes that reach every kernel (tests/mx_kernels.py): against the plain form in 64 bits, with
scale bytes of 255 and at their ends, and with outputs at any address.

Bounds are those of test_gpu_mx.py, of which the plain form is.  A scale byte of 255 makes NaN of its row of results
(weights: its column, and of a gated pair either half) and leaves the bits of every other result."""

from __future__ import annotations

import numpy as np
import pytest

from mx_kernels import DENSE, EXPERTS, kernel_of
from oracle import mx
from test_gpu_mx import _cuda, _plain, _product, _weights

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _values(codes, scales):
    """mx.dequantize on the GPU."""
    levels = torch.tensor([*mx.LEVELS, *-mx.LEVELS], dtype=torch.float64, device="cuda")
    v = levels[torch.stack([codes & 15, codes >> 4], -1).flatten(-2).int()]
    return v * torch.exp2(scales.double() - 127).repeat_interleave(32, -1)


def test_values_are_the_oracles(gpu_ctx):
    c, s = _weights((7,), 96, 1)
    assert np.array_equal(_values(c.cuda(), s.cuda()).cpu().numpy(), mx.dequantize(c.numpy(), s.numpy()))


class Call:
    """A dense product (rows a number) or one by expert (rows a list)."""

    def __init__(self, rows, M, K, gated):
        dense = isinstance(rows, int)
        self.n, self.M, self.K, self.gated = rows if dense else sum(rows), M, K, gated
        self.width = M // 2 if gated else M
        self.bounds = None if dense else [0, *np.cumsum(rows).tolist()]
        self.offsets = None if dense else torch.tensor(self.bounds, dtype=torch.int32, device="cuda")
        seed = self.n + M + K
        self.x = _cuda(_weights((self.n,), K, seed, 120, 130))
        self.lead = (M,) if dense else (len(rows), M)
        self.w = _cuda(_weights(self.lead, K, seed + 1))
        g = torch.Generator().manual_seed(seed)
        self.bias = torch.randn(*self.lead, generator=g).cuda()
        self.residual = torch.randn(self.n, self.width, generator=g).to(torch.bfloat16).cuda()

    def run(self, ctx, act, x=None, w=None, **kw):
        return _product(ctx, x or self.x, w or self.w, act, offsets=self.offsets, **kw)

    def groups(self):
        """(rows, the part of the weights they meet) in turn."""
        if self.bounds is None:
            return [(slice(0, self.n), ())]
        return [(slice(a, b), (e,)) for e, (a, b) in enumerate(zip(self.bounds, self.bounds[1:])) if a < b]


CALLS = [pytest.param(s, gated, id=f"{'-'.join(map(str, s))}-{gated}") for s in DENSE for gated in (False, True)]
CALLS += [pytest.param(s, gated, id=f"{len(s[0])}x{sum(s[0])}-{s[1]}-{s[2]}-{gated}") for s in EXPERTS
          for gated in (False, True)]


@pytest.mark.parametrize("shape,gated", CALLS)
def test_product(gpu_ctx, shape, gated):
    c = Call(*shape, gated)
    for act in ("swiglu", "situ") if gated else ("none", "gelu_tanh"):
        got = c.run(gpu_ctx, act, bias=c.bias, residual=c.residual)
        for rows, e in c.groups():
            y, bound = _plain(_values(c.x[0][rows], c.x[1][rows]), _values(c.w[0][e], c.w[1][e]), c.bias[e].double(), act,
                              c.residual[rows].double())
            off = (got[rows].double() - y).abs()
            assert bool((off <= bound).all()), (act, e, float((off / bound).max()))
        at = c.residual.clone()
        assert torch.equal(c.run(gpu_ctx, act, bias=c.bias, residual=at, y=at), got)


@pytest.mark.parametrize("shape,gated", CALLS)
def test_bad_blocks(gpu_ctx, shape, gated):
    """In the first, a middle and the last block of the first, a middle and the last row."""
    c = Call(*shape, gated)
    act, kb, half = "swiglu" if gated else "none", c.K // 32, c.M // 2
    clean = c.run(gpu_ctx, act)
    assert not bool(torch.isnan(clean).any())
    xs, nan = c.x[1].clone(), torch.zeros_like(clean, dtype=torch.bool)
    for row, block in ((0, 0), (c.n // 2, kb // 2), (c.n - 1, kb - 1)):
        xs[row, block] = 255
        nan[row] = True
    y = c.run(gpu_ctx, act, x=(c.x[0], xs))
    assert torch.equal(torch.isnan(y), nan) and torch.equal(y[~nan], clean[~nan])
    ws, nan = c.w[1].clone(), torch.zeros_like(nan)
    for rows, e in c.groups()[-2:]:
        for row, block in ((0, kb - 1), (half + 1, kb // 2), (c.M // 3, min(16, kb - 1)), (c.M - 1, 0)):
            ws[(*e, row, block)] = 255
            nan[rows, row % c.width] = True
    y = c.run(gpu_ctx, act, w=(c.w[0], ws))
    assert torch.equal(torch.isnan(y), nan) and torch.equal(y[~nan], clean[~nan])


@pytest.mark.parametrize("shape,gated", CALLS)
def test_scales_at_their_ends(gpu_ctx, shape, gated):
    """Ones times 2^-127 and 2^127: sums past fp32 are infinite, below it zero, subnormal terms count."""
    c = Call(*shape, gated)
    for t in (c.x[0], c.w[0]):
        t.fill_(0x22)
    for a, b in ((0, 254), (254, 0), (0, 127), (254, 254), (0, 0)):
        z = torch.tensor(c.K * 2.0 ** (a + b - 254), dtype=torch.float64)
        want = float(z * torch.sigmoid(z) * z if gated else z)
        y = c.run(gpu_ctx, "swiglu" if gated else "none", x=(c.x[0], torch.full_like(c.x[1], a)),
                  w=(c.w[0], torch.full_like(c.w[1], b))).double()
        if want > 2.0 ** 128:
            assert bool(torch.isinf(y).all()) and bool((y > 0).all()), (a, b)
        else:
            assert bool(((y - want).abs() <= want * 2.0 ** -7 + 2.0 ** -134).all()), (a, b, float(y[0, 0]), want)


@pytest.mark.parametrize("shape,gated", CALLS)
def test_outputs_at_any_address(gpu_ctx, shape, gated):
    c = Call(*shape, gated)
    act, size = "swiglu" if gated else "none", c.n * c.width
    want = c.run(gpu_ctx, act, bias=c.bias, residual=c.residual)
    for shift in (1, 4):
        buf, rbuf = (torch.full((size + 16,), 7, dtype=torch.bfloat16, device="cuda") for _ in range(2))
        y, r = (t[shift:shift + size].view(c.n, c.width) for t in (buf, rbuf))
        r.copy_(c.residual)
        bias = torch.empty(c.bias.numel() + 1, device="cuda")[1:].view(c.bias.shape)
        bias.copy_(c.bias)
        c.run(gpu_ctx, act, bias=bias, residual=r, y=y)
        assert torch.equal(y, want), shift
        assert bool((buf[:shift] == 7).all()) and bool((buf[shift + size:] == 7).all())


@pytest.mark.parametrize("shape,gated", [(s, g) for s in DENSE + EXPERTS if s[2] % 512 == 0 for g in (False, True)])
def test_scales_at_any_address(gpu_ctx, shape, gated):
    """Scales that do not start on 16 bytes take the kernel of K that is not whole windows: within the bound of the sums'
    order (each side's own bound)."""
    c = Call(*shape, gated)
    rows = c.n, c.M, c.K, 0 if c.bounds is None else len(c.bounds) - 1
    act = "swiglu" if gated else "none"
    want = c.run(gpu_ctx, act).double()
    moved = []
    for s in (c.x[1], c.w[1]):
        buf = torch.zeros(s.numel() + 16, dtype=torch.uint8, device="cuda")
        moved.append(buf[3:3 + s.numel()].view(s.shape))
        moved[-1].copy_(s)
    got = c.run(gpu_ctx, act, x=(c.x[0], moved[0]), w=(c.w[0], moved[1])).double()
    if kernel_of(*rows) == kernel_of(*rows, aligned=False):
        assert torch.equal(got, want)
    for group, e in c.groups():
        bound = _plain(_values(c.x[0][group], c.x[1][group]), _values(c.w[0][e], c.w[1][e]), None, act, None)[1]
        assert bool(((got[group] - want[group]).abs() <= 2 * bound).all())
