"""GPU: reservations that do not fit, and what works after them."""

from __future__ import annotations

import numpy as np
import pytest

from oracle import q4nx as Q

pytestmark = pytest.mark.gpu

torch = pytest.importorskip("torch")


def _matrix(ctx, M, K):
    c, s, m = Q.quantize(np.random.default_rng(1).normal(0, 0.02, (M, K)).astype(np.float32))
    return ctx.upload_matrix(Q.pack_gemv(c, s, m), M, K)


def test_calls_after_a_reservation_that_does_not_fit(gpu_ctx):
    """An allocation that fails is that call's error alone: the next launches do not report it again."""
    M, K, T = 512, 2048, 64 * 81
    mat = _matrix(gpu_ctx, M, K)
    mat.reserve_act(T)
    st = torch.cuda.current_stream()
    x = torch.randn(T, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
    want, y = (torch.zeros(T, M, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    few = torch.zeros(3, M, dtype=torch.bfloat16, device="cuda")
    mat.linear_act_dev(x, T, want, stream=st)
    for call in (lambda: mat.linear_act_dev(x, T, y, stream=st), lambda: mat.linear_act_dev(x[:3], 3, few, stream=st)):
        with pytest.raises(RuntimeError, match="hipMalloc"):
            mat.reserve_act(2 ** 31 - 1)  # 8.8 TB
        call()
    torch.cuda.synchronize()
    assert torch.equal(y, want) and bool(few.any())
    mat.free()


def test_growth_that_fits_only_as_asked(gpu_ctx):
    """A reservation a little larger than the one before asks for twice that one; where only the size asked for
    fits, that is what it gets."""
    from raon_npu_amd import Context

    M, K, gib = 512, 2048, 2 ** 30
    ctx = Context(0)
    mat = _matrix(ctx, M, K)
    rows = 4 * gib // (2 * K)  # 4 GiB of rows in fp16
    mat.reserve_act(rows)
    torch.cuda.synchronize()
    torch.cuda.empty_cache()
    free = torch.cuda.mem_get_info()[0]
    fill = torch.empty(free - 7 * gib, dtype=torch.uint8, device="cuda")  # 8 GiB and more do not fit, 5 do
    try:
        mat.reserve_act(rows * 5 // 4)
        x = torch.randn(64 * 81, K, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).cuda()
        y = torch.zeros(64 * 81, M, dtype=torch.bfloat16, device="cuda")
        mat.linear_act_dev(x, 64 * 81, y, stream=torch.cuda.current_stream())
        torch.cuda.synchronize()
        assert bool((y != 0).any(1).all())
        with pytest.raises(RuntimeError, match="hipMalloc"):
            mat.reserve_act(2 * rows)
    finally:
        del fill
        torch.cuda.empty_cache()
    ctx.close()
