"""The weight gradient from an 8-bit checkpoint against code * scale in 64 bits: what the expansion
to bf16 on the way into the tensor core may cost, and what it costs (csrc/wgrad.cuh)."""
from __future__ import annotations

import pytest
import torch

from residual_inputs import U32, UBF16, assert_close, dequant_rows64, grads, mn_major, quant_rows, tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(1, 16, 128), (65, 48, 384), (1003, 32, 1024), (777, 1024, 1024), (5001, 144, 1152),
                                   (4099, 2064, 896)])
def test_against_the_codes_values(cuda_device, M, N, K):
    from ltx_kernels.blockwise import ops
    zero = (M // 2,) if M > 2 else ()
    xq, xs = quant_rows(tokens(M, K, 41, zero).float())
    g = grads(M, N, 42, zero).to(cuda_device)
    qd, sd = xq.to(cuda_device), mn_major(xs.to(cuda_device))
    dw = ops.wgrad_1x128(g, qd, sd)
    gd, xd = g.double(), dequant_rows64(qd, sd)
    want, size = gd.t() @ xd, gd.abs().t() @ xd.abs()
    # each code * scale rounded to bf16 once, the sums in fp32 (one step of 2^-22 of the running size
    # per 16 tokens and per split), the output rounded
    tol = want.abs() * (UBF16 + 2 * U32) + size * (UBF16 + (M / 16 + 70) * 2.0 ** -22)
    assert_close(dw, want, tol, f"{M, N, K}")
    # Independent roundings: in the root mean square of the sum no more than half a step spread
    # evenly, 2^-8 / sqrt(3), of the terms' root sum of squares, and the same of the output.
    rms = torch.sqrt(gd.square().t() @ xd.square())
    err = ((dw.double() - want).norm() / want.norm()).item()
    bar = UBF16 / 3 ** 0.5 * (1 + (rms.norm() / want.norm()).item()) + (M / 16 + 70) * 2.0 ** -22 * (size.norm() / want.norm()).item()
    assert err <= bar, (err, bar)
