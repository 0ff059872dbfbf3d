"""The activation's gradient over every finite input: far beyond where the derivative has become
0 or 1, up to the largest value a checkpoint can hold (csrc/activation.cuh)."""
from __future__ import annotations

import pytest
import torch

from residual_inputs import (U32, UBF16, act_grad64, assert_close, dequant_rows64, grads, mn_major, quant_rows)

pytestmark = pytest.mark.gpu

# As for moderate inputs: act' = s + q (1 - s) s.  Where s has become 1 or 0 both terms are exact; on
# the way there s is off by at most 2^-24 beside a q of at most 50, 2^-18.4.
GRAD_ABS = 1.5 * 2.0 ** -18
SIZES = (1.0, 4.0, 5.5, 7.0, 10.0, 15.0, 17.0, 33.0, 90.0, 130.0, 1e4, 1e12, 1.3e13, 1e15, 1e19, 1e25, 1e30, 3.3e38)


def _z(M, seed):
    """One magnitude and sign a 1x128 group: columns 256 i hold +SIZES[i], 256 i + 128 hold -SIZES[i],
    spread by 2 % within the group."""
    g = torch.Generator().manual_seed(seed)
    size = torch.tensor(SIZES, dtype=torch.float64).repeat_interleave(2) * torch.tensor([1.0, -1.0] * len(SIZES))
    z = size.repeat_interleave(128) * (0.98 + 0.02 * torch.rand(M, 128 * 2 * len(SIZES), generator=g))
    return z.float()


@pytest.mark.parametrize("act", ("gelu_tanh", "silu"))
@pytest.mark.parametrize("M", [1, 33, 65, 700])  # few rows straight from memory, more through the ring
def test_backward_extremes(cuda_device, M, act):
    from ltx_kernels.blockwise import ops
    zq, zs = quant_rows(_z(M, 71))
    N = zq.shape[1]
    dy = grads(M, N, 72).to(cuda_device)
    qd, sd = zq.to(cuda_device), mn_major(zs.to(cuda_device))
    dz, dq, ds, db = ops.act_backward(dy, qd, sd, act, quantize=True, dbias=True)
    only = ops.act_backward(dy, qd, sd, act)[0]
    z64, dy64 = dequant_rows64(qd, sd), dy.double()
    want = dy64 * act_grad64(z64, act)
    assert torch.isfinite(want).all()
    assert_close(dz, want, want.abs() * UBF16 + dy64.abs() * GRAD_ABS, "dz")
    assert torch.equal(only, dz)
    # beyond 32 the derivative is 1 or 0 to fp32
    assert torch.equal(dz[z64 > 32], dy[z64 > 32])
    assert (dz[z64 < -110] == 0).all()
    scale = ds.double().repeat_interleave(128, 1)
    x = want / scale
    extra = dy64.abs() * GRAD_ABS / scale
    tol = torch.maximum(x.abs() * 2.0 ** -4, torch.full_like(x, 2.0 ** -10)) + 2 * extra + x.abs() * 2.0 ** -20
    assert ((dq.double() - x).abs() <= tol).all()
    steps = M / 2 + 32 + M / 64 + 32  # the longest chain of additions
    assert_close(db, want.sum(0), (want.abs() * steps * U32 + dy64.abs() * GRAD_ABS).sum(0), "dbias")


@pytest.mark.parametrize("act", ("gelu_tanh", "silu"))
@pytest.mark.parametrize("M", [5, 300])
def test_backward_nan_keeps_to_its_group(cuda_device, M, act):
    from ltx_kernels.blockwise import ops
    zq, zs = quant_rows(_z(M, 73))
    zs[2, 3] = float("nan")
    dy = grads(M, zq.shape[1], 74).to(cuda_device)
    dz, dq, ds, db = ops.act_backward(dy, zq.to(cuda_device), mn_major(zs.to(cuda_device)), act, quantize=True,
                                      dbias=True)
    lost = torch.zeros(M, zq.shape[1], dtype=torch.bool, device=cuda_device)
    lost[2, 3 * 128:4 * 128] = True
    assert torch.equal(torch.isnan(dz), lost) and torch.equal(torch.isnan(dq.float()), lost)
    assert torch.equal(torch.isnan(ds), lost[:, ::128]) and torch.equal(torch.isnan(db), lost.any(0))
