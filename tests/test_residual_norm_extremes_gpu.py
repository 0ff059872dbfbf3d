"""The RMS norm at its ends: all-zero rows with and without an epsilon (csrc/residual_norm.cuh)."""
from __future__ import annotations

import pytest
import torch

from residual_inputs import tokens

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H", [128, 1152, 4096, 16384])
def test_zero_rows(cuda_device, H):
    """With an epsilon they give zeros; without one they have no norm, and keep that to themselves."""
    from ltx_kernels.blockwise import ops
    x = tokens(9, H, 1, zero_rows=(2, 8)).to(cuda_device)
    zero = torch.zeros(9, dtype=torch.bool, device=cuda_device)
    zero[2], zero[8] = True, True
    q, s, _, rstd = ops.rms_norm_quantize(x)
    y, _, _ = ops.rms_norm_quantize(x, quantize=False)
    assert torch.isfinite(rstd).all() and torch.isfinite(s).all() and (s > 0).all()
    assert (q[zero].float() == 0).all() and (y[zero] == 0).all()
    q, s, _, rstd = ops.rms_norm_quantize(x, eps=0.0)
    y, _, _ = ops.rms_norm_quantize(x, eps=0.0, quantize=False)
    assert torch.isinf(rstd[zero]).all() and torch.isfinite(rstd[~zero]).all()
    for t in (q.float(), s, y):
        assert torch.isnan(t[zero]).all() and torch.isfinite(t[~zero]).all()
