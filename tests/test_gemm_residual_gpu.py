"""Blockwise FP8 GEMM with bias, activation and residual in its epilogue against a 64-bit
evaluation (csrc/gemm.cuh, kAct >= 0)."""
from __future__ import annotations

import pytest
import torch

from residual_inputs import (U32, UBF16, act64, assert_close, dequant_rows64, dequant_weight64, gen, mn_major,
                             quant_rows, quant_weight, tokens)

pytestmark = pytest.mark.gpu


def _problem(M, N, K, dev, seed=0):
    aq, asc = quant_rows(tokens(M, K, seed + 51).float())
    wq, wsc = quant_weight(torch.randn(N, K, generator=gen(seed + 52)) / K ** 0.5)
    b = 0.1 * torch.randn(N, generator=gen(seed + 53))
    r = tokens(M, N, seed + 54)
    return aq.to(dev), mn_major(asc.to(dev)), wq.to(dev), wsc.to(dev), b.to(dev), r.to(dev)


def _want(aq, asc, wq, wsc, b, r, act):
    a, w = dequant_rows64(aq, asc), dequant_weight64(wq, wsc)
    z = a @ w.t()
    size = a.abs() @ w.abs().t()
    if b is not None:
        z = z + b.double()
    y = act64(z, act)
    if r is not None:
        y = y + r.double()
    K = a.shape[1]
    # products of codes are exact; K/32 tensor-core steps and K/128 scaled additions (two
    # roundings each) lose at most 2^-22 of the running size; the activations' slope is at
    # most 1.13 and their own error 2^-15 of the value; one rounding of the sum and one to bf16
    tol = y.abs() * (UBF16 + U32) + 1.13 * (K / 32 + 3 * K / 128 + 2) * 2.0 ** -22 * size
    if act is not None:
        tol = tol + act64(z, act).abs() * 2.0 ** -15
    return y, tol


@pytest.mark.parametrize("M,N,K", [
    (1, 128, 128), (1, 4096, 4096),    # single tokens: one tile, and split-K
    (7, 1024, 2048), (33, 384, 128), (129, 640, 1152),
    (8, 256, 1152), (9, 128, 128), (16, 384, 2176), (16, 4096, 4096), (17, 256, 1152),  # the streaming kernel's ends
    (12, 8192, 4224),                  # its widest weight passed
    (257, 4096, 512),                  # more than half of a wave of tiles
    (2100, 1152, 256),                 # several row tiles, ragged, N ends inside a tile
    (1280, 4096, 8192),                # the last rows split over K
    (4000, 4096, 256),                 # several tiles a CTA: the next residual loads behind a store
])
@pytest.mark.parametrize("act", [None, "gelu_tanh", "silu"])
@pytest.mark.parametrize("res", [True, False])
def test_against_64_bits(cuda_device, M, N, K, act, res):
    from ltx_kernels.blockwise import ops
    aq, asc, wq, wsc, b, r = _problem(M, N, K, cuda_device)
    r = r if res else None
    out = ops.gemm_residual(aq, asc, wq, wsc, b, residual=r, activation=act)
    again = ops.gemm_residual(aq, asc, wq, wsc, b, residual=r, activation=act)
    torch.cuda.synchronize()
    assert torch.equal(out, again), "not repeatable"
    y, tol = _want(aq, asc, wq, wsc, b, r, act)
    assert_close(out, y, tol)


def test_options(cuda_device):
    """No bias, no split, a strided or misaligned residual, and the residual updated in place."""
    from ltx_kernels.blockwise import ops
    for M, N, K in ((3, 512, 1152), (13, 384, 640), (70, 512, 4096), (700, 4096, 256)):
        aq, asc, wq, wsc, b, r = _problem(M, N, K, cuda_device, seed=7)
        y, tol = _want(aq, asc, wq, wsc, None, r, None)
        assert_close(ops.gemm_residual(aq, asc, wq, wsc, residual=r), y, tol)
        y, tol = _want(aq, asc, wq, wsc, b, r, "silu")
        want = ops.gemm_residual(aq, asc, wq, wsc, b, residual=r, activation="silu")
        assert_close(ops.gemm_residual(aq, asc, wq, wsc, b, residual=r, activation="silu", split_k=False), y, tol)
        wide = torch.zeros(M, N + 64, dtype=torch.bfloat16, device=cuda_device)
        for off in (16, 5):
            wide[:, off:off + N] = r
            assert torch.equal(ops.gemm_residual(aq, asc, wq, wsc, b, residual=wide[:, off:off + N],
                                                 activation="silu"), want)
        inplace = r.clone()
        assert ops.gemm_residual(aq, asc, wq, wsc, b, residual=inplace, activation="silu", out=inplace) is inplace
        assert torch.equal(inplace, want)
    e = ops.gemm_residual(aq[:0], asc[:0], wq, wsc, b, residual=r[:0])
    assert e.shape == (0, N)


def test_rows_keep_to_themselves(cuda_device):
    """A NaN in a token's codes or residual reaches only its row; untouched memory behind the
    last row stays as it was."""
    from ltx_kernels.blockwise import ops
    M, N, K = 130, 512, 512
    aq, asc, wq, wsc, b, r = _problem(M, N, K, cuda_device, seed=9)
    want = ops.gemm_residual(aq, asc, wq, wsc, b, residual=r, activation="gelu_tanh")
    bad = aq.clone()
    bad.view(torch.uint8)[5, 3] = 0x7F
    rbad = r.clone()
    rbad[77, 9] = float("nan")
    buf = torch.full((M + 70, N), 3.0, dtype=torch.bfloat16, device=cuda_device)
    out = ops.gemm_residual(bad, asc, wq, wsc, b, residual=rbad, activation="gelu_tanh", out=buf[:M])
    assert torch.isnan(out[5]).all() and torch.isnan(out[77, 9]) and torch.isnan(out).sum() == N + 1
    keep = ~torch.isnan(out)
    assert torch.equal(out[keep], want[keep]) and (buf[M:] == 3.0).all()


def test_other_epilogues_unchanged(cuda_device):
    """activation=None without a residual rounds bf16(acc + bias), as ops.gemm does: same bits."""
    from ltx_kernels.blockwise import ops
    for M, N, K in ((1, 512, 4096), (300, 1024, 512), (1280, 4096, 8192)):
        aq, asc, wq, wsc, b, _ = _problem(M, N, K, cuda_device, seed=11)
        assert torch.equal(ops.gemm_residual(aq, asc, wq, wsc, b), ops.gemm(aq, asc, wq, wsc, b))
