"""Activation with an 8-bit checkpoint of its input and its gradient, the weight gradient
from an 8-bit checkpoint, and the weight's transpose, against 64-bit evaluations
(csrc/act_checkpoint.cuh, csrc/wgrad.cuh)."""
from __future__ import annotations

import ctypes

import pytest
import torch

from residual_inputs import (U32, UBF16, act64, act_grad64, assert_close, assert_quantised, dequant_rows64, gen, grads,
                             mn_major, quant_rows, quant_weight, tokens)

pytestmark = pytest.mark.gpu

ACTS = ("gelu_tanh", "silu")


def _z(M, N, seed, zero_rows=()):
    z = 2.0 * torch.randn(M, N, generator=gen(seed))
    for r in zero_rows:
        z[r] = 0
    return z.to(torch.bfloat16)


# act(z) = z / (1 + 2^a): the argument a has three roundings of up to |a| <= 126 (values below
# 2^-126 of z vanish), so 2^a is off by 3 * 126 * ln2 * 2^-24 < 2^-15; the two approximate
# instructions and the product add a few 2^-23.
ACT_REL = 2.0 ** -15 + 8 * U32


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N", [(1, 128), (1, 4096), (3, 384), (65, 1152), (130, 16384), (1003, 2048), (70000, 128)])
def test_save(cuda_device, M, N, act):
    from ltx_kernels.blockwise import ops
    zero = (M // 2,) if M > 2 else ()
    z = _z(M, N, 31, zero)
    yq, ys, zq, zs = ops.act_quantize_save(z.to(cuda_device), act)
    z64 = z.to(cuda_device).double()
    assert_quantised(zq, zs, z64, 0.0, "z")
    assert_quantised(yq, ys, act64(z64, act), ACT_REL, "y")
    for r in zero:
        assert (zq[r].float() == 0).all() and (yq[r].float() == 0).all()


@pytest.mark.parametrize("act", ACTS)
def test_save_extremes(cuda_device, act):
    """Far negative inputs vanish, far positive ones pass; NaN and infinity keep to their group."""
    from ltx_kernels.blockwise import ops
    z = _z(4, 256, 32)
    z[0, :128] = -torch.linspace(1, 1e4, 128).to(torch.bfloat16)
    z[1, :128] = torch.linspace(1, 1e30, 128).to(torch.bfloat16)
    z[2, 3] = float("nan")
    z[3, 200] = float("inf")
    yq, ys, zq, zs = ops.act_quantize_save(z.to(cuda_device), act)
    z64 = z.to(cuda_device).double()
    assert_quantised(yq[:2], ys[:2], act64(z64[:2], act), ACT_REL, "y")
    assert_quantised(zq[:2], zs[:2], z64[:2], 0.0, "z")
    assert torch.isnan(zs[2, 0]) and torch.isfinite(zs[2, 1]) and torch.isfinite(zs[3, 0]) and zs[3, 1] == float("inf")
    clean = _z(4, 256, 32)
    q0, s0, _, _ = ops.act_quantize_save(clean.to(cuda_device), act)
    assert torch.equal(yq[2, 128:].float(), q0[2, 128:].float()) and torch.equal(yq[3, :128].float(), q0[3, :128].float())


# act'(z) = s + z s (1 - s) u': both terms are at most 1.2 in size and carry the argument's
# error (2^-15 relative at the very most, where s or 1 - s is below 2^-100; 2^-19 for |z| <= 8).
GRAD_ABS = 1.5 * 2.0 ** -18


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("M,N", [(1, 128), (2, 4096), (37, 384), (64, 1152), (65, 256), (300, 1152), (1003, 2048), (40, 16384), (5000, 128)])
def test_backward(cuda_device, M, N, act):
    from ltx_kernels.blockwise import ops
    zero = (M // 2,) if M > 2 else ()
    zq, zs = quant_rows(_z(M, N, 33, zero).float())
    dy = grads(M, N, 34, zero)
    qd, sd, dyd = zq.to(cuda_device), mn_major(zs).to(cuda_device), dy.to(cuda_device)
    sd = mn_major(zs.to(cuda_device))
    dz, dq, ds, db = ops.act_backward(dyd, qd, sd, act, quantize=True, dbias=True)
    again = ops.act_backward(dyd, qd, sd, act, quantize=True, dbias=True)
    only = ops.act_backward(dyd, qd, sd, act)
    torch.cuda.synchronize()
    for a, b in zip((dz, dq, ds, db), again):
        assert torch.equal(a.float(), b.float()), "not repeatable"
    assert torch.equal(only[0], dz) and only[1] is None and only[2] is None and only[3] is None
    z64 = dequant_rows64(qd, sd)
    dy64 = dyd.double()
    want = dy64 * act_grad64(z64, act)
    assert_close(dz, want, want.abs() * UBF16 + dy64.abs() * GRAD_ABS, "dz")
    # the codes of dz: half a step, plus the gradient's error in units of the scale
    g = want.view(M, N // 128, 128)
    scale = ds.double().unsqueeze(-1)
    err = (dq.double().view_as(g) - g / scale).abs()
    x = (g / scale).abs()
    extra = (dy64.abs() * GRAD_ABS).view_as(g) / scale
    tol = torch.maximum(x * 2.0 ** -4, torch.full_like(x, 2.0 ** -10)) + 2 * extra + x * 2.0 ** -20
    assert (err <= tol).all()
    amax = g.abs().amax(-1)
    assert ((ds.double() * 448 - amax).abs() <= amax * 2.0 ** -20 + (dy64.abs() * GRAD_ABS).view_as(g).amax(-1)
            + 2.0 ** -110).all()
    # a thread adds at most every second row of its share (M / 2 of a single share is at most 32),
    # a block joins at most 32 rows, the shares (at most M / 2 of them) are summed in 32 chains
    steps = M / 2 + 32 + M / 64 + 32
    assert_close(db, want.sum(0), (want.abs() * steps * U32 + dy64.abs() * GRAD_ABS).sum(0), "dbias")


@pytest.mark.parametrize("act", ACTS)
def test_backward_is_the_forward_gradient(cuda_device, act):
    from ltx_kernels.blockwise import ops
    zq, zs = quant_rows(_z(2, 256, 35).float())
    dy = torch.ones(2, 256, dtype=torch.bfloat16)
    dz = ops.act_backward(dy.to(cuda_device), zq.to(cuda_device), mn_major(zs.to(cuda_device)), act)[0]
    z, step = dequant_rows64(zq, zs), 1e-4
    d = (act64(z + step, act) - act64(z - step, act)) / (2 * step)
    # the differences' error: third derivatives below 3, times step^2 / 6
    assert_close(dz.cpu(), d, d.abs() * UBF16 + GRAD_ABS + step ** 2, "dz")


def test_act_strided_empty_and_layouts(cuda_device):
    from ltx_kernels.blockwise import ops
    big = _z(50, 600, 36).to(cuda_device)
    a = ops.act_quantize_save(big[:, 8:520], "silu")
    b = ops.act_quantize_save(big[:, 8:520].contiguous(), "silu")
    c = ops.act_quantize_save(big[:, 8:520].reshape(5, 10, 512), "silu")
    for i in range(4):
        assert torch.equal(a[i].float(), b[i].float()) and torch.equal(c[i].float(), b[i].float())
    for M, N in ((300, 384), (130, 1152)):  # one column block, and two: rows fetched one by one
        zq, zs = quant_rows(_z(M, N, 38).float())
        zq, zs, wide = zq.to(cuda_device), mn_major(zs).to(cuda_device), grads(M, N + 40, 39).to(cuda_device)
        dy = wide[:, 8:N + 8]
        for x, y in zip(ops.act_backward(dy, zq, zs, "silu", quantize=True, dbias=True),
                        ops.act_backward(dy.contiguous(), zq, zs, "silu", quantize=True, dbias=True)):
            assert torch.equal(x.float(), y.float())
    dy = grads(50, 600, 37).to(cuda_device)
    d1 = ops.act_backward(dy[:, 3:515], a[2], a[3], "silu", quantize=True, dbias=True)
    d2 = ops.act_backward(dy[:, 3:515].contiguous(), a[2], a[3].t().contiguous(), "silu", quantize=True, dbias=True)
    for i in range(4):
        assert torch.equal(d1[i].float(), d2[i].float())
    e = torch.empty(0, 256, dtype=torch.bfloat16, device=cuda_device)
    yq, ys, zq, zs = ops.act_quantize_save(e)
    assert yq.shape == (0, 256) and ys.shape == (0, 2)
    dz, dq, ds, db = ops.act_backward(e, zq, zs, quantize=True, dbias=True)
    assert dz.shape == (0, 256) and (db == 0).all() and db.shape == (256,)


# ----------------------------------------------------------------------------- weight gradient
def _wgrad64(g, xb, alpha):
    """64-bit sum over the bf16 values the operator is defined on, and the sum of sizes."""
    gd, xd = g.double(), xb.double()
    return alpha * (gd.t() @ xd), abs(alpha) * (gd.abs().t() @ xd.abs())


def _wgrad_tol(want, size, M):
    # fp32 accumulation, at most one rounding or truncation (2^-22 of the running size) per
    # 16-token step of the tensor core and per split, then alpha and the output's rounding
    return want.abs() * (UBF16 + 2 * U32) + (M / 16 + 70) * 2.0 ** -22 * size


def test_wgrad_forms(cuda_device):
    """One CTA and the pair of CTAs, with and without a split over the tokens, each with tokens,
    rows and columns that end inside a tile."""
    from ltx_kernels import _lib
    from ltx_kernels.blockwise import ops
    seen = set()
    sms = torch.cuda.get_device_properties(cuda_device).multi_processor_count
    for M, N, K in ((333, 48, 384), (5001, 144, 1152), (77, 2064, 1152), (333, 2064, 384), (1001, 528, 2176),
                    (2001, 144, 896), (5001, 2064, 896), (2068, 832, 2176), (4175, 1536, 1920), (24577, 128, 640)):
        i = _lib.WgradPlanInfo()
        assert _lib.load().ltxfp8_wgrad_plan_for_sms(M, N, K, sms, ctypes.byref(i)) == _lib.OK
        seen.add((bool(i.pair), i.splits > 1))
        xq, xs = quant_rows(tokens(M, K, 46).float())
        g = grads(M, N, 47).to(cuda_device)
        qd, sd = xq.to(cuda_device), mn_major(xs.to(cuda_device))
        xb = (qd.float() * sd.repeat_interleave(128, 1)).to(torch.bfloat16)
        want, size = _wgrad64(g, xb, 1.0)
        for transposed in (False, True):
            a = ops.wgrad_1x128(g, qd, sd, transposed=transposed)
            b = ops.wgrad_bf16(g, xb, transposed=transposed)
            a, b = (a.t(), b.t()) if transposed else (a, b)
            assert_close(a, want, _wgrad_tol(want, size, M), f"{M, N, K}")
            assert torch.equal(a, b)
    assert len(seen) == 4, seen


@pytest.mark.parametrize("M,N,K", [
    (1, 16, 128),        # one token
    (63, 16, 256), (64, 32, 384), (65, 48, 128), (129, 256, 512), (200, 240, 640),
    (1000, 272, 256),    # two column tiles, the second ragged
    (513, 512, 1152),    # K ends inside a 256 tile
    (4099, 128, 256),    # split over tokens, ragged
    (9000, 16, 2048),
    (777, 1024, 1024),
    (640, 4096, 2048),   # several waves
])
def test_wgrad(cuda_device, M, N, K):
    from ltx_kernels.blockwise import ops
    zero = (M // 2,) if M > 2 else ()
    xq, xs = quant_rows(tokens(M, K, 41, zero).float())
    g = grads(M, N, 42, zero).to(cuda_device)
    qd, sd = xq.to(cuda_device), mn_major(xs.to(cuda_device))
    xb = (qd.float() * sd.repeat_interleave(128, 1)).to(torch.bfloat16)
    dw = ops.wgrad_1x128(g, qd, sd, alpha=0.5)
    again = ops.wgrad_1x128(g, qd, sd, alpha=0.5)
    dwt = ops.wgrad_1x128(g, qd, sd, alpha=0.5, transposed=True)
    db = ops.wgrad_bf16(g, xb, alpha=0.5)
    dbt = ops.wgrad_bf16(g, xb, alpha=0.5, transposed=True)
    torch.cuda.synchronize()
    want, size = _wgrad64(g, xb, 0.5)
    assert_close(dw, want, _wgrad_tol(want, size, M), "dw")
    assert torch.equal(dw, again) and torch.equal(dw, dwt.t()) and torch.equal(dw, db) and torch.equal(dw, dbt.t())


def test_wgrad_strided_empty_and_scale_layouts(cuda_device):
    from ltx_kernels.blockwise import ops
    M, N, K = 300, 64, 256
    xq, xs = quant_rows(tokens(M, K, 43).float())
    qd, sd = xq.to(cuda_device), mn_major(xs.to(cuda_device))
    big = grads(M, 200, 44).to(cuda_device)
    want = ops.wgrad_1x128(big[:, 16:80].contiguous(), qd, sd)
    for g in (big[:, 16:80], big[:, 16:80].reshape(3, 100, 64)):
        assert torch.equal(ops.wgrad_1x128(g, qd, sd), want)
    assert torch.equal(ops.wgrad_1x128(big[:, 16:80], qd.view(3, 100, K), sd.t().contiguous()), want)
    odd = big[:, 3:67]
    assert torch.equal(ops.wgrad_1x128(odd, qd, sd), ops.wgrad_1x128(odd.contiguous(), qd, sd))
    e = ops.wgrad_1x128(big[:0, :64], qd[:0], sd[:0])
    assert e.shape == (N, K) and (e == 0).all()


@pytest.mark.parametrize("N,K", [(128, 128), (256, 640), (1152, 384)])
def test_transpose_weight(cuda_device, N, K):
    from ltx_kernels.blockwise import ops
    w, s = quant_weight(torch.randn(N, K, generator=gen(45)))
    s = s * torch.rand(s.shape, generator=gen(46))
    wt, st = ops.transpose_weight_128x128(w.to(cuda_device), s.to(cuda_device))
    assert torch.equal(wt.cpu().view(torch.uint8), w.view(torch.uint8).t()) and torch.equal(st.cpu(), s.t())
