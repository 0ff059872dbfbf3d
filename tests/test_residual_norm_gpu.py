"""RMS norm with the residual's addition and an 8-bit output, and its gradient, against a
64-bit evaluation of their formulas (csrc/residual_norm.cuh)."""
from __future__ import annotations

import pytest
import torch

from residual_inputs import U32, UBF16, assert_close, assert_quantised, gen, grads, tokens

pytestmark = pytest.mark.gpu

EPS = 1e-6


def _gain(H, dtype, seed=5):
    return (1.0 + 0.2 * torch.randn(H, generator=gen(seed))).to(dtype)


# A row's sum of squares is a chain of at most 8 fused steps in a thread (16 with two runs),
# 2 joining steps, 5 shuffles and 16 warps: under 40 roundings of positive terms; the root
# halves them, and the mean, eps, root and quotient add four.
RSTD_REL = 24 * U32


def _forward64(x, r, w, dev):
    h = x if r is None else (x.float() + r.float()).to(torch.bfloat16)
    hd = h.to(dev).double()
    rstd = 1.0 / torch.sqrt(hd.square().mean(1) + EPS)
    y = hd * rstd[:, None]
    return h, rstd, y if w is None else y * w.to(dev).double()


@pytest.mark.parametrize("M,H,res,gain", [
    (1, 4096, True, torch.bfloat16),       # a single token
    (3, 128, True, torch.float32),         # one group a row, 8 lanes of a warp
    (37, 384, False, torch.bfloat16),      # three groups
    (130, 640, True, None),                # two warps a row, partly idle, no gain
    (65, 1152, False, torch.float32),
    (257, 2048, True, torch.bfloat16),
    (1003, 4096, False, None),
    (19, 5120, True, torch.float32),
    (7, 8192, False, torch.bfloat16),
    (5, 8320, True, torch.bfloat16),       # two runs a thread
    (4, 16384, True, torch.float32),       # the widest row
])
def test_forward(cuda_device, M, H, res, gain):
    from ltx_kernels.blockwise import ops
    zero = (M // 2,) if M > 2 else ()
    x = tokens(M, H, 1, zero)
    r = tokens(M, H, 2, zero) if res else None
    w = None if gain is None else _gain(H, gain)
    xd, rd, wd = (None if t is None else t.to(cuda_device) for t in (x, r, w))
    q, s, h, rstd = ops.rms_norm_quantize(xd, wd, rd, eps=EPS)
    y, h2, rstd2 = ops.rms_norm_quantize(xd, wd, rd, eps=EPS, quantize=False)
    torch.cuda.synchronize()
    h64, rstd64, y64 = _forward64(x, r, w, cuda_device)
    assert torch.equal(h.cpu(), h64) and torch.equal(h2.cpu(), h64)
    assert torch.equal(rstd, rstd2)
    assert_close(rstd, rstd64, rstd64 * RSTD_REL, "rstd")
    assert tuple(s.shape) == (M, H // 128) and s.stride() == (1, (M + 3) // 4 * 4)
    assert_quantised(q, s, y64, RSTD_REL + 2 * U32, "y")
    assert_close(y, y64, y64.abs() * (UBF16 + RSTD_REL + 2 * U32), "bf16 y")
    for z in zero:
        assert (q[z].float() == 0).all() and torch.isfinite(s[z]).all() and (s[z] > 0).all()


def test_forward_takes_strided_and_shaped_rows(cuda_device):
    """A column slice, a transposed view, a misaligned slice and a [b, s, h] tensor give what
    their contiguous copies give."""
    from ltx_kernels.blockwise import ops
    big = tokens(40, 1024, 3).to(cuda_device)
    w = _gain(512, torch.bfloat16).to(cuda_device)
    for x in (big[:, 256:768], big[::2, :512], big[:, 3:515], tokens(512, 40, 4).to(cuda_device).t(),
              big[:1].expand(8, 1024)[:, :512]):
        r = tokens(x.shape[0], 512, 6).to(cuda_device)
        for got, want in zip(ops.rms_norm_quantize(x, w, r), ops.rms_norm_quantize(x.contiguous(), w, r)):
            assert torch.equal(got.float(), want.float())
    x3 = big[:, :512].reshape(5, 8, 512)
    q, s, h, rstd = ops.rms_norm_quantize(x3, w)
    q2, s2, _, rstd2 = ops.rms_norm_quantize(big[:, :512].contiguous(), w)
    assert torch.equal(q.float(), q2.float()) and torch.equal(s, s2) and torch.equal(rstd, rstd2)
    assert q.shape == (40, 512) and h.shape == (40, 512)


def test_forward_keeps_bad_rows_to_themselves(cuda_device):
    """NaN and infinity stay in their rows; an infinite value makes its row NaN or zero as
    1 / sqrt(inf) = 0 says."""
    from ltx_kernels.blockwise import ops
    x = tokens(6, 1024, 7)
    clean = x.clone()
    x[1, 5] = float("nan")
    x[4, 9] = float("inf")
    q, s, _, rstd = ops.rms_norm_quantize(x.to(cuda_device))
    q0, s0, _, rstd0 = ops.rms_norm_quantize(clean.to(cuda_device))
    for r in (0, 2, 3, 5):
        assert torch.equal(q[r].float(), q0[r].float()) and torch.equal(s[r], s0[r]) and rstd[r] == rstd0[r]
    assert torch.isnan(q[1].float()).all() and torch.isnan(rstd[1])
    assert rstd[4] == 0


def test_forward_empty_and_in_place(cuda_device):
    from ltx_kernels import _lib as L
    from ltx_kernels.blockwise import ops
    q, s, h, rstd = ops.rms_norm_quantize(torch.empty(0, 256, dtype=torch.bfloat16, device=cuda_device))
    assert q.shape == (0, 256) and s.shape == (0, 2) and rstd.shape == (0,)
    x, r = tokens(33, 768, 8).to(cuda_device), tokens(33, 768, 9).to(cuda_device)
    want = ops.rms_norm_quantize(x, None, r)
    for target in (0, 1):  # h written over x, then over the residual
        xx, rr = x.clone(), r.clone()
        q, s = torch.empty_like(want[0]), torch.empty_like(want[1])
        L.check(L.load().ltxfp8_rms_norm_quantize(
            xx.data_ptr(), 768, rr.data_ptr(), 768, 33, 768, None, 0, 1e-6, (xx, rr)[target].data_ptr(), q.data_ptr(),
            s.data_ptr(), s.stride(1), None, None, torch.cuda.current_stream().cuda_stream))
        assert torch.equal((xx, rr)[target], want[2]) and torch.equal(q.float(), want[0].float())


def _backward64(dy, h, rstd, w, dh, dev):
    dyd, hd, r = dy.to(dev).double(), h.to(dev).double(), rstd.double()[:, None]
    xhat = hd * r
    g = dyd if w is None else dyd * w.to(dev).double()
    c = (g * xhat).mean(1, keepdim=True)
    dx = r * (g - xhat * c)
    # what the roundings inside scale with: the terms' sizes before they cancel
    size = r * (g.abs() + xhat.abs() * (g * xhat).abs().mean(1, keepdim=True))
    if dh is not None:
        dx = dx + dh.to(dev).double()
        size = size + dh.to(dev).double().abs()
    return dx, size, (dyd * xhat).sum(0), (dyd * xhat).abs().sum(0)


@pytest.mark.parametrize("M,H,res,gain", [
    (1, 4096, True, torch.bfloat16),
    (2, 128, False, torch.float32),
    (37, 384, True, torch.bfloat16),
    (130, 640, False, None),
    (1003, 1152, True, torch.float32),
    (2500, 2048, False, torch.bfloat16),   # more rows than resident blocks
    (1300, 4096, True, torch.float32),
    (19, 5120, True, torch.float32),
    (700, 8192, False, torch.bfloat16),
    (5, 8320, True, torch.bfloat16),
    (301, 16384, False, torch.float32),
])
def test_backward(cuda_device, M, H, res, gain):
    from ltx_kernels.blockwise import ops
    zero = (M // 2,) if M > 2 else ()
    h = tokens(M, H, 11, zero)
    dy = grads(M, H, 12, zero)
    dh = grads(M, H, 13) if res else None
    w = None if gain is None else _gain(H, gain)
    hd, dyd, dhd, wd = (None if t is None else t.to(cuda_device) for t in (h, dy, dh, w))
    rstd = torch.rsqrt(hd.float().square().mean(1) + EPS)
    dx, dw = ops.rms_norm_backward(dyd, hd, rstd, wd, dhd)
    dx2, dw2 = ops.rms_norm_backward(dyd, hd, rstd, wd, dhd)
    torch.cuda.synchronize()
    assert torch.equal(dx, dx2) and (dw is None or torch.equal(dw, dw2)), "not repeatable"
    dx64, size, dw64, dwabs = _backward64(dy, h, rstd, w, dh, cuda_device)
    # xhat, g, their product, the 40-step row sum, the mean, and four steps to dx
    assert_close(dx, dx64, dx64.abs() * UBF16 + 64 * U32 * size, "dx")
    if w is None:
        assert dw is None
    else:
        assert dw.dtype == gain and dw.shape == (H,)
        # a block (at least one an SM) adds at most M / 148 of its rows in turn, joins 8 row groups,
        # and the at most 296 blocks are summed in 32 chains; each product has two roundings of its own
        steps = M / 148 + 1 + 8 + 296 / 32 + 1 + 32 + 2
        tol = steps * U32 * dwabs + (dw64.abs() * UBF16 if gain == torch.bfloat16 else 0)
        assert_close(dw, dw64, tol, "dw")


def test_backward_is_the_forward_gradient(cuda_device):
    """Against central differences of the 64-bit forward, at a few coordinates."""
    from ltx_kernels.blockwise import ops
    M, H = 3, 256
    h, dy = tokens(M, H, 21), (grads(M, H, 22).float() * 1e4).to(torch.bfloat16)
    w = _gain(H, torch.float32)
    hd = h.to(cuda_device)
    rstd = torch.rsqrt(hd.float().square().mean(1) + EPS)
    dx, dw = ops.rms_norm_backward(dy.to(cuda_device), hd, rstd, w.to(cuda_device))

    def loss(hh, ww):
        return (dy.double() * hh * ww / torch.sqrt(hh.square().mean(1, keepdim=True) + EPS)).sum()

    step = 1e-5
    for m, i in ((0, 0), (1, 17), (2, 255)):
        e = torch.zeros(M, H, dtype=torch.float64)
        e[m, i] = step
        d = (loss(h.double() + e, w.double()) - loss(h.double() - e, w.double())) / (2 * step)
        # bf16 rounding of dx, and the differences' own error (third derivatives ~ 1, step^2)
        assert abs(dx[m, i].item() - d.item()) <= abs(d.item()) * UBF16 + 1e-5
        d = (loss(h.double(), w.double() + e[m]) - loss(h.double(), w.double() - e[m])) / (2 * step)
        assert abs(dw[i].item() - d.item()) <= 1e-5 * max(1.0, abs(d.item()))


def test_backward_empty_strided_and_bad_rows(cuda_device):
    from ltx_kernels.blockwise import ops
    w = _gain(256, torch.bfloat16).to(cuda_device)
    e = torch.empty(0, 256, dtype=torch.bfloat16, device=cuda_device)
    dx, dw = ops.rms_norm_backward(e, e, torch.empty(0, device=cuda_device), w)
    assert dx.shape == (0, 256) and (dw == 0).all()
    big = grads(30, 600, 23).to(cuda_device)
    h = tokens(30, 600, 24).to(cuda_device)
    rstd = torch.rand(30, device=cuda_device) + 0.5
    a = ops.rms_norm_backward(big[:, 8:264], h[:, 16:272], rstd, w, big[:, 5:261])
    b = ops.rms_norm_backward(big[:, 8:264].contiguous(), h[:, 16:272].contiguous(), rstd, w,
                              big[:, 5:261].contiguous())
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    bad = big[:, 8:264].clone()
    bad[3, 7] = float("nan")
    c = ops.rms_norm_backward(bad, h[:, 16:272], rstd, w, big[:, 5:261])
    keep = torch.arange(30, device=cuda_device) != 3
    assert torch.equal(c[0][keep], a[0][keep]) and torch.isnan(c[0][3]).all()
