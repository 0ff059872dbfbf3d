"""Inputs and 64-bit definitions for the residual-path and training operators' tests.

Tolerances count roundings: one rounding to a type t is off by at most
``torch.finfo(t).eps / 2`` of the value (fp32 2^-24, bf16 2^-8, e4m3 2^-4, or half its
subnormal spacing, 2^-10).
"""
from __future__ import annotations

import math

import torch

U32 = 2.0 ** -24
UBF16 = 2.0 ** -8
AMAX_MIN = 448.0 * 2.0 ** -126


def gen(seed: int) -> torch.Generator:
    return torch.Generator().manual_seed(seed)


def tokens(M: int, K: int, seed: int, zero_rows=()) -> torch.Tensor:
    """bf16 activations with a few channels much larger than the rest."""
    g = gen(seed)
    x = torch.randn(M, K, generator=g) * torch.exp(0.5 * torch.randn(K, generator=g))
    for r in zero_rows:
        x[r] = 0
    return x.to(torch.bfloat16)


def grads(M: int, N: int, seed: int, zero_rows=()) -> torch.Tensor:
    """bf16 gradients: small, token scales spread over a few octaves."""
    g = gen(seed)
    x = torch.randn(M, N, generator=g) * (1e-4 * torch.exp2(torch.randn(M, 1, generator=g)))
    for r in zero_rows:
        x[r] = 0
    return x.to(torch.bfloat16)


def quant_rows(v: torch.Tensor):
    """1x128 codes (e4m3) and (M, K/128) scales of a matrix."""
    M, K = v.shape
    g = v.float().view(M, K // 128, 128)
    amax = g.abs().amax(-1, keepdim=True).clamp_min(AMAX_MIN)
    q = (g * (448.0 / amax)).to(torch.float8_e4m3fn).view(M, K)
    return q, (amax / 448.0).view(M, K // 128)


def quant_weight(w: torch.Tensor):
    N, K = w.shape
    b = w.float().view(N // 128, 128, K // 128, 128)
    amax = b.abs().amax((1, 3), keepdim=True).clamp_min(AMAX_MIN)
    q = (b * (448.0 / amax)).to(torch.float8_e4m3fn).view(N, K)
    return q, (amax / 448.0).view(N // 128, K // 128).contiguous()


def mn_major(s: torch.Tensor) -> torch.Tensor:
    """(M, KB) scales with strides (1, M rounded up to 4), on s's device."""
    M, KB = s.shape
    out = torch.empty_strided((M, KB), (1, max(1, (M + 3) // 4 * 4)), dtype=torch.float32, device=s.device)
    out.copy_(s)
    return out


def dequant_rows64(q, s):
    return q.double() * s.double().repeat_interleave(128, 1)


def dequant_weight64(q, s):
    return q.double() * s.double().repeat_interleave(128, 0).repeat_interleave(128, 1)


def act64(z, act):
    if act == "gelu_tanh":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3)))
    if act == "silu":
        return z * torch.sigmoid(z)
    return z


def act_grad64(z, act):
    if act == "gelu_tanh":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z ** 3))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    s = torch.sigmoid(z)
    return s * (1 + z * (1 - s))


def assert_quantised(q, s, v, rel, what=""):
    """``(q, s)`` is the 1x128 quantisation of the 64-bit ``v`` computed with a relative
    error of at most ``rel``: every scale within rel + 3 roundings (floor, product with
    1/448, the constant's own), every code half an e4m3 step from v / scale plus the
    perturbation of v and of the scale's reciprocal (an approximate instruction, 2^-22)."""
    M, K = v.shape
    g = v.view(M, K // 128, 128)
    scale = g.abs().amax(-1).clamp_min(AMAX_MIN) / 448
    sd = s.double()
    assert ((sd - scale).abs() <= scale * (rel + 4 * U32)).all(), f"{what}: scales"
    x = (g / scale.unsqueeze(-1)).view(M, K)
    err = (q.double() - x).abs()
    tol = torch.maximum(x.abs() * 2.0 ** -4, torch.full_like(x, 2.0 ** -10)) + x.abs() * (2 * rel + 2.0 ** -21)
    assert (err <= tol).all(), f"{what}: codes, worst {(err - tol).max().item()}"


def assert_close(got, want, tol, what=""):
    err = (got.double() - want).abs()
    bad = ~(err <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} outside, worst excess {(err - tol).max().item():.3e}"
