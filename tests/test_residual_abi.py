"""The residual-path and training operators without a GPU: their entry points refuse bad
arguments before touching a device, the tensor-level calls refuse what they cannot take,
and the modules keep their parameters."""
from __future__ import annotations

import ctypes

import pytest
import torch

P = 4096  # a made-up aligned address: every call here returns before it is used


def _lib():
    from ltx_kernels import _lib as L
    return L, L.load()


def test_binding_is_built_and_complete():
    L, _ = _lib()
    b = L.binding()
    for f in ("rms_norm_quantize", "rms_norm_backward", "gemm_residual", "act_quantize_save", "act_backward",
              "wgrad_1x128", "wgrad_bf16", "check_capture"):
        assert callable(getattr(b, f))
    with pytest.raises(TypeError, match="positional"):
        b.act_quantize_save()


@pytest.mark.parametrize("kw,code", [
    (dict(H=100), "shape"), (dict(H=0), "shape"), (dict(H=16512), "shape"), (dict(M=-1), "shape"),
    (dict(x=None), "arg"), (dict(x_ld=64), "arg"), (dict(x=P + 2), "align"), (dict(x_ld=260), "align"),
    (dict(r=None), "arg"),            # h without a residual
    (dict(h=None), "arg"),            # a residual without h
    (dict(r_ld=12), "arg"), (dict(r=P + 8), "align"),
    (dict(q=None), "arg"),            # neither codes nor out
    (dict(out=P), "arg"),             # both
    (dict(sfa=None), "arg"), (dict(sfa_ld=3), "arg"), (dict(q=P + 8), "align"),
    (dict(w=P, wdt=2), "arg"), (dict(w=P + 4, wdt=0), "align"), (dict(eps=-1.0), "arg"), (dict(eps=float("nan")), "arg"),
])
def test_rms_norm_refusals(kw, code):
    L, lib = _lib()
    a = dict(x=P, x_ld=256, r=P, r_ld=256, M=4, H=256, w=None, wdt=0, eps=1e-6, h=P, q=P, sfa=P, sfa_ld=4, out=None,
             rstd=P)
    a.update(kw)
    rc = lib.ltxfp8_rms_norm_quantize(a["x"], a["x_ld"], a["r"], a["r_ld"], a["M"], a["H"], a["w"], a["wdt"], a["eps"],
                                      a["h"], a["q"], a["sfa"], a["sfa_ld"], a["out"], a["rstd"], None)
    assert rc == {"shape": L.ERR_UNSUPPORTED_SHAPE, "arg": L.ERR_INVALID_ARGUMENT, "align": L.ERR_MISALIGNED}[code]
    assert "rms_norm_quantize" in lib.ltxfp8_last_error().decode()


def test_empty_calls_are_no_ops_without_device():
    L, lib = _lib()
    assert lib.ltxfp8_rms_norm_quantize(None, 256, None, 0, 0, 256, None, 0, 1e-6, None, None, None, 0, None, None,
                                        None) == L.OK
    assert lib.ltxfp8_act_quantize_save(None, 256, 0, 256, 1, None, None, 0, None, None, 0, None) == L.OK


@pytest.mark.parametrize("kw,code", [
    (dict(H=128 * 129), "shape"), (dict(dy=None), "arg"), (dict(h=None), "arg"), (dict(rstd=None), "arg"),
    (dict(dx=None), "arg"), (dict(dh=P + 2), "align"), (dict(w=None), "arg"),
])
def test_rms_norm_backward_refusals(kw, code):
    L, lib = _lib()
    a = dict(dy=P, h=P, rstd=P, w=P, dh=P, H=256, dx=P, dw=P)
    a.update(kw)
    rc = lib.ltxfp8_rms_norm_backward(a["dy"], 256, a["h"], 256, a["rstd"], a["w"], 0, a["dh"], 256, 4, a["H"], a["dx"],
                                      a["dw"], P, 1 << 30, None)
    assert rc == {"shape": L.ERR_UNSUPPORTED_SHAPE, "arg": L.ERR_INVALID_ARGUMENT, "align": L.ERR_MISALIGNED}[code]


@pytest.mark.parametrize("kw,code", [
    (dict(M=0), "shape"), (dict(N=100), "shape"), (dict(K=200), "shape"), (dict(act=3), "arg"), (dict(act=-1), "arg"),
    (dict(D=None), "arg"), (dict(sfa_ld=7), "arg"), (dict(r_ld=128), "arg"), (dict(r=P + 2), "align"),
    (dict(r_ld=260), "align"), (dict(bias=P + 4), "align"),
])
def test_gemm_residual_refusals(kw, code):
    L, lib = _lib()
    a = dict(M=8, N=256, K=256, sfa_ld=8, r=P, r_ld=256, bias=None, D=2 * P, act=0)
    a.update(kw)
    rc = lib.ltxfp8_gemm_residual(P, P, a["sfa_ld"], P, P, a["bias"], a["r"], a["r_ld"], a["D"], a["M"], a["N"], a["K"],
                                  a["act"], None, 0, None)
    assert rc == {"shape": L.ERR_UNSUPPORTED_SHAPE, "arg": L.ERR_INVALID_ARGUMENT, "align": L.ERR_MISALIGNED}[code]


def test_act_and_wgrad_refusals():
    L, lib = _lib()
    S, A, M = L.ERR_UNSUPPORTED_SHAPE, L.ERR_INVALID_ARGUMENT, L.ERR_MISALIGNED
    save = lambda z=P, ld=256, N=256, act=1, yq=P, ys=P, ysld=4, zq=P, zsld=4: lib.ltxfp8_act_quantize_save(  # noqa: E731
        z, ld, 4, N, act, yq, ys, ysld, zq, P, zsld, None)
    assert save(N=100) == S and save(act=0) == A and save(act=7) == A and save(z=None) == A and save(ld=128) == A
    assert save(yq=None) == A and save(ysld=3) == A and save(zsld=3) == A and save(zq=P + 4) == M and save(z=P + 2) == M
    bwd = lambda dy=P, zq=P, act=1, dz=P, dzq=None, dzs=None: lib.ltxfp8_act_backward(  # noqa: E731
        dy, 256, zq, P, 4, 4, 256, act, dz, dzq, dzs, 4, None, None, 0, None)
    assert bwd(dy=None) == A and bwd(zq=None) == A and bwd(act=0) == A and bwd(dz=None) == A and bwd(dz=P + 2) == M
    assert bwd(dzq=P) == A  # codes without scales
    wg = lambda g=P, gld=64, x=P, xld=256, xs=P, xsld=8, out=P, m=8, n=64, k=256: lib.ltxfp8_wgrad(  # noqa: E731
        g, gld, x, xld, xs, xsld, 1.0, out, 0, m, n, k, None, 0, None)
    assert wg(n=24) == S and wg(n=0) == S and wg(k=200) == S and wg(m=-1) == S and wg(n=1 << 21) == S
    assert wg(g=None) == A and wg(x=None) == A and wg(out=None) == A and wg(gld=32) == A and wg(xld=128) == A
    assert wg(xsld=4) == A and wg(g=P + 2) == M and wg(gld=68) == M and wg(xld=264) == M and wg(out=P + 8) == M
    tr = lib.ltxfp8_transpose_weight_128x128
    assert tr(P, P, 100, 128, 2 * P, P, None) == S and tr(None, P, 128, 128, P, P, None) == A
    assert tr(P, P, 128, 128, P, P, None) == A and tr(P + 8, P, 128, 128, P, P, None) == M


@pytest.mark.parametrize("M,N,K", [(1, 16, 128), (6143, 32, 4096), (6144, 4096, 4096), (300, 1008, 640), (99999, 16, 128)])
def test_wgrad_plan(M, N, K):
    """The plan covers every token, fits its workspace's formula, and needs none for one split."""
    L, lib = _lib()
    i = L.WgradPlanInfo()
    assert lib.ltxfp8_wgrad_plan_for_sms(M, N, K, 148, ctypes.byref(i)) == L.OK
    assert 16 <= i.columns <= 256 and i.columns % 16 == 0 and i.columns <= max(64, N) and i.splits >= 1
    assert i.splits <= (M + 63) // 64
    tile_k = 512 if i.pair else 256
    tiles = -(-N // i.columns) * -(-K // tile_k)
    assert i.workspace_bytes == (tiles * i.splits * tile_k * i.columns * 4 if i.splits > 1 else 0)
    again = L.WgradPlanInfo()
    assert lib.ltxfp8_wgrad_plan_for_sms(M, N, K, 148, ctypes.byref(again)) == L.OK
    assert (again.columns, again.splits, again.pair) == (i.columns, i.splits, i.pair)
    assert lib.ltxfp8_wgrad_plan_for_sms(0, N, K, 148, ctypes.byref(i)) == L.ERR_INVALID_ARGUMENT
    assert lib.ltxfp8_wgrad_plan_for_sms(M, N, K, 0, ctypes.byref(i)) == L.ERR_INVALID_ARGUMENT


def test_in_place_needs_contiguous_rows():
    """Writing a result over a strided operand would overwrite its neighbours: refused."""
    L, lib = _lib()
    A = L.ERR_INVALID_ARGUMENT
    Q = 2 * P
    for h, xld, rld in ((P, 512, 256), (Q, 256, 512)):
        assert lib.ltxfp8_rms_norm_quantize(P, xld, Q, rld, 4, 256, None, 0, 1e-6, h, 3 * P, P, 4, None, None, None) == A
    for dx, h, dy_ld, dh_ld in ((P, Q, 512, 256), (3 * P, Q, 256, 512), (Q, Q, 256, 256)):
        assert lib.ltxfp8_rms_norm_backward(P, dy_ld, h, 256, P, None, 0, 3 * P, dh_ld, 4, 256, dx, None, None, 0,
                                            None) == A
    assert lib.ltxfp8_gemm_residual(P, P, 8, P, P, None, Q, 512, Q, 8, 256, 256, 0, None, 0, None) == A
    # results shifted against an operand by some rows
    assert lib.ltxfp8_gemm_residual(P, P, 8, P, P, None, Q, 256, Q + 512, 8, 256, 256, 0, None, 0, None) == A
    assert lib.ltxfp8_rms_norm_quantize(P, 256, Q, 256, 4, 256, None, 0, 1e-6, P + 512, 3 * P, P, 4, None, None, None) == A
    assert lib.ltxfp8_rms_norm_quantize(P, 256, None, 0, 4, 256, None, 0, 1e-6, None, None, None, 4, P + 1024, None,
                                        None) == A
    assert lib.ltxfp8_rms_norm_quantize(P, 256, Q, 256, 4, 256, None, 0, 1e-6, 3 * P, None, None, 4, 3 * P, None,
                                        None) == A  # out is h
    assert lib.ltxfp8_rms_norm_backward(P, 256, Q, 256, P, None, 0, None, 0, 4, 256, Q + 512, None, None, 0, None) == A
    assert lib.ltxfp8_act_backward(P, 256, Q, P, 4, 4, 256, 1, P + 512, None, None, 4, None, None, 0, None) == A
    assert lib.ltxfp8_act_backward(P, 512, Q, P, 4, 4, 256, 1, P, None, None, 4, None, None, 0, None) == A


def test_quantize_modes():
    L, lib = _lib()
    for mode, ok in ((L.QUANT_FINITE, True), (3, False), (L.QUANT_TORCH | L.QUANT_ZEROS, True),
                     (L.QUANT_TRITON | L.QUANT_ZEROS, True), (L.QUANT_FINITE | L.QUANT_ZEROS, False), (8, False),
                     (-1, False)):
        rc = lib.ltxfp8_quantize_1x128(16, 0, 128, 128, 16, 128, 16, 0, mode, None)
        assert (rc == L.OK) == ok
    # the reference's producers keep their two arithmetics
    assert lib.ltxfp8_gated_attention(16, 16, 1, 4, 256, 2, 16, 16, 4, None, L.QUANT_FINITE, None) \
        == L.ERR_INVALID_ARGUMENT


    w = lib.ltxfp8_quantize_weight_128x128_finite
    assert w(P, 0, 100, 128, P, P, None) == L.ERR_UNSUPPORTED_SHAPE and w(P, 3, 128, 128, P, P, None) == L.ERR_INVALID_ARGUMENT
    assert w(None, 0, 128, 128, P, P, None) == L.ERR_INVALID_ARGUMENT and w(P + 4, 0, 128, 128, P, P, None) == L.ERR_MISALIGNED


def test_check_capture():
    L, _ = _lib()
    t = torch.zeros(3, requires_grad=True)
    y = t * 2
    assert L.binding().check_capture("f", [t]) is None and y.requires_grad  # a host leaf has no stream
    with pytest.raises(TypeError, match="f"):
        L.binding().check_capture("f", [1])
    with pytest.raises(TypeError, match="list"):
        L.binding().check_capture("f", t)


def test_host_tensors_and_wrong_types_are_refused():
    from ltx_kernels.blockwise import fp8_linear_train, ops, pre_norm_feed_forward
    x = torch.zeros(4, 256, dtype=torch.bfloat16)
    q, s = torch.zeros(4, 256).to(torch.float8_e4m3fn), torch.ones(4, 2)
    w, ws = torch.zeros(128, 256).to(torch.float8_e4m3fn), torch.ones(1, 2)
    for call in (lambda: ops.rms_norm_quantize(x), lambda: ops.rms_norm_backward(x, x, torch.ones(4)),
                 lambda: ops.gemm_residual(q, s, w, ws), lambda: ops.act_quantize_save(x),
                 lambda: ops.act_backward(x, q, s), lambda: ops.wgrad_1x128(x, q, s), lambda: ops.wgrad_bf16(x, x),
                 lambda: ops.transpose_weight_128x128(w, ws), lambda: fp8_linear_train(x, (w, ws)),
                 lambda: pre_norm_feed_forward(x, (w, ws), (w.t().contiguous(), ws.t().contiguous()))):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(TypeError, match="must be a tensor"):
        ops.rms_norm_quantize(None)
    with pytest.raises(RuntimeError, match="expected bf16"):
        fp8_linear_train(x[:, :128], (w, ws))
    with pytest.raises(RuntimeError, match="w1"):
        pre_norm_feed_forward(x, (w, ws), (w, ws))


def test_module_parameters():
    from ltx_kernels.blockwise import BlockwiseFP8LoRALinear, BlockwiseFP8PreNormFeedForward
    ff = BlockwiseFP8PreNormFeedForward(256, device="cpu")
    assert sorted(ff.state_dict()) == ["norm_weight", "proj_in.bias", "proj_in.weight", "proj_in.weight_scale",
                                       "proj_out.bias", "proj_out.weight", "proj_out.weight_scale"]
    assert [n for n, p in ff.named_parameters() if p.requires_grad] == ["norm_weight"]
    lora = BlockwiseFP8LoRALinear(256, 128, 16, device="cpu")
    assert not any(p.requires_grad for p in lora.parameters())
