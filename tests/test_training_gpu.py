"""Training through the blockwise-FP8 linears: the operators run together, as a pre-norm
block's and a LoRA linear's step, against the sequence of operators they stand for and
against float64 autograd of the unquantised function."""
from __future__ import annotations

import pytest
import torch

from residual_inputs import (act64, dequant_weight64, gen, grads, quant_weight, tokens)

pytestmark = pytest.mark.gpu

# A rounding to e4m3 is off by at most 2^-4 of the value, uniformly spread at worst: 2^-4 / sqrt(3)
# in the root mean square.  Errors of independent roundings add at most linearly.
E4M3_RMS = 2.0 ** -4 / 3 ** 0.5


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return ((a - b).norm() / b.norm()).item()


def _weight(N, K, dev, seed):
    q, s = quant_weight(torch.randn(N, K, generator=gen(seed)) / K ** 0.5)
    return q.to(dev), s.to(dev)


def _leaf(t, dev):
    return t.to(dev).requires_grad_()


@pytest.mark.parametrize("lead,d,inner,act", [((2, 33), 256, 1024, "gelu_tanh"), ((130,), 384, 640, "silu"),
                                              ((1,), 128, 128, "gelu_tanh"), ((3, 300), 1024, 4096, "gelu_tanh")])
def test_pre_norm_block_step(cuda_device, lead, d, inner, act):
    """Forward and every gradient equal the operators run by hand, bit for bit, and lie within
    the 8-bit roundings of float64 autograd through the unquantised block."""
    from ltx_kernels import _lib as L
    from ltx_kernels.blockwise import ops, pre_norm_feed_forward
    M = 1
    for n in lead:
        M *= n
    x, r = _leaf(tokens(M, d, 1).view(*lead, d), cuda_device), _leaf(tokens(M, d, 2).view(*lead, d), cuda_device)
    nw = _leaf(1 + 0.2 * torch.randn(d, generator=gen(3)), cuda_device)
    m1 = _leaf(torch.randn(inner, d, generator=gen(4)) / d ** 0.5, cuda_device)
    m2 = _leaf((torch.randn(d, inner, generator=gen(5)) / inner ** 0.5).to(torch.bfloat16), cuda_device)
    b1, b2 = (_leaf(0.1 * torch.randn(n, generator=gen(6)), cuda_device) for n in (inner, d))
    dout = (grads(M, d, 7).view(*lead, d) * 1e3).to(cuda_device)
    out = pre_norm_feed_forward(x, m1, m2, residual=r, norm_weight=nw, b1=b1, b2=b2, activation=act)
    got = torch.autograd.grad(out, (x, r, nw, m1, m2, b1, b2), dout)

    with torch.no_grad():
        w1, s1 = ops.quantize_weight_128x128(m1)
        w2, s2 = ops.quantize_weight_128x128(m2)
        nq, ns, h, rstd = ops.rms_norm_quantize(x, nw, r)
        z = ops.gemm(nq, ns, w1, s1, b1)
        yq, ys, zq, zs = ops.act_quantize_save(z, act)
        assert torch.equal(out.view(M, d), ops.gemm_residual(yq, ys, w2, s2, b2, residual=h))
        g = dout.view(M, d)
        gq, gs = ops.quantize_1x128(g, L.QUANT_FINITE)
        dy = ops.gemm(gq, gs, *ops.transpose_weight_128x128(w2, s2))
        dz, dzq, dzs, db1 = ops.act_backward(dy, zq, zs, act, quantize=True, dbias=True)
        dn = ops.gemm(dzq, dzs, *ops.transpose_weight_128x128(w1, s1))
        dx, dnw = ops.rms_norm_backward(dn, h, rstd, nw, g)
        want = (dx.view(x.shape), dx.view(x.shape), dnw, ops.wgrad_1x128(dz, nq, ns).float(),
                ops.wgrad_1x128(g, yq, ys), db1, g.sum(0, dtype=torch.float32))
    for name, a, b in zip(("x", "residual", "norm_weight", "w1", "w2", "b1", "b2"), got, want):
        assert a.dtype == b.dtype and a.shape == b.shape and torch.equal(a, b), name

    # float64, with the weights as quantised (their gradients pass straight through)
    p = [t.detach().double().requires_grad_() for t in (x, r, nw, b1, b2)]
    v1, v2 = (dequant_weight64(*w).requires_grad_() for w in ((w1, s1), (w2, s2)))
    h64 = p[0] + p[1]
    n64 = h64 / torch.sqrt(h64.square().mean(-1, keepdim=True) + 1e-6) * p[2]
    o64 = h64 + act64(n64 @ v1.t() + p[3], act) @ v2.t() + p[4]
    ref = torch.autograd.grad(o64, (p[0], p[1], p[2], v1, v2, p[3], p[4]), dout.double())
    # roundings to 8 bits on the way: the output has two (the norm's and the activation's output);
    # dx: the gradient, z inside act' (slope |z act''| <= 1.5 of act'), the norm's output through z
    # (the same slope), dz; dw1: the gradient, z twice, the norm's output; dw2: the activation's
    # output and the norm's through it; db1: the gradient, z twice; db2: none (bf16 steps only)
    bars = {"x": 5, "residual": 5, "norm_weight": 5, "w1": 5, "w2": 2.5, "b1": 4, "b2": 0.01}
    assert _rel(out, o64) <= 2 * E4M3_RMS
    for (name, n), a, b in zip(bars.items(), got, ref):
        assert _rel(a, b) <= n * E4M3_RMS + 2 ** -8, (name, _rel(a, b))


def test_pre_norm_module(cuda_device):
    """Inference and training give the same output; frozen weights get no gradient; padded tokens
    stay finite; no gradient, no checkpoint."""
    from ltx_kernels.blockwise import BlockwiseFP8PreNormFeedForward
    torch.manual_seed(0)
    ff = BlockwiseFP8PreNormFeedForward(256, device=cuda_device)
    for lin, (n, k), seed in ((ff.proj_in, (1024, 256), 11), (ff.proj_out, (256, 1024), 12)):
        w, s = _weight(n, k, cuda_device, seed)
        lin.weight.data, lin.weight_scale.data = w, s
        lin.bias.data.zero_()
    x = tokens(70, 256, 13, zero_rows=(5, 69)).view(2, 35, 256).to(cuda_device)
    with torch.no_grad():
        y0 = ff(x, x)
    y = ff(x.requires_grad_(), x)
    assert torch.equal(y, y0) and y.requires_grad and not y0.requires_grad
    dout = grads(70, 256, 14, zero_rows=(5, 69)).view(2, 35, 256).to(cuda_device)
    y.backward(dout)
    assert torch.isfinite(x.grad).all() and torch.isfinite(ff.norm_weight.grad).all()
    assert (x.grad.view(70, 256)[5] == 0).all() and ff.proj_in.weight.grad is None
    assert torch.isfinite(y).all() and (y.view(70, 256)[5] == 0).all()
    empty = ff(x[:, :0].detach())
    assert empty.shape == (2, 0, 256)


@pytest.mark.parametrize("M,K,N,r", [(65, 256, 384, 16), (300, 512, 256, 32), (1, 128, 128, 64), (1030, 1024, 1152, 128)])
def test_lora_linear_step(cuda_device, M, K, N, r):
    from ltx_kernels import _lib as L
    from ltx_kernels.blockwise import BlockwiseFP8LoRALinear, ops
    from ltx_kernels.blockwise.functional import quant_mode_code
    layer = BlockwiseFP8LoRALinear(K, N, r, alpha=0.5, device=cuda_device)
    w, s = _weight(N, K, cuda_device, 21)
    layer.weight.data, layer.weight_scale.data = w, s
    layer.bias.data = 0.1 * torch.randn(N, generator=gen(22)).to(cuda_device)
    layer.lora_A.data = (torch.randn(r, K, generator=gen(23)) / K ** 0.5).to(torch.bfloat16).to(cuda_device)
    layer.lora_B.data = (torch.randn(N, r, generator=gen(24)) / r ** 0.5).to(torch.bfloat16).to(cuda_device)
    x = tokens(M, K, 25).to(cuda_device)
    frozen = layer(x)
    assert not frozen.requires_grad
    layer.lora_A.requires_grad_()
    layer.lora_B.requires_grad_()
    layer.bias.requires_grad_()
    x.requires_grad_()
    y = layer(x)
    dy = (grads(M, N, 26) * 1e3).to(cuda_device)
    got = torch.autograd.grad(y, (x, layer.lora_A, layer.lora_B, layer.bias), dy)
    assert torch.equal(y, frozen)

    with torch.no_grad():
        q, sc = ops.quantize_1x128(x, quant_mode_code())
        a, b = layer.lora_A, layer.lora_B
        u = ops.lora_a(dy, b.t().contiguous())
        gq, gs = ops.quantize_1x128(dy, L.QUANT_FINITE)
        wt, wts = ops.transpose_weight_128x128(w, s)
        ax = ops.lora_a(x, a)
        want = (ops.gemm(gq, gs, wt, wts, lora_ax=u, lora_b=a.t().contiguous(), lora_alpha=0.5),
                ops.wgrad_1x128(u, q, sc, alpha=0.5), ops.wgrad_bf16(ax, dy, alpha=0.5, transposed=True),
                dy.sum(0, dtype=torch.float32))
        for name, p, t in zip(("x", "A", "B", "bias"), got, want):
            assert p.dtype == t.dtype and p.shape == t.shape and torch.equal(p, t), name

    p = [t.detach().double().requires_grad_() for t in (x, layer.lora_A, layer.lora_B, layer.bias)]
    y64 = p[0] @ dequant_weight64(w, s).t() + 0.5 * (p[0] @ p[1].t()) @ p[2].t() + p[3]
    ref = torch.autograd.grad(y64, p, dy.double())
    # dx: the gradient's 8-bit rounding; dA: x's; dB: bf16 roundings of x A^T only; dbias: none
    for name, n, a_, b_ in zip(("x", "A", "B", "bias"), (1, 1, 0, 0), got, ref):
        assert _rel(a_, b_) <= n * E4M3_RMS + 3 * 2 ** -8, (name, _rel(a_, b_))


def test_linear_train_master_weight_and_residual(cuda_device):
    from ltx_kernels.blockwise import fp8_linear_train, ops
    M, K, N = 200, 512, 384
    x = _leaf(tokens(M, K, 31), cuda_device)
    m = _leaf(torch.randn(N, K, generator=gen(32)) / K ** 0.5, cuda_device)
    r = _leaf(tokens(M, N, 33), cuda_device)
    y = fp8_linear_train(x, m, residual=r)
    dy = (grads(M, N, 34) * 1e3).to(cuda_device)
    dx, dm, dr = torch.autograd.grad(y, (x, m, r), dy)
    assert torch.equal(dr, dy) and dm.dtype == torch.float32
    w, s = ops.quantize_weight_128x128(m.detach())
    v = dequant_weight64(w, s)
    assert _rel(y, x.double() @ v.t() + r.double()) <= E4M3_RMS + 2 ** -8
    assert _rel(dx, dy.double() @ v) <= E4M3_RMS + 2 ** -8
    assert _rel(dm, dy.double().t() @ x.double()) <= E4M3_RMS + 2 ** -8
    # fp32 gradients arriving at the output, and nothing to do for a frozen weight
    y2 = fp8_linear_train(x, (w, s)).float()
    (g2,) = torch.autograd.grad(y2, x, dy.float())
    assert torch.equal(g2, dx)


def test_memory_kept_is_8_bit(cuda_device):
    """What a trained linear keeps of its input: one byte a value and 1/32 of scales, not a bf16
    copy; nothing where no gradient reads it."""
    from ltx_kernels.blockwise import fp8_linear_train, pre_norm_feed_forward
    M, K, N = 8192, 2048, 128
    w = _weight(N, K, cuda_device, 41)
    m = _leaf(torch.randn(N, K, generator=gen(43)), cuda_device)
    kept = []

    def pack(t):
        if t.dim() == 2 and t.shape[0] == M:
            kept.append((t.dtype, t.numel() * t.element_size()))
        return t

    x = _leaf(tokens(M, K, 42), cuda_device)
    with torch.autograd.graph.saved_tensors_hooks(pack, lambda t: t):
        fp8_linear_train(x, m)
        assert sorted(str(d) for d, _ in kept) == ["torch.float32", "torch.float8_e4m3fn"]
        assert sum(b for _, b in kept) == M * K + M * K // 128 * 4
        kept.clear()
        fp8_linear_train(x, w)
        assert not kept
        # a frozen block: its input's h in bf16 and the activation's input in 8 bits
        pre_norm_feed_forward(x, _weight(256, K, cuda_device, 44), _weight(K, 256, cuda_device, 45))
        assert sum(b for _, b in kept) == 2 * M * K + M * 256 + M * 256 // 128 * 4


def test_gradients_of_any_layout(cuda_device):
    """Expanded, transposed and oddly sliced gradients and inputs, no tokens, the same tensor as
    input and residual."""
    from ltx_kernels.blockwise import fp8_linear_train, pre_norm_feed_forward
    M, K, N = 40, 256, 384
    m = _leaf(torch.randn(N, K, generator=gen(91)) / 16, cuda_device)
    wide = tokens(M, K + 24, 92).to(cuda_device)
    v = (grads(1, N, 93) * 1e3).to(cuda_device)
    gw = (grads(M, N + 8, 94) * 1e3).to(cuda_device)
    for x in (wide[:, 5:5 + K], wide[:, 8:8 + K], wide[:1, :K].expand(M, K)):
        x = x.detach().requires_grad_()
        xc = x.detach().contiguous().requires_grad_()
        for dy in (v.expand(M, N), gw[:, 3:3 + N], gw.t().contiguous().t()[:, :N]):
            got = torch.autograd.grad(fp8_linear_train(x, m), (x, m), dy)
            want = torch.autograd.grad(fp8_linear_train(xc, m), (xc, m), dy.contiguous())
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    w1, w2 = _weight(512, K, cuda_device, 95), _weight(K, 512, cuda_device, 96)
    x = _leaf(tokens(M, K, 97), cuda_device)
    y = pre_norm_feed_forward(x, w1, w2, residual=x)
    (both,) = torch.autograd.grad(y.sum(0).float() @ torch.ones(K, device=cuda_device), x)
    a, b = x.detach().clone().requires_grad_(), x.detach().clone().requires_grad_()
    ga, gb = torch.autograd.grad(pre_norm_feed_forward(a, w1, w2, residual=b).float().sum(), (a, b))
    assert torch.equal(ga, gb) and torch.equal(both, ga + gb)
    e = x.detach()[:0].requires_grad_()
    dx, dm = torch.autograd.grad(fp8_linear_train(e, m), (e, m), gw[:0, :N])
    assert dx.shape == (0, K) and (dm == 0).all()
    (dx,) = torch.autograd.grad(pre_norm_feed_forward(e, w1, w2), e, e)
    assert dx.shape == (0, K)


def test_zeros_stay_finite(cuda_device):
    """Padded tokens in a LoRA linear's training and zero-initialised master weights: finite
    outputs and gradients, the other tokens' as without them."""
    from ltx_kernels.blockwise import BlockwiseFP8LoRALinear, fp8_linear_train
    M, K, N, r = 70, 256, 384, 16
    layer = BlockwiseFP8LoRALinear(K, N, r, device=cuda_device)
    layer.weight.data, layer.weight_scale.data = _weight(N, K, cuda_device, 101)
    layer.bias.data.zero_()
    for p, shape, seed in ((layer.lora_A, (r, K), 102), (layer.lora_B, (N, r), 103)):
        p.data = torch.randn(shape, generator=gen(seed)).to(torch.bfloat16).to(cuda_device)
        p.requires_grad_()
    x = tokens(M, K, 104, zero_rows=(3, 69)).to(cuda_device)
    x[4, :128] = 0
    dy = (grads(M, N, 105, zero_rows=(3, 69)) * 1e3).to(cuda_device)
    y = layer(x)
    ga, gb = torch.autograd.grad(y, (layer.lora_A, layer.lora_B), dy)
    assert torch.isfinite(y).all() and torch.isfinite(ga).all() and torch.isfinite(gb).all()
    with torch.no_grad():
        full = torch.arange(M, device=cuda_device)[(x != 0).view(M, 2, 128).any(-1).all(-1)]
        assert torch.equal(y[full], layer(x[full])) and (y[3] == 0).all()
    m = torch.randn(N, K, generator=gen(106)) / 16
    m[:128] = 0
    m[128:256, 128:] = 0
    m = _leaf(m, cuda_device)
    xg = x.clone().requires_grad_()
    y = fp8_linear_train(xg, m)
    dx, dm = torch.autograd.grad(y, (xg, m), dy)
    assert (y[:, :128] == 0).all() and all(torch.isfinite(t).all() for t in (y, dx, dm))
    v = m.detach().double()
    assert _rel(dx, dy.double() @ v) <= 2 * E4M3_RMS + 2 ** -8 and _rel(y, x.double() @ v.t()) <= 2 * E4M3_RMS + 2 ** -8
    assert _rel(dm, dy.double().t() @ x.double()) <= E4M3_RMS + 2 ** -8


def test_quantisers_without_nan(cuda_device):
    """QUANT_ZEROS and finite weights: the same bytes but for groups without a finite scale,
    which become zeros; NaN and infinity stay what they were."""
    from ltx_kernels import _lib as L
    from ltx_kernels.blockwise import ops
    x = tokens(67, 384, 107).to(cuda_device)
    x[3], x[5, 128:256], x[9, 0], x[10, 1], x[11, :128] = 0, 0, float("nan"), float("inf"), 1e-37
    lost = torch.zeros(67, 3, dtype=torch.bool, device=cuda_device)
    lost[3], lost[5, 1], lost[11, 0] = True, True, True
    for mode in (L.QUANT_TORCH, L.QUANT_TRITON):
        (q0, s0), (q1, s1) = ops.quantize_1x128(x, mode), ops.quantize_1x128(x, mode | L.QUANT_ZEROS)
        a, b = q0.view(torch.uint8).view(67, 3, 128), q1.view(torch.uint8).view(67, 3, 128)
        assert torch.equal(a[~lost], b[~lost]) and (b[lost] & 0x7F == 0).all()
        assert torch.equal(s0[~lost].nan_to_num(7.0), s1[~lost].nan_to_num(7.0)) and (s1[lost] == 0).all()
    w = torch.randn(256, 384, generator=gen(108)).to(cuda_device)
    w[:128, 128:256], w[200, 300] = 0, float("nan")
    (q0, s0), (q1, s1) = ops.quantize_weight_128x128(w), ops.quantize_weight_128x128(w, finite=True)
    keep = torch.ones(256, 384, dtype=torch.bool, device=cuda_device)
    keep[:128, 128:256] = False
    a, b = q0.view(torch.uint8), q1.view(torch.uint8)
    assert torch.equal(a[keep], b[keep]) and (b[~keep] & 0x7F == 0).all() and s1[0, 1] == 0
    s0[0, 1] = 0
    assert torch.equal(s0.nan_to_num(7.0), s1.nan_to_num(7.0))


def test_step_in_a_cuda_graph(cuda_device):
    """Forward and backward captured after a warm-up on a side stream, replayed on new inputs."""
    from ltx_kernels.blockwise import fp8_linear_train, pre_norm_feed_forward
    M, d, inner, N = 300, 256, 512, 128
    w1, w2 = _weight(inner, d, cuda_device, 111), _weight(d, inner, cuda_device, 112)
    m = _leaf(torch.randn(N, d, generator=gen(113)) / 16, cuda_device)
    nw = _leaf(1 + 0.1 * torch.randn(d, generator=gen(114)), cuda_device)
    x = _leaf(tokens(M, d, 115), cuda_device)
    dy = (grads(M, N, 116) * 1e3).to(cuda_device)

    def step():
        return torch.autograd.grad(fp8_linear_train(pre_norm_feed_forward(x, w1, w2, norm_weight=nw), m), (x, nw, m), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    with torch.no_grad():
        x.copy_(tokens(M, d, 117))
        dy.copy_(grads(M, N, 118) * 1e3)
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b)


def test_capture_beside_a_living_eager_result_is_refused(cuda_device):
    """Its gradient nodes belong to the default stream, where a captured backward pass must not
    run: refused in the forward call, before anything of it is captured."""
    from ltx_kernels.blockwise import fp8_linear_train, pre_norm_feed_forward
    w1, w2 = _weight(256, 128, cuda_device, 121), _weight(128, 256, cuda_device, 122)
    x = _leaf(tokens(16, 128, 123), cuda_device)
    m = _leaf(torch.randn(128, 128, generator=gen(124)), cuda_device)
    y = fp8_linear_train(x, m)
    buf = torch.zeros(4, device=cuda_device)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        buf += 1
        with pytest.raises(RuntimeError, match="default stream"):
            fp8_linear_train(x, m)
        with pytest.raises(RuntimeError, match="default stream"):
            pre_norm_feed_forward(x, w1, w2)
    graph.replay()
    torch.cuda.synchronize()
    assert (buf == 1).all()
    (gx,) = torch.autograd.grad(y, x, torch.ones_like(y))  # the eager result is as good as before
    assert torch.isfinite(gx).all()


def test_operators_on_another_stream(cuda_device):
    """Every operator runs on the current stream: work queued behind a long one on a side
    stream sees its inputs, and agrees with the default stream's results."""
    from ltx_kernels.blockwise import ops
    x, r = tokens(300, 1024, 51).to(cuda_device), tokens(300, 1024, 52).to(cuda_device)
    w, s = _weight(512, 1024, cuda_device, 53)
    g = grads(300, 64, 54).to(cuda_device)

    def chain(a):
        q, sc, h, rstd = ops.rms_norm_quantize(a, None, r)
        z = ops.gemm_residual(q, sc, w, s, activation="silu")
        yq, ys, zq, zs = ops.act_quantize_save(z)
        dz, dq, ds, db = ops.act_backward(z, zq, zs, quantize=True, dbias=True)
        dw = ops.wgrad_1x128(g, q, sc)
        dx, _ = ops.rms_norm_backward(h, h, rstd, None, r)
        return [h, z, yq.float(), zq.float(), dz, dq.float(), ds, db, dw, dx]

    want = chain(x)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    late = torch.zeros_like(x)
    with torch.cuda.stream(side):
        big = torch.randn(4096, 4096, device=cuda_device)
        for _ in range(4):
            big = big @ big * 1e-3
        late.copy_(x)
        got = chain(late)
    side.synchronize()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


def test_two_threads_on_two_streams(cuda_device):
    """Calls from two host threads at once, each on its own stream: nothing is shared between them."""
    import threading

    from ltx_kernels.blockwise import ops
    w, s = _weight(384, 640, cuda_device, 131)
    ins = [(tokens(m, 640, 132 + m).to(cuda_device), grads(m, 384, 133 + m).to(cuda_device)) for m in (12, 700)]

    def chain(x, g):
        q, sc, h, rstd = ops.rms_norm_quantize(x, None, x)
        z = ops.gemm_residual(q, sc, w, s, residual=g, activation="silu")
        yq, ys, zq, zs = ops.act_quantize_save(z)
        dz, dq, ds, db = ops.act_backward(g, zq, zs, quantize=True, dbias=True)
        dx, dw = ops.rms_norm_backward(x, h, rstd, torch.ones(640, device=cuda_device), h)
        return [z, yq.float(), dz, ds, db, dx, dw, ops.wgrad_1x128(dz, q, sc)]

    want = [chain(*i) for i in ins]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()) as _:
                for _ in range(20):
                    got = chain(*ins[i])
                    torch.cuda.current_stream().synchronize()
                    if not all(torch.equal(a, b) for a, b in zip(got, want[i])):
                        bad.append(i)
        except Exception as e:  # noqa: BLE001
            bad.append(e)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not bad


def test_operators_in_cuda_graphs(cuda_device):
    """Captured once and replayed on new inputs, two graphs in turn: each has workspaces of its own."""
    from ltx_kernels.blockwise import ops
    M, H, N = 900, 1152, 512
    w, s = _weight(N, H, cuda_device, 61)
    nw = (1 + 0.1 * torch.randn(H, generator=gen(62))).to(cuda_device)

    def chain(x, r, g):
        q, sc, h, rstd = ops.rms_norm_quantize(x, nw, r)
        y = ops.gemm_residual(q, sc, w, s, residual=g, activation="gelu_tanh")
        yq, ys, zq, zs = ops.act_quantize_save(y)
        dz, dq, ds, db = ops.act_backward(g, zq, zs, quantize=True, dbias=True)
        dw = ops.wgrad_1x128(dz, q, sc)
        dl = ops.wgrad_1x128(dz[:, :32], q, sc)
        dx, dnw = ops.rms_norm_backward(r, h, rstd, nw, x)
        return [y, dz, dq.float(), ds, db, dw, dl, dx, dnw]

    sets = [(tokens(M, H, 63 + i).to(cuda_device), tokens(M, H, 73 + i).to(cuda_device),
             grads(M, N, 83 + i).to(cuda_device)) for i in range(4)]
    graphs = []
    for i in range(2):
        static = [t.clone() for t in sets[i]]
        chain(*static)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = chain(*static)
        graphs.append((graph, static, out))
    for rep in range(2):
        for i, (graph, static, out) in enumerate(graphs):
            for t, new in zip(static, sets[2 * rep + i]):
                t.copy_(new)
        for graph, _, _ in graphs:  # back to back: neither may use the other's scratch
            graph.replay()
        torch.cuda.synchronize()
        for i, (_, _, out) in enumerate(graphs):
            for a, b in zip(out, chain(*sets[2 * rep + i])):
                assert torch.equal(a, b)


def test_offsets_past_32_bits(cuda_device):
    """Element offsets beyond 2^31: the last rows of long inputs match a short call on them."""
    from ltx_kernels.blockwise import ops
    M, H = 262200, 8192  # 2.15e9 values
    x = torch.empty(M, H, dtype=torch.bfloat16, device=cuda_device)
    tail = tokens(64, H, 71).to(cuda_device)
    x[:64] = tail
    x[64:-64] = 0.5
    x[-64:] = tail
    q, s, h, rstd = ops.rms_norm_quantize(x)
    q0, s0, _, rstd0 = ops.rms_norm_quantize(tail)
    assert torch.equal(q[-64:].view(torch.uint8), q0.view(torch.uint8)) and torch.equal(s[-64:], s0)
    assert torch.equal(q[:64].view(torch.uint8), q0.view(torch.uint8)) and torch.equal(rstd[-64:], rstd0)
    yq, ys, zq, zs = ops.act_quantize_save(x)
    y0 = ops.act_quantize_save(tail)
    for a, b in ((yq, y0[0]), (zq, y0[2])):
        assert torch.equal(a[-64:].view(torch.uint8), b.view(torch.uint8))
    assert torch.equal(ys[-64:], y0[1]) and torch.equal(zs[-64:], y0[3])
    del yq, ys, q, s
    dz = ops.act_backward(x, zq, zs)[0]
    assert torch.equal(dz[-64:], ops.act_backward(tail, y0[2], y0[3])[0])
    del dz
    dx = ops.rms_norm_backward(x, x, rstd)[0]
    assert torch.equal(dx[-64:], ops.rms_norm_backward(tail, tail, rstd0)[0])
    del dx
    # the weight gradient reads codes past 2^31 as well: one token at the end carries all of g
    g = torch.zeros(M, 16, dtype=torch.bfloat16, device=cuda_device)
    g[-1] = 1.0
    dw = ops.wgrad_1x128(g, zq, zs)
    assert torch.equal(dw, ops.wgrad_1x128(g[-64:], y0[2], y0[3]))
