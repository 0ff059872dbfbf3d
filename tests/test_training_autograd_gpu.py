"""How the training functions stand in an autograd graph: gradients with storage of their own,
outputs that can be modified in place, layers above and below, captures."""
from __future__ import annotations

import pytest
import torch

from residual_inputs import act64, dequant_weight64, gen, grads, quant_weight, tokens

pytestmark = pytest.mark.gpu

# e4m3's rounding in the root mean square, at worst uniformly spread over half a step
E4M3_RMS = 2.0 ** -4 / 3 ** 0.5


def _rel(a, b):
    a, b = a.detach().double(), b.detach().double()
    return ((a - b).norm() / b.norm()).item()


def _weight(N, K, dev, seed):
    q, s = quant_weight(torch.randn(N, K, generator=gen(seed)) / K ** 0.5)
    return q.to(dev), s.to(dev)


def _leaf(t, dev):
    return t.to(dev).requires_grad_()


def _bf16(*shape, seed, scale=1.0):
    return (scale * torch.randn(*shape, generator=gen(seed))).to(torch.bfloat16)


# ----------------------------------------------------------------------------- storage
@pytest.mark.parametrize("lead", [(24,), (2, 12)])
@pytest.mark.parametrize("lora", [False, True])
def test_residual_gradients_have_their_own_storage(cuda_device, lead, lora):
    """Two linears, each with a residual of its own, summed; three steps accumulate into the
    leaves: each gradient is three times one step's, and the caller's gradient is untouched."""
    from ltx_kernels.blockwise import fp8_linear_train
    K, N = 128, 256
    w = _weight(N, K, cuda_device, 1)
    ab = (_bf16(16, K, seed=2).to(cuda_device), _bf16(N, 16, seed=3).to(cuda_device), 0.5) if lora else None
    x = tokens(24, K, 4).view(*lead, K).to(cuda_device)
    r1, r2 = (_leaf(tokens(24, N, s).view(*lead, N), cuda_device) for s in (5, 6))
    dy = (grads(24, N, 7).view(*lead, N) * 1e3).to(cuda_device)
    kept = dy.clone()
    for _ in range(3):
        y = fp8_linear_train(x, w, lora=ab, residual=r1) + fp8_linear_train(x, w, lora=ab, residual=r2)
        y.backward(dy)
    assert torch.equal(dy, kept)
    want = kept + kept + kept  # bf16, as the accumulation rounds
    assert torch.equal(r1.grad, want) and torch.equal(r2.grad, want)
    assert r1.grad.data_ptr() != r2.grad.data_ptr()
    # the output's gradient handed in directly
    r1.grad = r2.grad = None
    for _ in range(2):
        fp8_linear_train(x, w, lora=ab, residual=r1).backward(dy)
    assert torch.equal(dy, kept) and torch.equal(r1.grad, kept + kept) and r1.grad.data_ptr() != dy.data_ptr()


def test_block_gradients_have_their_own_storage(cuda_device):
    """x and the residual of a block share the values of their gradient, not its memory."""
    from ltx_kernels.blockwise import pre_norm_feed_forward
    d, inner = 128, 256
    w1, w2 = _weight(inner, d, cuda_device, 11), _weight(d, inner, cuda_device, 12)
    x, r = (_leaf(tokens(24, d, s).view(2, 12, d), cuda_device) for s in (13, 14))
    dy = (grads(24, d, 15).view(2, 12, d) * 1e3).to(cuda_device)
    kept = dy.clone()
    grad = torch.autograd.grad(pre_norm_feed_forward(x, w1, w2, residual=r), x, dy)[0]
    for _ in range(3):
        pre_norm_feed_forward(x, w1, w2, residual=r).backward(dy)
    assert torch.equal(dy, kept) and x.grad.data_ptr() != r.grad.data_ptr()
    want = grad + grad + grad
    assert torch.equal(x.grad, want) and torch.equal(r.grad, want)


# ----------------------------------------------------------------------------- in place
@pytest.mark.parametrize("lead", [(24,), (2, 12)])
@pytest.mark.parametrize("which", ["linear", "lora", "block"])
def test_outputs_can_be_modified_in_place(cuda_device, lead, which):
    """``y += skip`` and an in-place activation on the output: the same gradients as out of place."""
    from ltx_kernels.blockwise import fp8_linear_train, pre_norm_feed_forward
    K = 128
    w1, w2 = _weight(256, K, cuda_device, 21), _weight(K, 256, cuda_device, 22)
    a, b = _leaf(_bf16(16, K, seed=23), cuda_device), _leaf(_bf16(256, 16, seed=24), cuda_device)
    x = _leaf(tokens(24, K, 25).view(*lead, K), cuda_device)
    call = {"linear": lambda: fp8_linear_train(x, w1), "lora": lambda: fp8_linear_train(x, w1, lora=(a, b, 0.5)),
            "block": lambda: pre_norm_feed_forward(x, w1, w2)}[which]
    skip = _leaf(tokens(24, call().shape[-1], 26).view(*lead, -1), cuda_device)
    dy = (grads(24, skip.shape[-1], 27).view(*lead, -1) * 1e3).to(cuda_device)
    y = call()
    y += skip
    y.relu_()
    got = torch.autograd.grad(y, (x, skip), dy)
    z = torch.relu(call() + skip)
    want = torch.autograd.grad(z, (x, skip), dy)
    assert torch.equal(y, z) and y.shape == (*lead, skip.shape[-1])
    for p, q in zip(got, want):
        assert torch.equal(p, q)


# ----------------------------------------------------------------------------- LoRA and residual
@pytest.mark.parametrize("lead", [(130,), (2, 65)])
def test_lora_with_residual(cuda_device, lead):
    """The linear with LoRA is rounded to bf16, then the residual added and rounded again; the
    gradients are the linear's, and the output's own gradient for the residual."""
    from ltx_kernels.blockwise import fp8_linear_train
    M, K, N, r = 130, 256, 384, 32
    w, s = _weight(N, K, cuda_device, 31)
    x, res = _leaf(tokens(M, K, 32).view(*lead, K), cuda_device), _leaf(tokens(M, N, 33).view(*lead, N), cuda_device)
    a, b = _leaf(_bf16(r, K, seed=34, scale=K ** -0.5), cuda_device), _leaf(_bf16(N, r, seed=35, scale=r ** -0.5),
                                                                              cuda_device)
    bias = _leaf(0.1 * torch.randn(N, generator=gen(36)), cuda_device)
    dy = (grads(M, N, 37).view(*lead, N) * 1e3).to(cuda_device)
    y = fp8_linear_train(x, (w, s), bias, lora=(a, b, 0.5), residual=res)
    got = torch.autograd.grad(y, (x, a, b, bias, res), dy)
    y0 = fp8_linear_train(x, (w, s), bias, lora=(a, b, 0.5))
    assert torch.equal(y, y0 + res)
    for p, q in zip(got, (*torch.autograd.grad(y0, (x, a, b, bias), dy), dy)):
        assert torch.equal(p, q) and p.shape == q.shape
    p = [t.detach().double().requires_grad_() for t in (x, a, b, bias, res)]
    y64 = p[0] @ dequant_weight64(w, s).t() + 0.5 * (p[0] @ p[1].t()) @ p[2].t() + p[3] + p[4]
    ref = torch.autograd.grad(y64, p, dy.double())
    # the output: x's 8-bit rounding, x A^T's and the two of the sum in bf16
    assert _rel(y, y64) <= E4M3_RMS + 3 * 2 ** -8
    for name, n, g, t in zip(("x", "A", "B", "bias", "residual"), (1, 1, 0, 0, 0), got, ref):
        assert _rel(g, t) <= n * E4M3_RMS + 3 * 2 ** -8, (name, _rel(g, t))


# ----------------------------------------------------------------------------- captures
def test_inference_capture_beside_a_living_eager_result(cuda_device):
    """Without gradients nothing of a capture reaches a leaf's gradient node: evaluating a block in
    a CUDA graph while a training step's loss is alive."""
    from ltx_kernels.blockwise import fp8_linear_train, pre_norm_feed_forward
    w1, w2 = _weight(256, 128, cuda_device, 41), _weight(128, 256, cuda_device, 42)
    nw = _leaf(torch.ones(128), cuda_device)
    m = _leaf(torch.randn(128, 128, generator=gen(43)), cuda_device)
    x = tokens(16, 128, 44).to(cuda_device)
    y = fp8_linear_train(pre_norm_feed_forward(x, w1, w2, norm_weight=nw), m)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    refused = None
    with torch.no_grad(), torch.cuda.graph(graph):
        try:
            z = fp8_linear_train(pre_norm_feed_forward(x, w1, w2, norm_weight=nw), m)
        except RuntimeError as e:
            refused = e
    assert refused is None, refused
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(z, y) and not z.requires_grad
    for g in torch.autograd.grad(y, (nw, m), torch.ones_like(y)):
        assert torch.isfinite(g).all()


# ----------------------------------------------------------------------------- frozen linear
def _linear(N, K, dev, seed, bias=True):
    from ltx_kernels.blockwise import BlockwiseFP8Linear
    layer = BlockwiseFP8Linear(K, N, bias=bias, device=dev)
    layer.weight.data, layer.weight_scale.data = _weight(N, K, dev, seed)
    if bias:
        layer.bias.data = 0.1 * torch.randn(N, generator=gen(seed + 1)).to(dev)
    return layer


def _lora(N, K, r, dev, seed):
    from ltx_kernels.blockwise import BlockwiseFP8LoRALinear
    layer = BlockwiseFP8LoRALinear(K, N, r, alpha=0.5, device=dev)
    layer.weight.data, layer.weight_scale.data = _weight(N, K, dev, seed)
    layer.bias.data.zero_()
    layer.lora_A.data = _bf16(r, K, seed=seed + 1, scale=K ** -0.5).to(dev)
    layer.lora_B.data = _bf16(N, r, seed=seed + 2, scale=r ** -0.5).to(dev)
    layer.lora_A.requires_grad_()
    layer.lora_B.requires_grad_()
    return layer


@pytest.mark.parametrize("mode", ["triton", "torch"])
@pytest.mark.parametrize("lead,bias", [((2, 65), True), ((1, 1), False), ((3, 100), True)])
def test_gradient_through_a_frozen_linear(cuda_device, lead, bias, mode):
    """An adapter below a frozen linear gets the gradient that float64 autograd gives; the
    linear's output keeps its bits; its own parameters get none."""
    from ltx_kernels.blockwise import functional
    old = functional.get_quant_mode()
    functional.set_quant_mode(mode)
    try:
        d, k, n, r = 256, 384, 256, 16
        low, top = _lora(k, d, r, cuda_device, 61), _linear(n, k, cuda_device, 64, bias)
        M = lead[0] * lead[1]
        x = tokens(M, d, 66).view(*lead, d).to(cuda_device)
        dy = (grads(M, n, 67).view(*lead, n) * 1e3).to(cuda_device)
        h = low(x)
        y = top(h)
        with torch.no_grad():
            assert torch.equal(y, top(h)) and torch.equal(y, top(low(x)))
        assert y.requires_grad and y.shape == (*lead, n)
        got = torch.autograd.grad(y, (low.lora_A, low.lora_B, h), dy)
        assert top.weight.grad is None
        p = [t.detach().double().requires_grad_() for t in (low.lora_A, low.lora_B)]
        h64 = x.double() @ dequant_weight64(low.weight, low.weight_scale).t() + 0.5 * (x.double() @ p[0].t()) @ p[1].t()
        y64 = h64 @ dequant_weight64(top.weight, top.weight_scale).t()
        ref = torch.autograd.grad(y64, (*p, h64), dy.double())
        # dy's 8-bit rounding for h; x's besides for A; bf16 roundings
        for name, e, g, t in zip(("A", "B", "h"), (2, 1, 1), got, ref):
            assert _rel(g, t) <= e * E4M3_RMS + 4 * 2 ** -8, (name, _rel(g, t))
    finally:
        functional.set_quant_mode(old)


def test_frozen_linear_with_padded_tokens(cuda_device):
    """All-zero tokens count as zeros where gradients flow (NaN without), so that they do not reach
    the gradients of the others; a trainable bias gets its gradient."""
    lin = _linear(256, 128, cuda_device, 81, bias=False)
    x = _leaf(tokens(20, 128, 87, zero_rows=(3, 19)).view(1, 20, 128), cuda_device)
    y = lin(x)
    dy = (grads(20, 256, 88, zero_rows=(3, 19)).view(1, 20, 256) * 1e3).to(cuda_device)
    (g,) = torch.autograd.grad(y, x, dy)
    assert torch.isfinite(y).all() and torch.isfinite(g).all() and (y[0, 3] == 0).all() and (g[0, 3] == 0).all()
    lin = _linear(256, 128, cuda_device, 89)
    lin.bias.requires_grad_()
    y = lin(x.detach()[:, 4:10])
    y.backward(torch.ones_like(y))
    assert torch.equal(lin.bias.grad, torch.full((256,), 6.0, device=cuda_device))


def test_frozen_linear_takes_what_it_took(cuda_device):
    """Quantised inputs, inputs without a gradient and no-grad calls run as before."""
    from ltx_kernels.blockwise.functional import blockwise_quantize_triton
    lin = _linear(256, 128, cuda_device, 91)
    x = tokens(20, 128, 96).view(1, 20, 128).to(cuda_device)
    y = lin(x)
    assert not y.requires_grad
    assert torch.equal(lin(blockwise_quantize_triton(x)), y)
    with torch.no_grad():
        z = lin(x.clone().requires_grad_())
    assert torch.equal(z, y) and not z.requires_grad


# ----------------------------------------------------------------------------- frozen feed-forward
@pytest.mark.parametrize("mode", ["triton", "torch"])
@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("lead,bias", [((2, 65), True), ((1, 1), False), ((400,), True)])
def test_gradient_through_a_frozen_feed_forward(cuda_device, lead, bias, fused, mode):
    from ltx_kernels.blockwise import BlockwiseFP8FeedForward, functional
    old = functional.get_quant_mode()
    functional.set_quant_mode(mode)
    try:
        d, inner, n, r = 256, 512, 384, 16
        low = _lora(d, d, r, cuda_device, 71)
        ff = BlockwiseFP8FeedForward.from_linears(_linear(inner, d, cuda_device, 74, bias),
                                                  _linear(n, inner, cuda_device, 76, bias))
        ff.fused_epilogue = fused
        M = 1
        for i in lead:
            M *= i
        x = tokens(M, d, 78).view(*lead, d).to(cuda_device)
        dy = (grads(M, n, 79).view(*lead, n) * 1e3).to(cuda_device)
        h = low(x)
        y = ff(h)
        with torch.no_grad():
            assert torch.equal(y, ff(h))
        assert y.requires_grad and y.shape == (*lead, n)
        got = torch.autograd.grad(y, (low.lora_A, low.lora_B, h), dy)
        p = [t.detach().double().requires_grad_() for t in (low.lora_A, low.lora_B)]
        h64 = x.double() @ dequant_weight64(low.weight, low.weight_scale).t() + 0.5 * (x.double() @ p[0].t()) @ p[1].t()
        b1, b2 = ((l.bias.double() if bias else 0.0) for l in (ff.proj_in, ff.proj_out))
        z64 = h64 @ dequant_weight64(ff.proj_in.weight, ff.proj_in.weight_scale).t() + b1
        y64 = act64(z64, "gelu_tanh") @ dequant_weight64(ff.proj_out.weight, ff.proj_out.weight_scale).t() + b2
        ref = torch.autograd.grad(y64, (*p, h64), dy.double())
        # h: dy, dz and z's three (its checkpoint and h's codes below it, slope |z act''| <= 1.5 of act');
        # A: x's besides
        for name, e, g, t in zip(("A", "B", "h"), (6, 5, 5), got, ref):
            assert _rel(g, t) <= e * E4M3_RMS + 4 * 2 ** -8, (name, _rel(g, t))
        assert _rel(y, y64) <= 2.5 * E4M3_RMS + 2 ** -8
    finally:
        functional.set_quant_mode(old)


def test_frozen_feed_forward_with_padded_tokens(cuda_device):
    from ltx_kernels.blockwise import BlockwiseFP8FeedForward
    ff = BlockwiseFP8FeedForward.from_linears(_linear(512, 128, cuda_device, 83, bias=False),
                                              _linear(128, 512, cuda_device, 85, bias=False))
    x = _leaf(tokens(20, 128, 87, zero_rows=(3, 19)).view(1, 20, 128), cuda_device)
    y = ff(x)
    dy = (grads(20, 128, 88, zero_rows=(3, 19)).view(1, 20, 128) * 1e3).to(cuda_device)
    (g,) = torch.autograd.grad(y, x, dy)
    assert torch.isfinite(y).all() and torch.isfinite(g).all() and (y[0, 3] == 0).all() and (g[0, 3] == 0).all()
    ff.proj_in.register_parameter("bias", torch.nn.Parameter(torch.zeros(512, device=cuda_device)))
    ff.proj_out.register_parameter("bias", torch.nn.Parameter(torch.zeros(128, device=cuda_device)))
    y = ff(x.detach()[:, 4:10])
    y.backward(torch.ones_like(y))
    assert torch.equal(ff.proj_out.bias.grad, torch.full((128,), 6.0, device=cuda_device))
    assert torch.isfinite(ff.proj_in.bias.grad).all() and (ff.proj_in.bias.grad != 0).any()


def test_frozen_feed_forward_takes_what_it_took(cuda_device):
    from ltx_kernels.blockwise import BlockwiseFP8FeedForward
    from ltx_kernels.blockwise.functional import blockwise_quantize_triton
    ff = BlockwiseFP8FeedForward.from_linears(_linear(512, 128, cuda_device, 92), _linear(128, 512, cuda_device, 94))
    x = tokens(20, 128, 96).view(1, 20, 128).to(cuda_device)
    y = ff(x)
    assert not y.requires_grad
    assert torch.equal(ff(blockwise_quantize_triton(x)), y)
    with torch.no_grad():
        z = ff(x.clone().requires_grad_())
    assert torch.equal(z, y) and not z.requires_grad
    empty = ff(x[:, :0].clone().requires_grad_())
    assert empty.shape == (1, 0, 128)
    assert torch.autograd.grad(empty.sum(), empty, allow_unused=True)[0] is not None
def test_gelu_quantiser_without_nan(cuda_device):
    """QUANT_ZEROS in the GELU quantiser: the same bytes but for groups without a finite scale."""
    from ltx_kernels import _lib as L
    from ltx_kernels.blockwise import ops
    x = tokens(67, 384, 107).to(cuda_device)
    x[3], x[5, 128:256], x[7, :128], x[9, 0] = 0, -40, -1e-37, float("nan")
    lost = torch.zeros(67, 3, dtype=torch.bool, device=cuda_device)
    lost[3], lost[5, 1], lost[7, 0] = True, True, True
    for mode in (L.QUANT_TORCH, L.QUANT_TRITON):
        (q0, s0), (q1, s1) = (ops.gelu_tanh_quantize_1x128(x, m) for m in (mode, mode | L.QUANT_ZEROS))
        a, b = q0.view(torch.uint8).view(67, 3, 128), q1.view(torch.uint8).view(67, 3, 128)
        assert torch.equal(a[~lost], b[~lost]) and (b[lost] & 0x7F == 0).all()
        assert torch.equal(s0[~lost].nan_to_num(7.0), s1[~lost].nan_to_num(7.0)) and (s1[lost] == 0).all()
    with pytest.raises(RuntimeError, match="unknown mode"):
        ops.gelu_tanh_quantize_1x128(x, L.QUANT_FINITE)


def test_frozen_layers_in_a_cuda_graph(cuda_device):
    """An adapter's step through frozen layers, captured after a warm-up on a side stream and
    replayed on new inputs."""
    from ltx_kernels.blockwise import BlockwiseFP8FeedForward
    low, lin = _lora(256, 256, 16, cuda_device, 121), _linear(256, 256, cuda_device, 124)
    ff = BlockwiseFP8FeedForward.from_linears(_linear(512, 256, cuda_device, 126), _linear(256, 512, cuda_device, 128))
    x = tokens(64, 256, 130).view(2, 32, 256).to(cuda_device)
    dy = (grads(64, 256, 131) * 1e3).view(2, 32, 256).to(cuda_device)

    def step():
        return torch.autograd.grad(ff(lin(low(x))), (low.lora_A, low.lora_B), dy)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    x.copy_(tokens(64, 256, 132).view(2, 32, 256))
    graph.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, step()):
        assert torch.equal(a, b) and torch.isfinite(a).all()
