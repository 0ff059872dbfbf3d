"""Training through the blockwise-FP8 linears with 8-bit activation checkpoints.

The forward GEMMs read their input as e4m3 codes with 1x128 scales; those codes are what
the backward pass keeps -- one byte a value (plus 1/32 of scales) in place of a bf16 copy --
for the weight gradients (``ops.wgrad_1x128``) and for the activation's gradient
(``ops.act_backward``).  Input gradients are blockwise-FP8 GEMMs on the transposed weight,
with the incoming gradient quantised 1x128 (``dX = dY W``).  All-zero tokens (padding)
quantise to zeros here.

* :func:`fp8_linear_train` -- one linear: frozen e4m3 weight, with or without LoRA factors to
  train, or a bf16 / fp32 master weight that is quantised per call and gets a gradient;
* :func:`pre_norm_feed_forward` -- a whole un-gated pre-norm block, ``h + W2 act(W1 norm(h))``
  with ``h = x + residual``, whose intermediate tensors are kept in 8 bits only;
* :class:`BlockwiseFP8PreNormFeedForward` -- that block as a module;
* :func:`frozen_linear`, :func:`frozen_feed_forward` -- what ``BlockwiseFP8Linear`` and
  ``BlockwiseFP8FeedForward`` run where their input or a bias requires a gradient.

No reference counterpart: the reference's blockwise linear is forward-only
(ltx-kernels/src/ltx_kernels/blockwise/linear.py:82-104).
"""
from __future__ import annotations

from typing import Optional, Tuple, Union

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from .. import _lib as L
from . import ops
from .functional import quant_mode_code
from .linear import BlockwiseFP8Linear

Weight = Union[torch.Tensor, Tuple[torch.Tensor, torch.Tensor]]


def _fp8_weight(weight: Weight, name: str) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor]]:
    """(codes, scales, master): a frozen ``(e4m3, scales)`` pair, or a float master weight
    quantised 128x128 now."""
    if isinstance(weight, (tuple, list)):
        q, s = weight
        if q.dtype != torch.float8_e4m3fn:
            raise RuntimeError(f"{name}: a frozen weight must be (float8_e4m3fn, scales), got {q.dtype}")
        return q, s, None
    if weight.dtype not in (torch.float32, torch.bfloat16):
        raise RuntimeError(f"{name}: a master weight must be fp32 or bf16, got {weight.dtype}")
    q, s = ops.quantize_weight_128x128(weight.detach(), finite=True)
    return q, s, weight


def _rows(t: torch.Tensor, width: int) -> torch.Tensor:
    """[..., width] as [M, width] with 16-byte aligned rows (a copy only where it has none: an
    expanded or oddly sliced tensor)."""
    t = t.reshape(-1, width)
    if t.shape[0] and (t.stride(1) != 1 or t.data_ptr() % 16
                       or (t.shape[0] > 1 and (t.stride(0) < width or t.stride(0) % 8))):
        t = t.clone(memory_format=torch.contiguous_format)
    return t


def _empty_output(x: torch.Tensor, N: int) -> Tuple[torch.Tensor, torch.Tensor]:
    """A bf16 result [..., N] for x [..., K], and its rows [M, N].  The operators write the rows and the
    Function returns the result: a view of what they return could not be modified in place."""
    out = torch.empty((*x.shape[:-1], N), dtype=torch.bfloat16, device=x.device)
    return out, out.view(-1, N)


def _check_capture(name: str, *leaves: Optional[torch.Tensor]) -> None:
    """Refuse, while a CUDA graph is captured with gradients enabled, leaves whose gradient node was
    made on the default stream and is still alive (an earlier eager result that has not been
    released): autograd would run that node on the default stream, which a capture forbids, and the
    error ends the process from its backward thread."""
    if torch.is_grad_enabled() and torch.cuda.is_current_stream_capturing():
        L.binding().check_capture(name, [t for t in leaves if t is not None and t.is_leaf and t.requires_grad])


def _column_sum(g: torch.Tensor) -> torch.Tensor:
    return g.sum(0, dtype=torch.float32)


def _dgrad(g: torch.Tensor, w_q: torch.Tensor, w_s: torch.Tensor, **lora) -> torch.Tensor:
    """dX = dY W in FP8: the gradient quantised 1x128, the weight transposed."""
    gq, gs = ops.quantize_1x128(g, L.QUANT_FINITE)
    wt, wts = ops.transpose_weight_128x128(w_q, w_s)
    return ops.gemm(gq, gs, wt, wts, **lora)


def _bf16_grad(g: torch.Tensor, width: int) -> torch.Tensor:
    return _rows(g.to(torch.bfloat16), width)


class _LinearTrain(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, master, bias, lora_a, lora_b, residual, w_q, w_s, alpha, quant_mode, plain):
        K, N = x.shape[-1], w_q.shape[0]
        x2 = _rows(x, K)
        q, s = ops.quantize_1x128(x2, quant_mode)
        ax = a = b = None
        y, rows = _empty_output(x, N)
        if lora_a is not None:
            a, b = lora_a.to(torch.bfloat16), lora_b.to(torch.bfloat16)
            ax = ops.lora_a(x2, a)
            ops.gemm(q, s, w_q, w_s, bias, out=rows, lora_ax=ax, lora_b=b, lora_alpha=alpha)
            if residual is not None:
                y += residual
        elif plain:
            ops.gemm(q, s, w_q, w_s, bias, out=rows)
        else:
            ops.gemm_residual(q, s, w_q, w_s, bias, out=rows,
                              residual=None if residual is None else residual.reshape(-1, N))
        # Only what the wanted gradients read: the codes for the weight or A, x A^T for B.
        need_x, need_w, _, need_a, need_b = ctx.needs_input_grad[:5]
        if not (need_w or need_a):
            q = s = None
        ctx.save_for_backward(q, s, w_q, w_s, ax if need_b else None, a, b)
        ctx.alpha = alpha
        ctx.x_meta = (x.shape, x.dtype)
        ctx.master_dtype = None if master is None else master.dtype
        ctx.lora_dtypes = (None, None) if lora_a is None else (lora_a.dtype, lora_b.dtype)
        return y

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        q, s, w_q, w_s, ax, a, b = ctx.saved_tensors
        need_x, need_w, need_bias, need_a, need_b, need_r = ctx.needs_input_grad[:6]
        g = _bf16_grad(dy, w_q.shape[0])
        dx = dw = dbias = da = db = dr = None
        u = None
        if a is not None and (need_x or need_a):
            u = ops.lora_a(g, b.t().contiguous())  # dY B, [M, r]
        if need_x:
            if a is not None:
                dx = _dgrad(g, w_q, w_s, lora_ax=u, lora_b=a.t().contiguous(), lora_alpha=ctx.alpha)
            else:
                dx = _dgrad(g, w_q, w_s)
            dx = dx.view(ctx.x_meta[0])
        if need_w:
            dw = ops.wgrad_1x128(g, q, s).to(ctx.master_dtype)
        if need_bias:
            dbias = _column_sum(g)
        if need_a:
            da = ops.wgrad_1x128(u, q, s, alpha=ctx.alpha).to(ctx.lora_dtypes[0])
        if need_b:
            db = ops.wgrad_bf16(ax, g, alpha=ctx.alpha, transposed=True).to(ctx.lora_dtypes[1])
        if need_r:
            # The tensor itself: a view of it would be a new object over the same memory, which autograd
            # takes over as a leaf's .grad although the caller, or another leaf, still holds dy.
            dr = dy
        return dx, dw, dbias, da, db, dr, None, None, None, None, None


def _check_x(x: torch.Tensor, K: int, name: str) -> None:
    if x.dtype != torch.bfloat16 or x.dim() < 1 or x.shape[-1] != K:
        raise RuntimeError(f"{name}: expected bf16 [..., {K}], got {x.dtype} {tuple(x.shape)}")
    if not x.is_cuda:
        raise RuntimeError(f"{name}: ltx-2_b200 kernels need CUDA (sm_100) tensors, got {x.device}")


def _check_bias(bias: Optional[torch.Tensor], N: int, name: str) -> None:
    if bias is not None and (bias.dtype != torch.float32 or tuple(bias.shape) != (N,)):
        raise RuntimeError(f"{name}: bias must be fp32 [{N}], got {bias.dtype} {tuple(bias.shape)}")


def fp8_linear_train(x: torch.Tensor, weight: Weight, bias: Optional[torch.Tensor] = None, *,
                     lora: Optional[Tuple[torch.Tensor, torch.Tensor, float]] = None,
                     residual: Optional[torch.Tensor] = None, quant_mode: int = L.QUANT_FINITE) -> torch.Tensor:
    """Differentiable blockwise-FP8 linear, ``x W^T + bias [+ alpha (x A^T) B^T] [+ residual]``.

    ``x`` bf16 ``[..., K]``.  ``weight`` is a frozen ``(e4m3 [N, K], fp32 scales [N/128, K/128])``
    pair or a bf16 / fp32 master weight ``[N, K]``, which is quantised for this call and
    receives the gradient ``dY^T x~``.  ``bias`` fp32 ``[N]``.  ``lora = (A [r, K], B [N, r],
    alpha)``, r a multiple of 16 up to 256, used in bf16.  ``residual`` bf16 of the output's shape:
    added in the GEMM's epilogue before the only rounding; with ``lora`` by an addition of its own to
    the linear's bf16 result, a second rounding.

    What the backward pass keeps of ``x`` is its e4m3 codes and scales (``x~``, where the weight
    or A wants a gradient), and with LoRA ``x A^T``; the weight is not copied.  The gradient of
    ``x`` is a blockwise-FP8 GEMM of the quantised output gradient.  Gradients of a master weight and
    of the LoRA factors are rounded to bf16, from fp32 sums over ``x~`` in bf16 (code * scale rounded
    once), also where the parameter is fp32.  ``quant_mode``: of ``x``, as ``ops.quantize_1x128``
    takes it."""
    name = "fp8_linear_train"
    shape = weight[0].shape if isinstance(weight, (tuple, list)) else weight.shape
    if len(shape) != 2:
        raise RuntimeError(f"{name}: expected a 2-D weight, got shape {tuple(shape)}")
    N, K = shape
    _check_x(x, K, name)
    _check_bias(bias, N, name)
    la = lb = None
    alpha = 1.0
    if lora is not None:
        la, lb, alpha = lora
        r = la.shape[0]
        if tuple(la.shape) != (r, K) or tuple(lb.shape) != (N, r):
            raise RuntimeError(f"{name}: LoRA factors must be A [r, {K}] and B [{N}, r]")
    if residual is not None:
        _check_x(residual, N, f"{name}: residual")
        if residual.shape[:-1] != x.shape[:-1]:
            raise RuntimeError(f"{name}: residual has shape {tuple(residual.shape)}, x {tuple(x.shape)}")
    _check_capture(name, x, None if isinstance(weight, (tuple, list)) else weight, bias, la, lb, residual)
    w_q, w_s, master = _fp8_weight(weight, name)
    return _LinearTrain.apply(x, master, bias, la, lb, residual, w_q, w_s, float(alpha),
                              quant_mode, False)


def frozen_linear(x: torch.Tensor, weight: torch.Tensor, weight_scale: torch.Tensor,
                  bias: Optional[torch.Tensor]) -> torch.Tensor:
    """The differentiable forward of :class:`BlockwiseFP8Linear`: its inference GEMM and quantiser,
    so its output bits (but zeros for an all-zero 1x128 group of x), and gradients of x and the bias."""
    _check_x(x, weight.shape[1], "BlockwiseFP8Linear")
    _check_capture("BlockwiseFP8Linear", x, bias)
    return _LinearTrain.apply(x, None, bias, None, None, None, weight, weight_scale, 1.0,
                              quant_mode_code() | L.QUANT_ZEROS, True)


class _FrozenFeedForward(torch.autograd.Function):
    """The differentiable forward of BlockwiseFP8FeedForward: its quantisers and GEMMs, and 8-bit
    codes of the hidden state for the activation's gradient."""

    @staticmethod
    def forward(ctx, x, b1, b2, w1, s1, w2, s2, quant_mode):
        q, s = ops.quantize_1x128(_rows(x, x.shape[-1]), quant_mode)
        z = ops.gemm(q, s, w1, s1, b1)
        yq, ys = ops.gelu_tanh_quantize_1x128(z, quant_mode)
        out, rows = _empty_output(x, w2.shape[0])
        ops.gemm(yq, ys, w2, s2, b2, out=rows)
        need_x, need_b1, _ = ctx.needs_input_grad[:3]
        zq, zs = ops.quantize_1x128(z, L.QUANT_FINITE) if need_x or need_b1 else (None, None)
        ctx.save_for_backward(zq, zs, w1, s1, w2, s2)
        ctx.shape = x.shape
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        zq, zs, w1, s1, w2, s2 = ctx.saved_tensors
        need_x, need_b1, need_b2 = ctx.needs_input_grad[:3]
        g = _bf16_grad(dout, w2.shape[0])
        dx = db1 = None
        if need_x or need_b1:
            _, dzq, dzs, db1 = ops.act_backward(_dgrad(g, w2, s2), zq, zs, "gelu_tanh", quantize=need_x, dbias=need_b1)
            if need_x:
                w1t, s1t = ops.transpose_weight_128x128(w1, s1)
                dx = ops.gemm(dzq, dzs, w1t, s1t).view(ctx.shape)
        return dx, db1, _column_sum(g) if need_b2 else None, None, None, None, None, None


def frozen_feed_forward(x: torch.Tensor, up: BlockwiseFP8Linear, down: BlockwiseFP8Linear) -> torch.Tensor:
    """The differentiable forward of :class:`BlockwiseFP8FeedForward`: the same output bits (but zeros
    for an all-zero 1x128 group of x or of the hidden state), and gradients of x and the biases."""
    _check_x(x, up.weight.shape[1], "BlockwiseFP8FeedForward")
    _check_capture("BlockwiseFP8FeedForward", x, up.bias, down.bias)
    return _FrozenFeedForward.apply(x, up.bias, down.bias, up.weight, up.weight_scale, down.weight, down.weight_scale,
                                    quant_mode_code() | L.QUANT_ZEROS)


class _PreNormFeedForward(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, norm_weight, m1, b1, m2, b2, w1, s1, w2, s2, activation, eps, train):
        K = x.shape[-1]
        x2 = x.reshape(-1, K)
        r2 = None if residual is None else residual.reshape(-1, K)
        nq, ns, h, rstd = ops.rms_norm_quantize(x2, norm_weight, r2, eps=eps)
        z = ops.gemm(nq, ns, w1, s1, b1)
        # Only what the wanted gradients read: y's codes for W2, z's for all that lies below the
        # activation, the normalised input's for W1, h and rstd for the norm and its inputs.
        need_x, need_r, need_nw, need_w1, need_b1, need_w2, _ = ctx.needs_input_grad[:7] if train else (False,) * 7
        below = need_x or need_r or need_nw
        yq, ys, zq, zs = ops.act_quantize_save(z, activation, save=below or need_w1 or need_b1)
        out, rows = _empty_output(x, K)
        ops.gemm_residual(yq, ys, w2, s2, b2, residual=h, out=rows)
        if train:
            keep = lambda want, *ts: ts if want else (None,) * len(ts)  # noqa: E731
            ctx.save_for_backward(*keep(need_w1, nq, ns), *keep(below, h, rstd), zq, zs, *keep(need_w2, yq, ys),
                                  norm_weight, w1, s1, w2, s2)
        ctx.activation = activation
        ctx.shape = x.shape
        ctx.master_dtypes = tuple(None if m is None else m.dtype for m in (m1, m2))
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dout):
        nq, ns, h, rstd, zq, zs, yq, ys, norm_weight, w1, s1, w2, s2 = ctx.saved_tensors
        need_x, need_r, need_nw, need_w1, need_b1, need_w2, need_b2 = ctx.needs_input_grad[:7]
        g = _bf16_grad(dout, w2.shape[0])
        dx = dnw = dw1 = db1 = dw2 = db2 = None
        if need_w2:
            dw2 = ops.wgrad_1x128(g, yq, ys).to(ctx.master_dtypes[1])
        if need_b2:
            db2 = _column_sum(g)
        below = need_x or need_r or need_nw
        if below or need_w1 or need_b1:
            dy = _dgrad(g, w2, s2)
            dz, dzq, dzs, db1 = ops.act_backward(dy, zq, zs, ctx.activation, quantize=below, dbias=need_b1)
            if need_w1:
                dw1 = ops.wgrad_1x128(dz, nq, ns).to(ctx.master_dtypes[0])
            if below:
                w1t, s1t = ops.transpose_weight_128x128(w1, s1)
                dn = ops.gemm(dzq, dzs, w1t, s1t)
                dx, dnw = ops.rms_norm_backward(dn, h, rstd, norm_weight, g)
                dx = dx.view(ctx.shape)
        return (dx if need_x else None, dx if need_r else None, dnw if need_nw else None, dw1, db1, dw2, db2,
                None, None, None, None, None, None, None)


def pre_norm_feed_forward(x: torch.Tensor, w1: Weight, w2: Weight, *, residual: Optional[torch.Tensor] = None,
                          norm_weight: Optional[torch.Tensor] = None, b1: Optional[torch.Tensor] = None,
                          b2: Optional[torch.Tensor] = None, activation: str = "gelu_tanh",
                          eps: float = 1e-6) -> torch.Tensor:
    """An un-gated pre-norm feed-forward block: ``h + W2 act(W1 norm(h) + b1) + b2`` with
    ``h = bf16(x + residual)`` and ``norm(h) = h / sqrt(mean(h^2) + eps) * norm_weight``.

    ``x``, ``residual`` bf16 ``[..., d]``; ``w1`` [inner, d] and ``w2`` [d, inner] each a frozen
    ``(e4m3, scales)`` pair or a bf16 / fp32 master weight that gets a gradient; ``norm_weight``
    fp32 or bf16 ``[d]``; ``b1``, ``b2`` fp32; ``activation`` ``"gelu_tanh"`` or ``"silu"``.
    Differentiable in x, residual, norm_weight, master weights (whose gradients are rounded to bf16, as
    :func:`fp8_linear_train`'s) and biases.  The backward pass
    keeps h in bf16, the activation's input in 8 bits and, for the gradients of w1 and w2, the
    normalised input and the activation's output in 8 bits; without gradients nothing is kept
    and the activation's input is not quantised."""
    name = "pre_norm_feed_forward"
    sh1, sh2 = (w[0].shape if isinstance(w, (tuple, list)) else w.shape for w in (w1, w2))
    if len(sh1) != 2 or tuple(sh2) != (sh1[1], sh1[0]):
        raise RuntimeError(f"{name}: w1 [inner, d] and w2 [d, inner] expected, got {tuple(sh1)} and {tuple(sh2)}")
    inner, d = sh1
    _check_x(x, d, name)
    if residual is not None:
        _check_x(residual, d, f"{name}: residual")
        if residual.shape != x.shape:
            raise RuntimeError(f"{name}: residual has shape {tuple(residual.shape)}, x {tuple(x.shape)}")
    _check_bias(b1, inner, f"{name}: b1")
    _check_bias(b2, d, f"{name}: b2")
    _check_capture(name, x, residual, norm_weight, b1, b2,
                   *(w for w in (w1, w2) if not isinstance(w, (tuple, list))))
    q1, s1, m1 = _fp8_weight(w1, f"{name}: w1")
    q2, s2, m2 = _fp8_weight(w2, f"{name}: w2")
    # What only the backward pass reads is not written when no gradient is wanted.
    train = torch.is_grad_enabled() and any(t is not None and t.requires_grad
                                            for t in (x, residual, norm_weight, m1, b1, m2, b2))
    return _PreNormFeedForward.apply(x, residual, norm_weight, m1, b1, m2, b2, q1, s1, q2, s2, activation, float(eps),
                                     train)


class BlockwiseFP8PreNormFeedForward(nn.Module):
    """:func:`pre_norm_feed_forward` over frozen blockwise-FP8 linears: the un-gated pre-norm
    feed-forward block (``norm`` -> ``proj_in`` -> activation -> ``proj_out`` -> + residual),
    in four to six launches for inference.  The norm's gain is a trainable fp32 parameter; the linears'
    parameters keep :class:`BlockwiseFP8Linear`'s names, layout and ``requires_grad=False``
    (their fp32 biases can be made trainable)."""

    def __init__(self, dim: int, mult: int = 4, bias: bool = True, activation: str = "gelu_tanh", eps: float = 1e-6,
                 device=None):
        super().__init__()
        inner = int(dim * mult)
        self.norm_weight = nn.Parameter(torch.ones(dim, device=device, dtype=torch.float32))
        self.proj_in = BlockwiseFP8Linear(dim, inner, bias=bias, device=device)
        self.proj_out = BlockwiseFP8Linear(inner, dim, bias=bias, device=device)
        self.activation = activation
        self.eps = eps

    @classmethod
    def from_linears(cls, up: BlockwiseFP8Linear, down: BlockwiseFP8Linear,
                     norm_weight: Optional[torch.Tensor] = None, activation: str = "gelu_tanh",
                     eps: float = 1e-6) -> "BlockwiseFP8PreNormFeedForward":
        ff = cls.__new__(cls)
        nn.Module.__init__(ff)
        if norm_weight is None:
            norm_weight = torch.ones(up.in_features, device=up.weight.device, dtype=torch.float32)
        ff.norm_weight = norm_weight if isinstance(norm_weight, nn.Parameter) else nn.Parameter(norm_weight)
        ff.proj_in, ff.proj_out = up, down
        ff.activation, ff.eps = activation, eps
        return ff

    def forward(self, x: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
        up, down = self.proj_in, self.proj_out
        return pre_norm_feed_forward(x, (up.weight, up.weight_scale), (down.weight, down.weight_scale),
                                     residual=residual, norm_weight=self.norm_weight, b1=up.bias, b2=down.bias,
                                     activation=self.activation, eps=self.eps)
