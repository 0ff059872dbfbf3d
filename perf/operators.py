"""Cases of the training-side and residual-path operators: what is measured, in plain torch and through the kernels.

Four operators around the blockwise-FP8 linear, sizes from the DiT's 4096-wide video and 2048-wide audio streams;
``op`` of a case names the operator and its direction:

* RMS norm with the residual's addition: ``rms_norm`` (h = bf16(x + residual), the norm with a gain as 1x128 e4m3
  codes and scales) and ``rms_norm_bwd`` (its gradient plus the residual stream's own, and the gain's)
* ``gemm_residual``: bf16(act(A W^T + bias) + residual) on blockwise-FP8 operands
* the activation with its 8-bit checkpoint: ``act_save`` (quantised for the next GEMM, its input kept in 8 bits) and
  ``act_bwd`` (its gradient from that checkpoint, in bf16 and in 8 bits, and the bias gradient)
* ``wgrad``: a weight's (or a LoRA factor's) gradient from the 8-bit checkpoint of the layer's input
"""
import math
import os
import sys

import torch

own = False

_E4M3_MAX = 448.0
_AMAX_MIN = 448.0 * 2.0 ** -126  # an all-zero group keeps a normal scale
_EPS = 1e-6
_SQRT_2_PI = math.sqrt(2.0 / math.pi)
_KAPPA = 0.044715


def listed():
    return [
        # a handful of tokens through one norm: the latency of a call
        {"name": "rms_norm_8x4096", "op": "rms_norm", "m": 8, "h": 4096, "residual": True, "pad": 0},
        # the audio stream's width, an odd number of tokens with padded (all-zero) ones, no residual
        {"name": "rms_norm_1003x2048_pad", "op": "rms_norm", "m": 1003, "h": 2048, "residual": False, "pad": 11},
        # the FFN workload's tokens, video stream
        {"name": "rms_norm_24576x4096", "op": "rms_norm", "m": 24576, "h": 4096, "residual": True, "pad": 0},
        # gradient of the audio stream's norm, odd token count, fp32 gain
        {"name": "rms_norm_bwd_1003x2048", "op": "rms_norm_bwd", "m": 1003, "h": 2048, "residual": False,
         "w32": True, "pad": 11},
        # gradient of the video stream's norm at the FFN workload's tokens
        {"name": "rms_norm_bwd_24576x4096", "op": "rms_norm_bwd", "m": 24576, "h": 4096, "residual": True,
         "w32": False, "pad": 0},
        # a few tokens through the attention output projection and the residual stream
        {"name": "gemm_residual_7x4096x4096", "op": "gemm_residual", "m": 7, "n": 4096, "k": 4096,
         "act": "none", "residual": True},
        # the single-linear workload with an activation and a residual, ragged rows
        {"name": "gemm_residual_silu_6143x4096x4096", "op": "gemm_residual", "m": 6143, "n": 4096, "k": 4096,
         "act": "silu", "residual": True},
        # the FFN's down projection onto the residual stream
        {"name": "gemm_residual_24576x4096x16384", "op": "gemm_residual", "m": 24576, "n": 4096, "k": 16384,
         "act": "none", "residual": True},
        # the FFN's hidden state in training: quantised for the down projection, its input kept in 8 bits
        {"name": "act_save_6144x16384", "op": "act_save", "m": 6144, "n": 16384, "act": "gelu_tanh", "pad": 0},
        # ... and its gradient, ragged
        {"name": "act_bwd_6143x16384", "op": "act_bwd", "m": 6143, "n": 16384, "act": "gelu_tanh", "pad": 9},
        # gradient of a rank-32 LoRA factor over the video stream
        {"name": "wgrad_lora32_6143x32x4096", "op": "wgrad", "m": 6143, "n": 32, "k": 4096, "pad": 9},
        # gradient of a full 4096 x 4096 weight
        {"name": "wgrad_6144x4096x4096", "op": "wgrad", "m": 6144, "n": 4096, "k": 4096, "pad": 0},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _mult(rng, unit, lo, hi):
    return unit * max(lo // unit, min(hi // unit, int(round(_log_int(rng, lo, hi) / unit))))


def draw(rng):
    op = rng.choice(["rms_norm", "rms_norm_bwd", "gemm_residual", "act_save", "act_bwd", "wgrad"])
    m = _log_int(rng, 1, 24576)
    pad = rng.choice([0, 0, max(1, m // 50)]) if m > 1 else 0
    if op == "rms_norm":
        return {"op": op, "m": m, "h": _mult(rng, 128, 128, 8192), "residual": rng.random() < 0.6, "pad": pad}
    if op == "rms_norm_bwd":
        return {"op": op, "m": m, "h": _mult(rng, 128, 128, 8192), "residual": rng.random() < 0.6,
                "w32": rng.random() < 0.5, "pad": pad}
    if op == "act_save":
        return {"op": op, "m": m, "n": _mult(rng, 128, 128, 16384), "act": rng.choice(["gelu_tanh", "silu"]),
                "pad": pad}
    if op == "act_bwd":
        return {"op": op, "m": m, "n": _mult(rng, 128, 128, 16384), "act": rng.choice(["gelu_tanh", "silu"]),
                "pad": pad}
    if op == "gemm_residual":
        return {"op": op, "m": m, "n": _mult(rng, 128, 128, 8192), "k": _mult(rng, 128, 128, 8192),
                "act": rng.choice(["none", "gelu_tanh", "silu"]), "residual": rng.random() < 0.7}
    if rng.random() < 0.5:  # a LoRA factor: rank 16 .. 256
        n = 16 * rng.choice([1, 2, 3, 4, 6, 8, 12, 16])
    else:
        n = _mult(rng, 128, 128, 8192)
    return {"op": op, "m": m, "n": n, "k": _mult(rng, 128, 128, 8192), "pad": pad}


# ----------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return g


def _randn(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _tokens(g, m, h):
    """Residual-stream values: a few channels much larger than the rest, as trained transformers have."""
    chan = torch.exp(0.5 * _randn(g, h))
    return (_randn(g, m, h) * chan).to(torch.bfloat16)


def _grads(g, m, n):
    """Gradients: small, with token scales that spread over a few octaves."""
    return (_randn(g, m, n) * (1e-4 * torch.exp2(_randn(g, m, 1)))).to(torch.bfloat16)


def _pad_rows(t, pad):
    """The last `pad` rows are padding."""
    if pad:
        t[t.shape[0] - pad:] = 0
    return t


def _mn_major(s):
    """(M, KB) scales in the layout the GEMM reads: strides (1, M rounded up to 4)."""
    m, kb = s.shape
    out = torch.empty_strided((m, kb), (1, (m + 3) // 4 * 4), dtype=torch.float32, device=s.device)
    out.copy_(s)
    return out


def _quant_rows(v):
    """1x128 codes and scales of an fp32 matrix."""
    m, k = v.shape
    g = v.view(m, k // 128, 128)
    amax = g.abs().amax(-1, keepdim=True).clamp_min(_AMAX_MIN)
    q = (g * (_E4M3_MAX / amax)).to(torch.float8_e4m3fn)
    return q.view(m, k), (amax / _E4M3_MAX).view(m, k // 128)


def _quant_weight(w):
    """128x128 codes and scales of an fp32 matrix."""
    n, k = w.shape
    b = w.view(n // 128, 128, k // 128, 128)
    amax = b.abs().amax((1, 3), keepdim=True).clamp_min(_AMAX_MIN)
    q = (b * (_E4M3_MAX / amax)).to(torch.float8_e4m3fn)
    return q.view(n, k), (amax / _E4M3_MAX).view(n // 128, k // 128).contiguous()


def prepare(case, seed):
    g = _gen(seed)
    op, m = case["op"], case["m"]
    st = dict(case)
    if op in ("rms_norm", "rms_norm_bwd"):
        h = case["h"]
        st["x"] = _pad_rows(_tokens(g, m, h), case["pad"])
        w = 1.0 + 0.2 * _randn(g, h)
        if op == "rms_norm":
            st["w"] = w.to(torch.bfloat16)
            st["r"] = _pad_rows(_tokens(g, m, h), case["pad"]) if case["residual"] else None
        else:
            st["w"] = w if case["w32"] else w.to(torch.bfloat16)
            st["dy"] = _pad_rows(_grads(g, m, h), case["pad"])
            st["dh"] = _pad_rows(_grads(g, m, h), case["pad"]) if case["residual"] else None
            st["rstd"] = torch.rsqrt(st["x"].float().square().mean(-1) + _EPS)
    elif op == "gemm_residual":
        n, k = case["n"], case["k"]
        st["a"], s = _quant_rows(_tokens(g, m, k).float())
        st["sfa"] = _mn_major(s)
        st["w"], st["sfb"] = _quant_weight(_randn(g, n, k) / math.sqrt(k))
        st["bias"] = 0.1 * _randn(g, n)
        st["r"] = _tokens(g, m, n) if case["residual"] else None
    elif op == "act_save":
        st["z"] = _pad_rows((1.5 * _randn(g, m, case["n"])).to(torch.bfloat16), case["pad"])
    elif op == "act_bwd":
        st["zq"], s = _quant_rows(_pad_rows(1.5 * _randn(g, m, case["n"]), case["pad"]))
        st["zs"] = _mn_major(s)
        st["dy"] = _pad_rows(_grads(g, m, case["n"]), case["pad"])
    else:
        st["xq"], s = _quant_rows(_pad_rows(_tokens(g, m, case["k"]).float(), case["pad"]))
        st["xs"] = _mn_major(s)
        st["g"] = _pad_rows(_grads(g, m, case["n"]), case["pad"])
    return st


# ----------------------------------------------------------------------------- plain forms
def _dequant_rows(q, s):
    m, k = q.shape
    return (q.float().view(m, k // 128, 128) * s.unsqueeze(-1)).view(m, k)


def _dequant_weight(q, s):
    n, k = q.shape
    return (q.float().view(n // 128, 128, k // 128, 128) * s.view(n // 128, 1, k // 128, 1)).view(n, k)


def _act(z, act):
    if act == "gelu_tanh":
        return 0.5 * z * (1.0 + torch.tanh(_SQRT_2_PI * (z + _KAPPA * z * z * z)))
    if act == "silu":
        return z / (1.0 + torch.exp(-z))
    return z


def _act_grad(z, act):
    if act == "gelu_tanh":
        t = torch.tanh(_SQRT_2_PI * (z + _KAPPA * z * z * z))
        return 0.5 * (1.0 + t) + 0.5 * z * (1.0 - t * t) * _SQRT_2_PI * (1.0 + 3.0 * _KAPPA * z * z)
    s = 1.0 / (1.0 + torch.exp(-z))
    return s * (1.0 + z * (1.0 - s))


def _plain(st):
    op = st["op"]
    if op == "rms_norm":
        h = st["x"] if st["r"] is None else (st["x"].float() + st["r"].float()).to(torch.bfloat16)
        v = h.float()
        rstd = torch.rsqrt(v.square().mean(-1) + _EPS)
        q, s = _quant_rows(v * rstd.unsqueeze(-1) * st["w"].float())
        return {"q": q, "scales": s, "h": h, "rstd": rstd}
    if op == "rms_norm_bwd":
        rstd = st["rstd"].unsqueeze(-1)
        xhat = st["x"].float() * rstd
        dy = st["dy"].float()
        g = dy * st["w"].float()
        dx = rstd * (g - xhat * (g * xhat).mean(-1, keepdim=True))
        if st["dh"] is not None:
            dx = dx + st["dh"].float()
        return {"dx": dx.to(torch.bfloat16), "dw": (dy * xhat).sum(0).to(st["w"].dtype)}
    if op == "gemm_residual":
        z = torch.matmul(_dequant_rows(st["a"], st["sfa"]), _dequant_weight(st["w"], st["sfb"]).t()) + st["bias"]
        y = _act(z, st["act"])
        if st["r"] is not None:
            y = y + st["r"].float()
        return {"out": y.to(torch.bfloat16)}
    if op == "act_save":
        z = st["z"].float()
        yq, ys = _quant_rows(_act(z, st["act"]))
        zq, zs = _quant_rows(z)
        return {"yq": yq, "ys": ys, "zq": zq, "zs": zs}
    if op == "act_bwd":
        dz = st["dy"].float() * _act_grad(_dequant_rows(st["zq"], st["zs"]), st["act"])
        q, s = _quant_rows(dz)
        return {"dz": dz.to(torch.bfloat16), "dzq": q, "dzs": s, "dbias": dz.sum(0)}
    dw = torch.matmul(st["g"].float().t(), _dequant_rows(st["xq"], st["xs"]))
    return {"dw": dw.to(torch.bfloat16)}


# ----------------------------------------------------------------------------- the framework's kernels
_ops = None


def _kernels():
    global _ops
    if _ops is None:
        pkg = os.path.join(os.getcwd(), "ltx-2_b200")
        if pkg not in sys.path:
            sys.path.insert(0, pkg)
        from ltx_kernels.blockwise import ops
        _ops = ops
    return _ops


def _own(st):
    k = _kernels()
    op = st["op"]
    if op == "rms_norm":
        q, s, h, rstd = k.rms_norm_quantize(st["x"], st["w"], st["r"], eps=_EPS)
        return {"q": q, "scales": s, "h": h, "rstd": rstd}
    if op == "rms_norm_bwd":
        dx, dw = k.rms_norm_backward(st["dy"], st["x"], st["rstd"], st["w"], st["dh"])
        return {"dx": dx, "dw": dw}
    if op == "gemm_residual":
        return {"out": k.gemm_residual(st["a"], st["sfa"], st["w"], st["sfb"], st["bias"], residual=st["r"],
                                       activation=None if st["act"] == "none" else st["act"])}
    if op == "act_save":
        yq, ys, zq, zs = k.act_quantize_save(st["z"], st["act"])
        return {"yq": yq, "ys": ys, "zq": zq, "zs": zs}
    if op == "act_bwd":
        dz, dzq, dzs, dbias = k.act_backward(st["dy"], st["zq"], st["zs"], st["act"], quantize=True, dbias=True)
        return {"dz": dz, "dzq": dzq, "dzs": dzs, "dbias": dbias}
    return {"dw": k.wgrad_1x128(st["g"], st["xq"], st["xs"])}


def run(state):
    return _own(state) if own else _plain(state)


# ----------------------------------------------------------------------------- what a pass cannot do without
def work(case):
    op, m = case["op"], case["m"]
    if op in ("rms_norm", "rms_norm_bwd"):
        e = m * case["h"]
        if op == "rms_norm":
            return {"bytes": e * (2 + 1 + (4 if case["residual"] else 0)) + 4 * e // 128 + 4 * m + 2 * case["h"],
                    "flops": 6 * e}
        wb = 4 if case["w32"] else 2
        return {"bytes": e * (6 + (2 if case["residual"] else 0)) + 4 * m + 2 * wb * case["h"], "flops": 10 * e}
    if op == "gemm_residual":
        n, k = case["n"], case["k"]
        return {"bytes": m * k + n * k + 4 * m * k // 128 + n * k // 4096 + 4 * n
                + m * n * (4 if case["residual"] else 2), "flops": 2 * m * n * k}
    if op == "act_save":
        e = m * case["n"]
        return {"bytes": 4 * e + 8 * e // 128, "flops": 12 * e}
    if op == "act_bwd":
        e = m * case["n"]
        return {"bytes": 6 * e + 8 * e // 128 + 4 * case["n"], "flops": 20 * e}
    n, k = case["n"], case["k"]
    return {"bytes": 2 * m * n + m * k + 4 * m * k // 128 + 2 * n * k, "flops": 2 * m * n * k}


# ----------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    """The definitions in float64.  Where an output is 8-bit codes, the value before its rounding to e4m3
    stands here (in units of the group's scale), so that both sides' distance is that of a rounding."""
    st = prepare(case, seed)
    op, m = case["op"], case["m"]
    d = torch.float64

    def codes(v):
        k = v.shape[1] // 128
        v = v.reshape(m, k, 128)
        top = torch.maximum(v.abs().max(dim=-1).values, torch.tensor(_AMAX_MIN, dtype=d, device=v.device))
        scale = top / 448
        return (v / scale[:, :, None]).reshape(m, k * 128), scale

    def rows(q, s):
        return q.to(d) * s.to(d).repeat_interleave(128, dim=1)

    def sigmoid_arg(z):
        # gelu_tanh(z) = z * sigmoid(2 u), silu(z) = z * sigmoid(z)
        if case["act"] == "gelu_tanh":
            c = 2 * math.sqrt(2 / math.pi)
            return c * (z + 0.044715 * z ** 3), c * (1 + 3 * 0.044715 * z ** 2)
        return z, torch.ones_like(z)

    if op == "rms_norm":
        h = st["x"].to(d)
        if st["r"] is not None:
            h = (h + st["r"].to(d)).to(torch.bfloat16).to(d)  # the normalised value is the stored one
        rstd = (h.pow(2).sum(1) / case["h"] + _EPS).pow(-0.5)
        q, s = codes(h * rstd[:, None] * st["w"].to(d))
        return {"q": q, "scales": s, "h": h, "rstd": rstd}
    if op == "rms_norm_bwd":
        r = st["rstd"].to(d)[:, None]
        h, dy, w = st["x"].to(d), st["dy"].to(d), st["w"].to(d)
        dot = (dy * w * h).sum(1, keepdim=True) / case["h"]
        dx = r * dy * w - h * (r ** 3) * dot
        if st["dh"] is not None:
            dx = dx + st["dh"].to(d)
        return {"dx": dx, "dw": torch.einsum("mh,mh->h", dy, h * r)}
    if op == "gemm_residual":
        wd = st["w"].to(d) * st["sfb"].to(d).repeat_interleave(128, 0).repeat_interleave(128, 1)
        out = torch.empty(m, case["n"], dtype=d, device="cuda")
        for i in range(0, m, 4096):
            z = rows(st["a"][i:i + 4096], st["sfa"][i:i + 4096]) @ wd.T + st["bias"].to(d)
            if case["act"] != "none":
                z = z * torch.sigmoid(sigmoid_arg(z)[0])
            out[i:i + 4096] = z if st["r"] is None else z + st["r"][i:i + 4096].to(d)
        return {"out": out}
    if op == "act_save":
        z = st["z"].to(d)
        yq, ys = codes(z * torch.sigmoid(sigmoid_arg(z)[0]))
        zq, zs = codes(z)
        return {"yq": yq, "ys": ys, "zq": zq, "zs": zs}
    if op == "act_bwd":
        z = rows(st["zq"], st["zs"])
        u, du = sigmoid_arg(z)
        sg = torch.sigmoid(u)
        dz = st["dy"].to(d) * (sg + z * sg * torch.sigmoid(-u) * du)
        q, s = codes(dz)
        return {"dz": dz, "dzq": q, "dzs": s, "dbias": dz.sum(0)}
    dw = torch.zeros(case["n"], case["k"], dtype=d, device="cuda")
    for i in range(0, m, 4096):
        dw += st["g"][i:i + 4096].to(d).T @ rows(st["xq"][i:i + 4096], st["xs"][i:i + 4096])
    return {"dw": dw}
