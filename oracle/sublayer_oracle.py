"""Plain fp64 forms of the cross-attention sublayer's operators, with bounds on
what a kernel may be off (test infrastructure only).

Every bound counts the roundings the kernels make, each at most half a step
relative to the value: bf16 2^-8, fp32 2^-24 (sums of n terms: n steps), e4m3
2^-4 (or half its smallest step, 2^-10 of the scale).
"""

from __future__ import annotations

import math

import torch

BF16_HALF = 2.0 ** -8
FP32 = 1e-5  # fp32 chains of these kernels: exp2, scores and sums of a few thousand terms, well below bf16_half


def cross_attention(q, k, v, lens=None):
    """fp64 ``(o, lse (base 2), p, keep)`` of q [B, H, Lq, D], k and v [B, Hkv, Lk, D]."""
    B, H, Lq, D = q.shape
    G, Lk = H // k.shape[1], k.shape[2]
    keep = torch.ones(B, Lk, dtype=torch.bool)
    if lens is not None:
        keep = torch.arange(Lk)[None] < torch.as_tensor(lens).clamp(0, Lk)[:, None]
    # what the masked states hold has no effect: drop it before it is multiplied
    k64 = torch.where(keep[:, None, :, None], k.double(), 0.0).repeat_interleave(G, 1)
    v64 = torch.where(keep[:, None, :, None], v.double(), 0.0).repeat_interleave(G, 1)
    s = q.double() @ k64.transpose(2, 3) / math.sqrt(D)
    s = s.masked_fill(~keep[:, None, None, :], -math.inf)
    lse = torch.logsumexp(s, -1)
    p = torch.where(keep[:, None, None, :], torch.exp(s - lse[..., None]), 0.0)
    p = torch.nan_to_num(p, nan=0.0) if bool((~keep).all(1).any()) else p
    return p @ v64, lse * math.log2(math.e), p, k64, v64


def cross_attention_bound(q, k, v, lens=None):
    """``(o, |error| allowed)``: P rounded to bf16 before P V, the result rounded to bf16."""
    o, lse, p, _, v64 = cross_attention(q, k, v, lens)
    mag = p @ v64.abs()
    return o, lse, BF16_HALF * (mag + o.abs()) * 1.01 + FP32 * mag


def cross_attention_grads(q, k, v, do, lens=None):
    """``{name: (gradient, |error| allowed)}``.  The kernels round P and dS to bf16
    where they feed a product, take delta from the rounded output, and round the
    gradients to bf16."""
    B, H, Lq, D = q.shape
    Hkv = k.shape[1]
    o, _, p, k64, v64 = cross_attention(q, k, v, lens)
    _, _, o_err = cross_attention_bound(q, k, v, lens)
    do64, q64 = do.double(), q.double()
    dp = do64 @ v64.transpose(2, 3)
    delta = (do64 * o).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # |dS| off by: its rounding, delta's error, fp32 sums
    dp_mag = do64.abs() @ v64.abs().transpose(2, 3)
    ds_err = BF16_HALF * 1.01 * ds.abs() + p * (do64.abs() * o_err).sum(-1, keepdim=True) * 1.01 + FP32 * p * (
        dp_mag + (do64 * o).abs().sum(-1, keepdim=True))
    scale = 1 / math.sqrt(D)

    def grouped(t):  # sum over the query heads of a key head
        return t.view(B, Hkv, H // Hkv, *t.shape[2:]).sum(2)

    dq, dq_e = ds @ k64 * scale, ds_err @ k64.abs() * scale
    dk, dk_e = grouped(ds.transpose(2, 3) @ q64) * scale, grouped(ds_err.transpose(2, 3) @ q64.abs()) * scale
    dv = grouped(p.transpose(2, 3) @ do64)
    dv_e = grouped(p.transpose(2, 3) @ do64.abs()) * (BF16_HALF * 1.01 + FP32)
    mag_q, mag_k = ds.abs() @ k64.abs() * scale, grouped(ds.abs().transpose(2, 3) @ q64.abs()) * scale
    return {"dq": (dq, dq_e + BF16_HALF * dq.abs() * 1.01 + FP32 * mag_q),
            "dk": (dk, dk_e + BF16_HALF * dk.abs() * 1.01 + FP32 * mag_k),
            "dv": (dv, dv_e + BF16_HALF * dv.abs() * 1.01)}


def add_rms_norm(x, w, eps, res=None):
    """``(h in its own type, y fp64, r fp64)``; h as the stream stores it."""
    h = x if res is None else (x.float() + res.float()).to(res.dtype)
    h64 = h.double()
    r = (h64.square().mean(-1, keepdim=True) + eps).rsqrt()
    return h, h64 * r * w.double(), r


def add_rms_norm_grads(x, w, eps, dy, res=None, dh=None):
    """fp64 ``(dh total, its fp32 error scale, dw, sum of |terms| of dw)``."""
    h, _, r = add_rms_norm(x, w, eps, res)
    u = h.double() * r
    g = dy.double() * w.double()
    c = (g * u).mean(-1, keepdim=True)
    d = r * (g - u * c)
    mag = r * (g.abs() + u.abs() * (g * u).abs().mean(-1, keepdim=True))
    if dh is not None:
        d, mag = d + dh.double(), mag + dh.double().abs()
    t = (dy.double() * u).reshape(-1, x.shape[-1])
    return d, mag, t.sum(0), t.abs().sum(0)


def block_scales(y, block):
    """``max|y|/448 + 1e-12`` over each ``block`` columns (None: the row) of fp64 ``y [M, K]``."""
    parts = y.split(block or y.shape[1], 1)
    return torch.stack([t.abs().amax(1) for t in parts], 1) / 448.0 + 1e-12


def spread(scale, K, block):
    """Scales ``[M, nb]`` repeated over their columns."""
    return scale.repeat_interleave(block or K, 1)[:, :K]


def gemm_fp8_block(xq, xs, wq, ws, bias=None):
    """``(out fp64, |error| allowed)``: fp32 sums over 128 products and the K blocks,
    one step (2^-23) each at the magnitude of the terms, and the bf16 rounding."""
    K, N = xq.shape[1], wq.shape[0]
    x = xq.double() * spread(xs.double(), K, 128)
    w = wq.double() * spread(ws.double().repeat_interleave(128, 0)[:N], K, 128)
    out = x @ w.t()
    mag = x.abs() @ w.abs().t()
    if bias is not None:
        out = out + bias.double()
        mag = mag + bias.double().abs()
    return out, BF16_HALF * out.abs() * 1.01 + (128 + xs.shape[1] + 2) * 2.0 ** -23 * mag
