"""Training path of the RoLa layer on the B200 kernels.

The reference trains ``WanSelfAttentionRoLa`` through its non-fused forward
(sparkdiffusion/networks/wan_rola_attention.py:452-559): eager q/k/v
projections, ``WanRMSNorm`` (wan2pt1.py:188-206), ``rope_apply``
(wan2pt1.py:156-185), the low-rank branch (``_lowrank_attn``,
wan_rola_attention.py:329-391) and the gated fusion in PyTorch, and the
block-sparse softmax attention from the external SLA package:
``get_block_map`` for the selection and ``_attention.apply`` for the forward
and backward (wan_rola_attention.py:293-327).  Here the selection runs on the
B200 selection kernels and the attention's forward (with the row
log-sum-exp) and backward on the tcgen05 kernels (``BlockSparseAttention``);
the eager parts stay eager PyTorch, as in the reference.  There is no
fallback: the attention raises without the CUDA library.

``add_rms_norm`` and ``cross_attention`` are the differentiable operators of the
block's next sublayer.  A backward of any of these functions may be captured
into a CUDA graph as long as no eager autograd graph of the same leaf tensors is
alive (PyTorch would order the captured backward after the eager graph's stream).
"""

from __future__ import annotations

import torch
import torch.nn.functional as F
from torch.autograd.function import once_differentiable

from . import _lib, ops


def select_blocks(q: torch.Tensor, k: torch.Tensor, topk_ratio: float, blk: int):
    """Block selection of ``q, k [B, H, L, 128]`` (post-RoPE, bf16): mean
    pooling, smooth-K centre, fp32 scores, top-k with ties toward the lower
    index — the semantics of the reference's ``get_block_map``
    (fused_sparse_attn.py:179-198 restates it for the fused path).  Returns
    ``(lut [B*H, NB, topk], topk, paired)``; ``paired`` is the block-64 table
    the attention kernels take (None for block 128)."""
    B, H, L, _ = q.shape
    NB = (L + blk - 1) // blk
    topk = ops.topk_count(topk_ratio, NB)
    with torch.no_grad():
        pq = ops.mean_pool(q, blk)
        pk = ops.mean_pool(k, blk, center=ops.smooth_k_center(k, blk))
        lut = ops.block_select(pq, pk, topk)
        paired = None
        if blk == 64:
            paired = torch.empty(B * H, (NB + 1) // 2, 2 * topk + 1, device=q.device, dtype=torch.int32)
            _lib.call("rola_b200_pair_blocks", ops._ptr(lut), B * H, NB, topk, ops._ptr(paired), ops._stream())
    return lut, topk, paired


class BlockSparseAttention(torch.autograd.Function):
    """o = block-sparse softmax attention of ``q, k, v [B, H, L, 128]`` (bf16)
    over the selection ``lut``; backward on the B200 kernels.  The counterpart
    of SLA's ``_attention.apply(q, k, v, sparse_map, lut, real_topk, BLKQ,
    BLKK)`` (wan_rola_attention.py:320-321)."""

    @staticmethod
    def forward(ctx, q, k, v, lut, paired, blk: int, topk: int):
        o, lse = ops.sparse_attention_fwd_lse(q, k, v, lut if blk == 128 else paired, blk, topk)
        ctx.save_for_backward(q, k, v, o, lse, lut, paired if paired is not None else lut)
        ctx.blk, ctx.topk = blk, topk
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse, lut, paired = ctx.saved_tensors
        dq, dk, dv = ops.sparse_attention_bwd(q, k, v, o, do, lut, paired if ctx.blk == 64 else None, lse, ctx.blk,
                                              ctx.topk)
        return dq, dk, dv, None, None, None, None


def sparse_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, topk_ratio: float, blkq: int,
                     blkk: int) -> torch.Tensor:
    """The reference's ``_sparse_attn`` (wan_rola_attention.py:293-327) on the
    B200 kernels: ``q, k, v [B, H, L, 128]`` -> ``o [B, H, L, 128]`` in the
    input dtype, differentiable in q, k and v."""
    if blkq != blkk or blkq not in (64, 128):
        raise ValueError("the B200 attention kernels support blkq == blkk in (64, 128)")
    if not q.is_cuda:
        raise RuntimeError("the B200 training path runs on CUDA tensors only")
    dt = q.dtype
    qb, kb, vb = (t.to(torch.bfloat16) for t in (q, k, v))
    lut, topk, paired = select_blocks(qb.detach(), kb.detach(), topk_ratio, blkq)
    o = BlockSparseAttention.apply(qb, kb, vb, lut, paired, blkq, topk)
    return o.to(dt)


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float) -> torch.Tensor:
    """``WanRMSNorm.forward`` (wan2pt1.py:200-206): fp32 normalisation, cast back, times the weight."""
    xf = x.float()
    return (xf * torch.rsqrt(xf.pow(2).mean(dim=-1, keepdim=True) + eps)).type_as(x) * weight


def rope_apply(x: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """``rope_apply`` (wan2pt1.py:156-185): interleaved pairs rotated in fp32 by
    the raw angles ``freqs [L, D/2]``; ``x [B, L, H, D]``."""
    B, L, H, D = x.shape
    f = freqs[:L].reshape(L, D // 2)
    c = torch.cos(f).float()[None, :, None, :]
    s = torch.sin(f).float()[None, :, None, :]
    xf = x.float()
    e, o = xf[..., 0::2], xf[..., 1::2]
    return torch.stack([e * c - o * s, e * s + o * c], dim=-1).flatten(-2).to(x.dtype)


def rope_rank(x: torch.Tensor, freqs: torch.Tensor, rank: int) -> torch.Tensor:
    """Truncated interleaved RoPE of the low-rank features ``x [B, H, L, rank]``
    (``_apply_rope_rank``, wan_rola_attention.py:329-364): angles cast to the
    data dtype, the first ``min(rank/2, D/2)`` pairs rotated, the rest unchanged."""
    L = x.shape[2]
    rd = min(rank // 2, freqs.shape[-1])
    f = freqs[:L, :rd].to(x.dtype)
    c, s = torch.cos(f), torch.sin(f)
    x1, x2 = x[..., : 2 * rd].unflatten(-1, (-1, 2)).unbind(-1)
    rot = torch.stack([x1 * c - x2 * s, x1 * s + x2 * c], dim=-1).flatten(-2)
    if 2 * rd < rank:
        rot = torch.cat([rot, x[..., 2 * rd:]], dim=-1)
    return rot


def lowrank_attention(layer, qn: torch.Tensor, kn: torch.Tensor, v: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """``_lowrank_attn`` (wan_rola_attention.py:366-391) over ``[B, H, L, D]``:
    SiLU projections to the rank, truncated RoPE, O = Q_lr (K_lr^T V), RMS-normed."""
    q_lr = rope_rank(F.silu(layer.proj_q(qn)), freqs, layer.rola_rank)
    k_lr = rope_rank(F.silu(layer.proj_k(kn)), freqs, layer.rola_rank)
    out = q_lr @ (k_lr.transpose(-2, -1) @ v)
    return F.rms_norm(out, [out.shape[-1]])


def training_attention_core(layer, x: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """The reference's non-fused forward up to (not including) ``self.o``
    (wan_rola_attention.py:481-545): differentiable in x and every parameter."""
    b, s, _ = x.shape
    n, d = layer.num_heads, layer.head_dim
    q = layer.q(x)
    k = layer.k(x)
    if layer.qk_norm:
        q = rms_norm(q, layer.norm_q.weight, layer.norm_q.eps)
        k = rms_norm(k, layer.norm_k.weight, layer.norm_k.eps)
    q = q.view(b, s, n, d)
    k = k.view(b, s, n, d)
    v = layer.v(x).view(b, s, n, d)
    q_rope = rope_apply(q, freqs)
    k_rope = rope_apply(k, freqs)
    v_bhld = v.transpose(1, 2)
    o_s = sparse_attention(q_rope.transpose(1, 2), k_rope.transpose(1, 2), v_bhld, layer.rola_topk_ratio,
                           layer.rola_blkq, layer.rola_blkk)
    o_l = lowrank_attention(layer, q.transpose(1, 2), k.transpose(1, 2), v_bhld, freqs)
    x_bhld = x.view(b, s, n, d).transpose(1, 2)
    gate = torch.sigmoid(layer.gate_proj(x_bhld) + layer.gate_bias)
    o_s_scale = (o_s.pow(2).mean(dim=-1, keepdim=True) + 1e-5).sqrt()
    fused = o_s.float() / o_s_scale.float() + gate * o_l.float()
    out_bhld = (fused * o_s_scale.float()).to(o_l.dtype)
    return out_bhld.transpose(1, 2).reshape(b, s, n * d)


def dense_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> torch.Tensor:
    """Dense softmax attention of ``q, k, v [B, H, L, 128]``, differentiable:
    the block-sparse kernels with every 128-token key block selected."""
    if not q.is_cuda:
        raise RuntimeError("the B200 training path runs on CUDA tensors only")
    B, H, L, _ = q.shape
    NB = (L + 127) // 128
    lut = ops._full_lut(B * H, NB, q.device)
    dt = q.dtype
    o = BlockSparseAttention.apply(*(t.to(torch.bfloat16) for t in (q, k, v)), lut, None, 128, NB)
    return o.to(dt)


def dense_training_forward(layer, x: torch.Tensor, freqs: torch.Tensor) -> torch.Tensor:
    """``WanSelfAttention.forward``'s differentiable route (wan2pt1.py:313-328)
    with the attention on the B200 kernels: projections, ``WanRMSNorm``, ``rope_apply``,
    dense attention, ``self.o``."""
    b, s, _ = x.shape
    n, d = layer.num_heads, layer.head_dim
    q, k = layer.q(x), layer.k(x)
    if layer.qk_norm:
        q = rms_norm(q, layer.norm_q.weight, layer.norm_q.eps)
        k = rms_norm(k, layer.norm_k.weight, layer.norm_k.eps)
    q = rope_apply(q.view(b, s, n, d), freqs)
    k = rope_apply(k.view(b, s, n, d), freqs)
    v = layer.v(x).view(b, s, n, d)
    o = dense_attention(q.transpose(1, 2), k.transpose(1, 2), v.transpose(1, 2))
    return layer.o(o.transpose(1, 2).reshape(b, s, n * d))


def _differentiable_once(backward):
    """``once_differentiable`` where a graph of the gradient is asked for (its
    own differentiation then raises); without one, nothing around the kernels."""
    once = once_differentiable(backward)

    def run(ctx, *grads):
        return once(ctx, *grads) if torch.is_grad_enabled() else backward(ctx, *grads)

    return run


class AddRMSNorm(torch.autograd.Function):
    """``ops.add_rms_norm`` with its backward kernel; saves h and the row factors."""

    @staticmethod
    def forward(ctx, x, weight, eps: float, residual):
        rstd = x.new_empty(x.numel() // max(1, x.shape[-1]), dtype=torch.float32)
        y, h = ops.add_rms_norm(x, weight, eps, residual, rstd=rstd)
        ctx.save_for_backward(h, weight, rstd)
        ctx.x_dtype, ctx.res_dtype = x.dtype, None if residual is None else residual.dtype
        ctx.set_materialize_grads(False)
        return (y, h) if residual is not None else y

    @staticmethod
    @_differentiable_once
    def backward(ctx, dy, dh=None):
        h, weight, rstd = ctx.saved_tensors
        if dy is None:
            dy = torch.zeros(h.shape, device=h.device, dtype=torch.bfloat16)
        dx, dres, dw = ops.add_rms_norm_bwd(h, weight, rstd, dy, dh, ctx.x_dtype, ctx.res_dtype,
                                            need_dw=ctx.needs_input_grad[1])
        return dx, dw, None, dres


def add_rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: torch.Tensor | None = None):
    """Differentiable ``ops.add_rms_norm``: ``(y, h)``, gradients to ``x``,
    ``residual`` and ``weight``, one kernel each way."""
    if not x.is_cuda:
        raise RuntimeError("the B200 training path runs on CUDA tensors only")
    out = AddRMSNorm.apply(x, weight, eps, residual)
    return out if residual is not None else (out, x)


class CrossAttention(torch.autograd.Function):
    """``ops.cross_attention`` with its backward kernels."""

    @staticmethod
    def forward(ctx, q, k, v, kv_lens):
        o, lse = ops.cross_attention_fwd_lse(q, k, v, kv_lens)
        ctx.save_for_backward(q, k, v, o, lse, kv_lens)
        return o

    @staticmethod
    @_differentiable_once
    def backward(ctx, do):
        q, k, v, o, lse, lens = ctx.saved_tensors
        B, H, Lq, _ = q.shape
        lens = None if lens is None else lens.contiguous()
        return (*ops._cross_bwd(q.get_device(), (B, H, k.shape[1], Lq, k.shape[2]), q, k, v, o, do, lse, lens), None)


def cross_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                    kv_lens: torch.Tensor | None = None) -> torch.Tensor:
    """Differentiable attention of ``q [B, H, Lq, 128]`` to the states ``k, v
    [B, Hkv, Lk, 128]`` (``ops.cross_attention``), in the input dtype; beside
    ``dense_attention``, which takes one length.  With ``kv_lens`` at most 65536
    sequences where a gradient is asked for (the backward kernels' limit)."""
    if (kv_lens is not None and q.shape[0] > ops.MAX_BWD_LENS and torch.is_grad_enabled()
            and any(t.requires_grad for t in (q, k, v))):
        raise ValueError(f"cross_attention: {q.shape[0]} sequences of their own lengths, the backward takes at most "
                         f"{ops.MAX_BWD_LENS}")
    if not q.is_cuda:
        raise RuntimeError("the B200 training path runs on CUDA tensors only")
    dt, bf16 = q.dtype, torch.bfloat16
    o = CrossAttention.apply(*(t if t.dtype is bf16 else t.to(bf16) for t in (q, k, v)), kv_lens)
    return o if dt is bf16 else o.to(dt)
