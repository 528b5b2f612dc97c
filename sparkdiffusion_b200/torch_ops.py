"""``torch.ops.rola_b200.*``: the B200 kernels as PyTorch custom operators.

The Wan inference entry points compile the whole model
(``torch.compile(model, ...)``, sparkdiffusion/utils/inference_optimization.py:122).
Each op here is opaque to Dynamo/Inductor: its real implementation launches
librola_b200 kernels through the C ABI (``ops``), and a fake (meta) kernel
gives output shapes and dtypes for tracing, so a compiled graph holds one node
per op instead of tracing into ctypes calls on ``data_ptr()``.  The drop-in
layers call these ops.

Ops (inputs and layouts as in ``ops``; outputs are new tensors):

* ``qkv_gemm(x2d, w, bias?) -> [M, N]`` bf16 (the QKV projection and ``self.o``);
* ``attention_core(x, w_qkv, b_qkv?, cos_sin, lr_cos, lr_sin, rope_dim, norm_wq?,
  norm_wk?, proj_q, proj_k, gate_w, gate_b, num_heads, topk, eps, blk=128, w_scale?) -> [B, L, H*D]``
  (``w_scale`` given: ``w_qkv`` is float8_e4m3fn, the reference's FP8 mode)
  bf16: ``fused_forward`` minus ``self.o`` (wan_rola_attention.py:414-446);
* ``block_select(pooled_q, pooled_k, topk) -> [B*H, NBq, topk]`` int32;
* ``fused_sparse_attn(q, k, v, topk_ratio, blkq, blkk, num_heads) -> [B, H, L, D]``
  (fused_sparse_attn.py:151-215);
* ``dense_attention(q, k, v, num_heads) -> [B, H, L, D]``;
* ``cross_attention(q, k, v, kv_lens?) -> [B, H, Lq, D]`` (a view of a token-major tensor);
* ``add_rms_norm(x, residual, weight, eps) -> (y, h)`` and
  ``add_rms_norm_e4m3(x, residual, weight, eps) -> (yq, scale, h)`` (a scale per 128 columns);
* ``quantize_blocks_e4m3(x) -> (xq, scale)`` and
  ``gemm_fp8_block(xq, x_scale, wq, w_scale, bias?) -> [M, N]`` bf16.
"""

from __future__ import annotations

from typing import Optional

import torch

from . import ops

BF16 = torch.bfloat16
Tensor = torch.Tensor


@torch.library.custom_op("rola_b200::qkv_gemm", mutates_args=())
def qkv_gemm(x2d: Tensor, w: Tensor, bias: Optional[Tensor]) -> Tensor:
    return ops.qkv_gemm(x2d, w, bias)


@qkv_gemm.register_fake
def _(x2d, w, bias):
    return x2d.new_empty(x2d.shape[0], w.shape[0], dtype=BF16)


@torch.library.custom_op("rola_b200::attention_core", mutates_args=())
def attention_core(x: Tensor, w_qkv: Tensor, b_qkv: Optional[Tensor], cos_sin: Tensor, lr_cos: Tensor,
                   lr_sin: Tensor, rope_dim: int, norm_wq: Optional[Tensor], norm_wk: Optional[Tensor],
                   proj_q: Tensor, proj_k: Tensor, gate_w: Tensor, gate_b: Tensor, num_heads: int, topk: int,
                   eps: float, blk: int = 128, w_scale: Optional[Tensor] = None) -> Tensor:
    return ops.rola_attention_core(x, w_qkv, b_qkv, cos_sin, lr_cos, lr_sin, rope_dim, norm_wq, norm_wk, proj_q,
                                   proj_k, gate_w, gate_b, num_heads, blk, topk, eps, w_scale=w_scale)


@attention_core.register_fake
def _(x, w_qkv, b_qkv, cos_sin, lr_cos, lr_sin, rope_dim, norm_wq, norm_wk, proj_q, proj_k, gate_w, gate_b,
      num_heads, topk, eps, blk=128, w_scale=None):
    return x.new_empty(x.shape, dtype=BF16)


@torch.library.custom_op("rola_b200::block_select", mutates_args=())
def block_select(pooled_q: Tensor, pooled_k: Tensor, topk: int) -> Tensor:
    return ops.block_select(pooled_q, pooled_k, topk)


@block_select.register_fake
def _(pooled_q, pooled_k, topk):
    B, H, NBq, _ = pooled_q.shape
    return pooled_q.new_empty(B * H, NBq, topk, dtype=torch.int32)


@torch.library.custom_op("rola_b200::fused_sparse_attn", mutates_args=())
def fused_sparse_attn(q: Tensor, k: Tensor, v: Tensor, topk_ratio: float, blkq: int, blkk: int,
                      num_heads: int) -> Tensor:
    return ops.fused_sparse_attn(q, k, v, topk_ratio, blkq, blkk, num_heads)


@fused_sparse_attn.register_fake
def _(q, k, v, topk_ratio, blkq, blkk, num_heads):
    BH, L, D = q.shape
    return v.new_empty(BH // num_heads, num_heads, L, D)


@torch.library.custom_op("rola_b200::dense_attention", mutates_args=())
def dense_attention(q: Tensor, k: Tensor, v: Tensor, num_heads: int) -> Tensor:
    return ops.dense_attention(q, k, v, num_heads)


@dense_attention.register_fake
def _(q, k, v, num_heads):
    BH, L, D = q.shape
    return v.new_empty(BH // num_heads, num_heads, L, D)


@torch.library.custom_op("rola_b200::cross_attention", mutates_args=())
def cross_attention(q: Tensor, k: Tensor, v: Tensor, kv_lens: Optional[Tensor]) -> Tensor:
    return ops.cross_attention(q, k, v, kv_lens)


@cross_attention.register_fake
def _(q, k, v, kv_lens):
    B, H, Lq, D = q.shape
    return q.new_empty_strided((B, H, Lq, D), (Lq * H * D, D, H * D, 1))


@torch.library.custom_op("rola_b200::add_rms_norm", mutates_args=())
def add_rms_norm(x: Tensor, residual: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor]:
    return ops.add_rms_norm(x, weight, eps, residual)


@add_rms_norm.register_fake
def _(x, residual, weight, eps):
    return x.new_empty(x.shape, dtype=BF16), x.new_empty(x.shape, dtype=residual.dtype)


def _scales_like(x: Tensor) -> Tensor:
    """The layout ``ops`` gives block scales: rows (flattened) innermost."""
    lead, nb = x.shape[:-1], (x.shape[-1] + ops.SCALE_BLOCK - 1) // ops.SCALE_BLOCK
    strides, step = [], 1
    for n in reversed(lead):
        strides.insert(0, step)
        step = step * n
    return x.new_empty_strided((*lead, nb), (*strides, step), dtype=torch.float32)


@torch.library.custom_op("rola_b200::add_rms_norm_e4m3", mutates_args=())
def add_rms_norm_e4m3(x: Tensor, residual: Tensor, weight: Tensor, eps: float) -> tuple[Tensor, Tensor, Tensor]:
    return ops.add_rms_norm_e4m3(x, weight, eps, residual)


@add_rms_norm_e4m3.register_fake
def _(x, residual, weight, eps):
    return x.new_empty(x.shape, dtype=ops.E4M3), _scales_like(x), x.new_empty(x.shape, dtype=residual.dtype)


@torch.library.custom_op("rola_b200::quantize_blocks_e4m3", mutates_args=())
def quantize_blocks_e4m3(x: Tensor) -> tuple[Tensor, Tensor]:
    return ops.quantize_blocks_e4m3(x)


@quantize_blocks_e4m3.register_fake
def _(x):
    return x.new_empty(x.shape, dtype=ops.E4M3), _scales_like(x)


@torch.library.custom_op("rola_b200::gemm_fp8_block", mutates_args=())
def gemm_fp8_block(xq: Tensor, x_scale: Tensor, wq: Tensor, w_scale: Tensor, bias: Optional[Tensor]) -> Tensor:
    return ops.gemm_fp8_block(xq, x_scale, wq, w_scale, bias)


@gemm_fp8_block.register_fake
def _(xq, x_scale, wq, w_scale, bias):
    return xq.new_empty(xq.shape[0], wq.shape[0], dtype=BF16)
