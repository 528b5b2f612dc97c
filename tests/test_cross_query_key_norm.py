"""The norm without a residual as the query and key norm of the cross-attention:
projection -> norm over all heads -> attention to the states, and back."""

import pytest
import torch

from oracle import sublayer_oracle as orc
from sparkdiffusion_b200 import _lib, ops, train

BF16, F32 = torch.bfloat16, torch.float32
B, L, LK, H, DIM, LENS, EPS = 2, 140, 90, 3, 384, (90, 33), 1e-6


def _within(got, ref, tol, what):
    worst = ((got.detach().cpu().double() - ref).abs() / (tol + 1e-30)).max().item()
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


def _heads(t):
    return t.view(B, -1, H, 128).transpose(1, 2)


@pytest.mark.gpu
def test_query_and_key_norm_in_the_sublayer():
    """Each stage from the GPU's own previous one, against the fp64 form; forward and backward."""
    g = torch.Generator().manual_seed(31)
    x, ctx = torch.randn(B * L, DIM, generator=g).to(BF16), torch.randn(B * LK, DIM, generator=g).to(BF16)
    weights = [(torch.randn(DIM, DIM, generator=g) * DIM ** -0.5).cuda() for _ in range(3)]
    norms = [(1 + 0.2 * torch.randn(DIM, generator=g)).cuda().requires_grad_(True) for _ in range(2)]
    do = torch.randn(B, H, L, 128, generator=g).to(BF16)
    lens = torch.tensor(LENS, dtype=torch.int32, device="cuda")
    xq, cq = ops.quantize_blocks_e4m3(x.cuda()), ops.quantize_blocks_e4m3(ctx.cuda())
    q, k, v = (ops.gemm_fp8_block(*t, *ops.quantize_tiles_e4m3(w)) for t, w in zip((xq, cq, cq), weights))
    v = _heads(v.view(B, LK, DIM))

    # inference: the norm gives the input itself as its second result
    served = []
    for t, w in zip((q, k), norms):
        y, h = ops.add_rms_norm(t.view(B, -1, DIM), w.detach(), EPS)
        assert h.data_ptr() == t.data_ptr() and h.shape == y.shape
        _, ref, _ = orc.add_rms_norm(t.cpu().view(B, -1, DIM), w.detach().cpu(), EPS)
        _within(y, ref, (orc.BF16_HALF + orc.FP32) * ref.abs() * 1.01, "norm")
        served.append(_heads(y))
    o = ops.cross_attention(*served, v, lens)

    # training: the same bits, and the gradients through both operators
    leaves = [t.view(B, -1, DIM).clone().requires_grad_(True) for t in (q, k)]
    normed = [train.add_rms_norm(t, w, EPS)[0] for t, w in zip(leaves, norms)]
    o2 = train.cross_attention(*(_heads(t) for t in normed), v, lens)
    assert torch.equal(o, o2.detach())
    ref, _, tol = orc.cross_attention_bound(*(t.cpu() for t in (*served, v)), LENS)
    _within(o, ref, tol, "attention")
    dn = torch.autograd.grad(o2, normed, do.cuda(), retain_graph=True)
    grads = torch.autograd.grad(o2, (*leaves, *norms), do.cuda())
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    bounds = orc.cross_attention_grads(*(t.cpu() for t in (*served, v)), do, LENS)
    for i, name in enumerate(("dq", "dk")):
        _within(_heads(dn[i]), *bounds[name], name)
        d, mag, dw, dw_mag = orc.add_rms_norm_grads(leaves[i].detach().cpu(), norms[i].detach().cpu(), EPS, dn[i].cpu())
        _within(grads[i], d, orc.FP32 * mag + orc.BF16_HALF * 1.01 * d.abs(), f"norm of {name}")
        _within(grads[2 + i], dw, orc.FP32 * dw_mag, f"weight of {name}")
