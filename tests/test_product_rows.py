"""What a row of the block-scaled e4m3 product depends on: the operands' sizes (they
choose the kernel and with it the order in which the K blocks are added) and its
own values, not those of the other rows."""

import pytest
import torch

from sparkdiffusion_b200 import _lib, ops

E4M3 = torch.float8_e4m3fn

# sizes for each way the product is cut: few rows, whole narrow tiles, K blocks shared by CTAs, rounds of
# wide tiles, these and a rest
PRODUCTS = [(7, 264, 1040), (16, 1536, 1536), (129, 136, 272), (200, 1000, 4112), (3500, 2560, 272), (1300, 3904, 2064)]


@pytest.mark.gpu
@pytest.mark.parametrize("M, N, K", PRODUCTS)
def test_product_row_depends_on_no_other_row(M, N, K):
    """With the sizes fixed, other values (NaN too) in the other rows leave a row's bits as they are."""
    g = torch.Generator().manual_seed(3)

    def operand(rows, per):
        x = (torch.randn(rows, K, generator=g) * 60).clamp(-448, 448).to(E4M3)
        return x.cuda(), (torch.rand(-(-rows // per), -(-K // 128), generator=g) * 0.02 + 0.001).cuda()

    (xq, xs), (yq, ys), (wq, ws) = operand(M, 1), operand(M, 1), operand(N, 128)
    out = ops.gemm_fp8_block(xq, xs, wq, ws)
    keep = torch.tensor(sorted({0, M // 2, M - 1}), device="cuda")
    ys[1] = float("nan")
    yq.view(torch.uint8)[keep], ys[keep] = xq.view(torch.uint8)[keep], xs[keep]
    assert torch.equal(ops.gemm_fp8_block(yq, ys, wq, ws)[keep], out[keep])
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
