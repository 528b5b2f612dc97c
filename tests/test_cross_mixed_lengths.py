"""Attention to another sequence's states over batches in which sequences of one
64-key step, of several and without keys follow one another in a CTA's items."""

import pytest
import torch

from oracle import sublayer_oracle as orc
from sparkdiffusion_b200 import _lib, ops, train

BF16 = torch.bfloat16
MIXED = {
    # H, Hkv, Lq, Lk, lens: more items than SMs, so that every CTA meets several lengths
    "short_and_long": (8, 8, 300, 400, (1, 400, 64, 65, 2, 399, 63, 129) * 2),
    "short_between_empty": (4, 4, 260, 330, (64, 0, 330, 0, 3, 128, 0, 7, 200, 64, 1, 330) * 2),
    "shared_heads": (10, 2, 130, 200, (10, 200, 64, 66, 33, 1, 150, 2, 64, 64)),
    "short_only": (6, 3, 500, 64, (64, 1, 17, 2, 63, 30, 64, 5)),
}


@pytest.mark.gpu
@pytest.mark.parametrize("case", sorted(MIXED))
def test_gradients_over_mixed_lengths(case):
    H, Hkv, Lq, Lk, lens = MIXED[case]
    B = len(lens)
    g = torch.Generator().manual_seed(5)
    q, do = (torch.randn(B, H, Lq, 128, generator=g).to(BF16) for _ in range(2))
    k, v = (torch.randn(B, Hkv, Lk, 128, generator=g).to(BF16) for _ in range(2))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = train.cross_attention(*leaves, torch.tensor(lens, dtype=torch.int32, device="cuda"))
    runs = [torch.autograd.grad(o, leaves, do.cuda(), retain_graph=True) for _ in range(8)]
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    ref = orc.cross_attention_grads(q, k, v, do, lens)
    for i, name in enumerate(("dq", "dk", "dv")):
        r, tol = ref[name]
        worst = ((runs[0][i].cpu().double() - r).abs() / (tol + 1e-30)).max().item()
        assert worst <= 1.0, f"{name}: {worst:.3f} of the bound"
        assert all(torch.equal(run[i], runs[0][i]) for run in runs), f"{name}: two runs differ"


@pytest.mark.gpu
def test_a_million_sequences():
    """Of one token and two states each: the bits of a call on each 65536 of them."""
    B, part = (1 << 20) + 7, 1 << 16
    g = torch.Generator("cuda").manual_seed(6)
    q, do = (torch.randn(B, 1, 1, 128, device="cuda", generator=g).to(BF16) for _ in range(2))
    k, v = (torch.randn(B, 1, 2, 128, device="cuda", generator=g).to(BF16) for _ in range(2))

    def step(at):
        leaves = [t[at].detach().requires_grad_(True) for t in (q, k, v)]
        o = train.cross_attention(*leaves)
        return (o.detach(), *torch.autograd.grad(o, leaves, do[at]))

    got = step(slice(None))
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    for b in range(0, B, part):
        for name, a, w in zip(("o", "dq", "dk", "dv"), got, step(slice(b, b + part))):
            assert torch.equal(a[b:b + part], w), (name, b)
    last = slice(B - 50, B)
    ref = orc.cross_attention_grads(*(t[last].cpu() for t in (q, k, v, do)))
    for name, a in zip(("dq", "dk", "dv"), got[1:]):
        r, tol = ref[name]
        assert bool(((a[last].cpu().double() - r).abs() <= tol + 1e-30).all()), name


def _ragged(B, device="cpu"):
    t = [torch.zeros(B, 1, 1, 128, device=device, dtype=BF16, requires_grad=True) for _ in range(3)]
    return t, torch.ones(B, device=device, dtype=torch.int32)


def test_too_many_lengths_are_refused_before_the_forward():
    """What the backward cannot take is refused when the gradient is asked for, not after the forward."""
    t, lens = _ragged(ops.MAX_BWD_LENS + 1)
    with pytest.raises(ValueError, match="65536"):
        train.cross_attention(*t, lens)
    with pytest.raises(RuntimeError, match="CUDA"):  # no gradient asked for: on to the next check
        train.cross_attention(*(x.detach() for x in t), lens)
    with pytest.raises(RuntimeError, match="CUDA"):
        train.cross_attention(*t)


@pytest.mark.gpu
def test_as_many_lengths_as_the_backward_takes():
    t, lens = _ragged(ops.MAX_BWD_LENS, "cuda")
    dq, dk, dv = torch.autograd.grad(train.cross_attention(*t, lens).sum(), t)
    assert bool((dv == 1).all()) and bool((dq == 0).all()) and bool((dk == 0).all())
    many, lens = _ragged(ops.MAX_BWD_LENS + 1, "cuda")
    with torch.no_grad():
        assert bool((train.cross_attention(*many, lens) == 0).all())
    assert _lib.device_status() == 0
