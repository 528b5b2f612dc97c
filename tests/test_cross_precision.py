"""How precise the cross-attention sublayer's kernels are, in norms: the attention's
output and gradients against the error of the roundings that the kernels make,
made in fp64; the running maximum where it moves in every tile.

The elementwise bounds of ``oracle/sublayer_oracle.py`` add up magnitudes, so they
hold for every element and leave room for a mistake of a few per cent in all of
them together.  In the norm over many elements independent roundings do not add
up so: the error is what the same roundings give in fp64, but for the fp32 sums
(2^-24 each, some 1e-6 of the norm) and chance: with 10^4 roundings or more, the
norm of their errors is within some 2 % of its mean.  10 % are allowed for both."""

import math

import pytest
import torch

from oracle import sublayer_oracle as orc
from sparkdiffusion_b200 import _lib, train

gpu = pytest.mark.gpu
BF16 = torch.bfloat16
CHANCE, FP32_SUMS = 1.1, 1e-5


def _round(t):
    return t.float().to(BF16).double()


def _cross(q, k, v, do, lens, ds_times=1.0, delta_times=1.0, delta_from_o=None):
    """The kernels' steps in fp64 with their roundings to bf16: ``{name: result}``.  A factor on dS or
    delta, or delta taken from the rounded output everywhere, are mistakes to be found."""
    B, H, Lq, D = q.shape
    Hkv = k.shape[1]
    _, _, p, k64, v64 = orc.cross_attention(q, k, v, lens)
    do64 = do.double()
    # P in the forward is scaled to the row's maximum before it is rounded
    top = p.amax(-1, keepdim=True).clamp_min(1e-300)
    o = _round(_round(p / top) @ v64 * top)
    dp = do64 @ v64.transpose(2, 3)
    few = torch.tensor([n <= 64 for n in (lens or [k.shape[2]] * B)])[:, None, None, None]
    from_o, from_p = (do64 * o).sum(-1, keepdim=True), (p * dp).sum(-1, keepdim=True)
    delta = from_o if delta_from_o else torch.where(few, from_p, from_o)
    ds = _round(p * (dp - delta * delta_times) * ds_times)

    def grouped(t):
        return t.view(B, Hkv, H // Hkv, *t.shape[2:]).sum(2)

    scale = 1 / math.sqrt(D)
    return {"o": o, "dq": _round(ds @ k64 * scale), "dk": _round(grouped(ds.transpose(2, 3) @ q.double()) * scale),
            "dv": _round(grouped(_round(p).transpose(2, 3) @ do64))}


CASES = {
    # Lk, lens
    "2_keys": (2, None),
    "40_keys": (40, None),
    "64_keys": (64, None),
    "65_keys": (65, None),
    "257_keys": (257, None),
    "512_keys": (512, None),
    "short_of_many": (300, (20, 64)),
    "ragged": (300, (300, 130)),
}


def _inputs(case):
    Lk, lens = CASES[case]
    g = torch.Generator().manual_seed(17)
    q, do = (torch.randn(2, 4, 600, 128, generator=g).to(BF16) for _ in range(2))
    k, v = (torch.randn(2, 2, Lk, 128, generator=g).to(BF16) for _ in range(2))
    return q, k, v, do, lens


def _exact(q, k, v, do, lens):
    ref = {n: r for n, (r, _) in orc.cross_attention_grads(q, k, v, do, lens).items()}
    return {"o": orc.cross_attention(q, k, v, lens)[0], **ref}


def _off(got, ref):
    return {n: ((got[n] - ref[n]).norm() / ref[n].norm()).item() for n in ref}


def _allowed(inputs, ref):
    return {n: CHANCE * e + FP32_SUMS for n, e in _off(_cross(*inputs), ref).items()}


@gpu
@pytest.mark.parametrize("case", sorted(CASES))
def test_attention_errs_by_its_roundings_alone(case):
    inputs = _inputs(case)
    q, k, v, do, lens = inputs
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = train.cross_attention(*leaves, None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda"))
    grads = torch.autograd.grad(o, leaves, do.cuda())
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    ref = _exact(*inputs)
    off = _off({n: t.detach().cpu().double() for n, t in zip(("o", "dq", "dk", "dv"), (o, *grads))}, ref)
    allowed = _allowed(inputs, ref)
    assert all(off[n] <= allowed[n] for n in off), (off, allowed)


@pytest.mark.parametrize("case", sorted(CASES))
def test_mistakes_in_the_gradient_are_found(case):
    """2 % on dS (at every length) and, where delta weighs enough, 3 % on delta: beyond the bound.
    The elementwise bounds let both pass."""
    inputs = _inputs(case)
    ref = _exact(*inputs)
    allowed = _allowed(inputs, ref)
    assert max(allowed.values()) < 0.004
    off = _off(_cross(*inputs, ds_times=1.02), ref)
    assert off["dq"] > 2 * allowed["dq"] and off["dk"] > 2 * allowed["dk"]
    off = _off(_cross(*inputs, delta_times=0.97), ref)
    assert off["dq"] > allowed["dq"] or off["dk"] > allowed["dk"]


def test_delta_from_the_rounded_output_is_found_over_two_keys():
    """Where dP and delta nearly cancel (over 20 to 64 keys the two differ by less than the bound)."""
    inputs = _inputs("2_keys")
    ref = _exact(*inputs)
    allowed, off = _allowed(inputs, ref), _off(_cross(*inputs, delta_from_o=True), ref)
    assert off["dq"] > allowed["dq"] or off["dk"] > allowed["dk"], (off, allowed)


@gpu
@pytest.mark.parametrize("slope", [80.0, 300.0])
def test_running_maximum_moves_in_every_tile(slope):
    """Row maxima that grow by 2^15 or 2^56 a tile of 128 keys: O and l are rescaled at every unit,
    by the factor of the unit before as well.

    The scores are large here, in powers of two up to s.  Each is off by 16 fp32 steps of its sum
    (8 accumulations of 16 products, two steps each), one of the scaled difference and one of the
    log-sum-exp: 18 * 2^-23 s, and P by ln 2 of that.  The output has P and l, the gradients P and
    the output in terms that the bounds count with 2^-8 of them: twice P's part over 2^-8 is added."""
    Lq, Lk = 150, 700
    g = torch.Generator().manual_seed(23)
    u = torch.nn.functional.normalize(torch.ones(128), dim=0)
    q, k, v, do = (torch.randn(1, 2, n, 128, generator=g) for n in (Lq, Lk, Lk, Lq))
    q = q * 0.3 + 8 * u
    k = k * 0.3 + (torch.arange(Lk) / Lk * slope)[:, None] * u
    q, k, v, do = (t.to(BF16) for t in (q, k, v, do))
    top = torch.stack([t.amax(-1) for t in (q.double() @ k.double().transpose(2, 3)).split(128, -1)])
    assert ((top[1:-1] - top[:-2]) / math.sqrt(128) * math.log2(math.e)).min() > 8  # each whole tile
    s = top.max().item() / math.sqrt(128) * math.log2(math.e)
    wider = 1 + 2 * math.log(2) * 18 * 2.0 ** -23 * s / orc.BF16_HALF
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = train.cross_attention(*leaves)
    grads = torch.autograd.grad(o, leaves, do.cuda())
    torch.cuda.synchronize()
    assert _lib.device_status() == 0
    ref, _, tol = orc.cross_attention_bound(q, k, v)
    assert bool(((o.detach().cpu().double() - ref).abs() <= wider * tol + 1e-30).all())
    for (name, (r, t)), got in zip(orc.cross_attention_grads(q, k, v, do).items(), grads):
        assert bool(((got.cpu().double() - r).abs() <= wider * t + 1e-30).all()), name
