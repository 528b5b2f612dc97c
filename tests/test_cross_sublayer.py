"""The cross-attention sublayer's operators against plain fp64 forms
(``oracle/sublayer_oracle.py``, which derives every tolerance from the roundings
the kernels make): norm with the residual's addition, block-scaled e4m3
quantisation and product, attention to another sequence's states; forward and
backward, and their refusals."""

import pytest
import torch

from oracle import sublayer_oracle as orc
from sparkdiffusion_b200 import _lib, ops, torch_ops, train  # noqa: F401  (torch_ops registers torch.ops.rola_b200.*)

gpu = pytest.mark.gpu
BF16, F32, E4M3 = torch.bfloat16, torch.float32, torch.float8_e4m3fn


def _randn(*shape, seed, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _within(got, ref, tol, what):
    got = got.detach().cpu().double()
    assert got.shape == ref.shape, (what, got.shape, ref.shape)
    assert bool(torch.isfinite(got).all()), f"{what}: not finite"
    worst = ((got - ref).abs() / (tol + 1e-30)).max().item() if ref.numel() else 0.0
    assert worst <= 1.0, f"{what}: {worst:.3f} of the bound"


def _ok():
    torch.cuda.synchronize()
    assert _lib.device_status() == 0


# ---------------------------------------------------------------- attention
ATTENTION = {
    # B, H, Hkv, Lq, Lk, kv_lens
    "one_one": (1, 1, 1, 1, 1, None),
    "two_keys": (1, 2, 2, 3, 2, None),
    "one_token_split": (2, 3, 3, 1, 5000, (4999, 37)),
    "one_token_groups": (2, 10, 2, 1, 1100, (1100, 513)),
    "one_token_groups_split": (2, 10, 2, 1, 2300, (2300, 130)),
    "few_rows_split": (1, 2, 2, 130, 3000, None),
    "packed_128_rows": (1, 8, 1, 16, 700, (641,)),
    "unpacked_136_rows": (1, 8, 1, 17, 700, (641,)),
    # runs that end in the midst of items, of one and two query tiles; empty and short sequences between
    "ragged_tokens": (6, 8, 2, 1, 3000, (0, 3000, 1, 129, 2999, 640)),
    "ragged_rows": (3, 4, 4, 200, 2100, (2100, 0, 300)),
    "fewer_tiles_than_runs": (4, 3, 3, 2, 4000, (5, 0, 130, 0)),
    "row_tail": (1, 2, 2, 129, 64, None),
    "key_tail": (2, 2, 1, 127, 257, (257, 129)),
    "empty_rows": (3, 2, 2, 70, 129, (0, 128, 129)),
    "all_empty": (2, 2, 2, 5, 40, (0, 0)),
    "one_key": (2, 2, 2, 200, 300, (1, 300)),
    "encoder": (1, 2, 2, 600, 512, None),
    # more items than SMs: CTAs walk several, with one and two query tiles, empty ones between
    "many_items": (5, 40, 40, 300, 200, (200, 0, 77, 1, 128)),
    "many_groups": (4, 40, 8, 130, 140, (140, 0, 139, 13)),
    # items of one step, four a CTA: every role runs across their ends
    "one_step_items": (1, 4, 4, 19000, 40, None),
    "clamped_lens": (3, 1, 1, 40, 50, (-3, 50, 99)),
}


def _attention_inputs(case, seed=0):
    B, H, Hkv, Lq, Lk, lens = ATTENTION[case]
    q = _randn(B, H, Lq, 128, seed=seed) * 1.5
    k, v = _randn(B, Hkv, Lk, 128, seed=seed + 1), _randn(B, Hkv, Lk, 128, seed=seed + 2)
    return q, k, v, _randn(B, H, Lq, 128, seed=seed + 3), lens


def _lens_gpu(lens):
    return None if lens is None else torch.tensor(lens, dtype=torch.int32, device="cuda")


@gpu
@pytest.mark.parametrize("case", sorted(ATTENTION))
def test_cross_attention(case):
    q, k, v, _, lens = _attention_inputs(case)
    o, lse = ops.cross_attention_fwd_lse(q.cuda(), k.cuda(), v.cuda(), _lens_gpu(lens))
    _ok()
    ref, ref_lse, tol = orc.cross_attention_bound(q, k, v, lens)
    _within(o, ref, tol, f"{case} o")
    B, H, Lq, _ = q.shape
    lse = lse.cpu().double().view(B, H, -1)
    assert bool((lse[..., Lq:] == float("inf")).all())
    dead = ref_lse == -float("inf")
    assert bool((lse[..., :Lq][dead] == float("inf")).all())
    # exp2, log2 and the sums in fp32: a few steps at the scores' magnitude
    assert (lse[..., :Lq] - ref_lse)[~dead].abs().max().item() <= 1e-4 if bool((~dead).any()) else True
    o2 = ops.cross_attention(q.cuda(), k.cuda(), v.cuda(), _lens_gpu(lens))
    assert torch.equal(o, o2)


@gpu
@pytest.mark.parametrize("case", sorted(ATTENTION))
def test_cross_attention_backward(case):
    q, k, v, do, lens = _attention_inputs(case, seed=10)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = train.cross_attention(*leaves, _lens_gpu(lens))
    grads = torch.autograd.grad(o, leaves, do.cuda(), retain_graph=True)
    again = torch.autograd.grad(o, leaves, do.cuda())
    _ok()
    ref = orc.cross_attention_grads(q, k, v, do, lens)
    for name, g, g2 in zip(("dq", "dk", "dv"), grads, again):
        _within(g, *ref[name], f"{case} {name}")
        assert torch.equal(g, g2), f"{case} {name}: two runs differ"


@gpu
def test_cross_attention_gradient_against_differences():
    """<grad, d> against (L(x + e d) - L(x - e d)) / 2e of the fp64 form, L = <o, do>: the
    kernel's own bound on each gradient, summed over the direction, plus the difference's e^2."""
    q, k, v, do, lens = _attention_inputs("key_tail", seed=20)
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(train.cross_attention(*leaves, _lens_gpu(lens)), leaves, do.cuda())
    ref = orc.cross_attention_grads(q, k, v, do, lens)
    for i, name in enumerate(("dq", "dk", "dv")):
        d = torch.randn(leaves[i].shape, generator=torch.Generator().manual_seed(30 + i)).double()

        def loss(e):
            t = [q.double(), k.double(), v.double()]
            t[i] = t[i] + e * d
            return (orc.cross_attention(*t, lens)[0] * do.double()).sum().item()

        slope = (loss(1e-4) - loss(-1e-4)) / 2e-4
        got = (grads[i].cpu().double() * d).sum().item()
        assert abs(got - slope) <= (ref[name][1] * d.abs()).sum().item() + 1e-4 * abs(slope), (name, got, slope)


@gpu
@pytest.mark.parametrize("fill", [float("nan"), float("inf"), -float("inf"), torch.finfo(BF16).min])
def test_cross_attention_ignores_what_masked_states_hold(fill):
    for case in ("key_tail", "empty_rows", "one_token_split", "many_groups"):
        q, k, v, do, lens = _attention_inputs(case, seed=40)
        kp, vp = k.clone(), v.clone()
        for b, n in enumerate(lens):
            kp[b, :, n:] = fill
            vp[b, :, n:] = fill
        runs = []
        for kk, vv in ((k, v), (kp, vp)):
            leaves = [t.cuda().requires_grad_(True) for t in (q, kk, vv)]
            o = train.cross_attention(*leaves, _lens_gpu(lens))
            runs.append((o.detach(), *torch.autograd.grad(o, leaves, do.cuda())))
        _ok()
        for name, a, b in zip(("o", "dq", "dk", "dv"), *runs):
            assert torch.equal(a, b), f"{case} {name}"


@gpu
def test_cross_attention_layouts():
    """Head views of one projection, head-major tensors, a broadcast batch, an unaligned base,
    size-1 dimensions with odd strides: the same bits as contiguous copies."""
    B, H, Lq, Lk = 2, 4, 150, 200
    q, do = _randn(B, Lq, H, 128, seed=1).cuda().transpose(1, 2), _randn(B, H, Lq, 128, seed=2).cuda()
    kv = _randn(B, Lk, 2, H, 128, seed=3).cuda()
    odd = torch.empty(B * H * Lk * 128 + 3, device="cuda", dtype=BF16)[3:].view(B, H, Lk, 128)
    odd.copy_(kv[:, :, 0].transpose(1, 2))
    views = {
        "packed": (q, kv[:, :, 0].transpose(1, 2), kv[:, :, 1].transpose(1, 2)),
        "broadcast": (q, kv[:1, :, 0].transpose(1, 2).expand(B, -1, -1, -1), kv[:1, :, 1].transpose(1, 2).expand(B, -1, -1, -1)),
        "one_head": (q[:, :1], kv[:, :, 0, :1].transpose(1, 2), kv[:, :, 1, :1].transpose(1, 2)),
        "unaligned": (q, odd, odd),
        "every_other": (q[:, ::2], kv[:, ::2, 0, ::2].transpose(1, 2), kv[:, ::2, 1, ::2].transpose(1, 2)),
        "odd_size_one": (torch.as_strided(q, (1, 1, Lq, 128), (3, 5, H * 128, 1)), kv[:1, :, 0, :1].transpose(1, 2),
                         torch.as_strided(kv, (1, 1, Lk, 128), (0, 7, 2 * H * 128, 1))),
    }
    for name, ts in views.items():
        d = do[: ts[0].shape[0], : ts[0].shape[1]]
        got = []
        for make in (lambda t: t, lambda t: t.contiguous()):
            leaves = [make(t).detach().requires_grad_(True) for t in ts]
            o = train.cross_attention(*leaves)
            got.append((o.detach(), *torch.autograd.grad(o, leaves, d)))
        _ok()
        for a, b in zip(*got):
            assert torch.equal(a, b), name


@gpu
def test_cross_attention_gradients_of_a_broadcast_input():
    """One sequence of states for the whole batch: its gradient is the sum over the batch."""
    B, H, Lq, Lk = 3, 2, 40, 90
    q, k, do = _randn(B, H, Lq, 128, seed=1), _randn(1, H, Lk, 128, seed=2), _randn(B, H, Lq, 128, seed=3)
    v = _randn(1, H, Lk, 128, seed=4)
    kg, vg = k.cuda().requires_grad_(True), v.cuda().requires_grad_(True)
    o = train.cross_attention(q.cuda(), kg.expand(B, -1, -1, -1), vg.expand(B, -1, -1, -1))
    dk, dv = torch.autograd.grad(o, (kg, vg), do.cuda())
    ref = orc.cross_attention_grads(q, k.expand(B, -1, -1, -1), v.expand(B, -1, -1, -1), do)
    for name, g in (("dk", dk), ("dv", dv)):
        r, tol = ref[name]
        r = r.sum(0, keepdim=True)
        # autograd adds the B bf16 gradients in bf16: B - 1 more roundings at the magnitude of the sum
        _within(g, r, tol.sum(0, keepdim=True) + B * orc.BF16_HALF * ref[name][0].abs().sum(0, keepdim=True), name)


@gpu
def test_cross_attention_streams_and_graph():
    """On a stream of its own, two calls at once on two streams, and captured and replayed with new
    inputs: the eager bits."""
    q, k, v, do, lens = _attention_inputs("one_token_split", seed=50)
    q, k, v, do, lens = q.cuda(), k.cuda(), v.cuda(), do.cuda(), _lens_gpu(lens)

    def step(q, k, v, do):
        leaves = [t.detach().requires_grad_(True) for t in (q, k, v)]
        o = train.cross_attention(*leaves, lens)
        return (o.detach(), *torch.autograd.grad(o, leaves, do))

    want = step(q, k, v, do)
    want2 = step(q * 2, k, v, do)
    s1, s2 = torch.cuda.Stream(), torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        a = step(q, k, v, do)
    with torch.cuda.stream(s2):
        b = step(q * 2, k, v, do)
    torch.cuda.synchronize()
    for x, y in zip(a + b, want + want2):
        assert torch.equal(x, y)
    buf = [t.clone() for t in (q, k, v, do)]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step(*buf)
    torch.cuda.current_stream().wait_stream(s)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = step(*buf)
    g.replay()
    torch.cuda.synchronize()
    for x, y in zip(out, want):
        assert torch.equal(x, y)
    buf[0].copy_(q * 2)
    g.replay()
    torch.cuda.synchronize()
    for x, y in zip(out, want2):
        assert torch.equal(x, y)
    _ok()


@gpu
def test_cross_attention_long_offsets():
    """States whose offsets pass 2^31 elements: the last head of a [1, L, H, 128] tensor of 2.2e9 elements."""
    H, Lk = 40, 430000
    k = torch.zeros(1, Lk, H, 128, device="cuda", dtype=BF16)
    assert k.numel() > 2 ** 31
    k[:, :, H - 1].copy_(torch.randn(1, Lk, 128, device="cuda", generator=torch.Generator("cuda").manual_seed(1)))
    kh = k.transpose(1, 2)[:, H - 1:]
    q = _randn(1, 1, 5, 128, seed=5).cuda()
    o = ops.cross_attention(q, kh, kh)
    _ok()
    p = torch.softmax(q.double() @ kh.double().transpose(2, 3) / 128 ** 0.5, -1)
    ref, mag = p @ kh.double(), p @ kh.double().abs()
    _within(o, ref.cpu(), (orc.BF16_HALF * (mag + ref.abs()) * 1.01 + orc.FP32 * mag).cpu(), "o")


@gpu
def test_cross_attention_long_rows():
    """Rows whose offsets pass 2^31 elements, against one state: o is v, and dv the sum of dO's rows."""
    L = (1 << 24) + 70
    q = torch.zeros(1, 1, L, 128, device="cuda", dtype=BF16)
    assert q.numel() > 2 ** 31
    q[:, :, -300:] = _randn(300, 128, seed=6).cuda()
    q.requires_grad_(True)
    k, v = (_randn(1, 1, 1, 128, seed=s).cuda().requires_grad_(True) for s in (7, 8))
    do = torch.zeros_like(q)
    do[:, :, -1] = _randn(128, seed=9).cuda()
    o = train.cross_attention(q, k, v)
    assert bool((o[:, :, -300:] == v).all()) and bool((o[:, :, ::4096] == v).all())
    dq, dk, dv = torch.autograd.grad(o, (q, k, v), do)
    _ok()
    assert torch.equal(dv[0, 0, 0], do[0, 0, -1])
    # dS = P (dP - delta): the same sum of 128 products twice, in fp32 in two orders
    eps = 2 * 128 * 2.0 ** -24 * (do[0, 0, -1].float() * v[0, 0, 0].float()).abs().sum().item()
    assert bool((dq[:, :, :-1] == 0).all())
    assert bool((dq[0, 0, -1].float().abs() <= eps * k[0, 0, 0].float().abs() * 128 ** -0.5 * 1.01).all())
    assert bool((dk[0, 0, 0].float().abs() <= eps * q[0, 0, -1].float().abs() * 128 ** -0.5 * 1.01).all())


@gpu
def test_norm_and_product_long_offsets():
    """Rows whose offsets pass 2^31 elements: the bits of a call on the last rows alone."""
    M, K = 140000, 16384
    x = torch.zeros(M, K, device="cuda", dtype=BF16)
    assert x.numel() > 2 ** 31
    x[-3:] = _randn(3, K, seed=1).cuda()
    w = _randn(K, seed=2).cuda()
    y, h = ops.add_rms_norm(x, w, 1e-6, x)
    y1, h1 = ops.add_rms_norm(x[-3:], w, 1e-6, x[-3:])
    assert torch.equal(y[-3:], y1) and torch.equal(h[-3:], h1) and bool((y[:: M // 7] == 0).all())
    rstd = torch.ones(M, device="cuda")
    dx, _, _ = ops.add_rms_norm_bwd(h, w, rstd, x, None, BF16, None, need_dw=False)
    assert torch.equal(dx[-3:], ops.add_rms_norm_bwd(h1, w, rstd[:3], x[-3:], None, BF16, None, need_dw=False)[0])
    del y, h, dx
    yq, s, _ = ops.add_rms_norm_e4m3(x, w)
    y1, s1, _ = ops.add_rms_norm_e4m3(x[-3:], w)
    assert torch.equal(yq[-3:].view(torch.uint8), y1.view(torch.uint8)) and torch.equal(s[-3:], s1)
    del x, yq
    (xq, xs), (wq, ws) = _quantized(200, 128, 1, 1), _quantized(32768, 128, 128, 2)
    xq, xs, wq, ws = _cuda(xq, xs, wq, ws)
    many = 70000
    tall = torch.zeros(many + 200, 128, device="cuda", dtype=torch.uint8)
    tall[many:] = xq.view(torch.uint8)
    out = ops.gemm_fp8_block(tall.view(E4M3), torch.cat([xs.new_ones(many, 1), xs]), wq, ws)
    assert out.numel() > 2 ** 31
    assert torch.equal(out[-200:], ops.gemm_fp8_block(xq, xs, wq, ws)) and bool((out[: many: 997] == 0).all())
    _ok()


@gpu
def test_norm_and_product_streams_and_graphs():
    """Two calls at once on two streams, and two captured graphs replayed in turn with new inputs: the eager bits."""
    xs = [_randn(257, 1536, seed=1 + i).cuda() for i in range(2)]
    res = [_randn(257, 1536, seed=5 + i, dtype=F32).cuda() for i in range(2)]
    w = (1 + 0.2 * _randn(1536, seed=3, dtype=F32)).cuda()
    wq, ws = ops.quantize_tiles_e4m3(_randn(520, 1536, seed=4).cuda())
    dy = _randn(257, 1536, seed=7).cuda()

    def step(x, r):
        leaves = [t.detach().requires_grad_(True) for t in (x, w, r)]
        y, h = train.add_rms_norm(leaves[0], leaves[1], 1e-6, leaves[2])
        yq, ys, _ = ops.add_rms_norm_e4m3(x, w, 1e-6, r)
        few = [ops.gemm_fp8_block(yq[:n], ys[:n], wq, ws) for n in (1, 257)]
        return (y.detach(), h.detach(), *few, *torch.autograd.grad((y, h), leaves, (dy, r)))

    want = [step(x, r) for x, r in zip(xs, res)]
    side = [torch.cuda.Stream() for _ in xs]
    torch.cuda.synchronize()
    got = []
    for s, x, r in zip(side, xs, res):
        with torch.cuda.stream(s):
            got.append(step(x, r))
    torch.cuda.synchronize()
    for a, b in zip(got, want):
        assert all(torch.equal(t, u) for t, u in zip(a, b))
    graphs = []
    for x, r in zip(xs, res):
        buf, g = (x.clone(), r.clone()), torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step(*buf)
        graphs.append((g, buf, out))
    for turn in range(2):
        for i, (g, buf, _) in enumerate(graphs):
            buf[0].copy_(xs[(i + turn) % 2])
            buf[1].copy_(res[(i + turn) % 2])
            g.replay()
        torch.cuda.synchronize()
        for i, (_, _, out) in enumerate(graphs):
            assert all(torch.equal(t, u) for t, u in zip(out, want[(i + turn) % 2]))
    _ok()


@gpu
def test_cross_attention_no_rows_or_states():
    z = lambda *s: torch.zeros(*s, device="cuda", dtype=BF16)  # noqa: E731
    assert ops.cross_attention(z(2, 3, 0, 128), z(2, 3, 5, 128), z(2, 3, 5, 128)).shape == (2, 3, 0, 128)
    q = _randn(2, 3, 4, 128, seed=1).cuda().requires_grad_(True)
    k = z(2, 3, 0, 128).requires_grad_(True)
    o = train.cross_attention(q, k, k)
    assert bool((o == 0).all())
    dq, dk = torch.autograd.grad(o.sum(), (q, k))
    assert bool((dq == 0).all()) and dk.shape == k.shape


@gpu
@pytest.mark.parametrize("order", ["rising", "falling", "one_late_peak"])
def test_cross_attention_running_maximum(order):
    """Row maxima that grow by more than 2^8 from tile to tile (and within one), fall, or come with
    one late key: the rescaling of O and l, in the forward and through its log-sum-exp in the backward."""
    B, H, Lq, Lk = 1, 2, 150, 700
    q, k, v, do = (_randn(B, H, n, 128, seed=80 + i, dtype=F32) for i, n in enumerate((Lq, Lk, Lk, Lq)))
    u = torch.nn.functional.normalize(torch.ones(128), dim=0)
    q = q * 0.3 + 8 * u
    grow = torch.arange(Lk) / Lk * 40 if order == "rising" else torch.arange(Lk, 0, -1) / Lk * 40
    if order == "one_late_peak":
        grow = torch.where(torch.arange(Lk) == Lk - 3, 30.0, 0.0)
    k = k * 0.3 + grow[:, None] * u  # scores up to about 8 * 40 / sqrt(128): 28, or 41 in powers of two
    q, k, v, do = (t.to(BF16) for t in (q, k, v, do))
    leaves = [t.cuda().requires_grad_(True) for t in (q, k, v)]
    o = train.cross_attention(*leaves)
    grads = torch.autograd.grad(o, leaves, do.cuda())
    _ok()
    ref, _, tol = orc.cross_attention_bound(q, k, v)
    _within(o, ref, tol, "o")
    bounds = orc.cross_attention_grads(q, k, v, do)
    for name, g in zip(("dq", "dk", "dv"), grads):
        _within(g, *bounds[name], name)


@gpu
def test_sublayer_operators_under_torch_compile():
    """The custom operators' fake kernels agree with the real ones in shape, type and layout."""
    q, k, v, _, lens = _attention_inputs("key_tail")
    x, r, w, eps = _norm_inputs("heads_12")
    (xq, xs), (wq, ws) = _quantized(40, 256, 1, 1), _quantized(64, 256, 128, 2)
    t = torch.ops.rola_b200
    for op, args in (
        (t.cross_attention, (*_cuda(q, k, v), _lens_gpu(lens))),
        (t.cross_attention, (*_cuda(q, k, v), None)),
        (t.add_rms_norm, (*_cuda(x, r, w), eps)),
        (t.add_rms_norm_e4m3, (*_cuda(x, r, w), eps)),
        (t.add_rms_norm_e4m3, (*(c.view(257, 2, 768) for c in _cuda(x, r)), w.cuda()[:768], eps)),
        (t.quantize_blocks_e4m3, _cuda(x)),
        (t.gemm_fp8_block, (*_cuda(xq, xs, wq, ws), None)),
    ):
        # (the schema test computes on its inputs and outputs, which e4m3 does not support)
        e4m3 = any(t.dtype is E4M3 for t in (args[0], *torch.utils._pytree.tree_leaves(op(*args))))
        torch.library.opcheck(op.default, args, test_utils=("test_faketensor",) if e4m3 else ("test_schema", "test_faketensor"))
    _ok()


# --------------------------------------------------------------------- norm
NORM = {
    # M, K, x, residual, weight
    "one_row": (1, 8, BF16, None, BF16),
    "narrow": (77, 40, BF16, BF16, BF16),
    "warp_rows": (130, 256, F32, F32, F32),
    "warp_rows_4": (9, 1000, BF16, F32, F32),
    "cta_rows": (33, 1032, F32, BF16, BF16),
    "heads_12": (257, 1536, BF16, BF16, BF16),
    "heads_40": (301, 5120, BF16, F32, F32),
    "heads_40_bf16": (3, 5120, BF16, BF16, BF16),
    "widest": (5, 16384, F32, None, F32),
    "many_rows": (9001, 128, BF16, BF16, F32),
}


def _norm_inputs(case, seed=0):
    M, K, xt, rt, wt = NORM[case]
    x = _randn(M, K, seed=seed, dtype=xt)
    r = None if rt is None else (_randn(M, K, seed=seed + 1, dtype=F32) * 3).to(rt)
    w = (1 + 0.2 * _randn(K, seed=seed + 2, dtype=F32)).to(wt)
    return x, r, w, 1e-6


def _cuda(*ts):
    return [None if t is None else t.cuda() for t in ts]


@gpu
@pytest.mark.parametrize("case", sorted(NORM))
def test_add_rms_norm(case):
    x, r, w, eps = _norm_inputs(case)
    xg, rg, wg = _cuda(x, r, w)
    rstd = torch.empty(x.shape[0], device="cuda")
    y, h = ops.add_rms_norm(xg, wg, eps, rg, rstd=rstd)
    _ok()
    h_ref, y_ref, r_ref = orc.add_rms_norm(x, w, eps, r)
    assert torch.equal(h.cpu(), h_ref) and h.dtype == h_ref.dtype
    _within(rstd[:, None], r_ref, orc.FP32 * r_ref, "rstd")
    _within(y, y_ref, (orc.BF16_HALF + orc.FP32) * y_ref.abs() * 1.01, "y")


@gpu
@pytest.mark.parametrize("block", [128, None])
@pytest.mark.parametrize("case", sorted(NORM))
def test_add_rms_norm_e4m3(case, block):
    x, r, w, eps = _norm_inputs(case, seed=5)
    yq, scale, h = ops.add_rms_norm_e4m3(*_cuda(x, w), eps, *_cuda(r), block=block)
    _ok()
    h_ref, y_ref, _ = orc.add_rms_norm(x, w, eps, r)
    assert torch.equal(h.cpu(), h_ref)
    s_ref = orc.block_scales(y_ref, block)
    s = scale.cpu().double().view(x.shape[0], -1)
    _within(s, s_ref, orc.FP32 * s_ref, "scale")
    full = orc.spread(s, x.shape[1], block)
    tol = torch.maximum(2.0 ** -4 * y_ref.abs(), 2.0 ** -10 * full) * 1.001 + orc.FP32 * full * 448
    _within(yq.cpu().double() * full, y_ref, tol, "yq")
    # a block's largest value is held at 448
    assert (yq.cpu().double().abs().view(x.shape[0], -1).amax(1) == 448).all()


@gpu
@pytest.mark.parametrize("case", sorted(NORM))
def test_add_rms_norm_backward(case):
    x, r, w, eps = _norm_inputs(case, seed=9)
    dy = _randn(*x.shape, seed=20)
    dh = None if r is None else _randn(*x.shape, seed=21, dtype=r.dtype)
    leaves = [t for t in (x, w, r) if t is not None]
    leaves = [t.cuda().requires_grad_(True) for t in leaves]
    y, h = train.add_rms_norm(leaves[0], leaves[1], eps, leaves[2] if r is not None else None)
    outs, gs = ((y, h), (dy.cuda(), dh.cuda())) if r is not None else ((y,), (dy.cuda(),))
    grads = torch.autograd.grad(outs, leaves, gs, retain_graph=True)
    again = torch.autograd.grad(outs, leaves, gs)
    _ok()
    d, mag, dw, dw_mag = orc.add_rms_norm_grads(x, w, eps, dy, r, dh)

    def tol(t, ref, m):
        return orc.FP32 * m + (orc.BF16_HALF * 1.01 * ref.abs() if t.dtype == BF16 else 0)

    _within(grads[0], d, tol(x, d, mag), "dx")
    _within(grads[1], dw, tol(w, dw, dw_mag), "dw")
    if r is not None:
        _within(grads[2], d, tol(r, d, mag), "dres")
    for a, b in zip(grads, again):
        assert torch.equal(a, b)


@gpu
def test_add_rms_norm_partial_gradients():
    """One of the two outputs unused, or no gradient asked of the weight."""
    x, r, w, eps = _norm_inputs("heads_12")
    dy, dh = _randn(*x.shape, seed=30), _randn(*x.shape, seed=31)
    xg, rg = x.cuda().requires_grad_(True), r.cuda().requires_grad_(True)
    y, h = train.add_rms_norm(xg, w.cuda(), eps, rg)
    gy = torch.autograd.grad(y, (xg, rg), dy.cuda(), retain_graph=True)
    gh = torch.autograd.grad(h, (xg, rg), dh.cuda())
    d, mag, _, _ = orc.add_rms_norm_grads(x, w, eps, dy, r)
    for g in gy:
        _within(g, d, orc.FP32 * mag + orc.BF16_HALF * 1.01 * d.abs(), "dy only")
    for g in gh:
        assert torch.equal(g.cpu(), dh)


@gpu
def test_add_rms_norm_gradient_against_differences():
    x, r, w, eps = _norm_inputs("narrow", seed=60)
    dy, dh = _randn(*x.shape, seed=61), _randn(*x.shape, seed=62)
    leaves = [t.cuda().requires_grad_(True) for t in (x, w, r)]
    grads = torch.autograd.grad(train.add_rms_norm(leaves[0], leaves[1], eps, leaves[2]), leaves, (dy.cuda(), dh.cuda()))
    h0 = orc.add_rms_norm(x, w, eps, r)[0].double()

    def loss(h, w):
        u = h * (h.square().mean(-1, keepdim=True) + eps).rsqrt()
        return ((u * w * dy.double()).sum() + (h * dh.double()).sum()).item()

    d, mag, dw, dw_mag = orc.add_rms_norm_grads(x, w, eps, dy, r, dh)
    dirs = [torch.randn(t.shape, generator=torch.Generator().manual_seed(70 + i)).double() for i, t in enumerate((x, w))]
    slope_h = (loss(h0 + 1e-5 * dirs[0], w.double()) - loss(h0 - 1e-5 * dirs[0], w.double())) / 2e-5
    slope_w = (loss(h0, w.double() + 1e-5 * dirs[1]) - loss(h0, w.double() - 1e-5 * dirs[1])) / 2e-5
    for g, slope, dd, ref, m in ((grads[0], slope_h, dirs[0], d, mag), (grads[2], slope_h, dirs[0], d, mag),
                                 (grads[1], slope_w, dirs[1], dw, dw_mag)):
        bound = ((orc.FP32 * m + orc.BF16_HALF * 1.01 * ref.abs()) * dd.abs()).sum().item() + 1e-5 * abs(slope)
        assert abs((g.cpu().double() * dd).sum().item() - slope) <= bound


@gpu
def test_add_rms_norm_layouts_and_extremes():
    base = _randn(64, 3, 520, seed=1).cuda()
    w = torch.ones(512, device="cuda")
    views = [base[:, 1, :512], base[:, 1, 8:], base[:, 1, 4:516], base[::2, :, :512]]
    for v in views:
        y, _ = ops.add_rms_norm(v, w)
        y2, _ = ops.add_rms_norm(v.contiguous(), w)
        assert y.shape == v.shape and torch.equal(y, y2)
    yq, s, _ = ops.add_rms_norm_e4m3(views[3], w)
    assert s.shape == (32, 3, 4) and yq.shape == views[3].shape
    # zero rows: y 0, scale 1e-12; a NaN stays in its row and its scale
    x = torch.zeros(4, 512, device="cuda", dtype=BF16)
    x[2, 7] = float("nan")
    x[3] = torch.finfo(BF16).max / 64  # squares beyond fp32: the row factor is 0, as the fp32 formula gives
    yq, s, _ = ops.add_rms_norm_e4m3(x, w)
    assert bool((yq[:2].float() == 0).all()) and bool((s[:2] == torch.tensor(1e-12)).all())
    assert bool(yq[2].float().isnan().all()) and bool(s[2].isnan().all())
    assert bool((ops.add_rms_norm(x, w)[0][3] == 0).all())
    e = torch.empty(0, 512, device="cuda", dtype=BF16)
    assert ops.add_rms_norm(e, w)[0].shape == (0, 512)
    assert ops.add_rms_norm_e4m3(e, w)[1].shape == (0, 4)
    _ok()


# ------------------------------------------------------------------ product
PRODUCT = {
    # M, N, K, bias
    "smallest": (1, 8, 16, True),
    "one_row": (1, 1000, 5120, True),
    "few_rows": (7, 136, 144, False),
    "rows_17": (17, 264, 1040, True),
    "rows_33": (33, 520, 400, False),
    "tile_tails": (129, 136, 272, True),
    "rows_300": (300, 1032, 1536, True),
    "rows_16_narrow": (16, 1536, 1536, False),
    "rows_16_wide": (16, 9000, 400, True),
    "tall": (2049, 24, 128, False),
    "many_tiles": (1500, 2600, 656, True),
    # rounds of narrow tiles; whole rounds of wide tiles and the rest as narrow ones, shared by CTAs or not
    "narrow_rounds": (12524, 384, 144, True),
    "rest_shared": (1300, 3904, 2064, True),
    "rest_not_shared": (4990, 5000, 400, False),
    # a tile shared by 2, 3 and 4 CTAs, even and uneven runs of K blocks
    "shared_by_2": (130, 3800, 2064, True),
    "shared_by_3": (100, 5000, 3088, False),
    "shared_by_4": (200, 1000, 4112, True),
    # several tiles a CTA, of both widths
    "persistent_narrow": (2000, 2600, 144, True),
    "persistent_wide": (3500, 2560, 272, False),
}


def _quantized(M, K, rows, seed):
    """e4m3 values of wide range and fp32 scales of a [M, K] operand (scales per ``rows`` x 128)."""
    g = torch.Generator().manual_seed(seed)
    q = (torch.randn(M, K, generator=g) * 60).clamp(-448, 448).to(E4M3)
    s = torch.exp(torch.randn((M + rows - 1) // rows, (K + 127) // 128, generator=g)) * 0.01
    return q, s


@gpu
@pytest.mark.parametrize("case", sorted(PRODUCT))
def test_gemm_fp8_block(case):
    M, N, K, has_bias = PRODUCT[case]
    (xq, xs), (wq, ws) = _quantized(M, K, 1, 1), _quantized(N, K, 128, 2)
    bias = _randn(N, seed=3) if has_bias else None
    out = ops.gemm_fp8_block(*_cuda(xq, xs, wq, ws, bias))
    _ok()
    ref, tol = orc.gemm_fp8_block(xq, xs, wq, ws, bias)
    _within(out, ref, tol, case)
    # the scales' layout does not change the bits, nor do other rows of the batch
    xs_t = xs.cuda().t().contiguous().t()
    assert torch.equal(out, ops.gemm_fp8_block(xq.cuda(), xs_t, *_cuda(wq, ws, bias)))


@gpu
@pytest.mark.parametrize("case", ["shared_by_4", "rest_shared"])
def test_gemm_fp8_block_shared_tiles_on_streams_and_in_a_graph(case):
    """Tiles whose K blocks several CTAs share: two calls at once, and captured and replayed with new operands."""
    M, N, K, _ = PRODUCT[case]
    ops1, ops2 = (_cuda(*_quantized(M, K, 1, 10 + i), *_quantized(N, K, 128, 20 + i)) for i in range(2))
    want = [ops.gemm_fp8_block(*o) for o in (ops1, ops2)]
    side = [torch.cuda.Stream(), torch.cuda.Stream()]
    torch.cuda.synchronize()
    got = []
    for s, o in zip(side, (ops1, ops2)):
        with torch.cuda.stream(s):
            got.append([ops.gemm_fp8_block(*o) for _ in range(4)][-1])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    buf, g = [t.clone() for t in ops1], torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = ops.gemm_fp8_block(*buf)
    for o, w in ((ops1, want[0]), (ops2, want[1])):
        for b, t in zip(buf, o):
            b.copy_(t)
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, w)
    _ok()


@gpu
def test_gemm_fp8_block_nan_stays_in_its_row():
    (xq, xs), (wq, ws) = _quantized(200, 256, 1, 1), _quantized(64, 256, 128, 2)
    xs[5, 1] = float("nan")
    out = ops.gemm_fp8_block(*_cuda(xq, xs, wq, ws))
    assert bool(out[5].isnan().all()) and int(out.isnan().sum()) == 64
    _ok()


@gpu
def test_quantize_blocks_and_tiles():
    for dtype in (BF16, F32):
        for M, K in ((1, 8), (130, 264), (7, 5120), (300, 128)):
            x = _randn(M, K, seed=M, dtype=dtype)
            xq, s = ops.quantize_blocks_e4m3(x.cuda())
            s_ref = orc.block_scales(x.double(), 128)
            _within(s, s_ref, 2.0 ** -22 * s_ref, "scale")
            full = orc.spread(s.cpu().double(), K, 128)
            tol = torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * full) * 1.001
            _within(xq.cpu().double() * full, x.double(), tol, "xq")
            wq, ws = ops.quantize_tiles_e4m3(x.cuda())
            ref = torch.stack([r.abs().amax(0) for r in orc.block_scales(x.double(), 128).split(128, 0)])
            assert ws.shape == ((M + 127) // 128, (K + 127) // 128)
            _within(ws, ref, 2.0 ** -22 * ref, "tile scale")
            full = orc.spread(ws.cpu().double().repeat_interleave(128, 0)[:M], K, 128)
            tol = torch.maximum(2.0 ** -4 * x.double().abs(), 2.0 ** -10 * full) * 1.001
            _within(wq.cpu().double() * full, x.double(), tol, "wq")
    _ok()


# ----------------------------------------------------------------- together
@gpu
def test_sublayer_strings_together():
    """Residual + norm -> e4m3 -> projections -> attention to the states -> e4m3 -> output
    projection: every stage from the GPU's own previous one, against the fp64 form."""
    B, L, H, Lk, dim = 2, 150, 2, 77, 256
    x, res = _randn(B, L, dim, seed=1), _randn(B, L, dim, seed=2)
    ctx = _randn(B, Lk, dim, seed=3)
    w = (1 + 0.1 * _randn(dim, seed=4, dtype=F32)).to(BF16)
    lens = (77, 30)
    ws = [ops.quantize_tiles_e4m3((_randn(dim, dim, seed=5 + i) * dim ** -0.5).cuda()) for i in range(4)]
    yq, ys, h = ops.add_rms_norm_e4m3(*_cuda(x, w), 1e-6, *_cuda(res))
    cq, cs = ops.quantize_blocks_e4m3(ctx.cuda().view(-1, dim))

    def project(tq, ts, i):
        out = ops.gemm_fp8_block(tq, ts, *ws[i])
        ref, tol = orc.gemm_fp8_block(*(t.cpu() for t in (tq, ts, *ws[i])))
        _within(out, ref, tol, f"projection {i}")
        return out

    q = project(yq.view(-1, dim), ys.reshape(B * L, -1), 0).view(B, L, H, 128).transpose(1, 2)
    k = project(cq, cs, 1).view(B, Lk, H, 128).transpose(1, 2)
    v = project(cq, cs, 2).view(B, Lk, H, 128).transpose(1, 2)
    o = ops.cross_attention(q, k, v, _lens_gpu(lens))
    ref, _, tol = orc.cross_attention_bound(q.cpu(), k.cpu(), v.cpu(), lens)
    _within(o, ref, tol, "attention")
    out = project(*ops.quantize_blocks_e4m3(o.transpose(1, 2).reshape(B * L, dim)), 3)
    assert out.shape == (B * L, dim)
    _ok()


# ----------------------------------------------------------------- refusals
def _refused(match, fn, *a, **kw):
    with pytest.raises(ValueError, match=match):
        fn(*a, **kw)


def test_refuses_cpu_tensors():
    t = torch.zeros(1, 1, 4, 128, dtype=BF16)
    _refused("CUDA", ops.cross_attention, t, t, t)
    _refused("CUDA", ops.add_rms_norm, t, torch.ones(128))
    _refused("CUDA", ops.add_rms_norm_e4m3, t, torch.ones(128))
    _refused("CUDA", ops.quantize_blocks_e4m3, t[0, 0])
    _refused("CUDA", ops.quantize_tiles_e4m3, t[0, 0])
    _refused("CUDA", ops.gemm_fp8_block, t[0, 0], t[0, 0], t[0, 0], t[0, 0])
    for fn in (lambda: train.cross_attention(t, t, t), lambda: train.add_rms_norm(t, torch.ones(128))):
        with pytest.raises(RuntimeError, match="CUDA"):
            fn()


@gpu
def test_refuses_bad_arguments():
    z = lambda *s, dt=BF16: torch.zeros(*s, device="cuda", dtype=dt)  # noqa: E731
    q, k = z(2, 4, 8, 128), z(2, 4, 16, 128)
    _refused("128", ops.cross_attention, z(2, 4, 8, 64), k, k)
    _refused("bf16 q", ops.cross_attention, q.float(), k, k)
    _refused("multiple", ops.cross_attention, q, z(2, 3, 16, 128), z(2, 3, 16, 128))
    _refused("share a shape", ops.cross_attention, q, k, z(2, 4, 15, 128))
    _refused("share a shape", ops.cross_attention, q, z(1, 4, 16, 128), z(1, 4, 16, 128))
    _refused("kv_lens", ops.cross_attention, q, k, k, torch.ones(2, device="cuda", dtype=torch.int64))
    _refused("kv_lens", ops.cross_attention, q, k, k, torch.ones(3, device="cuda", dtype=torch.int32))
    _refused("CUDA", ops.cross_attention, q, k, k, torch.ones(2, dtype=torch.int32))
    o, lse = ops.cross_attention_fwd_lse(q, k, k)
    _refused("lse", ops.cross_attention_bwd, q, k, k, o, o, lse[:1])
    _refused("shape", ops.cross_attention_bwd, q, k, k, o, o[:, :2], lse)
    x, w = z(4, 256), torch.ones(256, device="cuda")
    _refused("multiple of 8", ops.add_rms_norm, z(4, 252), torch.ones(252, device="cuda"))
    _refused("16384", ops.add_rms_norm, z(1, 16392), torch.ones(16392, device="cuda"))
    _refused("residual", ops.add_rms_norm, x, w, 1e-6, z(3, 256))
    _refused("weight", ops.add_rms_norm, x, w[:8])
    _refused("required", ops.add_rms_norm, x.half(), w)
    _refused("rstd", ops.add_rms_norm, x, w, 1e-6, None, torch.zeros(3, device="cuda"))
    _refused("block", ops.add_rms_norm_e4m3, x, w, block=64)
    _refused("multiple of 8", ops.quantize_blocks_e4m3, z(4, 252))
    (xq, xs), (wq, ws) = (_cuda(*_quantized(4, 256, r, 1)) for r in (1, 128))
    wq = wq.repeat(4, 1)
    _refused("e4m3", ops.gemm_fp8_block, x, xs, wq, ws)
    _refused("does not match", ops.gemm_fp8_block, xq, xs, wq[:, :128].contiguous(), ws)
    _refused("x_scale", ops.gemm_fp8_block, xq, xs[:, :1], wq, ws)
    _refused("w_scale", ops.gemm_fp8_block, xq, xs, wq, ws.repeat(2, 1))
    _refused("multiple of 16", ops.gemm_fp8_block, xq, xs, wq[:12], ws)
    _refused("bias", ops.gemm_fp8_block, xq, xs, wq, ws, z(4))
    g = torch.ones(4, 256, device="cuda", dtype=BF16, requires_grad=True)
    y, _ = train.add_rms_norm(g, w)
    (d,) = torch.autograd.grad(y.float().square().sum(), g, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        d.sum().backward()


def test_c_entries_validate_without_gpu():
    """Bad arguments are refused on the host, before any launch; workspace sizes are 0 for bad sizes."""
    import ctypes

    lib = _lib.load_library()
    p, odd = ctypes.c_void_p(256), ctypes.c_void_p(258)
    inv = _lib.ROLA_ERR_INVALID

    def err():
        return lib.rola_b200_last_error()

    def norm(M=4, K=256, x=p, ld=256, res=None, h=None, y=p):
        return lib.rola_b200_add_rms_norm(x, 0, ld, res, 0, 256, p, 0, M, K, 1e-6, h, y, None, None)

    assert norm(K=252) == inv and b"multiple of 8" in err()
    assert norm(M=0) == inv and norm(ld=128) == inv and norm(x=odd) == inv and norm(y=None) == inv
    assert norm(res=p) == inv and b"go together" in err()
    assert lib.rola_b200_add_rms_norm_e4m3(p, 0, 256, None, 0, 0, p, 0, 4, 256, 1e-6, None, p, p, 2, 1, 64, None) == inv
    assert lib.rola_b200_add_rms_norm_bwd(p, 0, 256, p, 0, p, p, 256, None, 0, 0, 4, 256, p, 0, None, 0, p, p, 1, None) == inv
    assert b"workspace" in err()
    assert lib.rola_b200_add_rms_norm_bwd_workspace(4, 252) == 0 < lib.rola_b200_add_rms_norm_bwd_workspace(4, 256)
    gemm = lambda M, N, K, out=p: lib.rola_b200_gemm_fp8_block(p, p, 1, 4, p, p, None, out, M, N, K, None)  # noqa: E731
    assert gemm(4, 12, 256) == inv and gemm(4, 16, 250) == inv and gemm(0, 16, 256) == inv and gemm(4, 16, 256, odd) == inv

    def cross(B=1, H=2, Hkv=2, Lq=4, Lk=4, st=128, ws=None, nb=0):
        s = (1024, st, 256)
        return lib.rola_b200_cross_attn(p, *s, p, *s, p, *s, None, B, H, Hkv, Lq, Lk, p, *s, None, ws, nb, None)

    assert cross(Hkv=3) == inv and cross(Lq=0) == inv and cross(st=0) == inv and cross(st=-128) == inv and cross(st=12) == inv
    assert lib.rola_b200_cross_attn_workspace(1, 1, 1, 1, 100000) > 0
    assert cross(Lk=100000) == inv and b"workspace" in err()
    assert lib.rola_b200_cross_attn_workspace(1, 3, 2, 1, 100) == 0 == lib.rola_b200_cross_attn_bwd_workspace(0, 1, 1, 1, 1)
    assert lib.rola_b200_cross_attn_bwd_workspace(1, 1, 1, 1, 1) > 0
