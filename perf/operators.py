"""What the operators of a DiT block's cross-attention sublayer cost on a B200.

Three operators that such a sublayer strings together, each beside its kind in
this package: the root-mean-square norm with the residual's addition (output in
bf16, or in e4m3 with scales; forward and backward), the matrix product of e4m3
operands with one scale per block of 128, and the attention to an encoder's
states of another length (forward and backward).

``run`` computes a case in elementary torch operations in fp32 (``own`` false)
or calls this package (``own`` true); ``exact`` restates it in fp64.
"""

import math

import torch

own = False

D = 128  # head dim of every attention in this package
BLK = 128  # values that share a scale
EPS = 1e-6
DIM = 5120  # 40 heads of 128
BF16, F32, F64, E4M3 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
TYPES = {"bf16": BF16, "fp32": F32}

# the largest attention and product below: no drawn case costs more
MAX_SCORES = 40 * 32760 * 512
MAX_PRODUCT = 32760 * 15360 * 5120
MAX_NORM = 32760 * 5120


def listed():
    return [
        # --- attention to the encoder's states ---
        # a 480P video's 32760 tokens attend to 512 text states, 40 heads: one block of one denoising step
        {"name": "attend 480P to 512", "op": "attend", "train": False, "B": 1, "H": 40, "G": 1, "Lq": 32760, "Lk": 512,
         "lens": ""},
        # conditional and unconditional prompt as a batch of two, unpadded lengths far apart
        {"name": "attend two prompts", "op": "attend", "train": False, "B": 2, "H": 12, "G": 1, "Lq": 32760, "Lk": 512,
         "lens": "387,1"},
        # one new token per sequence over long states, five query heads to a key head: latency and bandwidth
        {"name": "attend one token", "op": "attend", "train": False, "B": 4, "H": 40, "G": 5, "Lq": 1, "Lk": 8190,
         "lens": "8190,511,4097,6000"},
        # a training step of the attention on a small clip
        {"name": "attend train clip", "op": "attend", "train": True, "B": 1, "H": 12, "G": 1, "Lq": 1536, "Lk": 257,
         "lens": ""},
        # a training step at 480P
        {"name": "attend train 480P", "op": "attend", "train": True, "B": 1, "H": 40, "G": 1, "Lq": 32760, "Lk": 512,
         "lens": ""},
        # --- norm with the residual's addition ---
        # a few rows in a serving loop, straight to e4m3: latency
        {"name": "norm e4m3 4 rows", "op": "norm", "train": False, "M": 4, "K": DIM, "x": "bf16", "res": "bf16",
         "out": "block"},
        # every token of a 480P video, e4m3 with a scale per 128 values for the product below
        {"name": "norm e4m3 480P", "op": "norm", "train": False, "M": 32760, "K": DIM, "x": "bf16", "res": "bf16",
         "out": "block"},
        # the same in bf16 at the width of the 12-head model, on an odd number of rows
        {"name": "norm bf16 12 heads", "op": "norm", "train": False, "M": 16381, "K": 1536, "x": "bf16", "res": "bf16",
         "out": "bf16"},
        # a training step: bf16 branch added to an fp32 residual stream, gradients of both and of the weight
        {"name": "norm train 480P", "op": "norm", "train": True, "M": 32760, "K": DIM, "x": "bf16", "res": "fp32",
         "out": "bf16"},
        # --- product with a scale per block of 128 ---
        # one row through the QKV projection: reads the weight once
        {"name": "product 1 row", "op": "product", "M": 1, "N": 15360, "K": DIM, "bias": True},
        # an encoder's states through a projection, odd number of rows
        {"name": "product 1001 rows", "op": "product", "M": 1001, "N": DIM, "K": DIM, "bias": True},
        # every token of a 480P video through the QKV projection
        {"name": "product 480P", "op": "product", "M": 32760, "N": 15360, "K": DIM, "bias": True},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["attend", "attend", "norm", "product"])
    if op == "attend":
        while True:
            G, Hkv = rng.choice([1, 1, 1, 2, 5, 8]), rng.choice([1, 2, 5, 8, 12, 40])
            B, Lq, Lk = rng.randint(1, 6), _log(rng, 1, 32760), _log(rng, 1, 8192)
            # over a single key the gradients of q and k vanish: a training step has two at least
            train = rng.random() < 0.5 and Lk > 1
            if Hkv * G <= 40 and B * Hkv * G * Lq * Lk <= MAX_SCORES:
                break
        lens = ""
        if rng.random() < 0.6:
            lens = ",".join(str(rng.choice([0, 1, Lk, rng.randint(0, Lk), rng.randint(0, Lk), rng.randint(0, Lk)]))
                            for _ in range(B))
            if max(int(n) for n in lens.split(",")) < (2 if train else 1):
                lens = ",".join([str(Lk)] * B)
        return {"op": "attend", "train": train, "B": B, "H": Hkv * G, "G": G, "Lq": Lq, "Lk": Lk,
                "lens": lens}
    if op == "norm":
        while True:
            M, K = _log(rng, 1, 75600), 8 * _log(rng, 1, 1024)
            if M * K <= MAX_NORM:
                break
        train = rng.random() < 0.4
        return {"op": "norm", "train": train, "M": M, "K": K, "x": rng.choice(["bf16", "bf16", "fp32"]),
                "res": rng.choice(["bf16", "fp32", "none"]),
                "out": "bf16" if train else rng.choice(["bf16", "block", "row"])}
    while True:
        M, N, K = _log(rng, 1, 75600), 8 * _log(rng, 1, 1920), 16 * _log(rng, 1, 960)
        if M * N * K <= MAX_PRODUCT:
            break
    return {"op": "product", "M": M, "N": N, "K": K, "bias": rng.random() < 0.5}


def _lens(case):
    return [int(n) for n in case["lens"].split(",")] if case["lens"] else [case["Lk"]] * case["B"]


def _blocks(n):
    return -(-n // BLK)


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*shape, dtype=F32):
        return torch.randn(*shape, generator=g, device="cuda", dtype=F32).to(dtype)

    s = {"case": case}
    if case["op"] == "attend":
        # heads of token-major projections, as the sublayer's linears leave them
        B, H, Hkv = case["B"], case["H"], case["H"] // case["G"]

        def heads(L, n):
            return randn(B, L, n * D, dtype=BF16).view(B, L, n, D).transpose(1, 2)

        s["q"], s["k"], s["v"] = heads(case["Lq"], H), heads(case["Lk"], Hkv), heads(case["Lk"], Hkv)
        s["lens"] = torch.tensor(_lens(case), dtype=torch.int32, device="cuda") if case["lens"] else None
        if case["train"]:
            s["do"] = heads(case["Lq"], H)
            for n in "qkv":
                s[n].requires_grad_(True)
    elif case["op"] == "norm":
        M, K = case["M"], case["K"]
        s["x"] = randn(M, K, dtype=TYPES[case["x"]])
        s["res"] = None
        if case["res"] != "none":
            # a residual stream some blocks deep: larger than the branch, a few channels far larger
            res = randn(M, K).mul_(3.0)
            res[:, :: 97] *= 12.0
            s["res"] = res.to(TYPES[case["res"]])
        s["w"] = (1.0 + 0.2 * randn(K)).to(BF16 if not case["train"] else F32)
        if case["train"]:
            s["dy"] = randn(M, K, dtype=BF16)
            for n in ("x", "res", "w"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
            s["dh"] = None if s["res"] is None else randn(M, K, dtype=TYPES[case["res"]])
    else:
        M, N, K = case["M"], case["N"], case["K"]
        x = randn(M, K).mul_(torch.exp(0.5 * randn(M, 1)))
        w = randn(N, K).mul_(K ** -0.5)
        s["xq"], s["xs"] = _quantized(x, 1)
        s["wq"], s["ws"] = _quantized(w, BLK)
        # the scales of a row block lie side by side, as the quantising kernels leave them
        s["xs"] = s["xs"].t().contiguous().t()
        s["bias"] = randn(N, dtype=BF16) if case["bias"] else None
    return s


def _quantized(t, rows):
    """e4m3 values of ``t [M, K]`` with one scale per ``rows`` x 128 block, and the scales."""
    M, K = t.shape
    m, k = -(-M // rows), _blocks(K)
    p = torch.zeros(m * rows, k * BLK, device=t.device, dtype=F32)
    p[:M, :K] = t
    p = p.view(m, rows, k, BLK)
    scale = p.abs().amax((1, 3)) / 448.0 + 1e-12
    q = (p / scale[:, None, :, None]).clamp_(-448.0, 448.0).to(E4M3)
    return q.view(m * rows, k * BLK)[:M, :K].contiguous(), scale


def run(s):
    return {"attend": _attend, "norm": _norm, "product": _product}[s["case"]["op"]](s)


# --------------------------------------------------------------------- attention
def _attend(s):
    case, q, k, v, lens = s["case"], s["q"], s["k"], s["v"], s["lens"]
    if own:
        from sparkdiffusion_b200 import ops, train

        if not case["train"]:
            return {"o": ops.cross_attention(q, k, v, lens)}
        o = train.cross_attention(q, k, v, lens)
        dq, dk, dv = torch.autograd.grad(o, (q, k, v), s["do"])
        return {"o": o.detach(), "dq": dq, "dk": dk, "dv": dv}
    B, H, Lq, _ = q.shape
    Hkv, Lk, G = k.shape[1], k.shape[2], case["G"]
    with torch.no_grad():
        # the G query heads of a key head as rows of one product
        q32 = q.float().reshape(B, Hkv, G * Lq, D)
        k32, v32 = k.float(), v.float()
        p = (q32 @ k32.transpose(2, 3)).mul_(D ** -0.5)
        dead = None
        if lens is not None:
            dead = (torch.arange(Lk, device=q.device)[None, :] >= lens[:, None])[:, None, None, :]
            p.masked_fill_(dead, -math.inf)
        top = p.amax(-1, keepdim=True)
        p = p.sub_(torch.where(torch.isinf(top), 0.0, top)).exp_()
        p.div_(p.sum(-1, keepdim=True).clamp_min(1e-30))  # a row without keys: all zero
        o = p @ v32
        out = {"o": o.reshape(B, H, Lq, D).to(BF16)}
        if not case["train"]:
            return out
        do = s["do"].float().reshape(B, Hkv, G * Lq, D)
        out["dv"] = (p.transpose(2, 3) @ do).to(BF16)
        ds = do @ v32.transpose(2, 3)
        ds.sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(D ** -0.5)
        out["dk"] = (ds.transpose(2, 3) @ q32).to(BF16)
        out["dq"] = (ds @ k32).reshape(B, H, Lq, D).to(BF16)
        return out


# -------------------------------------------------------------------------- norm
def _norm(s):
    case, x, res, w = s["case"], s["x"], s["res"], s["w"]
    if own:
        from sparkdiffusion_b200 import ops, train

        if case["train"]:
            y, h = train.add_rms_norm(x, w, EPS, res)
            if res is None:
                dx, dw = torch.autograd.grad(y, (x, w), s["dy"])
                return {"y": y.detach(), "dx": dx, "dw": dw}
            dx, dres, dw = torch.autograd.grad((y, h), (x, res, w), (s["dy"], s["dh"]))
            return {"y": y.detach(), "h": h.detach(), "dx": dx, "dres": dres, "dw": dw}
        if case["out"] == "bf16":
            y, h = ops.add_rms_norm(x, w, EPS, res)
            out = {"y": y}
        else:
            yq, scale, h = ops.add_rms_norm_e4m3(x, w, EPS, res, block=BLK if case["out"] == "block" else None)
            out = {"y": yq, "scale": scale}
        return out if res is None else {**out, "h": h}
    with torch.no_grad():
        h = x if res is None else (x.float() + res.float()).to(res.dtype)  # the stream is kept in its own type
        h32, w32 = h.float(), w.float()
        rstd = torch.rsqrt(h32.square().mean(-1, keepdim=True) + EPS)
        unit = h32 * rstd
        y = unit * w32
        out = {} if res is None else {"h": h}
        if case["out"] == "bf16":
            out["y"] = y.to(BF16)
        else:
            M, K = y.shape
            k = _blocks(K) if case["out"] == "block" else 1
            span = BLK if case["out"] == "block" else K
            if k * span > K:
                p = torch.zeros(M, k * span, device=y.device)
                p[:, :K] = y
                y = p
            y = y.view(M, k, span)
            scale = y.abs().amax(-1) / 448.0 + 1e-12
            out["y"] = (y * (1.0 / scale)[..., None]).clamp_(-448.0, 448.0).view(M, k * span)[:, :K].to(E4M3)
            out["scale"] = scale if case["out"] == "block" else scale[:, 0]
        if case["train"]:
            dy = s["dy"].float()
            out["dw"] = (dy * unit).sum(0)
            g = dy.mul_(w32)
            dh = (g - unit * (g * unit).mean(-1, keepdim=True)) * rstd
            if res is not None:
                dh += s["dh"].float()
                out["dres"] = dh.to(res.dtype)
            out["dx"] = dh.to(x.dtype)
        return out


# ----------------------------------------------------------------------- product
def _product(s):
    if own:
        from sparkdiffusion_b200 import ops

        return {"out": ops.gemm_fp8_block(s["xq"], s["xs"], s["wq"], s["ws"], s["bias"])}
    K, N = s["xq"].shape[1], s["wq"].shape[0]
    x = s["xq"].float() * s["xs"].repeat_interleave(BLK, 1)[:, :K]
    w = s["wq"].float() * s["ws"].repeat_interleave(BLK, 0)[:N].repeat_interleave(BLK, 1)[:, :K]
    out = x @ w.t()
    if s["bias"] is not None:
        out += s["bias"].float()
    return {"out": out.to(BF16)}


# -------------------------------------------------------------------------- work
def work(case):
    if case["op"] == "attend":
        B, H, Hkv, Lq = case["B"], case["H"], case["H"] // case["G"], case["Lq"]
        keys = sum(_lens(case))
        rows, states = 2 * B * H * Lq * D, 2 * Hkv * keys * D
        if not case["train"]:  # q in, o out; k, v in; two products
            return {"bytes": 2 * rows + 2 * states, "flops": 4 * D * H * Lq * keys}
        # and do in, dq, dk, dv out; five more products
        return {"bytes": 4 * rows + 2 * states + 4 * B * Hkv * case["Lk"] * D, "flops": 14 * D * H * Lq * keys}
    if case["op"] == "norm":
        M, K = case["M"], case["K"]
        bx = 2 if case["x"] == "bf16" else 4
        br = {"bf16": 2, "fp32": 4, "none": 0}[case["res"]]
        by = 2 if case["out"] == "bf16" else 1
        per, extra = bx + 2 * br + by, 2 * K
        if case["out"] == "block":
            extra += 4 * M * _blocks(K)
        elif case["out"] == "row":
            extra += 4 * M
        if case["train"]:  # dy and dh in, dx and dres out, weight and its gradient in fp32
            per, extra = per + 2 + br + bx + br, 8 * K
        return {"bytes": M * K * per + extra, "flops": M * K * (16 if case["train"] else 6)}
    M, N, K = case["M"], case["N"], case["K"]
    return {"bytes": M * K + N * K + 2 * M * N + 4 * _blocks(K) * (M + _blocks(N)) + (2 * N if case["bias"] else 0),
            "flops": 2 * M * N * K}


# ------------------------------------------------------------------------- exact
def exact(case, seed):
    with torch.no_grad():
        s = {k: v.detach() if isinstance(v, torch.Tensor) else v for k, v in prepare(case, seed).items()}
        return {"attend": _exact_attend, "norm": _exact_norm, "product": _exact_product}[case["op"]](case, s)


def _exact_attend(case, s):
    """Head by head over the valid keys alone: softmax from the log-sum-exp, and its Jacobian."""
    q, k, v, G = s["q"], s["k"], s["v"], case["G"]
    o = torch.zeros(q.shape, dtype=F64, device="cuda")
    dq = torch.zeros(q.shape, dtype=F64, device="cuda") if case["train"] else None
    dk, dv = (torch.zeros(k.shape, dtype=F64, device="cuda") if case["train"] else None for _ in range(2))
    for b, n in enumerate(_lens(case)):
        if n == 0:
            continue
        for h in range(case["H"]):
            kk, vv, qq = k[b, h // G, :n].to(F64), v[b, h // G, :n].to(F64), q[b, h].to(F64)
            a = torch.einsum("id,jd->ij", qq, kk) / math.sqrt(D)
            w = torch.exp(a - torch.logsumexp(a, 1)[:, None])
            o[b, h] = torch.einsum("ij,jd->id", w, vv)
            if case["train"]:
                do = s["do"][b, h].to(F64)
                dv[b, h // G, :n] += torch.einsum("ij,id->jd", w, do)
                dw = torch.einsum("id,jd->ij", do, vv)
                da = w * (dw - torch.einsum("ij,ij->i", w, dw)[:, None]) / math.sqrt(D)
                dq[b, h] = torch.einsum("ij,jd->id", da, kk)
                dk[b, h // G, :n] += torch.einsum("ij,id->jd", da, qq)
    return {"o": o, "dq": dq, "dk": dk, "dv": dv} if case["train"] else {"o": o}


def _exact_norm(case, s):
    x, res, w = s["x"].to(F64), s["res"], s["w"].to(F64)
    h = x if res is None else (x + res.to(F64)).to(res.dtype).to(F64)
    n = torch.linalg.vector_norm(h, dim=1, keepdim=True)
    r = torch.sqrt(n * n / case["K"] + EPS)
    y = h / r * w
    out = {} if res is None else {"h": h}
    if case["out"] == "bf16":
        out["y"] = y
    else:
        parts = y.split(BLK if case["out"] == "block" else case["K"], 1)
        scales = [p.abs().max(1).values / 448.0 + 1e-12 for p in parts]
        out["y"] = torch.cat([(p / c[:, None]).float().to(E4M3).to(F64) for p, c in zip(parts, scales)], 1)
        out["scale"] = torch.stack(scales, 1) if case["out"] == "block" else scales[0]
    if case["train"]:
        dy = s["dy"].to(F64)
        out["dw"] = torch.einsum("mk,mk->k", dy, h / r)
        g = dy * w
        dh = g / r - h * (torch.einsum("mk,mk->m", g, h)[:, None] / (case["K"] * r ** 3))
        if res is not None:
            dh = dh + s["dh"].to(F64)
            out["dres"] = dh
        out["dx"] = dh
    return out


def _exact_product(case, s):
    M, N, K = case["M"], case["N"], case["K"]
    ws = s["ws"].to(F64)
    w = s["wq"].to(F64)
    for i in range(_blocks(N)):
        for j in range(_blocks(K)):
            w[i * BLK:(i + 1) * BLK, j * BLK:(j + 1) * BLK] *= ws[i, j]
    out = torch.empty(M, N, dtype=F64, device="cuda")
    col = torch.arange(K, device="cuda") // BLK
    for m in range(0, M, 4096):
        x = s["xq"][m:m + 4096].to(F64) * s["xs"][m:m + 4096].to(F64)[:, col]
        out[m:m + 4096] = x @ w.t()
    return {"out": out + s["bias"].to(F64) if s["bias"] is not None else out}
