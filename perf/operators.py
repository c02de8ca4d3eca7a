"""What the attention, layer norm and gradient clipping operators are timed on.

Each case is one pass of one operator: ``"op"`` is ``"attention"``
(``npf.ops.differential_attention``), ``"norm"`` (``npf.ops.layer_norm``) or
``"clip"`` (``npf.ops.clip_grad_norm_``).  ``own`` chooses between the plain
torch form and the framework's operator.
"""

import math

import torch

own = False

_TYPES = {
    "float32": torch.float32,
    "bfloat16": torch.bfloat16,
    "float16": torch.float16,
}


def listed():
    return [
        # -- differential attention ------------------------------------- #
        # training step of a 1D attentive model: 32 tasks, 50 contexts, 128
        # targets, r_dim 128 as 4 heads of two 16-wide maps; many tiny problems
        dict(name="attn 1d train fp32", op="attention", train=True,
             dtype="float32", B=32, H=4, Hk=4, Q=128, K=50, D=16, short=1.0),
        # self-attention over the 32x32 pixels of an image batch
        dict(name="attn image train bf16", op="attention", train=True,
             dtype="bfloat16", B=16, H=4, Hk=4, Q=1024, K=1024, D=16,
             short=1.0),
        # the same in single precision at a smaller batch, padded contexts
        dict(name="attn image train fp32", op="attention", train=True,
             dtype="float32", B=4, H=4, Hk=4, Q=1024, K=819, D=16, short=0.0),
        # long sequences, key heads shared by four query heads
        dict(name="attn long train bf16", op="attention", train=True,
             dtype="bfloat16", B=2, H=16, Hk=4, Q=4096, K=4096, D=64,
             short=1.0),
        # prediction over padded contexts, one of them empty; odd lengths
        dict(name="attn ragged fwd fp16", op="attention", train=False,
             dtype="float16", B=7, H=8, Hk=8, Q=333, K=2049, D=48, short=0.0),
        # one new target at a time against long contexts of unequal lengths
        dict(name="attn single token bf16", op="attention", train=False,
             dtype="bfloat16", B=8, H=8, Hk=2, Q=1, K=32768, D=64, short=0.5),
        # -- layer norm --------------------------------------------------- #
        # one small task served alone: 50 contexts of r_dim 128
        dict(name="norm task fwd fp32", op="norm", train=False,
             dtype="float32", rows=50, width=128, residual=True),
        # the norm of each head of the 1D training step
        dict(name="norm heads train fp32", op="norm", train=True,
             dtype="float32", rows=32 * 128 * 4, width=32, residual=False),
        # a wide model's residual norm, training
        dict(name="norm wide train bf16", op="norm", train=True,
             dtype="bfloat16", rows=16384, width=4096, residual=True),
        # odd width
        dict(name="norm odd train fp16", op="norm", train=True,
             dtype="float16", rows=5001, width=1001, residual=False),
        # -- gradient clipping -------------------------------------------- #
        # a 1D attentive model: about 250 thousand parameters in 32 tensors,
        # gradients as views of the data-parallel buffer
        dict(name="clip small flat fp32", op="clip", dtype="float32",
             layers=16, width=125, flat=True),
        # a large model's gradients, each a tensor of its own
        dict(name="clip large bf16", op="clip", dtype="bfloat16", layers=24,
             width=3201, flat=False),
    ]


def _spread(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["attention", "attention", "norm", "clip"])
    dtype = rng.choice(["float32", "bfloat16", "float16"])
    wide = dtype == "float32"
    if op == "norm":
        width = _spread(rng, 16, 8192)
        rows = _spread(rng, 1, min(65536, (1 << (25 if wide else 26)) // width))
        return dict(op=op, train=rng.random() < 0.7, dtype=dtype, rows=rows,
                    width=width, residual=rng.random() < 0.5)
    if op == "clip":
        layers = rng.randint(2, 24)
        width = _spread(rng, 20, 2200 if wide else 3200)
        return dict(op=op, dtype=dtype, layers=layers, width=width,
                    flat=rng.random() < 0.5)
    D = rng.choice([8, 16, 20, 24, 32, 48, 64, 96, 128])
    Hk = rng.choice([1, 2, 4, 8])
    H = Hk * rng.choice([1, 1, 2, 4])
    kind = rng.choice(["train", "train", "fwd", "token"])
    B = _spread(rng, 1, 32)
    if kind == "token":
        Q, K = rng.randint(1, 4), _spread(rng, 64, 65536)
        while B * Hk * K * D > (1 << 26):
            K = K // 2 + 1
    else:
        Q, K = _spread(rng, 16, 4096), _spread(rng, 16, 4096)
        # no more than the largest listed case computes, or its maps hold
        most = (1 << 35) // (6 if wide else 1) // (H * D)
        while B > 1 and B * Q * K > most:
            B = B // 2
        while B * Q * K > most or B * H * Q * K > (1 << 29):
            Q, K = Q // 2 + 1, K // 2 + 1
    return dict(op=op, train=kind == "train", dtype=dtype, B=B, H=H, Hk=Hk,
                Q=Q, K=K, D=D, short=rng.choice([1.0, 0.5, 0.0]))


def _lengths(case):
    """Keys of each batch entry, from `short` of them up to all."""
    B, K, short = case["B"], case["K"], case["short"]
    if B == 1:
        return [K]
    return [int(K * (short + (1.0 - short) * b / (B - 1))) for b in range(B)]


def _shapes(case):
    """The gradients of a stack of linear layers: weights and biases."""
    w = case["width"]
    return [s for i in range(case["layers"]) for s in ((w, w), (w + i,))]


def _sizes(case):
    return [math.prod(s) for s in _shapes(case)]


def prepare(case, seed):
    dev = torch.device("cuda")
    g = torch.Generator(dev).manual_seed(seed)
    dt = _TYPES[case["dtype"]]

    def normal(*shape, std=1.0, mean=0.0):
        x = torch.randn(*shape, generator=g, device=dev)
        return (x * std + mean).to(dt)

    s = dict(case)
    if case["op"] == "attention":
        B, H, Hk, Q, K, D = (case[n] for n in ("B", "H", "Hk", "Q", "K", "D"))
        # as the projections leave them: [B, L, heads * size], split by a view
        s["q"] = normal(B, Q, H, 2 * D).transpose(1, 2)
        s["k"] = normal(B, K, Hk, 2 * D).transpose(1, 2)
        s["v"] = normal(B, K, Hk, 2 * D).transpose(1, 2)
        # about where training starts it
        s["lam"] = normal(H, std=0.03, mean=0.25)
        s["lengths"] = None
        if case["short"] < 1.0:
            s["lengths"] = torch.tensor(
                _lengths(case), dtype=torch.int32, device=dev
            )
        if case["train"]:
            s["dout"] = normal(B, Q, H, 2 * D).transpose(1, 2)
            for n in ("q", "k", "v", "lam"):
                s[n].requires_grad_(True)
    elif case["op"] == "norm":
        rows, width = case["rows"], case["width"]
        s["x"] = normal(rows, width, std=1.5, mean=0.3)
        s["res"] = normal(rows, width) if case["residual"] else None
        s["w"] = normal(width, std=0.1, mean=1.0)
        s["b"] = normal(width, std=0.1)
        if case["train"]:
            s["dy"] = normal(rows, width)
            for n in ("x", "res", "w", "b"):
                if s[n] is not None:
                    s[n].requires_grad_(True)
    else:
        sizes = _sizes(case)
        if case["flat"]:
            s["flat"] = normal(sum(sizes), std=0.02)
            grads = list(s["flat"].split(sizes))
        else:
            grads = [normal(n, std=0.02) for n in sizes]
        s["params"] = []
        for grad, shape in zip(grads, _shapes(case)):
            p = torch.empty(shape, dtype=dt, device=dev, requires_grad=True)
            p.grad = grad.view(shape)
            s["params"].append(p)
        # the limit follows the norm down, so that each pass has to clip
        s["limit"] = 0.5 * 0.02 * math.sqrt(sum(sizes))
    return s


# ----------------------------- plain forms ------------------------------- #


def _plain_attention(s):
    q, k, v = (s[n].detach().float() for n in ("q", "k", "v"))
    lam = s["lam"].detach().float()[None, :, None, None]
    B, H, Q, D2 = q.shape
    Hk, K = k.shape[1], k.shape[2]
    G, D = H // Hk, D2 // 2
    scale = 1.0 / math.sqrt(D)
    # the query heads that share a key head stand in one axis with the queries
    q = q.reshape(B, Hk, G * Q, D2)
    k1, k2 = k[..., :D].contiguous(), k[..., D:].contiguous()
    q1, q2 = q[..., :D].contiguous(), q[..., D:].contiguous()
    lam = lam.expand(B, H, Q, 1).reshape(B, Hk, G * Q, 1)
    live = None
    if s["lengths"] is not None:
        at = torch.arange(K, device=q.device)
        live = (at[None] < s["lengths"][:, None])[:, None, None, :]

    def softmax(x):
        if live is not None:
            x = x.masked_fill(~live, float("-inf"))
        m = x.amax(-1, keepdim=True).clamp_min(torch.finfo(x.dtype).min)
        e = (x - m).exp()
        return e / e.sum(-1, keepdim=True).clamp_min(1e-30)

    p1 = softmax((q1 @ k1.transpose(-1, -2)) * scale)
    p2 = softmax((q2 @ k2.transpose(-1, -2)) * scale)
    a = p1 - lam * p2
    dt = s["q"].dtype
    out = {"out": (a @ v).reshape(B, H, Q, D2).to(dt)}
    if not s["train"]:
        return out
    do = s["dout"].float().reshape(B, Hk, G * Q, D2)
    out["dv"] = (a.transpose(-1, -2) @ do).to(dt)
    del a
    da = do @ v.transpose(-1, -2)
    d1 = (p1 * da).sum(-1, keepdim=True)
    d2 = (p2 * da).sum(-1, keepdim=True)
    ds1 = p1 * (da - d1) * scale
    ds2 = -lam * p2 * (da - d2) * scale
    dq = torch.cat([ds1 @ k1, ds2 @ k2], -1)
    dk = torch.cat([ds1.transpose(-1, -2) @ q1, ds2.transpose(-1, -2) @ q2], -1)
    out["dq"] = dq.reshape(B, H, Q, D2).to(dt)
    out["dk"] = dk.to(dt)
    # a long sum of both signs
    dlam = -(d2.double().reshape(B, H, Q).sum((0, 2)))
    out["dlam"] = dlam.to(dt)
    return out


def _plain_norm(s):
    x = s["x"].detach().float()
    dt = s["x"].dtype
    if s["res"] is not None:
        x = x + s["res"].detach().float()
    w, b = s["w"].detach().float(), s["b"].detach().float()
    c = x - x.mean(-1, keepdim=True)
    r = 1.0 / ((c * c).mean(-1, keepdim=True) + 1e-5).sqrt()
    h = c * r
    out = {"y": (h * w + b).to(dt)}
    if not s["train"]:
        return out
    dy = s["dy"].float()
    g = dy * w
    dx = r * (g - g.mean(-1, keepdim=True) - h * (g * h).mean(-1, keepdim=True))
    out["dx"] = dx.to(dt)
    if s["res"] is not None:
        out["dres"] = out["dx"]
    out["dw"] = (dy * h).sum(0).to(dt)
    out["db"] = dy.sum(0).to(dt)
    return out


def _plain_clip(s, limit):
    if s["flat"] is not False:
        grads = [s["flat"]]
    else:
        grads = [p.grad for p in s["params"]]
    total = torch.stack([g.float().square().sum() for g in grads]).sum().sqrt()
    c = (limit / (total + 1e-6)).clamp(max=1.0)
    for g in grads:
        g.copy_(g.float() * c)
    return total


# ------------------------------- one pass -------------------------------- #


def run(state):
    s = state
    if s["op"] == "attention":
        if not own:
            return _plain_attention(s)
        from npf import ops

        if not s["train"]:
            out = ops.differential_attention(
                s["k"], s["q"], s["v"], s["lam"], key_lengths=s["lengths"]
            )
            return {"out": out}
        out = ops.differential_attention(
            s["k"], s["q"], s["v"], s["lam"], key_lengths=s["lengths"]
        )
        dq, dk, dv, dlam = torch.autograd.grad(
            out, (s["q"], s["k"], s["v"], s["lam"]), s["dout"]
        )
        return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}
    if s["op"] == "norm":
        if not own:
            return _plain_norm(s)
        from npf import ops

        y = ops.layer_norm(s["x"], s["w"], s["b"], residual=s["res"])
        if not s["train"]:
            return {"y": y}
        if s["res"] is None:
            dx, dw, db = torch.autograd.grad(y, (s["x"], s["w"], s["b"]), s["dy"])
            return {"y": y, "dx": dx, "dw": dw, "db": db}
        dx, dres, dw, db = torch.autograd.grad(
            y, (s["x"], s["res"], s["w"], s["b"]), s["dy"]
        )
        return {"y": y, "dx": dx, "dres": dres, "dw": dw, "db": db}
    s["limit"] *= 0.999
    if own:
        from npf import ops

        total = ops.clip_grad_norm_(s["params"], s["limit"])
    else:
        total = _plain_clip(s, s["limit"])
    if s["flat"] is not False:
        return {"norm": total, "grads": s["flat"]}
    return {"norm": total, "grads": [p.grad for p in s["params"]]}


def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["op"] == "attention":
        B, H, Hk, Q, D = (case[n] for n in ("B", "H", "Hk", "Q", "D"))
        keys = sum(_lengths(case)) if case["short"] < 1.0 else B * case["K"]
        row = 2 * D * size
        data = 2 * B * H * Q * row + 2 * keys * Hk * row
        flops = 2 * H * Q * keys * 4 * D
        if case["train"]:
            data = 2 * data
            flops = 3 * flops
        return {"bytes": data, "flops": flops}
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        parts = 2 + int(case["residual"]) + (2 if case["train"] else 0)
        return {"bytes": n * size * parts, "flops": n * (23 if case["train"] else 8)}
    n = sum(_sizes(case))
    # the norm has to be whole before the first value is scaled
    return {"bytes": 2 * n * size, "flops": 3 * n}


# ------------------------ the definition in 64 bits ---------------------- #


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "attention":
        return _exact_attention(case, s)
    if case["op"] == "norm":
        return _exact_norm(s)
    s["limit"] *= 0.999
    if case["flat"]:
        g = s["flat"].double()
        total = torch.linalg.vector_norm(g)
        return {"norm": total, "grads": g * min(1.0, s["limit"] / float(total + 1e-6))}
    gs = [p.grad.double() for p in s["params"]]
    total = math.sqrt(sum(float((g ** 2).sum()) for g in gs))
    c = min(1.0, s["limit"] / (total + 1e-6))
    return {"norm": torch.tensor(total, dtype=torch.float64), "grads": [g * c for g in gs]}


def _exact_attention(case, s):
    B, H, Hk, Q, K, D = (case[n] for n in ("B", "H", "Hk", "Q", "K", "D"))
    q, k, v, lam = (s[n].detach().double() for n in ("q", "k", "v", "lam"))
    out = torch.zeros(B, H, Q, 2 * D, dtype=torch.float64, device=q.device)
    if case["train"]:
        dq, dk, dv = torch.zeros_like(q), torch.zeros_like(k), torch.zeros_like(v)
        dlam = torch.zeros_like(lam)
    lengths = _lengths(case) if case["short"] < 1.0 else [K] * B
    for b in range(B):
        n = lengths[b]
        if n == 0:
            continue
        for h in range(H):
            c = h // (H // Hk)
            leaves = [q[b, h], k[b, c, :n], v[b, c, :n], lam[h]]
            leaves = [t.detach().clone().requires_grad_(case["train"]) for t in leaves]
            qh, kh, vh, lh = leaves
            maps = [
                torch.softmax(
                    torch.mm(qh[:, i:i + D], kh[:, i:i + D].t()) / D ** 0.5, -1
                )
                for i in (0, D)
            ]
            o = torch.mm(maps[0], vh) - lh * torch.mm(maps[1], vh)
            out[b, h] = o.detach()
            if case["train"]:
                gq, gk, gv, gl = torch.autograd.grad(
                    o, leaves, s["dout"][b, h].double()
                )
                dq[b, h] = gq
                dk[b, c, :n] += gk
                dv[b, c, :n] += gv
                dlam[h] += gl
    if not case["train"]:
        return {"out": out}
    return {"out": out, "dq": dq, "dk": dk, "dv": dv, "dlam": dlam}


def _exact_norm(s):
    names = [n for n in ("x", "res", "w", "b") if s[n] is not None]
    t = {n: s[n].detach().double().requires_grad_(s["train"]) for n in names}
    z = t["x"] + t["res"] if "res" in t else t["x"]
    var, mean = torch.var_mean(z, dim=-1, correction=0, keepdim=True)
    y = torch.addcmul(t["b"], (z - mean) * torch.rsqrt(var + 1e-5), t["w"])
    if not s["train"]:
        return {"y": y}
    grads = torch.autograd.grad(y, [t[n] for n in names], s["dy"].double())
    return {"y": y.detach(), **{"d" + n: g for n, g in zip(names, grads)}}
