"""Differential attention, layer norm and gradient clipping: the operators
against their definitions in 64 bits, their refusals, and their use together.

Tolerances are bounds, elementwise, on what rounding can do.  With u half a
step of the inputs' type (finfo.eps / 2) and e = 2^-24 that of fp32:

- a stored value v is off by u |v| on top of what its computation is off, or,
  below the type's smallest normal value t, by half of the step there, u t (of
  fp16: 2^-11 2^-14 = 2^-25, which small gradients and map values do reach),
  and exponents of fp32 below 2^-126 become zero, so no less than that;
- a sum of n terms held in fp32 is off by at most n e sum|terms|, whatever its
  order, and a product of sums carries its factors' errors along.
"""

import math

import pytest
import torch

from npf import ops
from npf.architectures import get_attender
from npf.ops import functional as F_ops

E32 = 2.0 ** -24


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def lowest_step(dtype):
    """Half of the distance of values below the smallest normal one, or what
    an fp32 exponent loses where it becomes zero."""
    return max(half_step(dtype) * torch.finfo(dtype).tiny, 2.0 ** -126)


def assert_within(got, want, bound, name):
    got = got.detach().double().cpu()
    assert got.shape == want.shape, (name, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{name} has values that are not finite"
    off = (got - want).abs()
    worst = (off - bound).max().item() if off.numel() else -1.0
    assert worst <= 0, (
        f"{name}: off by {off.max().item():.3g}, {worst:.3g} over its bound "
        f"({(off > bound).sum().item()} of {off.numel()} values)"
    )


# --------------------------------------------------------------------------- #
# layer norm
# --------------------------------------------------------------------------- #


def norm_oracle(x, residual, weight, bias, eps, dy, out_dtype):
    """Values and bounds, in fp64, from the inputs as they are stored."""
    u, low = half_step(out_dtype), lowest_step(out_dtype)
    x, dy = x.double(), dy.double()
    z = x if residual is None else x + residual.double()
    zabs = x.abs() if residual is None else x.abs() + residual.double().abs()
    D, R = z.shape[-1], z.shape[0]
    w = torch.ones(D).double() if weight is None else weight.double()
    b = torch.zeros(D).double() if bias is None else bias.double()
    mean = z.mean(-1, keepdim=True)
    c = z - mean
    var = (c * c).mean(-1, keepdim=True)
    rstd = (var + eps).rsqrt()
    h = c * rstd
    # errors: of the mean (a sum of D), of a centred value, of rstd, of h
    e_mean = (D + 2) * E32 * zabs.mean(-1, keepdim=True)
    e_c = e_mean + 2 * E32 * (zabs + mean.abs())
    e_var = 2 * (c.abs() * e_c).mean(-1, keepdim=True) + (D + 3) * E32 * var \
        + (e_c * e_c).mean(-1, keepdim=True)
    r_rel = 0.5 * e_var / (var + eps) + 4 * E32
    e_h = rstd * e_c + h.abs() * (r_rel + 2 * E32)
    y = h * w + b
    e_y = e_h * w.abs() + 3 * E32 * (h.abs() * w.abs() + b.abs())
    out = {"y": (y, e_y + u * (y.abs() + e_y) + low)}
    g = dy * w
    m1, m2 = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    e_m1 = (D + 3) * E32 * g.abs().mean(-1, keepdim=True)
    e_m2 = (g.abs() * e_h).mean(-1, keepdim=True) \
        + (D + 4) * E32 * (g * h).abs().mean(-1, keepdim=True)
    inner = g - m1 - h * m2
    e_in = e_m1 + h.abs() * e_m2 + e_h * m2.abs() \
        + 4 * E32 * (g.abs() + m1.abs() + (h * m2).abs())
    dx = rstd * inner
    e_dx = rstd * e_in + dx.abs() * (r_rel + 2 * E32)
    out["dx"] = (dx, e_dx + u * (dx.abs() + e_dx) + low)
    dw, db = (dy * h).sum(0), dy.sum(0)
    e_dw = (dy.abs() * e_h).sum(0) + (R + 3) * E32 * (dy * h).abs().sum(0)
    e_db = (R + 3) * E32 * dy.abs().sum(0)
    for n, t, v, e in (("dw", weight, dw, e_dw), ("db", bias, db, e_db)):
        if t is not None:
            e = e + half_step(t.dtype) * (v.abs() + e) + lowest_step(t.dtype)
        out[n] = (v, e)
    return out


def norm_inputs(rows, width, dtype, wtype, residual, seed=0, mean=0.3):
    g = torch.Generator().manual_seed(seed)
    x = (torch.randn(rows, width, generator=g) * 1.5 + mean).to(dtype)
    r = torch.randn(rows, width, generator=g).to(dtype) if residual else None
    w = (1 + 0.1 * torch.randn(width, generator=g)).to(wtype)
    b = (0.1 * torch.randn(width, generator=g)).to(wtype)
    dy = torch.randn(rows, width, generator=g).to(dtype)
    return x, r, w, b, dy


def run_norm(device, x, r, w, b, dy, eps=1e-5):
    leaves = [None if t is None else t.to(device).requires_grad_(True)
              for t in (x, r, w, b)]
    y = ops.layer_norm(leaves[0], leaves[2], leaves[3], eps=eps, residual=leaves[1])
    live = [t for t in leaves if t is not None]
    grads = torch.autograd.grad(y, live, dy.to(device))
    got = dict(zip([n for n, t in zip(("dx", "dr", "dw", "db"), leaves)
                    if t is not None], grads))
    got["y"] = y
    return got


def check_norm(got, want):
    for n, t in got.items():
        assert_within(t, *want["dx" if n == "dr" else n], n)


class TestLayerNorm:
    @pytest.mark.parametrize("rows,width", [(1, 1), (5, 7), (3, 64), (9, 33)])
    @pytest.mark.parametrize("residual", [False, True])
    def test_composed(self, rows, width, residual):
        args = norm_inputs(rows, width, torch.float32, torch.float32, residual)
        check_norm(run_norm("cpu", *args),
                   norm_oracle(args[0], args[1], args[2], args[3], 1e-5, args[4],
                               torch.float32))

    def test_gradient_against_differences(self):
        x, r, w, b, _ = norm_inputs(4, 6, torch.float64, torch.float64, True)
        for t in (x, r, w, b):
            t.requires_grad_(True)
        assert torch.autograd.gradcheck(
            lambda x, r, w, b: ops.layer_norm(x, w, b, residual=r), (x, r, w, b)
        )

    def test_refusals(self):
        x = torch.randn(3, 8)
        with pytest.raises(ValueError, match="last axis"):
            ops.layer_norm(torch.randn(3, 0))
        with pytest.raises(ValueError, match="last axis"):
            ops.layer_norm(torch.tensor(1.0))
        with pytest.raises(TypeError, match="floating"):
            ops.layer_norm(torch.ones(3, 8, dtype=torch.int32))
        with pytest.raises(ValueError, match="weight"):
            ops.layer_norm(x, torch.ones(7))
        with pytest.raises(ValueError, match="bias"):
            ops.layer_norm(x, torch.ones(8), torch.ones(1, 8))
        with pytest.raises(ValueError, match="residual"):
            ops.layer_norm(x, residual=torch.randn(1, 8))
        with pytest.raises(TypeError, match="residual"):
            ops.layer_norm(x, residual=torch.randn(3, 8, dtype=torch.float64))
        with pytest.raises(TypeError, match="bias"):
            ops.layer_norm(x, torch.ones(8), torch.ones(8, dtype=torch.float64))

    # widths around the borders between the kernels' layouts: groups of lanes,
    # a wave, a block, a loop; vectors of 4 and 8 values that end inside a row
    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("rows,width", [
        (1, 1), (3, 2), (70, 5), (129, 16), (33, 31), (1000, 32), (257, 33),
        (65, 128), (40, 255), (40, 257), (1, 512), (37, 513), (19, 1000),
        (7, 1024), (5, 1025), (300, 1001), (6, 2049), (4, 4096), (3, 4099),
        (3, 8193), (2, 16384), (2, 16391), (3, 40001),
    ])
    def test_kernel(self, dtype, rows, width):
        residual = (rows + width) % 2 == 0
        args = norm_inputs(rows, width, dtype, dtype, residual, seed=width)
        check_norm(run_norm("cuda", *args),
                   norm_oracle(*args[:4], 1e-5, args[4], dtype))

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("width", [24, 300, 1500])
    def test_kernel_fp32_weights(self, dtype, width):
        args = norm_inputs(50, width, dtype, torch.float32, True)
        check_norm(run_norm("cuda", *args),
                   norm_oracle(*args[:4], 1e-5, args[4], dtype))

    @pytest.mark.gpu
    @pytest.mark.parametrize("width", [32, 640, 5000])
    def test_kernel_without_weights(self, width):
        x, r, _, _, dy = norm_inputs(50, width, torch.float32, torch.float32, True)
        want = norm_oracle(x, r, None, None, 1e-5, dy, torch.float32)
        check_norm(run_norm("cuda", x, r, None, None, dy), want)

    @pytest.mark.gpu
    @pytest.mark.parametrize("width", [20, 700])
    def test_weight_or_bias_alone(self, width):
        x, r, w, b, dy = norm_inputs(30, width, torch.bfloat16, torch.bfloat16, False)
        zero = torch.zeros_like(b)
        want = norm_oracle(x, None, w, zero, 1e-5, dy, torch.bfloat16)
        check_norm(run_norm("cuda", x, None, w, None, dy), want)
        want = norm_oracle(x, None, None, b, 1e-5, dy, torch.bfloat16)
        check_norm(run_norm("cuda", x, None, None, b, dy), want)

    @pytest.mark.gpu
    def test_weights_of_other_types(self):
        for wtype in (torch.float16, torch.float64):
            args = norm_inputs(30, 70, torch.float32, wtype, True)
            check_norm(run_norm("cuda", *args),
                       norm_oracle(*args[:4], 1e-5, args[4], torch.float32))

    @pytest.mark.gpu
    def test_residual_and_its_gradient(self):
        x = torch.randn(6, 24, device="cuda", requires_grad=True)
        r = torch.randn(6, 24, device="cuda", requires_grad=True)
        dy = torch.randn(6, 24, device="cuda")
        ops.layer_norm(x, residual=r).backward(dy)
        assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()
        # the same tensor twice: its gradients add up
        z = x.detach().clone().requires_grad_(True)
        ops.layer_norm(z, residual=z).backward(dy)
        one = x.detach().clone().requires_grad_(True)
        ops.layer_norm(one, residual=x.detach()).backward(dy)
        assert torch.equal(z.grad, 2 * one.grad)

    @pytest.mark.gpu
    @pytest.mark.parametrize("width", [8, 96, 2000])
    def test_one_of_the_gradients(self, width):
        x, r, w, b, dy = (None if t is None else t.cuda() for t in norm_inputs(
            70, width, torch.float32, torch.float32, True))
        full = run_norm("cuda", x, r, w, b, dy)
        for name, at in (("dx", 0), ("dr", 1), ("dw", 2), ("db", 3)):
            leaves = [t.detach() for t in (x, r, w, b)]
            leaves[at].requires_grad_(True)
            y = ops.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
            (grad,) = torch.autograd.grad(y, leaves[at], dy)
            assert torch.equal(grad, full[name]), name
            leaves[at].requires_grad_(False)

    @pytest.mark.gpu
    def test_differentiable_once(self):
        x = torch.randn(3, 8, device="cuda", requires_grad=True)
        w = torch.randn(8, device="cuda", requires_grad=True)
        y = ops.layer_norm(x, w)
        (dx,) = torch.autograd.grad(y.sum(), x, create_graph=True)
        assert torch.equal(dx, torch.autograd.grad(ops.layer_norm(x, w).sum(), x)[0])
        with pytest.raises(RuntimeError, match="layer_norm is differentiable once"):
            dx.square().sum().backward()

    @pytest.mark.gpu
    def test_no_rows(self):
        x = torch.randn(2, 0, 8, device="cuda", requires_grad=True)
        w = torch.ones(8, device="cuda", requires_grad=True)
        y = ops.layer_norm(x, w)
        assert y.shape == (2, 0, 8)
        y.sum().backward()
        assert x.grad.shape == x.shape and torch.equal(w.grad, torch.zeros_like(w))

    @pytest.mark.gpu
    def test_strides(self):
        base = torch.randn(6, 5, 3, 48, device="cuda")
        views = [base[..., 1:41], base.transpose(0, 1), base.permute(3, 0, 1, 2),
                 base[::2], base[:, :, :1].expand(-1, -1, 4, -1),
                 base.flatten()[1:1 + 24 * 40].view(24, 40)]
        for v in views:
            assert torch.equal(ops.layer_norm(v), ops.layer_norm(v.contiguous()))
            w = torch.randn(2 * v.shape[-1], device="cuda")[::2]
            assert torch.equal(ops.layer_norm(v, w),
                               ops.layer_norm(v.contiguous(), w.contiguous()))

    @pytest.mark.gpu
    def test_rows_of_equal_values_and_not_finite(self):
        for width in (16, 700, 20000):
            x = torch.full((4, width), 3.0, device="cuda")
            x[1, 0], x[2, width - 1] = float("nan"), float("inf")
            y = ops.layer_norm(x, bias=torch.full((width,), 0.5, device="cuda"))
            assert torch.equal(y[0], torch.full_like(y[0], 0.5))
            assert torch.equal(y[3], y[0])
            assert y[1].isnan().all() and y[2].isnan().all()

    @pytest.mark.gpu
    def test_far_mean(self):
        # a mean a thousand times the spread: the bounds grow with it and hold
        args = norm_inputs(20, 900, torch.float32, torch.float32, False, mean=1500.0)
        check_norm(run_norm("cuda", *args),
                   norm_oracle(*args[:4], 1e-5, args[4], torch.float32))

    @pytest.mark.gpu
    def test_refusals_of_the_kernel(self):
        x = torch.randn(3, 8, device="cuda")
        with pytest.raises(ValueError):
            ops.layer_norm(x, torch.ones(8))  # on the CPU
        with pytest.raises(TypeError):
            ops.layer_norm(x.double())
        with pytest.raises(ValueError):
            ops.layer_norm(x, residual=torch.randn(3, 8))


# --------------------------------------------------------------------------- #
# differential attention
# --------------------------------------------------------------------------- #


def attn_inputs(B, H, Hk, Q, K, D, Dv, dtype, seed=0, lam_each=True):
    g = torch.Generator().manual_seed(seed)

    def t(*shape):
        return torch.randn(*shape, generator=g).to(dtype)

    lam = 0.3 + 0.2 * torch.randn(H, generator=g)
    return dict(
        keys=t(B, Hk, K, 2 * D), queries=t(B, H, Q, 2 * D), values=t(B, Hk, K, Dv),
        lam=lam if lam_each else lam[0].clone(), dout=t(B, H, Q, Dv),
    )


def attn_oracle(a, scale=None, lengths=None):
    """Values and bounds in fp64; sums over keys and sizes are held in fp32,
    the maps and their gradients are rounded to the inputs' type once."""
    dtype = a["queries"].dtype
    u, low = half_step(dtype), lowest_step(dtype)
    k, q, v, do = (a[n].double() for n in ("keys", "queries", "values", "dout"))
    B, H, Q, D2 = q.shape
    Hk, K = k.shape[1:3]
    D, Dv, G = D2 // 2, v.shape[-1], H // Hk
    scale = 1 / math.sqrt(D) if scale is None else scale
    lam = a["lam"].double().expand(H).reshape(1, H, 1, 1)
    live = torch.ones(B, 1, 1, K, dtype=torch.bool)
    if lengths is not None:
        live = torch.arange(K) < torch.as_tensor(lengths).reshape(B, 1, 1, 1)
    k = k.masked_fill(~live.transpose(-1, -2), 0)
    v = v.masked_fill(~live.transpose(-1, -2), 0)
    kg, vg = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    P, rel = [], []
    for s in (slice(0, D), slice(D, D2)):
        qi, ki = q[..., s], kg[..., s]
        S = (qi @ ki.transpose(-1, -2)) * scale
        p = S.masked_fill(~live, -1e300).softmax(-1) * live
        mag = (qi.abs() @ ki.abs().transpose(-1, -2)) * scale
        top = mag.masked_fill(~live, 0).amax(-1, keepdim=True) if K else mag.sum(-1, keepdim=True)
        # of a probability, relative: its score, the largest score, the sum
        # of exponents, the exponent itself
        rel.append(2 * (D + 8) * E32 * (1 + top) + (K + 16) * E32)
        P.append(p)
    A = P[0] - lam * P[1]
    W = [P[0], lam.abs() * P[1]]  # magnitudes
    out, vabs = A @ vg, vg.abs()
    O2 = P[1] @ vg
    # rounding of both maps before they are subtracted or after, whichever
    # (a map's value is at least 1 / its sum of exponents times what is
    # rounded, so a lowest step there is at most one here)
    e_map = sum(w * (2 * u + r) for w, r in zip(W, rel)) + live * low * (1 + lam.abs())
    sums = (K + 4) * E32 * ((W[0] + W[1]) @ vabs)
    e_out = e_map @ vabs + sums
    e_o2 = (P[1] * (2 * u + rel[1]) + live * low) @ vabs + (K + 4) * E32 * (P[1] @ vabs)
    b_out = e_out + u * (out.abs() + e_out) + low
    b_o2 = e_o2 + u * (O2.abs() + e_o2) + low
    res = {"out": (out, b_out)}

    def grouped(x):
        return x.reshape(B, Hk, G, *x.shape[2:]).sum(2)

    Gd = do @ vg.transpose(-1, -2)
    Gabs = do.abs() @ vabs.transpose(-1, -2)
    d1 = ((P[0] * Gd).sum(-1, keepdim=True))
    d2 = ((P[1] * Gd).sum(-1, keepdim=True))
    e_d2 = (do.abs() * b_o2).sum(-1, keepdim=True) \
        + (Dv + 4) * E32 * (do.abs() * O2.abs()).sum(-1, keepdim=True)
    e_d1 = (do.abs() * (b_out + lam.abs() * b_o2)).sum(-1, keepdim=True) \
        + (Dv + 6) * E32 * (do.abs() * (out.abs() + 2 * (lam * O2).abs())).sum(-1, keepdim=True)
    dq, dk, e_dq, e_dk = [], [], [], []
    for i, s in enumerate((slice(0, D), slice(D, D2))):
        sign = torch.ones_like(lam) if i == 0 else -lam
        d, e_d = (d1, e_d1) if i == 0 else (d2, e_d2)
        ds = sign * P[i] * (Gd - d) * live
        e_ds = sign.abs() * P[i] * ((u + rel[i] + 4 * E32) * (Gd - d).abs()
                                    + (1 + u) * (e_d + (Dv + 4) * E32 * (Gabs + d.abs())))
        # rounded before or after the scale
        e_ds = e_ds + live * low * max(1.0, 1 / scale)
        ki, qi = kg[..., s], q[..., s]
        dq.append(scale * ds @ ki)
        e_dq.append(scale * (e_ds + (K + 4) * E32 * ds.abs()) @ ki.abs())
        dk.append(grouped(scale * ds.transpose(-1, -2) @ qi))
        e_dk.append(grouped(scale * (e_ds + (G * Q + 4) * E32 * ds.abs()).transpose(-1, -2)
                            @ qi.abs()))
    dq, dk, e_dq, e_dk = (torch.cat(t, -1) for t in (dq, dk, e_dq, e_dk))
    dv = grouped(A.transpose(-1, -2) @ do)
    e_dv = grouped((e_map + (G * Q + 4) * E32 * (W[0] + W[1])).transpose(-1, -2) @ do.abs())
    dlam, e_dlam = -d2.sum((0, 2, 3)), e_d2.sum((0, 2, 3))
    if a["lam"].dim() == 0:
        dlam, e_dlam = dlam.sum(), e_dlam.sum()
    ul = half_step(a["lam"].dtype)
    for n, x, e, r in (("dq", dq, e_dq, u), ("dk", dk, e_dk, u), ("dv", dv, e_dv, u),
                       ("dlam", dlam, e_dlam, ul)):
        t = a["lam"].dtype if n == "dlam" else dtype
        res[n] = (x, e + r * (x.abs() + e) + lowest_step(t))
    return res


def run_attn(device, a, scale=None, lengths=None, lengths_type=torch.int32):
    t = {n: x.to(device).requires_grad_(n != "dout") for n, x in a.items()}
    if lengths is not None:
        lengths = torch.tensor(lengths, dtype=lengths_type, device=device)
    out = ops.differential_attention(t["keys"], t["queries"], t["values"], t["lam"],
                                     scale=scale, key_lengths=lengths)
    names = ("keys", "queries", "values", "lam")
    grads = torch.autograd.grad(out, [t[n] for n in names], t["dout"])
    return dict(zip(("dk", "dq", "dv", "dlam"), grads), out=out)


def check_attn(got, want):
    for n, t in got.items():
        assert_within(t, *want[n], n)


SIZES = [
    # B, H, Hk, Q, K, D, Dv
    (1, 1, 1, 1, 1, 1, 1),
    (2, 1, 1, 1, 70, 16, 32),
    (2, 4, 2, 5, 3, 8, 16),
    (1, 2, 1, 33, 31, 16, 32),
    (3, 4, 4, 128, 50, 16, 32),
    (1, 3, 3, 65, 129, 5, 7),
    (2, 2, 2, 64, 64, 32, 64),
    (1, 4, 1, 100, 97, 33, 66),
    (1, 2, 2, 31, 200, 64, 128),
    (1, 6, 2, 70, 130, 80, 160),
    (1, 1, 1, 130, 260, 128, 256),
    (1, 2, 1, 3, 515, 128, 100),
    (2, 8, 1, 1, 300, 24, 48),
    # values wider or narrower than two maps
    (1, 2, 2, 40, 50, 16, 100),
    (1, 2, 1, 40, 50, 48, 16),
    (2, 2, 1, 50, 90, 96, 192),
    # one block of rows or keys: sums over a split axis
    (1, 2, 1, 600, 700, 16, 32),
    (1, 1, 1, 300, 1100, 64, 128),
    (1, 3, 1, 400, 530, 128, 256),
    (1, 2, 2, 257, 513, 20, 40),
]


class TestDifferentialAttention:
    @pytest.mark.parametrize("sizes", SIZES[:6])
    def test_composed(self, sizes):
        a = attn_inputs(*sizes, torch.float32)
        check_attn(run_attn("cpu", a), attn_oracle(a))

    @pytest.mark.parametrize("lengths", [[0, 3, 7], [7, 9, -2], [1, 0, 0]])
    def test_composed_lengths(self, lengths):
        a = attn_inputs(3, 2, 1, 4, 7, 4, 8, torch.float32)
        a["keys"][0, :, 6] = float("nan")
        a["values"][0, :, 6] = float("inf")
        lens = [min(max(n, 0), 7) for n in lengths]
        if lens[0] == 7:
            a = attn_inputs(3, 2, 1, 4, 7, 4, 8, torch.float32)
        check_attn(run_attn("cpu", a, lengths=lengths),
                   attn_oracle(a, lengths=lens))

    def test_composed_empty(self):
        for B, Q, K in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
            got = run_attn("cpu", attn_inputs(B, 2, 1, Q, K, 4, 8, torch.float32))
            assert got["out"].shape == (B, 2, Q, 8)
            assert not any(t.any() for t in got.values())

    def test_gradient_against_differences(self):
        a = attn_inputs(2, 2, 1, 3, 4, 2, 3, torch.float64)
        t = [a[n].double().requires_grad_(True)
             for n in ("keys", "queries", "values", "lam")]
        lens = torch.tensor([2, 0])
        for lengths in (None, lens):
            assert torch.autograd.gradcheck(
                lambda k, q, v, lam: ops.differential_attention(
                    k, q, v, lam, scale=0.7, key_lengths=lengths), t)

    def test_equal_maps_cancel(self):
        a = attn_inputs(1, 2, 2, 3, 5, 4, 8, torch.float32)
        a["queries"][..., 4:] = a["queries"][..., :4]
        a["keys"][..., 4:] = a["keys"][..., :4]
        out = ops.differential_attention(
            a["keys"], a["queries"], a["values"], torch.tensor(1.0))
        assert torch.equal(out, torch.zeros_like(out))

    def test_refusals(self):
        a = attn_inputs(2, 4, 2, 3, 5, 4, 8, torch.float32)
        k, q, v, lam = a["keys"], a["queries"], a["values"], a["lam"]
        f = ops.differential_attention
        bad = [
            (ValueError, (k[0], q, v, lam), {}),
            (ValueError, (k, q[..., :7], v, lam), {}),
            (ValueError, (k[..., :6], q, v, lam), {}),
            (ValueError, (k[:1], q, v, lam), {}),
            (ValueError, (k, q, v[:, :, :4], lam), {}),
            (ValueError, (k, q, v[:, :1], lam), {}),
            (ValueError, (k, q[:, :3], v, lam), {}),
            (ValueError, (k[:, :0], q, v[:, :0], lam), {}),
            (TypeError, (k.double(), q, v, lam), {}),
            (ValueError, (k, q, v, lam[:3]), {}),
            (ValueError, (k, q, v, 0.3), {}),
            (TypeError, (k, q, v, torch.tensor(1)), {}),
            (ValueError, (k, q, v, lam), dict(scale=0.0)),
            (ValueError, (k, q, v, lam), dict(scale=-1.0)),
            (ValueError, (k, q, v, lam), dict(scale=math.nan)),
            (ValueError, (k, q, v, lam), dict(scale=1e-30)),
            (ValueError, (k, q, v, lam), dict(key_lengths=torch.tensor([1]))),
            (TypeError, (k, q, v, lam), dict(key_lengths=torch.tensor([1.0, 2.0]))),
        ]
        for error, args, kwargs in bad:
            with pytest.raises(error):
                f(*args, **kwargs)

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("sizes", SIZES)
    def test_kernel(self, dtype, sizes):
        a = attn_inputs(*sizes, dtype, seed=sum(sizes))
        check_attn(run_attn("cuda", a), attn_oracle(a))

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
    @pytest.mark.parametrize("lengths", [[0, 3, 70], [129, 128, 0], [1, 33, 64], [-5, 400, 65]])
    @pytest.mark.parametrize("Q", [2, 90])
    def test_kernel_lengths(self, dtype, lengths, Q):
        a = attn_inputs(3, 4, 2, Q, 129, 16, 32, dtype)
        lens = [min(max(n, 0), 129) for n in lengths]
        for b, n in enumerate(lens):
            a["keys"][b, :, n:] = float("nan")
            a["values"][b, :, n:] = float("inf")
        for t in (torch.int32, torch.int64):
            got = run_attn("cuda", a, lengths=lengths, lengths_type=t)
            check_attn(got, attn_oracle(a, lengths=lens))
            for b, n in enumerate(lens):
                for g in ("dk", "dv"):
                    assert not got[g][b, :, n:].any()
                if n == 0:
                    assert not got["out"][b].any() and not got["dq"][b].any()

    @pytest.mark.gpu
    def test_scores_far_apart(self):
        # scores of several hundred: maps of one key, exponents that vanish
        for dtype in (torch.float32, torch.float16):
            a = attn_inputs(1, 2, 2, 40, 150, 16, 32, dtype)
            check_attn(run_attn("cuda", a, scale=30.0), attn_oracle(a, scale=30.0))

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
    def test_one_weight_for_all_heads(self, dtype):
        a = attn_inputs(2, 4, 2, 20, 30, 8, 16, dtype, lam_each=False)
        check_attn(run_attn("cuda", a), attn_oracle(a))
        a["lam"] = a["lam"].to(dtype)
        check_attn(run_attn("cuda", a), attn_oracle(a))

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
    def test_strides(self, dtype):
        g = torch.Generator().manual_seed(0)
        B, H, Hk, Q, K, D = 2, 4, 2, 37, 45, 16
        x = torch.randn(B, Q + K, 400, generator=g).to(dtype).cuda()
        # projections side by side in one buffer, at odd places
        q = x[:, :Q, 1:1 + H * 2 * D].unflatten(-1, (H, 2 * D)).transpose(1, 2)
        k = x[:, Q:, 131:131 + Hk * 2 * D].unflatten(-1, (Hk, 2 * D)).transpose(1, 2)
        v = x[:, Q:, 200:200 + Hk * 2 * D].unflatten(-1, (Hk, 2 * D)).transpose(1, 2)
        lam = torch.tensor([0.1, 0.2, 0.3, 0.4], device="cuda")
        dout = x[:, :Q, 7:7 + H * 2 * D].unflatten(-1, (H, 2 * D)).transpose(1, 2)

        def grads(q, k, v, lam, dout):
            q, k, v, lam = (t.detach().requires_grad_(True) for t in (q, k, v, lam))
            out = ops.differential_attention(k, q, v, lam)
            return (out, *torch.autograd.grad(out, (q, k, v, lam), dout))

        want = grads(q.contiguous(), k.contiguous(), v.contiguous(), lam,
                     dout.contiguous())
        last = [t.transpose(-1, -2).contiguous().transpose(-1, -2) for t in (q, k, v)]
        both = torch.stack([lam, lam], 1)[:, 1]
        for args in ((q, k, v, lam, dout), (*last, both, dout),
                     (q, k, v, lam, dout.transpose(-1, -2).contiguous().transpose(-1, -2))):
            for x1, x2 in zip(grads(*args), want):
                assert torch.equal(x1, x2)

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
    def test_aligned_and_not(self, dtype):
        # whole chunks at an odd place in memory take the loads that test each
        # lane's; the same products in the same order
        a = {n: t.cuda() for n, t in
             attn_inputs(1, 2, 1, 70, 150, 64, 128, dtype).items()}
        want = run_attn("cuda", a)

        def moved(t):
            room = torch.empty(t.numel() + 1, dtype=t.dtype, device="cuda")
            return room[1:].view(t.shape).copy_(t)

        got = run_attn("cuda", {n: t if n == "lam" else moved(t) for n, t in a.items()})
        for n in want:
            assert torch.equal(want[n], got[n]), n

    @pytest.mark.gpu
    @pytest.mark.parametrize("far", ["batch", "row"])
    def test_offsets_over_32_bits(self, far):
        # a cache whose entries stand more than 2^31 values apart
        a = attn_inputs(2, 2, 1, 3, 130, 16, 32, torch.bfloat16)
        step = {"batch": (2 ** 31 + 64, 32), "row": (64, 2 ** 24 + 32)}[far]
        room = torch.empty(step[0] + 260 * step[1] + 64, dtype=torch.bfloat16, device="cuda")
        t = {n: x.cuda() for n, x in a.items()}
        for i, n in enumerate(("keys", "values")):
            view = room.as_strided((2, 1, 130, 32), (step[0], 32, step[1], 1), 32 * i
                                   if far == "row" else 130 * 32 * i)
            t[n] = view.copy_(t[n])
        check_attn(run_attn("cuda", t), attn_oracle(a))

    @pytest.mark.gpu
    def test_broadcast_inputs(self):
        # one context set for a whole batch: gradients sum over it
        a = attn_inputs(3, 2, 2, 10, 20, 8, 16, torch.float32)
        a["keys"], a["values"] = (a[n][:1].expand(3, -1, -1, -1) for n in ("keys", "values"))
        want = attn_oracle(a)
        k, v = (a[n][:1].cuda().requires_grad_(True) for n in ("keys", "values"))
        q, lam = a["queries"].cuda(), torch.tensor(0.25).cuda().requires_grad_(True)
        lam4 = a["lam"].cuda()
        out = ops.differential_attention(k.expand(3, -1, -1, -1), q, v.expand(3, -1, -1, -1), lam4)
        dk, dv = torch.autograd.grad(out, (k, v), a["dout"].cuda())
        for name, got in (("dk", dk), ("dv", dv)):
            value, bound = want[name]
            add = 3 * E32 * value.abs().sum(0, keepdim=True)
            assert_within(got, value.sum(0, keepdim=True), bound.sum(0, keepdim=True) + add, name)
        same = lam.expand(2)
        out = ops.differential_attention(k, q[:1], v, same)
        (dlam,) = torch.autograd.grad(out, lam, a["dout"][:1].cuda())
        a1 = {n: t[:1] for n, t in a.items() if n != "lam"}
        a1["lam"] = torch.tensor(0.25)
        value, bound = attn_oracle(a1)["dlam"]
        assert_within(dlam, value, bound + 4 * E32 * value.abs(), "dlam")

    @pytest.mark.gpu
    def test_some_of_the_gradients(self):
        a = {n: t.cuda() for n, t in
             attn_inputs(2, 4, 2, 40, 50, 16, 32, torch.bfloat16).items()}
        full = run_attn("cuda", a)
        for want in (("dk",), ("dq",), ("dv",), ("dlam",), ("dk", "dlam"), ("dq", "dv")):
            t = {n: x.detach() for n, x in a.items()}
            names = {"dk": "keys", "dq": "queries", "dv": "values", "dlam": "lam"}
            for w in want:
                t[names[w]] = t[names[w]].clone().requires_grad_(True)
            out = ops.differential_attention(t["keys"], t["queries"], t["values"], t["lam"])
            for w, g in zip(want, torch.autograd.grad(out, [t[names[w]] for w in want], t["dout"])):
                assert torch.equal(g, full[w]), w

    @pytest.mark.gpu
    def test_differentiable_once(self):
        a = {n: t.cuda().requires_grad_(True) for n, t in
             attn_inputs(1, 1, 1, 3, 5, 4, 8, torch.float32).items()}
        out = ops.differential_attention(a["keys"], a["queries"], a["values"], a["lam"])
        (dq,) = torch.autograd.grad(out.sum(), a["queries"], create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            dq.sum().backward()

    @pytest.mark.gpu
    def test_empty(self):
        for B, Q, K in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
            a = attn_inputs(B, 2, 1, Q, K, 4, 8, torch.float32)
            got = run_attn("cuda", a)
            assert got["out"].shape == (B, 2, Q, 8)
            assert not any(t.any() for t in got.values())

    @pytest.mark.gpu
    def test_runs_agree_bit_for_bit(self):
        a = attn_inputs(2, 8, 2, 3, 3000, 32, 64, torch.bfloat16)
        first, second = run_attn("cuda", a), run_attn("cuda", a)
        for n in first:
            assert torch.equal(first[n], second[n]), n

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("sizes", [
        (1, 2, 1, 1, 5000, 64, 128), (1, 8, 2, 2, 2500, 16, 32),
        (2, 1, 1, 17, 1777, 128, 256),
    ])
    def test_few_queries_many_keys(self, dtype, sizes):
        a = attn_inputs(*sizes, dtype)
        check_attn(run_attn("cuda", a), attn_oracle(a))
        lens = [sizes[4] - 999] * sizes[0]
        check_attn(run_attn("cuda", a, lengths=lens), attn_oracle(a, lengths=lens))

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
    @pytest.mark.parametrize("D", [8, 24, 64, 127, 128])
    @pytest.mark.parametrize("Q, K", [(3, 60), (9, 127), (70, 33), (129, 255)])
    def test_maps_meet_in_a_block(self, dtype, D, Q, K):
        # key axes that are not split, of blocks with few rows and with many
        a = attn_inputs(2, 2, 1, Q, K, D, 2 * D, dtype)
        check_attn(run_attn("cuda", a), attn_oracle(a))
        lens = [K // 2, 0]
        check_attn(run_attn("cuda", a, lengths=lens), attn_oracle(a, lengths=lens))
        t = {n: x.cuda() for n, x in a.items()}
        alone = ops.differential_attention(t["keys"], t["queries"], t["values"], t["lam"])
        # (without what a backward pass would need, and the same)
        assert torch.equal(alone, run_attn("cuda", a)["out"])

    @pytest.mark.gpu
    def test_refusals_of_the_kernel(self):
        a = {n: t.cuda() for n, t in
             attn_inputs(2, 2, 2, 3, 5, 4, 8, torch.float32).items()}
        k, q, v, lam = a["keys"], a["queries"], a["values"], a["lam"]
        f = ops.differential_attention
        with pytest.raises(TypeError):
            f(k.double(), q.double(), v.double(), lam)
        with pytest.raises(ValueError):
            f(k, q, v, lam.cpu())
        with pytest.raises(ValueError):
            f(k.cpu(), q, v, lam)
        with pytest.raises(ValueError):
            f(k, q, v, lam, key_lengths=torch.tensor([1, 2]))
        wide = torch.randn(1, 1, 2, 2 * 129, device="cuda")
        with pytest.raises(ValueError):
            f(wide, wide, wide[..., :8], lam[:1])
        with pytest.raises(ValueError):
            f(k, q, torch.randn(2, 2, 5, 300, device="cuda"), lam)

    @pytest.mark.gpu
    def test_sizes_at_the_end_of_31_bits(self):
        f = ops.differential_attention
        k, lam = torch.zeros(1, 1, 1, 2, device="cuda"), torch.tensor(0.5, device="cuda")
        with pytest.raises(ValueError, match="too many rows"):
            f(k, k.expand(1, 1, 2 ** 31 - 64, 2), k, lam)
        with pytest.raises(ValueError, match="too many rows"):
            f(k.expand(1, 1, 2 ** 30, 2), k, k.expand(1, 1, 2 ** 30, 2), lam)
        bf16 = dict(dtype=torch.bfloat16, device="cuda")
        # a size whose low 32 bits would be one that is taken
        with pytest.raises(ValueError, match="1 to 256"):
            f(k.bfloat16(), k.bfloat16(), torch.empty(1, 1, 1, 2 ** 32 + 64, **bf16), lam)
        a = attn_inputs(1, 2, 1, 5, 9, 8, 16, torch.float32)
        room = torch.empty(2, 2 ** 31 + 8, **bf16)[:, 3]
        a["lam"] = room.copy_(a["lam"])
        want = attn_oracle({n: t.cpu() for n, t in a.items()})
        check_attn(run_attn("cuda", a), want)


# --------------------------------------------------------------------------- #
# gradient norm and clipping
# --------------------------------------------------------------------------- #


def params_of(shapes, dtype, device, seed=0, flat=False, std=1.0):
    g = torch.Generator().manual_seed(seed)
    grads = [(torch.randn(s, generator=g) * std).to(dtype).to(device) for s in shapes]
    if flat:
        sizes = [x.numel() for x in grads]
        buf = torch.cat([x.reshape(-1) for x in grads])
        grads = [x.view(s) for x, s in zip(buf.split(sizes), shapes)]
    params = []
    for x in grads:
        p = torch.zeros_like(x, requires_grad=True)
        p.grad = x
        params.append(p)
    return params


def check_clip(params, max_norm, p=2.0, **kwargs):
    before = [x.grad.detach().double().cpu() for x in params]
    every = torch.cat([x.reshape(-1) for x in before])
    want = torch.linalg.vector_norm(every, p)
    total = ops.clip_grad_norm_(params, max_norm, norm_type=p, **kwargs)
    assert total.dim() == 0
    # fp64 sums on the GPU, fp32 ones of the library on the CPU
    rel = 2 * E32 if total.is_cuda else (every.numel() + 4) * E32
    assert abs(total.double().item() - want.item()) <= rel * want.item()
    c = min(1.0, max_norm / (want.item() + 1e-6))
    for x, old in zip(params, before):
        u = half_step(x.grad.dtype)
        bound = old.abs() * c * ((rel + 3 * E32) * (1 + u) + u)
        assert_within(x.grad, old * c, bound + torch.finfo(x.grad.dtype).tiny, "grad")
        if c == 1.0:
            assert torch.equal(x.grad.double().cpu(), old)


SHAPES = [(3,), (1,), (128, 128), (128,), (0,), (33, 7), (4097,), (2, 3, 4, 5)]


class TestGradClip:
    @pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
    def test_composed(self, p):
        check_clip(params_of(SHAPES, torch.float32, "cpu"), 0.5, p)
        check_clip(params_of(SHAPES, torch.float32, "cpu"), 1e9, p)

    def test_refusals(self):
        params = params_of(SHAPES, torch.float32, "cpu")
        for norm_type in (0.0, 3.0, -math.inf, math.nan):
            with pytest.raises(ValueError, match="norm_type"):
                ops.clip_grad_norm_(params, 1.0, norm_type=norm_type)
        for max_norm in (-1.0, math.nan):
            with pytest.raises(ValueError, match="max_norm"):
                ops.clip_grad_norm_(params, max_norm)
        sparse = torch.zeros(4, requires_grad=True)
        sparse.grad = torch.ones(4).to_sparse()
        with pytest.raises(TypeError, match="dense"):
            ops.grad_norm(sparse)
        params[0].grad[0] = math.inf
        before = [p.grad.clone() for p in params]
        with pytest.raises(RuntimeError, match="inf"):
            ops.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
        assert all(torch.equal(a, p.grad) for a, p in zip(before, params))

    @pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
    def test_gradients_with_a_graph(self, device):
        # of a backward pass that is itself differentiated
        p = torch.tensor([3.0, 4.0], device=device, requires_grad=True)
        p.pow(2).sum().backward(create_graph=True)
        assert p.grad.requires_grad
        assert not ops.grad_norm([p]).requires_grad
        total = ops.clip_grad_norm_([p], 1.0)
        assert not total.requires_grad and abs(total.item() - 10.0) <= 10 * 4 * E32
        assert abs(p.grad.norm().item() - 1.0) <= 1e-6 + 16 * E32

    def test_nothing_to_clip(self):
        assert ops.clip_grad_norm_([], 1.0).item() == 0.0
        assert ops.grad_norm([torch.zeros(3, requires_grad=True)]).item() == 0.0

    @pytest.mark.gpu
    @pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
    @pytest.mark.parametrize("flat", [False, True])
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16,
                                       torch.float64])
    def test_kernel(self, dtype, flat, p):
        for max_norm in (0.5, 1e9, 0.0):
            check_clip(params_of(SHAPES, dtype, "cuda", flat=flat), max_norm, p)
        params = params_of(SHAPES, dtype, "cuda", flat=flat)
        total = ops.grad_norm(params, p)
        assert torch.equal(total, ops.clip_grad_norm_(params, 1.0, p))

    @pytest.mark.gpu
    def test_many_and_mixed(self):
        # more gradients than one launch takes, of every type, some not views
        # of one another's neighbours; one larger than a block's share
        params = []
        for i, dtype in enumerate((torch.float32, torch.bfloat16, torch.float16,
                                   torch.float64)):
            params += params_of([(n,) for n in range(1, 101)], dtype, "cuda", seed=i)
        params += params_of([(300007,)], torch.float32, "cuda", seed=9)
        check_clip(params, 3.0)

    @pytest.mark.gpu
    def test_large(self):
        params = params_of([(70000001,)], torch.bfloat16, "cuda", std=0.01)
        check_clip(params, 1.0)

    @pytest.mark.gpu
    def test_unaligned_and_dense_orders(self):
        x = torch.randn(5000, device="cuda")
        p = torch.zeros(4998, device="cuda", requires_grad=True)
        p.grad = x[1:4999]
        q = torch.zeros(40, 30, device="cuda", requires_grad=True)
        q.grad = torch.randn(30, 40, device="cuda").t()
        edge = x[[0, 4999]].clone()
        check_clip([p, q], 0.7)
        assert torch.equal(x[[0, 4999]], edge)

    @pytest.mark.gpu
    def test_squares_that_overflow_fp32(self):
        params = params_of([(50,)], torch.float32, "cuda", std=1e25)
        check_clip(params, 1.0)

    @pytest.mark.gpu
    def test_not_finite(self):
        for bad, rest in ((math.inf, 0.0), (math.nan, math.nan)):
            params = params_of([(50,), (60,)], torch.float32, "cuda")
            params[0].grad[7] = bad
            before = [p.grad.clone() for p in params]
            with pytest.raises(RuntimeError):
                ops.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
            for a, p in zip(before, params):
                assert torch.equal(a.nan_to_num(), p.grad.nan_to_num())
            total = ops.clip_grad_norm_(params, 1.0)
            assert torch.equal(total.cpu().nan_to_num(5.0), torch.tensor(bad).nan_to_num(5.0))
            assert params[0].grad[7].isnan()
            others = params[1].grad
            assert others.isnan().all() if math.isnan(rest) else not others.any()

    @pytest.mark.gpu
    def test_refusals_of_the_kernel(self):
        p = params_of([(50,)], torch.float32, "cuda")[0]
        with pytest.raises(ValueError, match="share memory"):
            ops.clip_grad_norm_([p, p], 1.0)
        q = torch.zeros(10, device="cuda", requires_grad=True)
        q.grad = p.grad[5:15]
        with pytest.raises(ValueError, match="share memory"):
            ops.clip_grad_norm_([p, q], 1.0)
        r = torch.zeros(10, device="cuda", requires_grad=True)
        r.grad = p.grad[:20:2]
        with pytest.raises(ValueError, match="dense"):
            ops.clip_grad_norm_([r], 1.0)
        with pytest.raises(ValueError, match="one GPU"):
            ops.clip_grad_norm_([p, *params_of([(3,)], torch.float32, "cpu")], 1.0)


# --------------------------------------------------------------------------- #
# together
# --------------------------------------------------------------------------- #


def composed(monkeypatch):
    """The framework's own switch for the composed path on a GPU."""
    monkeypatch.setenv("NPF_DISABLE_OPS", "layer_norm,differential_attention,grad_norm")


class TestAttenders:
    @pytest.mark.parametrize("name", ["differential", "differential_transformer"])
    @pytest.mark.parametrize("n_kv_heads", [None, 2])
    def test_shapes_and_gradients(self, name, n_kv_heads):
        torch.manual_seed(0)
        att = get_attender(name, 32, 32, 32, n_heads=4, n_kv_heads=n_kv_heads)
        keys, queries, values = (torch.randn(3, n, 32, requires_grad=True)
                                 for n in (7, 5, 7))
        out = att(keys, queries, values)
        assert out.shape == (3, 5, 32)
        out.square().sum().backward()
        for p in (*att.parameters(), keys, queries, values):
            assert p.grad is not None and torch.isfinite(p.grad).all()

    def test_padded_contexts_do_not_count(self):
        torch.manual_seed(0)
        att = get_attender("differential_transformer", 16, 16, 16, n_heads=2)
        keys, queries, values = (torch.randn(3, n, 16) for n in (7, 5, 7))
        lens = torch.tensor([7, 4, 0])
        out = att(keys, queries, values, key_lengths=lens)
        keys2, values2 = keys.clone(), values.clone()
        keys2[1, 4:], values2[1, 4:], keys2[2], values2[2] = 9.0, -9.0, 8.0, 7.0
        assert torch.equal(out, att(keys2, queries, values2, key_lengths=lens))
        alone = att(keys[1:2, :4], queries[1:2], values[1:2, :4])
        # products and sums of at most 16 terms of size 1, through two norms:
        # 64 roundings of values below 16
        assert (alone - out[1:2]).abs().max() <= 64 * 16 * E32

    @pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
    @pytest.mark.parametrize("name", ["differential", "differential_transformer"])
    @pytest.mark.parametrize("B, K, Q", [(2, 0, 3), (2, 3, 0), (0, 3, 2)])
    def test_nothing_to_attend(self, device, name, B, K, Q):
        att = get_attender(name, 16, 16, 16, n_heads=2).to(device)
        keys, queries, values = (torch.randn(B, n, 16, device=device, requires_grad=True)
                                 for n in (K, Q, K))
        out = att(keys, queries, values)
        assert out.shape == (B, Q, 16) and torch.isfinite(out).all()
        out.sum().backward()
        for p in (*att.parameters(), keys, queries, values):
            assert p.grad is not None and torch.isfinite(p.grad).all()

    def test_permutation_of_contexts(self):
        torch.manual_seed(0)
        att = get_attender("differential", 16, 16, 16, n_heads=2, depth=3)
        keys, queries, values = (torch.randn(2, n, 16) for n in (9, 4, 9))
        perm = torch.randperm(9)
        a, b = att(keys, queries, values), att(keys[:, perm], queries, values[:, perm])
        assert (a - b).abs().max() <= 64 * 16 * E32

    def test_refusals(self):
        for args, kw in (((30, 32, 32), {}), ((32, 30, 32), {}),
                         ((32, 32, 32), dict(n_kv_heads=3)), ((32, 32, 32), dict(depth=0))):
            with pytest.raises(ValueError):
                get_attender("differential", *args, n_heads=4, **kw)
        with pytest.raises(ValueError):
            get_attender("differential_transformer", 32, 32, 64, n_heads=4)

    def test_in_models(self):
        from npf import AttnCNP, AttnLNP, CNPFLoss, ELBOLossLNPF

        torch.manual_seed(0)
        X = torch.rand(2, 12, 1) * 2 - 1
        Y = torch.randn(2, 12, 1)
        for cls, loss, kw in ((AttnCNP, CNPFLoss, {}),
                              (AttnCNP, CNPFLoss, dict(
                                  is_self_attn=True, self_attention_kwargs=dict(
                                      attention="differential_transformer"))),
                              (AttnLNP, ELBOLossLNPF, dict(is_q_zCct=True))):
            m = cls(1, 1, r_dim=32, attention="differential_transformer", **kw)
            out = m(X[:, :5], Y[:, :5], X, Y)
            loss()(out, Y).backward()
            # lam's vectors learn
            assert m.attender.lam_vectors.grad.abs().sum() > 0


def training_step(device, dtype, seed=0):
    """One step as the trainer makes it, of an attentive model: loss, gradients
    and their norm, and the clipped gradients."""
    from npf import AttnCNP, CNPFLoss

    torch.manual_seed(seed)
    m = AttnCNP(1, 1, r_dim=64, attention="differential_transformer").to(device)
    g = torch.Generator().manual_seed(1)
    X = (torch.rand(4, 60, 1, generator=g) * 2 - 1).to(device)
    Y = torch.randn(4, 60, 1, generator=g).to(device)
    with torch.autocast("cuda", dtype=torch.bfloat16, enabled=dtype == torch.bfloat16):
        out = m(X[:, :37], Y[:, :37], X)
    loss = CNPFLoss()(out, Y)
    loss.backward()
    raw = [p.grad.clone() for p in m.parameters() if p.grad is not None]
    total = ops.clip_grad_norm_(m.parameters(), 0.1)
    done = [p.grad.clone() for p in m.parameters() if p.grad is not None]
    return loss.detach(), raw, total, done


class TestTogether:
    def test_trainer_clips(self):
        from npf import AttnCNP, CNPFLoss
        from npf.train import NPFTrainer

        def step(clip):
            torch.manual_seed(0)
            m = AttnCNP(1, 1, r_dim=16, attention="differential")
            t = NPFTrainer(m, CNPFLoss, optimizer=torch.optim.SGD, lr=1.0, device="cpu",
                           grad_clip_norm=clip)
            before = [p.detach().clone() for p in m.parameters()]
            g = torch.Generator().manual_seed(1)
            X = torch.rand(2, 9, 1, generator=g) * 2 - 1
            Y = torch.randn(2, 9, 1, generator=g)
            t.train_step(dict(X_cntxt=X[:, :4], Y_cntxt=Y[:, :4], X_trgt=X), Y)
            return torch.cat([(a - b).reshape(-1) for a, b in
                              zip(before, m.parameters())]).double()

        free, held = step(None), step(0.01)
        assert held.norm() <= 0.01 * 1.001 < free.norm()

    @pytest.mark.gpu
    def test_step_matches_the_composed_one(self, monkeypatch):
        loss, raw, total, done = training_step("cuda", torch.float32)
        composed(monkeypatch)
        loss2, raw2, total2, done2 = training_step("cuda", torch.float32)
        # both are fp32; sums of the same terms in other orders, through about
        # ten layers of at most 256 terms each
        n = 10 * 256 * E32
        assert abs(loss - loss2) <= n * abs(loss2)
        assert abs(total - total2) <= n * abs(total2)
        for a, b in zip(raw + done, raw2 + done2):
            assert (a - b).norm() <= n * max(b.norm(), total2 if b.norm() > 0.1 else 0.1)

    @pytest.mark.gpu
    def test_step_under_autocast(self):
        loss, raw, total, done = training_step("cuda", torch.bfloat16)
        assert torch.isfinite(loss) and torch.isfinite(total)
        clipped = torch.cat([g.reshape(-1) for g in done]).double().norm()
        assert clipped <= 0.1 * (1 + 4 * E32)
        assert all(torch.isfinite(g).all() for g in raw)

    @pytest.mark.gpu
    def test_trainer_graph_replays(self):
        from npf import AttnCNP, CNPFLoss
        from npf.train import NPFTrainer

        def losses(hipgraphs):
            torch.manual_seed(0)
            m = AttnCNP(1, 1, r_dim=32, attention="differential_transformer")
            t = NPFTrainer(m, CNPFLoss, device="cuda", grad_clip_norm=0.5,
                           hipgraphs=hipgraphs)
            g = torch.Generator().manual_seed(1)
            got = []
            for i in range(6):
                X = (torch.rand(4, 20, 1, generator=g) * 2 - 1).cuda()
                Y = torch.randn(4, 20, 1, generator=g).cuda()
                got.append(float(t.train_step(
                    dict(X_cntxt=X[:, :7], Y_cntxt=Y[:, :7], X_trgt=X), Y, _first=i == 0)))
            if hipgraphs:
                assert t._step_graphs is not None and t._step_graphs.graphs
            return torch.tensor(got).double()

        eager, graphed = losses(False), losses(True)
        # the same kernels on the same numbers
        assert torch.equal(eager, graphed)

    @pytest.mark.gpu
    def test_inference_graphs_of_two_streams(self):
        """Two captured calls replayed against eager work and one another."""
        sizes = [(2, 4, 2, 1, 4000, 16, 32), (1, 2, 2, 70, 50, 16, 32)]
        runs = []
        for i, s in enumerate(sizes):
            a = {n: t.cuda() for n, t in attn_inputs(*s, torch.bfloat16, seed=i).items()}
            w = torch.ones(s[-1], device="cuda")

            def call(a=a, w=w):
                out = ops.differential_attention(a["keys"], a["queries"], a["values"], a["lam"])
                return ops.layer_norm(out, w)

            with torch.no_grad():
                side = torch.cuda.Stream()
                side.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(side):
                    call()
                torch.cuda.current_stream().wait_stream(side)
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g):
                    out = call()
            runs.append((a, call, g, out))
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for i in range(4):
            for a, *_ in runs:
                a["queries"].normal_()
            for st, (_, _, g, _) in zip(streams, runs):
                st.wait_stream(torch.cuda.current_stream())
                with torch.cuda.stream(st):
                    g.replay()
            torch.cuda.synchronize()
            for _, call, _, out in runs:
                with torch.no_grad():
                    assert torch.equal(out, call())

    @pytest.mark.gpu
    def test_captured_training_call(self):
        """Forward and backward of both operators in one graph, replayed on new
        inputs between eager work."""
        a = {n: t.cuda() for n, t in
             attn_inputs(2, 4, 2, 140, 600, 16, 32, torch.bfloat16).items()}
        w = torch.randn(32, device="cuda")

        def call():
            t = {n: x.detach().requires_grad_(n != "dout") for n, x in a.items()}
            wg = w.detach().requires_grad_(True)
            out = ops.differential_attention(t["keys"], t["queries"], t["values"], t["lam"])
            out = ops.layer_norm(out, wg)
            leaves = [t[n] for n in ("keys", "queries", "values", "lam")] + [wg]
            return (out.detach(), *torch.autograd.grad(out, leaves, t["dout"]))

        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            call()
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            static = call()
        for i in range(4):
            for n in ("queries", "keys", "dout"):
                a[n].normal_()
            g.replay()
            torch.cuda.synchronize()
            for x, y in zip(static, call()):
                assert torch.equal(x, y)

    @pytest.mark.gpu
    def test_captured_clipping(self):
        params = params_of(SHAPES, torch.float32, "cuda")
        grads = [p.grad.clone() for p in params]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            ops.clip_grad_norm_(params, 0.5)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            total = ops.clip_grad_norm_(params, 0.5)
        for i in range(4):
            for p, x in zip(params, grads):
                p.grad.copy_(x * (i + 1))
            eager = params_of(SHAPES, torch.float32, "cuda")
            for p, x in zip(eager, grads):
                p.grad.copy_(x * (i + 1))
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(total, ops.clip_grad_norm_(eager, 0.5))
            for p, q in zip(params, eager):
                assert torch.equal(p.grad, q.grad)

    @pytest.mark.gpu
    def test_own_stream(self):
        a = {n: t.cuda() for n, t in
             attn_inputs(2, 2, 2, 64, 500, 32, 64, torch.float32).items()}
        want = ops.differential_attention(a["keys"], a["queries"], a["values"], a["lam"])
        s = torch.cuda.Stream()
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            k = a["keys"] * 2
            k /= 2
            got = ops.differential_attention(k, a["queries"], a["values"], a["lam"])
        torch.cuda.current_stream().wait_stream(s)
        assert torch.equal(got, want)
