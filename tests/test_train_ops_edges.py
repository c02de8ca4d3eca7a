"""Calls at the edges of differential attention, layer norm and gradient
clipping: types, values and ways of calling that ordinary use seldom meets.

Tolerances are those of test_train_ops: elementwise bounds on what rounding
can do.
"""

import math

import pytest
import torch

from npf import ops
from npf.architectures import get_attender
from test_train_ops import (E32, SHAPES, assert_within, attn_inputs, attn_oracle,
                            check_attn, check_clip, lowest_step, norm_inputs,
                            params_of, run_attn, run_norm)

HALF = [torch.bfloat16, torch.float16]


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
class TestComposedClip:
    """The composed form, whose sums and factor are held in more bits than
    16-bit gradients, like the kernels'."""

    @pytest.fixture(autouse=True)
    def composed(self, monkeypatch):
        monkeypatch.setenv("NPF_DISABLE_OPS", "grad_norm")

    @pytest.mark.parametrize("dtype", HALF)
    @pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
    def test_half(self, device, dtype, p):
        for max_norm in (0.5, 1e9, 0.0):
            check_clip(params_of(SHAPES, dtype, device), max_norm, p)
        params = params_of(SHAPES, dtype, device)
        assert ops.grad_norm(params, p).dtype == torch.float32

    def test_norm_over_the_types_largest(self, device):
        # finite gradients whose norm, about 1e5, no fp16 value holds
        params = params_of([(1000000,)], torch.float16, device, std=100.0)
        check_clip(params, 1.0, error_if_nonfinite=True)
        assert params[0].grad.any()

    def test_squares_that_overflow_fp32(self, device):
        check_clip(params_of([(50,)], torch.float32, device, std=1e25), 1.0)

    def test_mixed(self, device):
        params = []
        for i, dtype in enumerate((torch.bfloat16, torch.float32, torch.float16)):
            params += params_of([(n,) for n in range(1, 20)], dtype, device, seed=i)
        assert ops.grad_norm(params).dtype == torch.float32
        check_clip(params, 3.0)
        wide = params_of([(7,)], torch.float64, device)
        old = wide[0].grad.clone()
        want = torch.linalg.vector_norm(torch.cat(
            [p.grad.double().reshape(-1) for p in params + wide]))
        total = ops.clip_grad_norm_(params + wide, 1.0)
        assert total.dtype == torch.float64
        # 64-bit sums and products of 200 terms
        assert (total - want).abs() <= 256 * 2.0 ** -53 * want
        off = (wide[0].grad - old / (want + 1e-6)).abs()
        assert (off <= 256 * 2.0 ** -53 * old.abs()).all()


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("below", [1e-9, 1e-12, 0.5])
def test_clip_factors_next_to_one(device, below):
    # which fp32 does not tell from 1
    wide = params_of([(300,)], torch.float64, device)
    narrow = params_of([(200,)], torch.float32, device)
    old = [p.grad.clone() for p in wide + narrow]
    norm = torch.cat([g.double() for g in old]).norm()
    # (the factor's own 1e-6 is made up for)
    ops.clip_grad_norm_(wide + narrow, ((norm + 1e-6) * (1 - below)).item())
    # sums of 500 terms, a root, a quotient and products in 64 bits
    want = old[0] * (1 - below)
    assert ((wide[0].grad - want).abs() <= 512 * 2.0 ** -53 * want.abs()).all()
    want = old[1].double() * (1 - below)
    assert ((narrow[0].grad - want).abs() <= 2.5 * E32 * want.abs()).all()


class Oddly(torch.nn.Module):
    """A model whose gradients the clipping operator refuses, one way each."""

    def __init__(self, way, device="cpu"):
        super().__init__()
        dtype = torch.complex64 if way == "complex" else torch.float32
        self.a = torch.nn.Parameter(torch.full((3, 4), 0.5, dtype=dtype))
        self.b = torch.nn.Parameter(torch.full((3, 4), 2.0))
        both = torch.zeros(2, 3, 8, device=device)
        at = {"gaps": (both[0, :, ::2], both[1, :, 1::2]),
              "shared": (both[0, :, :4], both[0, :, :4])}.get(way)
        if at:
            for p, g in zip((self.a, self.b), at):
                p.register_post_accumulate_grad_hook(self.moved_to(g))

    @staticmethod
    def moved_to(place):
        def hook(p):
            p.grad = place.copy_(p.grad)
        return hook

    def forward(self, X):
        return (X @ self.a.abs() @ self.b.t()).square().mean()


class Itself(torch.nn.Module):
    def forward(self, out, y):
        return out


class TestTrainerClips:
    """Gradients that the operator refuses are clipped as they were before
    there was one."""

    @pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
    @pytest.mark.parametrize("way", ["complex", "gaps", "shared", "plain"])
    def test_as_the_library(self, device, way):
        from npf.train import NPFTrainer

        X = torch.linspace(-1, 1, 15).reshape(5, 3).to(device)
        t = NPFTrainer(Oddly(way, device), Itself, optimizer=torch.optim.SGD,
                       lr=1.0, device=device, grad_clip_norm=0.1)
        before = [p.detach().clone() for p in t.module.parameters()]
        t.train_step(dict(X=X), None)
        got = [b - p.detach() for b, p in zip(before, t.module.parameters())]
        m = Oddly(way, device).to(device)
        m(X).backward()
        total = torch.nn.utils.clip_grad_norm_(m.parameters(), 0.1)
        assert total > 0.1
        if way == "shared" and device == "cuda":
            # the library's one launch scales the same values twice at once
            assert all(torch.isfinite(g).all() for g in got)
            return
        for g, p in zip(got, m.parameters()):
            # norms of 24 terms, the factor and the step, in fp32
            assert ((g - p.grad).abs() <= 64 * E32 * (2.0 + p.grad.abs())).all()

    def test_negative_limits_are_the_librarys(self):
        from npf.train import NPFTrainer

        X = torch.linspace(-1, 1, 15).reshape(5, 3)
        t = NPFTrainer(Oddly("plain"), Itself, optimizer=torch.optim.SGD,
                       lr=0.0, device="cpu", grad_clip_norm=-0.1)
        t.train_step(dict(X=X), None)


# --------------------------------------------------------------------------- #
# differential attention: ranges of fp16
# --------------------------------------------------------------------------- #


def largest_map_gradient(a, scale):
    """The largest |P (G - delta)| of both maps, and 4 max|dO| max|V| max(1, |lam|)."""
    k, q, v, do = (a[n].double() for n in ("keys", "queries", "values", "dout"))
    G = q.shape[1] // k.shape[1]
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    D = q.shape[-1] // 2
    dA = do @ v.transpose(-1, -2)
    most = 0.0
    for s in (slice(0, D), slice(D, 2 * D)):
        P = (q[..., s] @ k[..., s].transpose(-1, -2) * scale).softmax(-1)
        dS = P * (dA - (P * dA).sum(-1, keepdim=True))
        most = max(most, dS.abs().max().item())
    reach = 4 * do.norm(dim=-1).max() * v.norm(dim=-1).max() * max(1.0, a["lam"].abs().max())
    return most, reach.item()


def scaled_oracle(a, scale, lengths=None):
    """attn_oracle where gradients of the maps are rounded as 2^e dS, with
    2^e reach between 2^14 and 2^15, so that 2^-25 2^-e is lost where it is
    small: results are linear in dout, and with dout 2^e as large the unscaled
    form loses the same."""
    _, reach = largest_map_gradient(a, scale)
    e = math.floor(14 - math.log2(reach))
    res = attn_oracle(dict(a, dout=a["dout"].double() * 2.0 ** e), scale, lengths)
    for n in ("dq", "dk", "dv", "dlam"):
        t = a["lam"].dtype if n == "dlam" else a["queries"].dtype
        value, bound = res[n]
        res[n] = (value * 2.0 ** -e, bound * 2.0 ** -e + lowest_step(t))
    return res


FP16_SIZES = [
    # B, H, Hk, Q, K, D, Dv: one launch for all gradients of the keys, or
    # several; whole 16-byte chunks or not; sums over split axes
    (1, 2, 1, 70, 90, 16, 32),
    (2, 4, 2, 33, 65, 20, 40),
    (1, 2, 1, 300, 700, 24, 48),
    (2, 2, 2, 40, 200, 64, 128),
    (1, 2, 1, 260, 530, 63, 100),
    (1, 2, 2, 130, 140, 128, 256),
]


class TestFp16Ranges:
    def inputs(self, sizes, dout, values, spread=1.0, scale=1 / 64):
        a = attn_inputs(*sizes, torch.float32)
        # scores of size 3
        size = math.sqrt(3 / scale / math.sqrt(sizes[5]))
        a["queries"] *= size
        a["keys"] *= size
        a["values"] *= values
        a["dout"] *= dout
        a["dout"][:, :, ::2] *= spread
        return {n: t if n == "lam" else t.half() for n, t in a.items()}, scale

    @pytest.mark.gpu
    @pytest.mark.parametrize("sizes", FP16_SIZES)
    def test_gradients_of_maps_over_the_largest_value(self, sizes):
        a, scale = self.inputs(sizes, 700.0, 24.0)
        most, _ = largest_map_gradient(a, scale)
        assert most > 65504
        want = scaled_oracle(a, scale)
        assert all(value.abs().max() < 60000 for n, (value, _) in want.items()
                   if n != "dlam")
        check_attn(run_attn("cuda", a, scale=scale), want)

    @pytest.mark.gpu
    @pytest.mark.parametrize("sizes", FP16_SIZES)
    def test_small_gradients_of_maps(self, sizes):
        # all of them below the smallest normal value, in part below its last step
        a, scale = self.inputs(sizes, 2.0 ** -13, 2.0 ** -6, scale=64.0)
        most, _ = largest_map_gradient(a, scale)
        assert most < 2.0 ** -14
        check_attn(run_attn("cuda", a, scale=scale), scaled_oracle(a, scale))

    @pytest.mark.gpu
    @pytest.mark.parametrize("sizes", FP16_SIZES[:4])
    def test_rows_of_unequal_size(self, sizes):
        a, scale = self.inputs(sizes, 0.5, 24.0, spread=1400.0)
        check_attn(run_attn("cuda", a, scale=scale), scaled_oracle(a, scale))
        B, K = sizes[0], sizes[4]
        lens = [0] * (B - 1) + [K - 7]
        check_attn(run_attn("cuda", a, scale=scale, lengths=lens),
                   scaled_oracle(a, scale, lengths=lens))

    @pytest.mark.gpu
    @pytest.mark.parametrize("sizes, last", [
        ((1, 1, 1, 3, 70001, 4, 8), (12000.0, 700.0)),
        ((1, 2, 1, 35000, 5, 4, 8), (300.0, 200.0)),
    ])
    def test_more_rows_than_chunks(self, sizes, last):
        # (norms of rows are taken in chunks, from 65536 rows on of several steps)
        a, scale = self.inputs(sizes, 0.5, 4.0)
        without = largest_map_gradient(a, scale)[1]
        # the largest at the very end, without which 2^e dS would be inf
        a["values"][:, :, -1], a["dout"][:, :, -1] = last
        most, _ = largest_map_gradient(a, scale)
        assert most * 2.0 ** (14 - math.log2(without)) > 65504
        check_attn(run_attn("cuda", a, scale=scale), scaled_oracle(a, scale))

    @pytest.mark.gpu
    @pytest.mark.parametrize("lam", [0.0, -40.0, 900.0])
    def test_weights_of_the_second_map(self, lam):
        a, scale = self.inputs(FP16_SIZES[0], 1.0, 1.0)
        a["lam"] = torch.tensor(lam)
        check_attn(run_attn("cuda", a, scale=scale), scaled_oracle(a, scale))

    @pytest.mark.gpu
    def test_weight_over_the_largest_value(self):
        # P_1 - lam P_2 passes 65504, what follows from it does not
        a, scale = self.inputs(FP16_SIZES[0], 2.0 ** -6, 2.0 ** -6)
        a["lam"] = torch.tensor([3e5, -2e5])
        want = scaled_oracle(a, scale)
        assert all(want[n][0].abs().max() < 60000 for n in ("out", "dq", "dk", "dv"))
        check_attn(run_attn("cuda", a, scale=scale), want)

    @pytest.mark.gpu
    @pytest.mark.parametrize("H, Hk, Q, K, D", [
        (1, 1, 1, 50000, 16), (2, 1, 130, 20000, 16), (1, 1, 200, 9000, 64),
        (1, 1, 40, 7000, 20), (1, 1, 3, 9000, 128),
    ])
    def test_many_small_map_values(self, H, Hk, Q, K, D):
        # One key with the weight 1, all others with e^-18, below 2^-25, which
        # is rounded to zero: most of a result is theirs, in both maps.
        k = torch.full((1, Hk, K, 2 * D), -18.0 / D).half()
        k[:, :, K // 3] = 0.0
        q = torch.ones(1, H, Q, 2 * D).half()
        v = torch.full((1, Hk, K, 2 * D), 16.0).half()
        v[:, :, K // 3] = 2.0 ** -9
        dout = torch.full((1, H, Q, 2 * D), 64.0).half()
        a = dict(keys=k, queries=q, values=v, lam=torch.tensor(0.25), dout=dout)
        got = run_attn("cuda", a, scale=1.0)
        P = k[0, 0, :, :D].double().sum(-1).softmax(-1)
        out = 0.75 * (P @ v[0, 0].double())
        # a map's values are rounded to half a step u each and below 2^-14 of
        # what is rounded, 2^-7 as large, to 2^-25; scores of 18 and sums of K
        # terms in fp32; both maps, weighted 1 and 1/4; the result once more
        u = 2.0 ** -11
        rel = u + 64 * E32 * 18 + 2 * (K + 16) * E32
        bound = 1.25 * ((P * rel + 2.0 ** -32) @ v[0, 0].double())
        want = out.expand(1, H, Q, 2 * D)
        assert_within(got["out"], want, (bound + u * out + 2.0 ** -25).expand_as(want), "out")
        # a gradient of the values: H Q rows of 64, with the same P
        dv = 0.75 * P[:, None] * 64.0 * (H // Hk) * Q
        rel = 2 * u + 64 * E32 * 18 + 2 * (K + 16 + H * Q) * E32
        bound = (1.25 / 0.75) * rel * dv + u * dv + 2.0 ** -25
        assert_within(got["dv"], dv.expand(1, Hk, K, 2 * D), bound.expand(1, Hk, K, 2 * D), "dv")

    @pytest.mark.gpu
    def test_scores_of_millions(self):
        # whose products' rounding is worth many powers of two: the largest
        # score's key alone counts, and the gradients of its map are zero
        a = attn_inputs(1, 2, 2, 70, 150, 16, 32, torch.float16)
        a["queries"] *= 1500.0
        a["keys"] *= 1500.0
        q, k = a["queries"].double(), a["keys"].double()
        first, second = (
            (q[..., s] @ k[..., s].transpose(-1, -2)).topk(2)
            for s in (slice(0, 16), slice(16, 32)))
        for scores in (first.values, second.values):
            # (fp32 sums of 16 terms of up to 2^26 are off by no more than 256)
            assert (scores[..., 0] - scores[..., 1]).min() > 1000
            assert 2 ** 24 < scores.max() < 2 ** 26
        first, second = first.indices[..., 0], second.indices[..., 0]
        pick = lambda i: a["values"].double().gather(
            2, i[..., None].expand(-1, -1, -1, 32))
        lam = a["lam"].double().reshape(1, 2, 1, 1)
        want = pick(first) - lam * pick(second)
        for lengths in (None, [150]):
            got = run_attn("cuda", a, scale=1.0, lengths=lengths)
            bound = 2.0 ** -11 * (3 * want.abs() + 2 * (lam * pick(second)).abs()) + 2.0 ** -24
            assert_within(got["out"], want, bound, "out")

    @pytest.mark.gpu
    def test_zeros_and_values_that_are_not_finite(self):
        a, scale = self.inputs((2, 2, 1, 40, 60, 16, 32), 1.0, 1.0)
        zero = dict(a, dout=torch.zeros_like(a["dout"]))
        got = run_attn("cuda", zero, scale=scale)
        assert not any(got[n].any() for n in ("dq", "dk", "dv", "dlam"))
        # one row's gradient: the rows and keys of the other entry stay
        want = scaled_oracle(a, scale)
        for bad in (math.inf, math.nan):
            b = dict(a, dout=a["dout"].clone())
            b["dout"][0, 1, 3, 5] = bad
            got = run_attn("cuda", b, scale=scale)
            assert not got["dk"][0].isfinite().any()
            assert not got["dq"][0, 1, 3].isfinite().any()
            for n in ("dq", "dk", "dv"):
                value, bound = want[n]
                assert_within(got[n][1], value[1], bound[1], n)
            rows = [i for i in range(40) if i != 3]
            value, bound = want["dq"]
            assert_within(got["dq"][0, 1, rows], value[0, 1, rows], bound[0, 1, rows], "dq")


# --------------------------------------------------------------------------- #
# what reads memory past torch's dispatcher refuses what the latter would do
# --------------------------------------------------------------------------- #


def calls(device):
    """name, call and a tensor that it takes, for each operator of the
    extension; the others' inputs are made beforehand."""
    g = torch.Generator().manual_seed(0)
    x = torch.randn(4, 8, generator=g).to(device)
    kqv = torch.randn(1, 2, 5, 8, generator=g).to(device)
    lam = torch.tensor(0.3, device=device)
    w = torch.ones(8, device=device)
    ext = ops.extension()

    def norm_of(grad):
        p = torch.zeros(grad.shape, device=device, requires_grad=True)
        p.grad = grad
        return ext.grad_norm([p], 2.0, 0.5)

    return [
        ("layer_norm x", lambda t: ext.layer_norm(t, None, w, None, 1e-5), x),
        ("layer_norm residual", lambda t: ext.layer_norm(x, t, None, None, 1e-5), x),
        ("layer_norm weight", lambda t: ext.layer_norm(x, None, t, None, 1e-5), w),
        ("layer_norm bias", lambda t: ext.layer_norm(x, None, None, t, 1e-5), w),
        ("differential_attention k",
         lambda t: ext.differential_attention(t, kqv, kqv, lam, 1.0, None), kqv),
        ("differential_attention q",
         lambda t: ext.differential_attention(kqv, t, kqv, lam, 1.0, None), kqv),
        ("differential_attention v",
         lambda t: ext.differential_attention(kqv, kqv, t, lam, 1.0, None), kqv),
        ("differential_attention lam",
         lambda t: ext.differential_attention(kqv, kqv, kqv, t, 1.0, None), lam),
        ("grad_norm", norm_of, x),
    ]


@pytest.mark.skipif(not ops.has_extension(), reason="the extension is not built")
@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
class TestPastTheDispatcher:
    # (on the CPU the refusals come before the one of CPU tensors)

    def test_forward_mode(self, device):
        import torch.autograd.forward_ad as fwad

        for name, call, t in calls(device):
            with fwad.dual_level():
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    call(fwad.make_dual(t, torch.ones_like(t)))
            if name != "grad_norm":
                with pytest.raises(NotImplementedError, match="wraps|forward-mode"):
                    torch.func.jvp(call, (t,), (torch.ones_like(t),))

    def test_traces(self, device):
        from torch.fx.experimental.proxy_tensor import make_fx

        for name, call, t in calls(device):
            with pytest.raises(NotImplementedError, match="traced"):
                torch.jit.trace(call, (t,), check_trace=False)
            for mode in ("real", "fake"):
                with pytest.raises(NotImplementedError, match="traced|wraps"):
                    make_fx(call, tracing_mode=mode)(t)

    def test_wrappers(self, device):
        for name, call, t in calls(device):
            if name != "grad_norm":
                with pytest.raises(NotImplementedError, match="wraps"):
                    torch.func.vmap(call)(torch.stack([t, t]))

    def test_gradients_of_gradients_in_forward_mode(self, device):
        import torch.autograd.forward_ad as fwad

        if device == "cpu":
            pytest.skip("a backward pass of the extension needs a GPU")
        x = torch.randn(4, 8, device=device, requires_grad=True)
        kqv = torch.randn(1, 2, 5, 8, device=device, requires_grad=True)
        lam = torch.tensor(0.3, device=device)
        for y, t in ((ops.layer_norm(x), x),
                     (ops.differential_attention(kqv, kqv, kqv[..., :4], lam), kqv)):
            with fwad.dual_level():
                dy = fwad.make_dual(torch.ones_like(y), torch.ones_like(y))
                with pytest.raises(NotImplementedError, match="forward-mode"):
                    torch.autograd.grad(y, t, dy)


@pytest.mark.skipif(not ops.has_extension(), reason="the extension is not built")
def test_fake_tensors_are_refused():
    # (which say that they are on a GPU, and have no memory)
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        x = torch.empty(4, 8, device="cuda")
        kqv = torch.empty(1, 2, 5, 8, device="cuda")
        lam = torch.empty((), device="cuda")
        p = torch.empty(4, 8, device="cuda", requires_grad=True)
        p.grad = x
        for call in (lambda: ops.layer_norm(x), lambda: ops.grad_norm([p]),
                     lambda: ops.clip_grad_norm_([p], 1.0),
                     lambda: ops.differential_attention(kqv, kqv, kqv, lam)):
            with pytest.raises(NotImplementedError, match="wraps"):
                call()


def test_composed_forward_mode():
    import torch.autograd.forward_ad as fwad

    x, t = torch.randn(4, 8).double(), torch.randn(4, 8).double()
    with fwad.dual_level():
        got = fwad.unpack_dual(ops.layer_norm(fwad.make_dual(x, t))).tangent
    want = (ops.layer_norm(x + 1e-6 * t) - ops.layer_norm(x - 1e-6 * t)) / 2e-6
    # differences of second order in 64 bits: 1e-12 of third derivatives, and
    # 2^-53 over the step
    assert (got - want).abs().max() <= 1e-8


# --------------------------------------------------------------------------- #
# rows without keys
# --------------------------------------------------------------------------- #

HERE = [("cpu", torch.float32)] + [
    pytest.param("cuda", t, marks=pytest.mark.gpu)
    for t in (torch.float32, torch.bfloat16, torch.float16)
]


class TestRowsWithoutKeys:
    """Batch entries without contexts: zeros, whatever stands in their places."""

    # few rows and many, sums over split axes, D 128
    SIZES = [(3, 2, 1, 5, 9, 4, 8), (3, 2, 1, 2, 300, 16, 32),
             (3, 2, 2, 140, 600, 16, 32), (3, 1, 1, 40, 70, 128, 256)]

    @pytest.mark.parametrize("device, dtype", HERE)
    @pytest.mark.parametrize("sizes", SIZES)
    @pytest.mark.parametrize("bad", [math.inf, math.nan])
    def test_gradients_that_are_not_finite(self, device, dtype, sizes, bad):
        a = attn_inputs(*sizes, dtype)
        lens = [sizes[4] // 2, 0, sizes[4]]
        zero = dict(a, dout=a["dout"].clone())
        zero["dout"][1] = 0.0
        want = run_attn(device, zero, lengths=lens)
        a["dout"][1] = bad
        got = run_attn(device, a, lengths=lens)
        for n in want:
            assert torch.equal(got[n], want[n]), n
        assert torch.isfinite(got["dlam"]).all()

    @pytest.mark.parametrize("device, dtype", HERE)
    @pytest.mark.parametrize("sizes", SIZES)
    @pytest.mark.parametrize("bad", [math.inf, math.nan])
    def test_weight_that_is_not_finite(self, device, dtype, sizes, bad):
        a = attn_inputs(*sizes, dtype)
        a["lam"][:] = bad
        got = run_attn(device, a, lengths=[sizes[4], 0, 1])
        for n in ("out", "dq", "dk", "dv"):
            assert torch.equal(got[n][1], torch.zeros_like(got[n][1])), n
        assert got["out"][0].isnan().all() or got["out"][0].isinf().any()


class TestNegatedViews:
    """Views whose memory holds the other sign (the imaginary part of a
    conjugate is one)."""

    @pytest.mark.gpu
    def test_attention(self):
        a = {n: t.cuda() for n, t in
             attn_inputs(2, 2, 1, 5, 9, 4, 1, torch.float32).items()}
        want = run_attn("cuda", a)

        def call(t):
            t = {n: x.detach().requires_grad_(True) for n, x in t.items()}
            out = ops.differential_attention(t["keys"], t["queries"], t["values"], t["lam"])
            names = ("keys", "queries", "values", "lam")
            grads = torch.autograd.grad(out, [t[n] for n in names], t["dout"].detach())
            return dict(zip(("dk", "dq", "dv", "dlam"), grads), out=out)

        for n in a:
            negated = torch._neg_view(-a[n])
            assert negated.is_neg()
            got = call(dict(a, **{n: negated}))
            for r in want:
                assert torch.equal(got[r], want[r]), (n, r)
        for n in ("values", "lam"):
            z = torch.complex(a[n], -a[n]).conj().imag
            assert z.is_neg() and torch.equal(z, a[n])
            got = call(dict(a, **{n: z}))
            for r in want:
                assert torch.equal(got[r], want[r]), (n, r)

    @pytest.mark.gpu
    def test_norm(self):
        args = [t.cuda() for t in norm_inputs(6, 20, torch.float32, torch.float32, True)]
        want = run_norm("cuda", *args)
        for i in range(5):
            some = list(args)
            some[i] = torch._neg_view(-args[i])
            leaves = [t.detach().requires_grad_(True) for t in some[:4]]
            y = ops.layer_norm(leaves[0], leaves[2], leaves[3], residual=leaves[1])
            got = dict(zip(("dx", "dr", "dw", "db"),
                           torch.autograd.grad(y, leaves, some[4])), y=y)
            for r in want:
                assert torch.equal(got[r], want[r]), (i, r)

    @pytest.mark.gpu
    def test_zeros_without_memory(self):
        # as torch makes them for gradients that are known to be zero
        zero = lambda *shape: torch._efficientzerotensor(shape, device="cuda")
        x = torch.randn(4, 8, device="cuda", requires_grad=True)
        assert torch.equal(ops.layer_norm(zero(4, 8)), torch.zeros(4, 8, device="cuda"))
        y = ops.layer_norm(x)
        (dx,) = torch.autograd.grad(y, x, zero(4, 8))
        assert torch.equal(dx, torch.zeros_like(dx))
        q = torch.randn(1, 1, 3, 8, device="cuda", requires_grad=True)
        lam = torch.tensor(0.25, device="cuda")
        out = ops.differential_attention(q, q, zero(1, 1, 3, 4), lam)
        assert torch.equal(out, torch.zeros_like(out))
        out = ops.differential_attention(q, q, q, lam)
        (dq,) = torch.autograd.grad(out, q, zero(1, 1, 3, 8))
        assert torch.equal(dq, torch.zeros_like(dq))
        p = torch.zeros(50, device="cuda", requires_grad=True)
        p.grad = zero(50)
        with pytest.raises(ValueError, match="dense"):
            ops.clip_grad_norm_([p], 1.0)

    @pytest.mark.gpu
    def test_gradients(self):
        p = torch.zeros(50, device="cuda", requires_grad=True)
        p.grad = torch._neg_view(torch.ones(50, device="cuda"))
        with pytest.raises(ValueError, match="dense"):
            ops.clip_grad_norm_([p], 1.0)


@pytest.mark.parametrize("device", ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)])
@pytest.mark.parametrize("disabled", ["", "differential_attention"])
def test_attention_under_autocast_keeps_its_types(device, disabled, monkeypatch):
    monkeypatch.setenv("NPF_DISABLE_OPS", disabled)
    a = attn_inputs(2, 2, 1, 5, 50, 8, 16, torch.float32)
    t = {n: x.to(device).requires_grad_(n != "dout") for n, x in a.items()}
    with torch.autocast(device, dtype=torch.bfloat16):
        out = ops.differential_attention(t["keys"], t["queries"], t["values"], t["lam"])
    assert out.dtype == torch.float32
    names = ("keys", "queries", "values", "lam")
    grads = torch.autograd.grad(out, [t[n] for n in names], t["dout"])
    check_attn(dict(zip(("dk", "dq", "dv", "dlam"), grads), out=out), attn_oracle(a))


# --------------------------------------------------------------------------- #
# launches that ordinary training steps do not make
# --------------------------------------------------------------------------- #

TYPES = [torch.float32, torch.bfloat16, torch.float16]


class TestOtherLaunches:
    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", TYPES)
    @pytest.mark.parametrize("D, Dv", [(4, 7), (64, 64), (64, 100), (128, 256), (20, 30)])
    @pytest.mark.parametrize("lengths", [None, [37, 0]])
    def test_gradients_of_keys_and_values_alone(self, dtype, D, Dv, lengths):
        # rows' sums without the kernel of dq; dk and dv each by itself
        a = attn_inputs(2, 4, 2, 45, 70, D, Dv, dtype)
        want = attn_oracle(a, lengths=lengths)
        lens = None if lengths is None else torch.tensor(lengths, device="cuda")
        for names in (("dk",), ("dv",), ("dk", "dv")):
            t = {n: x.cuda() for n, x in a.items()}
            leaves = [t[{"dk": "keys", "dv": "values"}[n]].requires_grad_(True) for n in names]
            out = ops.differential_attention(
                t["keys"], t["queries"], t["values"], t["lam"], key_lengths=lens)
            check_attn(dict(zip(names, torch.autograd.grad(out, leaves, t["dout"]))), want)

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", TYPES)
    @pytest.mark.parametrize("sizes", [
        (2, 2, 1, 700, 129, 16, 32), (2, 2, 1, 700, 600, 16, 32), (2, 1, 1, 600, 300, 64, 128),
        (2, 2, 2, 530, 140, 128, 200), (2, 4, 1, 150, 90, 20, 40),
    ])
    def test_lengths_and_queries_in_parts(self, dtype, sizes):
        # (a key head has at least 512 rows of queries: their axis is split)
        a = attn_inputs(*sizes, dtype)
        for lengths in ([0, sizes[4]], [sizes[4] - 1, 33]):
            check_attn(run_attn("cuda", a, lengths=lengths), attn_oracle(a, lengths=lengths))

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
    def test_one_weight_for_many_rows(self, dtype):
        a = attn_inputs(3, 4, 2, 1100, 40, 8, 16, dtype, lam_each=False)
        check_attn(run_attn("cuda", a), attn_oracle(a))
        # the key axis in parts, each with its own sums
        a = attn_inputs(1, 4, 2, 200, 1200, 8, 16, dtype, lam_each=False)
        check_attn(run_attn("cuda", a), attn_oracle(a))


class TestMostHeads:
    """Launches end at 2^32 threads, of which each head takes a block of its own."""

    def heads(self, n, Q, dtype=torch.bfloat16):
        row = torch.full((1, 1, 1, 2), 0.5, dtype=dtype, device="cuda")
        return row.expand(1, n, 1, 2), row.expand(1, n, Q, 2)

    @pytest.mark.gpu
    def test_refusals(self):
        lam = torch.tensor(0.25, device="cuda")
        for n, Q in ((2 ** 25 + 8, 1), (2 ** 23 + 8, 33)):
            k, q = self.heads(n, Q)
            with pytest.raises(ValueError, match="too many heads"):
                ops.differential_attention(k, q, k, lam)
        k, q = self.heads(2 ** 24 + 8, 1)
        lam.requires_grad_(True)
        with pytest.raises(ValueError, match="too many heads"):
            ops.differential_attention(k, q, k, lam)

    @pytest.mark.gpu
    def test_most(self):
        lam = torch.tensor(0.25, device="cuda", requires_grad=True)
        for dtype in (torch.bfloat16, torch.float16):
            k, q = self.heads(2 ** 22 + 3, 2, dtype)
            out = ops.differential_attention(k, q, k, lam)
            # one key: both maps are 1
            assert torch.equal(out, torch.full_like(out, 0.375))
            (dlam,) = torch.autograd.grad(out, lam, torch.ones_like(out))
            # -0.5 for each of 4 (2^22 + 3) values, in 64 bits and rounded
            assert dlam.item() == -2.0 * (2 ** 22 + 3)


    @pytest.mark.gpu
    def test_one_weight_each(self):
        # (1024 threads sum a head's part of the gradient: 2^22 heads a launch)
        n = 2 ** 22 + 5
        k, q = self.heads(n, 1)
        lam = torch.full((n,), 0.25, device="cuda", requires_grad=True)
        out = ops.differential_attention(k, q, k, lam)
        dout = torch.ones_like(out)
        dout[0, -1] = 3.0
        (dlam,) = torch.autograd.grad(out, lam, dout)
        want = torch.full((n,), -1.0, device="cuda")
        want[-1] = -3.0
        assert torch.equal(dlam, want)

    @pytest.mark.gpu
    def test_more_rows_than_a_launch_sums(self):
        # 2^25 rows a launch of the rows' sums, where no gradient needs the
        # kernel of dq: one key, whose map gives (1 - lam) dout to its value
        n = 2 ** 25 + 100
        k = torch.full((1, 1, 1, 2), 0.5, dtype=torch.bfloat16, device="cuda")
        v = k.clone().requires_grad_(True)
        q = k.expand(1, 1, n, 2)
        lam = torch.tensor(0.25, device="cuda")
        out = ops.differential_attention(k, q, v, lam)
        dout = torch.zeros_like(out)
        dout[0, 0, -1] = 3.0  # (of the second launch)
        kg = k.clone().requires_grad_(True)
        dv, = torch.autograd.grad(out, v, dout)
        assert torch.equal(dv, torch.full_like(dv, 2.25))
        out = ops.differential_attention(kg, q, v, lam)
        dk, = torch.autograd.grad(out, kg, dout)
        # the map's gradient is G - delta = 0
        assert torch.equal(dk, torch.zeros_like(dk))


class TestNotFinite:
    """Keys and values that count and are not finite."""

    SIZES = [(1, 2, 1, 70, 150, 16, 32), (1, 2, 1, 3, 700, 16, 32),
             (1, 2, 2, 40, 90, 128, 256), (1, 1, 1, 300, 600, 20, 40)]

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", TYPES)
    @pytest.mark.parametrize("sizes", SIZES)
    @pytest.mark.parametrize("place", ["first", "last"])
    def test_infinite_scores(self, dtype, sizes, place):
        # one key with -inf in both maps: rows of positive queries give it the
        # weight 0, as if it were not there; scores of the others are +inf
        D, at = sizes[5], 0 if place == "first" else sizes[4] - 1
        a = attn_inputs(*sizes, dtype)
        for c in (0, D):
            a["queries"][..., c] = a["queries"][..., c].abs() + 0.25
            a["queries"][:, :, 1::2, c] *= -1.0
        rest = [i for i in range(sizes[4]) if i != at]
        b = dict(a, keys=a["keys"][:, :, rest], values=a["values"][:, :, rest])
        want, bound = attn_oracle(b)["out"]
        a["keys"][:, :, at, 0] = a["keys"][:, :, at, D] = -math.inf
        got = run_attn("cuda", a)["out"]
        assert_within(got[:, :, ::2], want[:, :, ::2], bound[:, :, ::2], "out")
        assert got[:, :, 1::2].isnan().all()

    @pytest.mark.gpu
    @pytest.mark.parametrize("dtype", TYPES)
    @pytest.mark.parametrize("sizes", SIZES)
    def test_not_a_number(self, dtype, sizes):
        a = attn_inputs(*sizes, dtype)
        want, bound = attn_oracle(a)["out"]
        bad = dict(a, keys=a["keys"].clone())
        bad["keys"][0, 0, 33, 1] = math.nan
        got = run_attn("cuda", bad)["out"]
        assert got[0, 0].isnan().all()  # (a head of that key head's group)
        bad = dict(a, values=a["values"].clone())
        bad["values"][0, 0, 33, 3] = math.nan
        got = run_attn("cuda", bad)["out"]
        assert got[0, 0, :, 3].isnan().all()
        rest = [i for i in range(sizes[6]) if i != 3]
        assert_within(got[..., rest], want[..., rest], bound[..., rest], "out")


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", TYPES)
def test_training_calls_repeat_and_replay(dtype):
    """The same bits in every call, eager or replayed, with lengths and shared heads."""
    a = {n: t.cuda() for n, t in attn_inputs(2, 4, 2, 140, 600, 16, 32, dtype).items()}
    lens = torch.tensor([600, 411], dtype=torch.int32, device="cuda")

    def call():
        t = {n: x.detach().requires_grad_(n != "dout") for n, x in a.items()}
        out = ops.differential_attention(
            t["keys"], t["queries"], t["values"], t["lam"], key_lengths=lens)
        names = ("keys", "queries", "values", "lam")
        return (out.detach(), *torch.autograd.grad(out, [t[n] for n in names], t["dout"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        static = call()
    for i in range(4):
        for n, size in (("queries", 1.0), ("values", 10.0 ** i), ("dout", 30.0 ** (2 - i))):
            a[n].normal_().mul_(size)
        lens[1] = 411 - 200 * i if i < 3 else 0
        first = call()
        g.replay()
        torch.cuda.synchronize()
        for x, y, z in zip(static, first, call()):
            assert torch.equal(x, y) and torch.equal(x, z)
            assert torch.isfinite(x).all()


class TestSavedTensors:
    """Hooks of the program that take what a forward pass saves, and give it back."""

    CALLS = ["norm", "attention"]

    def call(self, which):
        g = torch.Generator().manual_seed(3)
        if which == "norm":
            t = [torch.randn(s, generator=g).cuda().requires_grad_(True)
                 for s in ((6, 24), (6, 24), (24,), (24,))]
            return ops.layer_norm(t[0], t[2], t[3], residual=t[1]), t
        a = attn_inputs(2, 2, 1, 5, 9, 4, 8, torch.float32)
        t = [a[n].cuda().requires_grad_(True) for n in ("keys", "queries", "values", "lam")]
        lens = torch.tensor([9, 4], device="cuda")
        return ops.differential_attention(*t, key_lengths=lens), t

    @pytest.mark.gpu
    @pytest.mark.parametrize("which", CALLS)
    def test_offloaded(self, which):
        y, t = self.call(which)
        want = torch.autograd.grad(y.square().sum(), t)
        with torch.autograd.graph.save_on_cpu():
            y, t = self.call(which)
        for x, z in zip(torch.autograd.grad(y.square().sum(), t), want):
            assert torch.equal(x, z)

    @pytest.mark.gpu
    @pytest.mark.parametrize("name", ["differential", "differential_transformer"])
    @pytest.mark.parametrize("reentrant", [False, True])
    def test_recomputed(self, name, reentrant):
        from torch.utils.checkpoint import checkpoint

        torch.manual_seed(0)
        att = get_attender(name, 32, 32, 32, n_heads=4).cuda()
        x = torch.randn(2, 9, 32, device="cuda", requires_grad=True)
        leaves = [x, *att.parameters()]

        def grads(out):
            for t in leaves:
                t.grad = None
            out.square().sum().backward()
            return [t.grad.clone() for t in leaves]

        want = grads(att(x, x, x))
        got = grads(checkpoint(lambda t: att(t, t, t), x, use_reentrant=reentrant))
        for a, b in zip(got, want):
            assert torch.equal(a, b)

    @pytest.mark.gpu
    @pytest.mark.parametrize("which", CALLS)
    @pytest.mark.parametrize("change", [
        lambda t: t.cpu(), lambda t: t.half() if t.is_floating_point() else t.short(),
        lambda t: t[:0], lambda t: torch._neg_view(t) if t.is_floating_point() else t.cpu(),
    ])
    def test_changed(self, which, change):
        # one saved tensor after the other comes back as it was not; none of
        # that reaches a kernel
        count = 0
        for at in range(20):
            seen = []

            def pack(t):
                seen.append(t)
                return (len(seen) - 1, t)

            def unpack(it):
                return change(it[1]) if it[0] == at else it[1]

            with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
                y, t = self.call(which)
            if at >= len(seen):
                break
            try:
                grads = torch.autograd.grad(y, t, torch.ones_like(y))
            except (ValueError, TypeError, RuntimeError):
                count += 1
            else:
                # (a weight or lam may be of another floating type)
                assert seen[at].dim() == 1 and seen[at].is_floating_point()
                assert change(seen[at]).dtype == torch.float16
                assert all(torch.isfinite(x).all() for x in grads)
        assert count >= 3


@pytest.mark.gpu
def test_inference_gradients_stay():
    p = torch.zeros(4, device="cuda", requires_grad=True)
    with torch.inference_mode():
        grad = torch.full((4,), 3.0, device="cuda")
    p.grad = grad
    with pytest.raises(RuntimeError, match="[Ii]nference"):
        ops.clip_grad_norm_([p], 1.0)
    assert torch.equal(grad.cpu(), torch.full((4,), 3.0))


@pytest.mark.gpu
def test_norm_of_the_widest_rows():
    # more columns than a launch's threads hold at 64 a column
    width = 2 ** 26 + 37
    x = torch.randn(1, width, device="cuda")
    w = torch.ones(width, device="cuda", requires_grad=True)
    b = torch.zeros(width, device="cuda", requires_grad=True)
    y = ops.layer_norm(x, w, b)
    dw, db = torch.autograd.grad(y, (w, b), torch.full_like(y, 2.0))
    # one row: the sums have one term each, and 2 h is exact
    assert torch.equal(dw, 2.0 * y[0].detach())
    assert torch.equal(db, torch.full_like(db, 2.0))
    var, mean = torch.var_mean(x.double(), correction=0)
    h = (x.double() - mean) * torch.rsqrt(var + 1e-5)
    # sums of 2^26 terms, 2^18 a thread one after the other
    assert (y - h).abs().max() <= 2 ** 18 * E32 * (1 + h.abs().max())
