"""Calls at the edges of differential attention, layer norm and gradient
clipping: types, values and ways of calling that ordinary use seldom meets.

Tolerances are those of test_train_ops: elementwise bounds on what rounding
can do.
"""

import math

import pytest
import torch

from npf import ops
from test_train_ops import E32, SHAPES, check_clip, params_of

HALF = [torch.bfloat16, torch.float16]


class TestComposedClip:
    """The composed form, whose sums and factor are held in more bits than
    16-bit gradients, like the kernels'."""

    @pytest.mark.parametrize("dtype", HALF)
    @pytest.mark.parametrize("p", [1.0, 2.0, math.inf])
    def test_half(self, dtype, p):
        for max_norm in (0.5, 1e9, 0.0):
            check_clip(params_of(SHAPES, dtype, "cpu"), max_norm, p)
        params = params_of(SHAPES, dtype, "cpu")
        assert ops.grad_norm(params, p).dtype == torch.float32

    def test_norm_over_the_types_largest(self):
        # finite gradients whose norm, about 1e5, no fp16 value holds
        params = params_of([(1000000,)], torch.float16, "cpu", std=100.0)
        check_clip(params, 1.0, error_if_nonfinite=True)
        assert params[0].grad.any()

    def test_squares_that_overflow_fp32(self):
        check_clip(params_of([(50,)], torch.float32, "cpu", std=1e25), 1.0)

    def test_mixed(self):
        params = []
        for i, dtype in enumerate((torch.bfloat16, torch.float32, torch.float16)):
            params += params_of([(n,) for n in range(1, 20)], dtype, "cpu", seed=i)
        assert ops.grad_norm(params).dtype == torch.float32
        check_clip(params, 3.0)
        wide = params_of([(7,)], torch.float64, "cpu")
        old = wide[0].grad.clone()
        want = torch.linalg.vector_norm(torch.cat(
            [p.grad.double().reshape(-1) for p in params + wide]))
        total = ops.clip_grad_norm_(params + wide, 1.0)
        assert total.dtype == torch.float64
        # 64-bit sums and products of 200 terms
        assert (total - want).abs() <= 256 * 2.0 ** -53 * want
        off = (wide[0].grad - old / (want + 1e-6)).abs()
        assert (off <= 256 * 2.0 ** -53 * old.abs()).all()
