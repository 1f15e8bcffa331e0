"""The modulated layer norm with shift and scale of different types and memory orders, against 64-bit arithmetic (bounds
of test_gpu_norm.py): each vector has to be read where it lies, also after one of them was converted to float32."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import assert_no_device_error, dev
from tests.ops64 import U, assert_within, randn
from tests.test_gpu_norm import EPS, _dx64, _inputs, _norm64, _sums64

pytestmark = pytest.mark.gpu
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


def _vector(batch, features, dtype, layout, seed):
    if layout == "columns":  # of a wider modulation output
        return randn((batch, 1, 6 * features), dtype, seed, 0.3).chunk(6, dim=-1)[seed % 6]
    if layout == "turned":  # dense, but features are not the inner dimension
        return randn((features, batch), dtype, seed, 0.3).t()
    if layout == "shared":
        return randn((1, 1, features), dtype, seed, 0.3)
    return randn((batch, features), dtype, seed, 0.3)


@pytest.mark.parametrize("layouts", [("columns", "columns"), ("columns", "packed"), ("packed", "columns"),
                                     ("turned", "turned"), ("turned", "columns"), ("shared", "columns")])
@pytest.mark.parametrize("dtypes", [(BF16, F32, BF16), (BF16, BF16, F32), (BF16, F16, F32), (F16, F32, F16), (F32, F32, BF16),
                                    (F32, BF16, F32), (F32, F16, BF16), (BF16, BF16, BF16)],
                         ids=lambda d: "-".join(str(t)[6:] for t in d))
@pytest.mark.parametrize("batch,tokens,features", [(3, 5, 64), (7, 2, 33)])
def test_modulation_of_mixed_types_and_orders(batch, tokens, features, dtypes, layouts):
    dtype, shift_dtype, scale_dtype = dtypes
    x = _inputs(batch * tokens, features, dtype, 7).view(batch, tokens, features).requires_grad_()
    shift = _vector(batch, features, shift_dtype, layouts[0], 8).requires_grad_()
    scale = _vector(batch, features, scale_dtype, layouts[1], 9).requires_grad_()
    dy = randn(x.shape, dtype, 10)
    y = cr.modulated_layer_norm(x, shift, scale, EPS)
    x0 = x.detach()
    w0 = (1 + scale.detach().double()).reshape(-1, 1, features).expand(batch, 1, features)
    b0 = shift.detach().reshape(-1, 1, features).expand(batch, 1, features)
    y64, slack, *_ = _norm64(x0, w0, b0)
    assert_within(y.detach(), y64, slack + U * y64.abs(), "y")  # 1 + scale is one more rounding
    dx, dshift, dscale = torch.autograd.grad(y, (x, shift, scale), dy)
    want, s = _dx64(x0, w0, b0, dy)
    _, _, h, _, r, *_ = _norm64(x0, w0, b0)
    g = (dy.double() * w0).abs()
    one = U * r * (g + g.mean(-1, keepdim=True) + h.abs() * (g * h.abs()).mean(-1, keepdim=True))
    assert_within(dx, want, s + one, "dx")
    dw64, sw, db64, sb = _sums64(x0, w0, b0, dy, (1,))
    if layouts[0] == "shared":  # one more sum, of the samples' own in the vector's type
        assert dshift.shape == shift.shape
    else:
        assert dshift.dtype == shift_dtype and dshift.shape == shift.shape
        assert_within(dshift.reshape(batch, features), db64, sb, "dshift")
    assert dscale.dtype == scale_dtype and dscale.shape == scale.shape
    assert_within(dscale.reshape(batch, features), dw64, sw, "dscale")
    assert_no_device_error()
