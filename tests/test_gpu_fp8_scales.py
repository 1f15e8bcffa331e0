"""The 8-bit floating-point product where the two scales of a block are far apart: what comes out is an ordinary number."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.fp8_64 import product64, values_of_blocks, values_of_rows
from tests.gpu_util import assert_no_device_error
from tests.ops64 import TINY, assert_within, randn

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("m", [1, 2, 5, 8, 40, 700])
@pytest.mark.parametrize("ew,ex", [(124, -110), (-110, 124), (-135, 100), (100, -135), (-125, 120), (60, 50), (-60, -70),
                                   (118, -118)])
def test_scales_far_apart(ew, ex, m, dtype):
    # magnitudes from 1 to 2 and one sign: the sums of codes are as large as they get
    w = (1 + randn((72, 400), torch.float32, 1).abs().clamp(max=1)) * 2.0 ** ew
    x = ((1 + randn((m, 400), torch.float32, 2).abs().clamp(max=0.99)) * 2.0 ** ex).to(dtype)
    qweight, wscales = cr.quantize_fp8_weight(w)
    codes, xscales = cr.quantize_fp8_blockwise(x)
    want, slack = product64(values_of_rows(codes, xscales), values_of_blocks(qweight, wscales))
    # sums below the normal range are rounded to multiples of 2^-149, once a block of 128 and warp
    slack = slack + 16 * TINY[torch.float32]
    for y in (cr.fp8_linear(x, qweight, wscales), cr.fp8_matmul(codes, qweight, xscales, wscales, output_dtype=dtype)):
        assert_within(y, want, slack, f"{m} tokens")
    assert_no_device_error()


@pytest.mark.parametrize("m", [1, 2, 8])
def test_scales_that_are_nan_beside_small_and_large_ones(m):
    w, x = randn((72, 400), torch.float32, 3), randn((m, 400), torch.float32, 4)
    qweight, wscales = cr.quantize_fp8_weight(w)
    codes, xscales = cr.quantize_fp8_blockwise(x)
    for byte in (0, 127, 254):
        for which in ("x", "w"):
            xs, ws = xscales.view(torch.uint8).clone(), wscales.view(torch.uint8).clone()
            (ws if which == "x" else xs).fill_(byte)
            if which == "x":
                xs[m - 1, 1] = 255
            else:
                ws[0, 2] = 255
            y = cr.fp8_matmul(codes, qweight, xs.view(torch.float8_e8m0fnu), ws.view(torch.float8_e8m0fnu),
                              output_dtype=torch.float32)
            assert torch.isnan(y[m - 1]).all()
            # A weight's scale of 2^127 takes blocks to 2^16 * 2^127 * 2^-8 and more, beyond float32: each is infinite, and two
            # of opposite signs make a NaN that is not the scale's.
            assert which == "w" or byte == 254 or not torch.isnan(y[:m - 1]).any()
