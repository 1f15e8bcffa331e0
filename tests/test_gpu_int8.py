"""The 8-bit linear (convrot_quantize_i8, convrot_i8_gemm, int8_linear, Int8Linear) against 64-bit arithmetic.

Bounds.  Codes of 16-bit inputs are exact (127 x has at most 18 bits, so the quotient's rounding decides as exact
arithmetic does); of float32 inputs 127 x is rounded once, 2^-24 relative, which moves a quotient of at most 127 by
less than 2e-5.  The dot is exact; its conversion, the two scales and the bias are four float32 roundings."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from convrot_mlx_b200 import _lib, adapter
from tests.gpu_util import assert_no_device_error, dev
from tests.ops64 import DTYPES, U, assert_within, codes64, randn

pytestmark = pytest.mark.gpu


def _weights(n, k, seed):
    return cr.quantize_int8_weight(randn((n, k), torch.float32, seed, 0.05))


def _check_codes(x, codes, scales, x64=None):
    q, want, s = codes64(x.double() if x64 is None else x64)
    if x.dtype == torch.float32 or x64 is not None:
        assert (codes.double() - q).abs().max() <= 0.5 + 2e-5
    else:
        assert torch.equal(codes.double(), want)
    assert ((scales.double() - s[:, 0]).abs() <= U * s[:, 0]).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", [(1, 1), (3, 15), (5, 16), (2, 4096), (7, 1997), (300, 768), (1, 15360),
                                           (2, 40001), (33, 131072)])
def test_codes(dtype, rows, features):
    x = randn((rows, features), dtype, rows + features)
    x[0, features // 2] *= 20
    codes, scales = cr.quantize_signed_int8_rowwise(x)
    assert codes.shape == (rows, features) and codes.stride(0) % 16 == 0
    _check_codes(x, codes, scales)
    assert codes.abs().amax(1).eq(127).all()


# every row shape of the quantizer's kernels: widths on either side of each, in vectors of 16 bytes, of two elements
# and of one; and rows enough that a CTA has several
ROW_SHAPES = [(3, f) for f in (31, 32, 34, 62, 66, 250, 256, 258, 510, 513, 1000, 1026, 2040, 2050, 2056, 4094, 4100, 4104,
                               8190, 8195, 8200, 16376, 16386, 16389, 16392, 32776)] + [(20000, 37), (20000, 64),
                                                                                      (9000, 130), (5000, 1032),
                                                                                      (3001, 2050)]


@pytest.mark.parametrize("scaled", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", ROW_SHAPES)
def test_codes_of_every_row_shape(dtype, rows, features, scaled):
    x = randn((rows, features), dtype, rows + features)
    factor = randn((features,), torch.float32, 5).abs() + 0.1 if scaled else None
    pitch = -(-features // 16) * 16
    codes = torch.full((rows, pitch), 99, dtype=torch.int8, device=dev())
    scales = torch.empty(rows, device=dev())
    _lib.call("convrot_quantize_i8", 0, x.data_ptr(), _lib.DTYPE_CODES[dtype], rows, features, features,
              None if factor is None else factor.data_ptr(), codes.data_ptr(), pitch, scales.data_ptr())
    assert codes[:, features:].eq(99).all()  # the padding is not touched
    _check_codes(x, codes[:, :features], scales, (x.float() * factor).double() if scaled else None)


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_strided_and_unaligned_rows(dtype):
    base = randn((9, 700), dtype, 3)
    for x in (base[:, 1:640], base[::2, 3:404], base[:, 8:520], base.t()[:600].t()):
        codes, scales = cr.quantize_signed_int8_rowwise(x)
        _check_codes(x, codes, scales)


def test_ties_round_to_even():
    # top = 4: x = top / 2 gives 63.5 -> 64, -top / 2 gives -64; other halves (2 j + 1) top / 254 are no bf16 value
    for top in (4.0, 3.0, 1.0078125, 0.0625, 2.0 ** 100, 2.0 ** -100):
        x = torch.zeros((1, 64), dtype=torch.bfloat16, device=dev())
        x[0, 0], x[0, 1], x[0, 2] = top, top / 2, -top / 2
        codes, _ = cr.quantize_signed_int8_rowwise(x)
        assert codes[0, :3].tolist() == [127, 64, -64]


def test_codes_of_extreme_rows():
    tiny, huge = 2.0 ** -149, torch.finfo(torch.float32).max
    x = torch.zeros((6, 100), device=dev())
    x[1, :3] = torch.tensor([tiny, -tiny, 0.0])
    x[2, :3] = torch.tensor([huge, -huge, huge / 127])
    x[3, 5] = float("inf")
    x[4, 7] = float("nan")
    x[5, :2] = torch.tensor([1e-30, 1e-38])
    x[3, 6], x[4, 8] = 1.0, float("-inf")
    codes, scales = cr.quantize_signed_int8_rowwise(x)
    assert codes[0].eq(0).all() and scales[0] == 0
    assert codes[1, :3].tolist() == [127, -127, 0]
    assert codes[2, :3].tolist() == [127, -127, 1] and torch.isfinite(scales[2])
    assert codes[3:5].eq(0).all() and torch.isnan(scales[3:5]).all()
    assert codes[5, :2].tolist() == [127, 0]


def _linear64(x, qweight, wscales, bias):
    """(y, bound of the float32 arithmetic) from the codes that the quantizer gives for x."""

    codes, scales = cr.quantize_signed_int8_rowwise(x.reshape(-1, x.shape[-1]))
    core = codes.double() @ qweight.double().T * scales.double()[:, None] * wscales.double()
    y = core if bias is None else core + bias.double()
    return y, 3.5 * U * core.abs() + U * y.abs()


SIZES = [(1, 1, 1), (1, 4096, 4096), (2, 33, 17), (5, 512, 640), (8, 1000, 264), (16, 2048, 96), (17, 129, 257),
         (64, 3000, 200), (65, 160, 1211), (127, 128, 128), (128, 256, 256), (129, 144, 259), (333, 1997, 1211),
         (257, 4160, 520), (600, 96, 2050), (1100, 1536, 1024),
         (1300, 300, 2100), (1300, 2103, 333), (300, 1997, 5001), (300, 5008, 1040), (2500, 130, 1000), (2500, 1000, 129),
         (4000, 1216, 1216), (5000, 128, 1100), (5000, 1100, 130), (40, 8192, 300), (100, 6000, 260), (16, 15000, 130),
         (3, 8200, 70), (1, 8208, 40), (7, 130, 9000), (2, 4100, 5000), (200, 64, 6000)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(dtype, m, k, n):
    qweight, wscales = _weights(n, k, 11)
    bias = randn((n,), torch.float32, 12) if (m + n) % 2 else None
    x = randn((m, k), dtype, 13)
    y = cr.int8_linear(x, qweight, wscales, bias)
    assert y.shape == (m, n) and y.dtype == dtype
    assert_within(y, *_linear64(x, qweight, wscales, bias), f"{m} {k} {n}")
    assert torch.equal(y, cr.int8_linear(x, qweight, wscales, bias))
    assert_no_device_error()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_input_gradient(dtype, m, k, n):
    qweight, wscales = _weights(n, k, 21)
    x = randn((m, k), dtype, 22).requires_grad_()
    dy = randn((m, n), dtype, 23, 0.1)
    y = cr.int8_linear(x, qweight, wscales)
    (dx,) = torch.autograd.grad(y, x, dy)
    assert dx.shape == x.shape and dx.dtype == dtype
    # the definition: dy * wscales in float32, quantized per token, times the codes of the weight
    g = (dy.float() * wscales).double()
    q, c, s = codes64(g)
    # a code may go either way where the float32 rounding of 127 g decides a half; each is worth one weight row
    near = ((q - q.floor() - 0.5).abs() < 2e-5).double()
    core = c @ qweight.double() * s
    assert_within(dx, core, 3.5 * U * core.abs() + near @ qweight.double().abs() * s, f"{m} {k} {n}")
    # and the gradient itself: half a code step of each token's dy, against every weight
    exact = g @ qweight.double()
    assert ((core - exact).abs() <= 0.5001 * s * qweight.double().abs().sum(0)).all()
    assert_no_device_error()


def test_gradient_against_differences():
    # y is linear in x up to half a code step of each of the two inputs, so a difference over a long step shows the
    # gradient: sum(dy * (y(x + v) - y(x))) = sum(dx * v) within those steps
    m, k, n = 19, 384, 200
    qweight, wscales = _weights(n, k, 31)
    x, v = randn((m, k), torch.float32, 32), randn((m, k), torch.float32, 33)
    dy = randn((m, n), torch.float32, 34)
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(cr.int8_linear(xr, qweight, wscales), xr, dy)
    d = cr.int8_linear(x + v, qweight, wscales).double() - cr.int8_linear(x, qweight, wscales).double()
    got, want = (dy.double() * d).sum(1), (dx.double() * v.double()).sum(1)
    w = (qweight.double() * wscales.double()[:, None]).abs()
    step = lambda t: t.double().abs().amax(1) / 254  # noqa: E731
    bound = (step(x + v) + step(x)) * (dy.double().abs() @ w).sum(1)
    bound += step(dy * wscales) * (v.double().abs() @ qweight.double().abs().T).sum(1)
    assert ((got - want).abs() <= 1.001 * bound + 1e-3).all()


def test_matmul_int32_extremes():
    # every product at its largest: the dot is 127 * 127 * k, near 2^31 at the largest k
    for k in (131072, 4096):
        codes = torch.full((3, k), 127, dtype=torch.int8, device=dev())
        codes[1] = -127
        codes[2, ::2] = -127
        w = torch.full((20, k), 127, dtype=torch.int8, device=dev())
        one = torch.ones(20, device=dev())
        y = cr.int8_matmul(codes, w, one[:3], one, output_dtype=torch.float32)
        want = float(127 * 127 * k)
        assert torch.equal(y[0], torch.full((20,), want, device=dev())) and torch.equal(y[1], -y[0])
        assert y[2].eq(0).all()


def test_matmul_copies_rows_off_the_pitch():
    codes = torch.randint(-127, 128, (40, 100), dtype=torch.int8, device=dev())
    w = torch.randint(-127, 128, (50, 100), dtype=torch.int8, device=dev())
    xs, ws = randn((40,), torch.float32, 1).abs(), randn((50,), torch.float32, 2).abs()
    want = codes.double() @ w.double().T * xs.double()[:, None] * ws.double()
    for a, b in ((codes, w), (codes[:, 3:90], w[:, 3:90]), (codes.t().contiguous().t(), w)):
        y = cr.int8_matmul(a, b, xs, ws, output_dtype=torch.float32)
        want = a.double() @ b.double().T * xs.double()[:, None] * ws.double()
        assert_within(y, want, 3 * U * want.abs())


@pytest.mark.parametrize("m", [3, 200])
def test_rows_that_are_not_finite(m):
    qweight, wscales = _weights(40, 96, 41)
    x = randn((m, 96), torch.bfloat16, 42)
    x[1, 5] = float("nan")
    x[2, 7] = float("inf")
    y = cr.int8_linear(x, qweight, wscales)
    assert torch.isnan(y[1:3]).all()
    assert torch.isfinite(torch.cat((y[:1], y[3:]))).all()


def test_leading_dimensions_empty_rows_and_expanded_gradients():
    qweight, wscales = _weights(48, 80, 51)
    x = randn((2, 3, 5, 80), torch.bfloat16, 52)
    y = cr.int8_linear(x, qweight, wscales)
    assert y.shape == (2, 3, 5, 48)
    assert torch.equal(y.reshape(-1, 48), cr.int8_linear(x.reshape(-1, 80), qweight, wscales))
    assert torch.equal(cr.int8_linear(x[0, 0, 0], qweight, wscales), y[0, 0, 0])
    e = torch.empty((0, 4, 80), dtype=torch.bfloat16, device=dev(), requires_grad=True)
    ye = cr.int8_linear(e, qweight, wscales)
    assert ye.shape == (0, 4, 48)
    assert torch.autograd.grad(ye.sum(), e)[0].shape == e.shape
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(cr.int8_linear(xr, qweight, wscales).sum(), xr)
    (dx2,) = torch.autograd.grad(cr.int8_linear(xr, qweight, wscales), xr, torch.ones_like(y))
    assert torch.equal(dx, dx2)


def test_module_and_swap():
    torch.manual_seed(5)
    dense = torch.nn.Sequential(torch.nn.Linear(100, 64), torch.nn.GELU(), torch.nn.Linear(64, 40, bias=False)).to(dev())
    x = randn((30, 100), torch.float32, 61)
    want = dense(x)
    names = adapter.replace_int8_linears(dense)
    assert names == ["0", "2"] and isinstance(dense[0], cr.Int8Linear) and dense[2].bias is None
    got = dense(x)
    assert (got - want).norm() / want.norm() < 0.03  # 8-bit steps of 4 operands, each about 1/254 of its largest
    state = dense.state_dict()
    other = torch.nn.Sequential(cr.Int8Linear(100, 64, device=dev()), torch.nn.GELU(),
                                cr.Int8Linear(64, 40, bias=False, device=dev()))
    other.load_state_dict(state)
    assert torch.equal(other(x), got)


def test_other_stream():
    qweight, wscales = _weights(256, 512, 71)
    x = randn((64, 512), torch.bfloat16, 72)
    want = cr.int8_linear(x, qweight, wscales)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = cr.int8_linear(x, qweight, wscales)
    side.synchronize()
    assert torch.equal(got, want)


def test_outputs_past_32_bits():
    m, n, k = 70001, 32768, 16
    qweight, wscales = _weights(n, k, 81)
    x = randn((m, k), torch.bfloat16, 82)
    y = cr.int8_linear(x, qweight, wscales)
    for rows in (slice(0, 3), slice(65534, 65540), slice(m - 3, m)):
        assert torch.equal(y[rows], cr.int8_linear(x[rows].clone(), qweight, wscales))
    assert_no_device_error()


def test_refusals():
    qweight, wscales = _weights(32, 64, 91)
    x = randn((4, 64), torch.bfloat16, 92)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        cr.int8_linear(x.double(), qweight, wscales)
    with pytest.raises(ValueError, match="CUDA"):
        cr.int8_linear(x.cpu(), qweight, wscales)
    with pytest.raises(ValueError, match="frozen"):
        cr.int8_linear(x, qweight, wscales.clone().requires_grad_())
    with pytest.raises(NotImplementedError, match="overflow the int32 dot"):
        cr.int8_linear(torch.zeros((1, 131073), dtype=torch.bfloat16, device=dev()),
                       torch.zeros((8, 131088), dtype=torch.int8, device=dev())[:, :131073], wscales[:8])
    lib = _lib.load()
    args = lambda stride, off: (_lib.ptr(qweight), stride, _lib.ptr(qweight), 64, 0, _lib.ptr(wscales), None, None,  # noqa: E731
                                _lib.ptr(x.view(torch.int8)[0, off:]), 2, 4, 4, 64, None)
    assert lib.convrot_i8_gemm(*args(65, 0)) == -1
    assert lib.convrot_i8_gemm(*args(64, 2)) == -1
