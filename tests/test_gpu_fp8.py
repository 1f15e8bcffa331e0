"""The 8-bit floating-point linear (convrot_quantize_fp8, convrot_quantize_fp8_weight, convrot_fp8_gemm, fp8_linear,
Fp8Linear) against 64-bit arithmetic.

Bounds.  Scales are powers of two, so x * 2^-e is exact and codes are one rounding of it: they have to be equal.  The
product's bound is in fp8_64.product64."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from convrot_mlx_b200 import _lib, adapter
from tests.fp8_64 import blocks64, product64, rows64, values_of_blocks, values_of_rows
from tests.gpu_util import assert_no_device_error, dev
from tests.ops64 import DTYPES, assert_within, randn

pytestmark = pytest.mark.gpu


def _uneven(shape, dtype, seed, scale=1.0):
    """Normal values whose columns differ by some powers of two."""

    return (randn(shape, torch.float32, seed, scale) * torch.exp2(randn(shape[-1:], torch.float32, seed + 1) * 2)).to(dtype)


def _weights(n, k, seed):
    return cr.quantize_fp8_weight(_uneven((n, k), torch.float32, seed, 0.05))


def _scale_bytes(e):
    return (e + 127).to(torch.uint8)


# --- quantizers ---------------------------------------------------------------


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", [(1, 1), (3, 15), (5, 16), (2, 127), (2, 128), (2, 129), (7, 1997), (300, 768),
                                           (1, 15360), (33, 4104), (1000, 130), (257, 513)])
def test_codes_of_rows(dtype, rows, features):
    x = _uneven((rows, features), dtype, rows + features)
    codes, scales = cr.quantize_fp8_blockwise(x)
    assert codes.shape == (rows, features) and codes.stride(0) % 16 == 0 and scales.stride(0) % 4 == 0
    want, e = rows64(x)
    assert torch.equal(codes.double(), want)
    assert torch.equal(scales.view(torch.uint8), _scale_bytes(e))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,k", [(1, 1), (127, 129), (128, 128), (129, 127), (300, 1000), (1000, 264), (257, 16)])
def test_codes_of_weights(dtype, n, k):
    w = _uneven((n, k), dtype, n + k)
    codes, scales = cr.quantize_fp8_weight(w)
    want, e = blocks64(w)
    assert torch.equal(codes.double(), want)
    assert torch.equal(scales.view(torch.uint8), _scale_bytes(e))


@pytest.mark.parametrize("dtype", DTYPES)
def test_codes_of_strided_and_unaligned_rows(dtype):
    base = _uneven((290, 700), dtype, 3)
    for x in (base[:, 1:640], base[::2, 3:404], base[:, 8:520], base.t()[:600].t(), base.t()):
        codes, scales = cr.quantize_fp8_blockwise(x)
        assert torch.equal(codes.double(), rows64(x)[0])
        codes, scales = cr.quantize_fp8_weight(x)
        assert torch.equal(codes.double(), blocks64(x)[0])


def test_codes_of_extreme_blocks():
    tiny, huge = 2.0 ** -149, torch.finfo(torch.float32).max
    x = torch.zeros((9, 300), device=dev())
    x[1, :3] = torch.tensor([tiny, -tiny, 0.0])
    x[2, :3] = torch.tensor([huge, -huge, huge / 300])
    x[3, 5], x[3, 200] = float("inf"), 1.0
    x[4, 7], x[4, 299] = float("nan"), 2.0
    x[5, :3] = torch.tensor([448.0, -448.0, 1.0])
    x[6, :3] = torch.tensor([448.00003, 2.0 ** -6, 2.0 ** -9])
    x[7, :4] = torch.tensor([256.0, 0.25, 2.0 ** -10, 2.0 ** -10 * 1.5])  # ties and steps at the bottom
    x[8, 128:131] = torch.tensor([1e-37, 1e-38, 3e-40])
    codes, scales = cr.quantize_fp8_blockwise(x)
    bytes_ = scales.view(torch.uint8)
    finite = [0, 1, 2, 5, 6, 7, 8]
    want, e = rows64(x[finite])
    assert torch.equal(codes[finite].double(), want)
    assert torch.equal(bytes_[finite], _scale_bytes(e))
    assert bytes_[3].tolist() == [255, 119, 0] and codes[3, 200] == 256.0 and codes[3, :128].double().eq(0).all()
    assert bytes_[4].tolist() == [255, 0, 120] and codes[4, :128].double().eq(0).all()
    w = torch.ones((130, 130), device=dev())
    w[3, 4], w[129, 5] = float("nan"), float("-inf")
    codes, scales = cr.quantize_fp8_weight(w)
    assert scales.view(torch.uint8).tolist() == [[255, 119], [255, 119]]
    assert codes[:, :128].double().eq(0).all() and codes[:, 128:].double().eq(256).all()


# --- product ------------------------------------------------------------------

SIZES = [(1, 1, 1), (1, 4096, 4096), (2, 33, 17), (5, 512, 640), (8, 1000, 264), (9, 140, 40), (16, 2048, 96),
         (17, 129, 257), (64, 3000, 200), (65, 160, 1211), (127, 128, 128), (128, 256, 256), (129, 144, 259),
         (451, 2203, 1301), (257, 4160, 520), (600, 96, 2050), (1100, 1536, 1024), (1300, 300, 2100), (1300, 2103, 333),
         (300, 1997, 5001), (300, 5008, 1040), (2500, 130, 1000), (2500, 1000, 129), (4000, 1216, 1216),
         (5000, 128, 1100), (5000, 1100, 130), (40, 8192, 300), (100, 6000, 260), (16, 15000, 130), (3, 8200, 70),
         (1, 8208, 40), (7, 130, 9000), (2, 4100, 5000), (200, 64, 6000), (8, 12300, 33), (4, 1, 300), (300, 1, 4)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_linear(dtype, m, k, n):
    qweight, wscales = _weights(n, k, 11)
    bias = randn((n,), torch.float32, 12) if (m + n) % 2 else None
    x = _uneven((m, k), dtype, 13)
    y = cr.fp8_linear(x, qweight, wscales, bias)
    assert y.shape == (m, n) and y.dtype == dtype
    a = values_of_rows(*cr.quantize_fp8_blockwise(x))
    assert_within(y, *product64(a, values_of_blocks(qweight, wscales), bias), f"{m} {k} {n}")
    assert torch.equal(y, cr.fp8_linear(x, qweight, wscales, bias))
    assert_no_device_error()


@pytest.mark.parametrize("m,k,n", [(30, 8192, 100), (30, 8193, 100), (300, 20000, 40), (4, 17000, 33)])
def test_float32_outputs_over_long_sums(m, k, n):
    # ranges of 8192 channels: each 256 steps, as product64 counts them, and the additions of the ranges
    qweight, wscales = _weights(n, k, 15)
    bias = randn((n,), torch.float32, 16)
    x = _uneven((m, k), torch.float32, 17).requires_grad_()
    y = cr.fp8_linear(x, qweight, wscales, bias)
    a, w = values_of_rows(*cr.quantize_fp8_blockwise(x)), values_of_blocks(qweight, wscales)
    want, _ = product64(a, w, bias)
    slack = (256 + 32 + 4) * 2.0 ** -22 * (a.abs() @ w.abs().T) + 2.0 ** -22 * want.abs()
    assert_within(y.detach(), want, slack)
    dy = _uneven((k, m), torch.float32, 18).t()[:, :].contiguous()
    back, bscales = cr.quantize_fp8_weight(w.T.float())  # a weight of k channels: the gradient sums over them
    z = torch.zeros((m, n), device=dev(), requires_grad=True)
    (dz,) = torch.autograd.grad(cr.fp8_linear(z, back, bscales), z, dy)
    a, w = values_of_rows(*cr.quantize_fp8_blockwise(dy)), values_of_blocks(back, bscales)
    assert_within(dz, a @ w, (256 + 32 + 4) * 2.0 ** -22 * (a.abs() @ w.abs()) + 2.0 ** -22 * (a @ w).abs())


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("m,k,n", SIZES)
def test_input_gradient(dtype, m, k, n):
    qweight, wscales = _weights(n, k, 21)
    x = randn((m, k), dtype, 22).requires_grad_()
    dy = _uneven((m, n), dtype, 23, 0.1)
    (dx,) = torch.autograd.grad(cr.fp8_linear(x, qweight, wscales), x, dy)
    assert dx.shape == x.shape and dx.dtype == dtype
    a, w = values_of_rows(*cr.quantize_fp8_blockwise(dy)), values_of_blocks(qweight, wscales)
    assert_within(dx, *product64(a, w.T), f"{m} {k} {n}")
    # and the gradient itself: half a step of each code of dy, against every weight (2^-4 of the code, or 2^-10 of the
    # block's scale, which is at most its largest magnitude / 224)
    top = torch.nn.functional.pad(dy.double(), (0, -n % 128)).unflatten(1, (-1, 128)).abs().amax(-1)
    slack = dy.double().abs() * 2.0 ** -4 + (top / 224 * 2.0 ** -10).repeat_interleave(128, 1)[:, :n]
    assert ((a @ w - dy.double() @ w).abs() <= slack @ w.abs() + 1e-30).all()
    assert_no_device_error()


def test_scales_of_every_block_are_applied():
    # one code of 1 in each block of a token, scales all different: the product spells them out.  Its terms lie between
    # 2^-17 and 2^17, more bits than float32 has, so the sums' bound applies.
    m, k, n = 150, 1400, 400
    kb, nb = 11, 4
    codes = torch.zeros((m, 1408), device=dev())
    e = (torch.arange(m, device=dev())[:, None] * 7 + torch.arange(kb, device=dev()) * 5) % 23 - 11
    we = (torch.arange(nb, device=dev())[:, None] * 3 + torch.arange(kb, device=dev()) * 2) % 13 - 6
    for b in range(kb):
        codes[torch.arange(m), torch.arange(m) % 100 + 128 * b if b < 10 else 128 * b + torch.arange(m) % 100] = 1.0
    codes = codes[:, :k].to(torch.float8_e4m3fn)
    weight = torch.ones((n, k), device=dev()).to(torch.float8_e4m3fn)
    xs, ws = _scale_bytes(e).view(torch.float8_e8m0fnu), _scale_bytes(we).view(torch.float8_e8m0fnu)
    want, slack = product64(values_of_rows(codes, xs), values_of_blocks(weight, ws))
    for rows in (1, 5, 16, 33, 64, 100, 150):
        y = cr.fp8_matmul(codes[:rows], weight, xs[:rows], ws, output_dtype=torch.float32)
        assert_within(y, want[:rows], slack[:rows], f"{rows} rows")


def test_gradient_against_differences():
    # y is linear in x up to the rounding of both codes (2^-4 of a value and 2^-10 of its block's largest / 224), so a
    # difference over a long step shows the gradient within those
    m, k, n = 19, 384, 200
    qweight, wscales = _weights(n, k, 31)
    x, v = randn((m, k), torch.float32, 32), randn((m, k), torch.float32, 33)
    dy = randn((m, n), torch.float32, 34)
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(cr.fp8_linear(xr, qweight, wscales), xr, dy)
    d = cr.fp8_linear(x + v, qweight, wscales).double() - cr.fp8_linear(x, qweight, wscales).double()
    got, want = (dy.double() * d).sum(1), (dx.double() * v.double()).sum(1)
    w = values_of_blocks(qweight, wscales).abs()
    step = lambda t: t.double().abs() * 2.0 ** -4 + t.double().abs().amax() * 2.0 ** -17  # noqa: E731
    bound = ((step(x + v) + step(x)) * (dy.double().abs() @ w)).sum(1) + (step(dy) @ w * v.double().abs()).sum(1)
    assert ((got - want).abs() <= 1.01 * bound).all()


def test_matmul_copies_rows_off_the_pitch():
    codes, xs = cr.quantize_fp8_blockwise(randn((40, 700), torch.float32, 1))
    w, ws = cr.quantize_fp8_weight(randn((50, 700), torch.float32, 2))
    want = cr.fp8_matmul(codes, w, xs, ws, output_dtype=torch.float32)
    odd = torch.empty((40, 701), dtype=torch.uint8, device=dev()).view(torch.float8_e4m3fn)[:, 1:]
    odd.copy_(codes)
    scales = torch.empty((40, 7), dtype=torch.uint8, device=dev())[:, 1:]
    scales.copy_(xs.view(torch.uint8))
    packed = xs.view(torch.uint8).contiguous()
    for a, b, s in ((odd, w.contiguous(), scales), (codes.t().contiguous().t(), w, packed), (codes, w, packed)):
        assert torch.equal(cr.fp8_matmul(a, b, s.view(torch.float8_e8m0fnu), ws, output_dtype=torch.float32), want)
    assert cr.fp8_matmul(codes[:0], w, xs[:0], ws, output_dtype=torch.bfloat16).shape == (0, 50)


@pytest.mark.parametrize("m", [1, 5, 40])
def test_weights_whose_storage_ends_with_the_last_row(m):
    # the padding of the rows holds NaN codes, that of the last row is not there
    n, k = 70, 203
    w, ws = _weights(n, k, 43)
    x = randn((m, k), torch.bfloat16, 44)
    want = cr.fp8_linear(x, w, ws)
    short = torch.full(((n - 1) * 208 + k,), 127, dtype=torch.uint8, device=dev()).view(torch.float8_e4m3fn)
    short = short.as_strided((n, k), (208, 1))
    short.copy_(w)
    assert torch.equal(cr.fp8_linear(x, short, ws), want)
    padded = torch.full((n, 208), 255, dtype=torch.uint8, device=dev()).view(torch.float8_e4m3fn)[:, :k]
    padded.copy_(w)
    assert torch.equal(cr.fp8_linear(x, padded, ws), want)
    codes, xs = cr.quantize_fp8_blockwise(x)
    assert torch.equal(cr.fp8_matmul(codes, short, xs, ws, output_dtype=torch.bfloat16),
                       cr.fp8_matmul(codes, w, xs, ws, output_dtype=torch.bfloat16))


@pytest.mark.parametrize("m", [3, 12, 200, 3000])
def test_rows_and_blocks_that_are_not_finite(m):
    qweight, wscales = _weights(300, 1400, 41)
    x = randn((m, 1400), torch.bfloat16, 42)
    x[1, 5] = float("nan")
    x[2, 1399] = float("inf")
    y = cr.fp8_linear(x, qweight, wscales)
    assert torch.isnan(y[1:3]).all()
    assert torch.isfinite(torch.cat((y[:1], y[3:]))).all()
    bad = wscales.view(torch.uint8).clone()
    bad[1, 3] = 255
    y = cr.fp8_linear(x[3:] if m > 3 else x[:1], qweight, bad.view(torch.float8_e8m0fnu))
    assert torch.isnan(y[:, 128:256]).all()
    assert torch.isfinite(y[:, :128]).all() and torch.isfinite(y[:, 256:]).all()


def test_extreme_scales():
    # the largest and smallest values: sums stay where float32 is
    for size in (2.0 ** 100, 2.0 ** -100, 2.0 ** -126):
        for m in (1, 40, 700):
            x = randn((m, 256), torch.float32, 45) * size
            qweight, wscales = cr.quantize_fp8_weight(randn((256, 256), torch.float32, 46))
            y = cr.fp8_linear(x, qweight, wscales)
            a = values_of_rows(*cr.quantize_fp8_blockwise(x))
            want, slack = product64(a, values_of_blocks(qweight, wscales))
            assert ((y.double() - want).abs() <= slack + 2.0 ** -140).all()


def test_leading_dimensions_empty_rows_and_expanded_gradients():
    qweight, wscales = _weights(48, 80, 51)
    x = randn((2, 3, 5, 80), torch.bfloat16, 52)
    y = cr.fp8_linear(x, qweight, wscales)
    assert y.shape == (2, 3, 5, 48)
    assert torch.equal(y.reshape(-1, 48), cr.fp8_linear(x.reshape(-1, 80), qweight, wscales))
    e = torch.empty((0, 4, 80), dtype=torch.bfloat16, device=dev(), requires_grad=True)
    ye = cr.fp8_linear(e, qweight, wscales)
    assert ye.shape == (0, 4, 48)
    assert torch.autograd.grad(ye.sum(), e)[0].shape == e.shape
    xr = x.clone().requires_grad_()
    (dx,) = torch.autograd.grad(cr.fp8_linear(xr, qweight, wscales).sum(), xr)
    (dx2,) = torch.autograd.grad(cr.fp8_linear(xr, qweight, wscales), xr, torch.ones_like(y))
    assert torch.equal(dx, dx2)
    with pytest.raises(RuntimeError, match="create_graph"):
        torch.autograd.grad(cr.fp8_linear(xr, qweight, wscales).sum(), xr, create_graph=True)


def test_graphs_kept_released_and_changed():
    qweight, wscales = _weights(48, 80, 53)
    x = randn((7, 80), torch.bfloat16, 54).requires_grad_()
    y = cr.fp8_linear(x, qweight, wscales)
    dy = torch.ones_like(y)
    (a,) = torch.autograd.grad(y, x, dy, retain_graph=True)
    (b,) = torch.autograd.grad(y, x, dy)
    assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="second time"):
        torch.autograd.grad(y, x, dy)
    y = cr.fp8_linear(x, qweight, wscales)
    qweight.view(torch.uint8).zero_()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        torch.autograd.grad(y, x, dy)
    cr.fp8_linear(x, qweight, wscales).sum().backward()
    assert x.grad.eq(0).all()
    with torch.no_grad():
        assert not cr.fp8_linear(x, qweight, wscales).requires_grad


def test_strided_inputs_and_gradients():
    qweight, wscales = _weights(200, 300, 55)
    base = randn((64, 700), torch.float16, 56)
    for x in (base[:, 3:303], base[:, 8:308], base.t()[:300, :].t(), base[::3, 100:400]):
        assert torch.equal(cr.fp8_linear(x, qweight, wscales), cr.fp8_linear(x.contiguous(), qweight, wscales))
    x = base[:, :300].clone().requires_grad_()
    dy = randn((200, 64), torch.float16, 57)
    (a,) = torch.autograd.grad(cr.fp8_linear(x, qweight, wscales), x, dy.t())
    (b,) = torch.autograd.grad(cr.fp8_linear(x, qweight, wscales), x, dy.t().contiguous())
    assert torch.equal(a, b)


def test_module_and_swap():
    torch.manual_seed(5)
    dense = torch.nn.Sequential(torch.nn.Linear(300, 164), torch.nn.GELU(), torch.nn.Linear(164, 40, bias=False)).to(dev())
    x = randn((30, 300), torch.float32, 61)
    want = dense(x)
    assert adapter.replace_fp8_linears(dense) == ["0", "2"]
    assert isinstance(dense[0], cr.Fp8Linear) and dense[2].bias is None
    got = dense(x)
    # four operands with steps of 2^-4 at most, 2.6% on average each: about 5%
    assert (got - want).norm() / want.norm() < 0.08
    other = torch.nn.Sequential(cr.Fp8Linear(300, 164, device=dev()), torch.nn.GELU(),
                                cr.Fp8Linear(164, 40, bias=False, device=dev()))
    other.load_state_dict(dense.state_dict())
    assert torch.equal(other(x), got)
    half = other.half()
    assert half[0].bias.dtype == torch.float32 and half[0].qweight.dtype == torch.uint8
    assert torch.equal(half(x), got)


def test_other_stream():
    qweight, wscales = _weights(256, 512, 71)
    for m in (2, 64, 3000):
        x = randn((m, 512), torch.bfloat16, 72)
        want = cr.fp8_linear(x, qweight, wscales)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = cr.fp8_linear(x, qweight, wscales)
        side.synchronize()
        assert torch.equal(got, want)


def test_calls_at_once():
    # products of every kernel on two streams, one after the other without waiting
    qweight, wscales = _weights(520, 1040, 77)
    inputs = [[randn((m, 1040), torch.bfloat16, 78 + m + i) for m in (1, 7, 40, 300, 3000)] for i in range(2)]
    want = [[cr.fp8_linear(x, qweight, wscales) for x in xs] for xs in inputs]
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        got = [[], []]
        for j in range(5):
            for i, stream in enumerate(streams):
                with torch.cuda.stream(stream):
                    got[i].append(cr.fp8_linear(inputs[i][j], qweight, wscales))
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for xs, ys in zip(got, want) for a, b in zip(xs, ys))
    assert_no_device_error()


def test_captured_forward_and_backward():
    qweight, wscales = _weights(264, 520, 73)
    for m in (2, 64, 1100):
        x = randn((m, 520), torch.bfloat16, 74).requires_grad_()
        dy = randn((m, 264), torch.bfloat16, 75)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            y = cr.fp8_linear(x, qweight, wscales)
            (dx,) = torch.autograd.grad(y, x, dy)
            del y, dx
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = cr.fp8_linear(x, qweight, wscales)
            (dx,) = torch.autograd.grad(y, x, dy)
        with torch.no_grad():
            x.copy_(randn((m, 520), torch.bfloat16, 76))
        graph.replay()
        fresh = x.detach().clone().requires_grad_()
        want = cr.fp8_linear(fresh, qweight, wscales)
        assert torch.equal(y, want)
        assert torch.equal(dx, torch.autograd.grad(want, fresh, dy)[0])


def test_offsets_past_32_bits():
    # outputs, then codes and inputs, beyond 2^31 bytes and values
    qweight, wscales = _weights(32768, 16, 81)
    x = randn((70001, 16), torch.bfloat16, 82)
    y = cr.fp8_linear(x, qweight, wscales)
    for rows in (slice(0, 3), slice(65534, 65540), slice(69998, 70001)):
        assert torch.equal(y[rows], cr.fp8_linear(x[rows].clone(), qweight, wscales))
    del y
    qweight, wscales = _weights(16, 32768, 83)
    x = randn((1, 32768), torch.bfloat16, 84).repeat(70001, 1)
    x[69999] *= -1
    y = cr.fp8_linear(x, qweight, wscales)
    assert torch.equal(y[:69999], y[:1].expand(69999, 16))
    assert torch.equal(y[69999], -y[0]) and torch.equal(y[70000], y[0])
    assert_no_device_error()


def test_refusals():
    qweight, wscales = _weights(32, 64, 91)
    x = randn((4, 64), torch.bfloat16, 92)
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        cr.fp8_linear(x.double(), qweight, wscales)
    with pytest.raises(ValueError, match="CUDA"):
        cr.fp8_linear(x.cpu(), qweight, wscales)
    with pytest.raises(ValueError, match="frozen"):
        cr.fp8_linear(x, qweight, wscales, torch.zeros(32, device=dev(), requires_grad=True))
    with pytest.raises(ValueError, match="2D input"):
        cr.quantize_fp8_blockwise(x[0])
    with pytest.raises(ValueError, match="activation scales"):
        cr.fp8_matmul(qweight, qweight, wscales, wscales, output_dtype=torch.float32)
