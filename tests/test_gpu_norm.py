"""Layer norm with its gradients (convrot_layer_norm, convrot_layer_norm_backward) against 64-bit arithmetic.

Bounds.  A float32 sum of F values in at most n sequential additions, a tree over 32 lanes and one over at most 32
warps has an error of at most (n + 12) U sum|v|, U = 2^-24; the kernels keep n <= F / 32 + 8 (a warp for a row), so
E = (F / 32 + 24) U bounds the relative error of every row sum against its sum of magnitudes.  With X = max|x| and
H = max|h| of a row:
  the mean is off by at most E X; the variance by at most 2 E var + (E X)^2, so rstd relatively by 1.1 E + (E X r)^2 + 2 U;
  h by dh = 1.1 r E X + |h| (1.2 E + (E X r)^2) + 4 U |h|;
  y by |w| dh + 2 U (|h w| + |b|).
  dx = r (g - E[g] - h E[g h]): with G = max|g| and GH = max|g h| a term-by-term sum of the same kinds.
  dw = sum dy h over R rows: at most (R + 600) U sum|dy h| + sum|dy| dh."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from convrot_mlx_b200 import _lib
from tests.gpu_util import assert_no_device_error, dev
from tests.ops64 import DTYPES, U, assert_within, randn

pytestmark = pytest.mark.gpu
EPS = 1e-6


def _norm64(x, w, b):
    """y and the bound of its arithmetic, h and its bound, rstd; w and b broadcast against x."""

    x = x.double()
    F = x.shape[-1]
    E = (F / 32 + 24) * U
    X = x.abs().amax(-1, keepdim=True)
    mean = x.mean(-1, keepdim=True)
    r = ((x - mean).square().mean(-1, keepdim=True) + EPS).rsqrt()
    h = (x - mean) * r
    rel = 1.2 * E + (E * X * r) ** 2 + 4 * U
    dh = 1.1 * r * E * X + h.abs() * rel
    w, b = w.double(), b.double()
    y = h * w + b
    return y, w.abs() * dh + 2 * U * ((h * w).abs() + b.abs()), h, dh, r, rel, E


def _dx64(x, w, b, dy):
    _, _, h, dh, r, rel, E = _norm64(x, w, b)
    g = dy.double() * w.double()
    m, mh = g.mean(-1, keepdim=True), (g * h).mean(-1, keepdim=True)
    dx = r * (g - m - h * mh)
    G = g.abs().mean(-1, keepdim=True)
    GH = (g * h).abs().mean(-1, keepdim=True)
    DH = (g.abs() * dh).mean(-1, keepdim=True)
    parts = 3 * U * g.abs() + (E + 2 * U) * G + h.abs() * ((E + 4 * U) * GH + DH) + dh * (mh.abs() + DH)
    return dx, r * parts + (rel + 4 * U) * r * (g.abs() + m.abs() + (h * mh).abs())


def _sums64(x, w, b, dy, over):
    _, _, h, dh, *_ = _norm64(x, w, b)
    d = dy.double()
    n = 1
    for a in over:
        n *= x.shape[a]
    E = (n + 600) * U
    dw, db = (d * h).sum(over), d.sum(over)
    return dw, E * (d * h).abs().sum(over) + (d.abs() * dh).sum(over), db, E * d.abs().sum(over)


SHAPES = [(1, 1), (3, 2), (4, 31), (8, 32), (5, 33), (8, 768), (300, 64), (7, 1153), (64, 3072), (33, 4100), (9, 8192),
          (3, 12289), (2, 40000), (500, 96), (1, 16384), (3000, 3072), (5000, 257), (2000, 130), (900, 1600), (700, 1602),
          (400, 5000), (301, 5001), (200, 6146), (90, 9216), (90, 9218), (70, 4609), (2500, 512), (1500, 320)]


def _inputs(rows, features, dtype, seed, offset=1.0):
    x = randn((rows, features), torch.float32, seed) + offset * randn((rows, 1), torch.float32, seed + 1)
    x[:, features // 3] *= 20
    return x.to(dtype)


@pytest.mark.parametrize("wide", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,features", SHAPES)
def test_affine(dtype, rows, features, wide):
    wdtype = torch.float32 if wide else dtype
    x = _inputs(rows, features, dtype, rows + features).requires_grad_()
    w = (1 + randn((features,), torch.float32, 3, 0.3)).to(wdtype).requires_grad_()
    b = randn((features,), wdtype, 4, 0.3).requires_grad_()
    dy = randn((rows, features), dtype, 5)
    y = cr.layer_norm(x, w, b, EPS)
    assert y.dtype == dtype
    x0, w0, b0 = x.detach(), w.detach(), b.detach()
    y64, slack, *_ = _norm64(x0, w0, b0)
    assert_within(y.detach(), y64, slack, "y")
    assert torch.equal(y.detach(), cr.layer_norm(x0, w0, b0, EPS))  # without a gradient: the same values
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert_within(dx, *_dx64(x0, w0, b0, dy), "dx")
    dw64, sw, db64, sb = _sums64(x0, w0, b0, dy, (0,))
    assert dw.dtype == wdtype and dw.shape == w.shape
    assert_within(dw, dw64, sw, "dw")
    assert_within(db, db64, sb, "db")
    assert_no_device_error()


# each number of threads of a row, at its ends, for vectors of one, two and sixteen bytes' worth of elements
ROW_SIZES = [255, 511, 512, 513, 514, 767, 768, 769, 1022, 1023, 1024, 1026, 1028, 1032, 1534, 1535, 1536, 1537, 1538, 1544, 2303,
             2304, 2305, 2306, 3070, 3071, 3073, 3074, 3080, 4606, 4607, 4608, 4610, 4616, 6144, 8191, 8192, 8193, 9214, 9224, 16382]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("features", ROW_SIZES)
def test_ends_of_the_row_shapes(dtype, features):
    test_affine(dtype, 37, features, False)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("offset", [1, 2, 5])
@pytest.mark.parametrize("rows,features", [(5, 64), (300, 1030), (3, 9001), (700, 9002), (2, 20001), (3, 30008), (2, 52000), (2, 110001)])
def test_tensors_that_start_anywhere(dtype, offset, rows, features):
    def at(t):
        return torch.cat([t.new_zeros(offset), t.flatten()])[offset:].view(t.shape)

    x = at(_inputs(rows, features, dtype, 61)).requires_grad_()
    w, b = at((1 + randn((features,), dtype, 62, 0.3)).to(dtype)).requires_grad_(), at(randn((features,), dtype, 63)).requires_grad_()
    dy = at(randn((rows, features), dtype, 64))
    y = cr.layer_norm(x, w, b, EPS)
    x0, w0, b0 = x.detach(), w.detach(), b.detach()
    y64, slack, *_ = _norm64(x0, w0, b0)
    assert_within(y.detach(), y64, slack, "y")
    dx, dw, db = torch.autograd.grad(y, (x, w, b), dy)
    assert_within(dx, *_dx64(x0, w0, b0, dy), "dx")
    dw64, sw, db64, sb = _sums64(x0, w0, b0, dy, (0,))
    assert_within(dw, dw64, sw, "dw")
    assert_within(db, db64, sb, "db")
    assert_no_device_error()


MOD_SHAPES = [(1, 1, 64), (3, 5, 257), (2, 700, 512), (8, 40, 3072), (5, 1, 33), (2, 3, 20000), (70, 9, 128), (300, 2, 40)]


@pytest.mark.parametrize("chunks", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("batch,tokens,features", MOD_SHAPES)
def test_modulated(dtype, batch, tokens, features, chunks):
    x = _inputs(batch * tokens, features, dtype, 7).view(batch, tokens, features).requires_grad_()
    if chunks:  # columns of one modulation output, as in a DiT block
        shift, scale = randn((batch, 1, 3 * features), dtype, 8, 0.3).chunk(3, dim=-1)[:2]
    else:
        shift, scale = randn((batch, features), dtype, 8, 0.3), randn((batch, features), dtype, 9, 0.3)
    shift, scale = shift.requires_grad_(), scale.requires_grad_()
    dy = randn(x.shape, dtype, 10)
    y = cr.modulated_layer_norm(x, shift, scale, EPS)
    x0 = x.detach()
    w0, b0 = (1 + scale.detach().double()).view(batch, 1, features), shift.detach().view(batch, 1, features)
    y64, slack, *_ = _norm64(x0, w0, b0)
    assert_within(y.detach(), y64, slack + U * y64.abs(), "y")  # 1 + scale is one more rounding
    dx, dshift, dscale = torch.autograd.grad(y, (x, shift, scale), dy)
    want, s = _dx64(x0, w0, b0, dy)
    g = (dy.double() * w0).abs()
    _, _, h, _, r, *_ = _norm64(x0, w0, b0)
    one = U * r * (g + g.mean(-1, keepdim=True) + h.abs() * (g * h.abs()).mean(-1, keepdim=True))
    assert_within(dx, want, s + one, "dx")
    dw64, sw, db64, sb = _sums64(x0, w0, b0, dy, (1,))
    assert dscale.shape == scale.shape and dshift.shape == shift.shape
    assert_within(dscale.view(batch, features), dw64, sw, "dscale")
    assert_within(dshift.view(batch, features), db64, sb, "dshift")
    assert_no_device_error()


@pytest.mark.parametrize("shared", ["both", "shift", "scale"])
def test_modulation_shared_by_the_batch(shared):
    b, t, f = 4, 6, 96
    x = randn((b, t, f), torch.float32, 1).requires_grad_()
    shift = randn((b if shared == "scale" else 1, 1, f), torch.float32, 2, 0.3).requires_grad_()
    scale = randn((b if shared == "shift" else 1, 1, f), torch.float32, 3, 0.3).requires_grad_()
    dy = randn((b, t, f), torch.float32, 4)
    y = cr.modulated_layer_norm(x, shift, scale, EPS)
    got = torch.autograd.grad(y, (x, shift, scale), dy)
    x64, sh64, sc64 = (v.detach().double().requires_grad_() for v in (x, shift, scale))
    y64 = torch.nn.functional.layer_norm(x64, (f,), eps=EPS) * (1 + sc64) + sh64
    want = torch.autograd.grad(y64, (x64, sh64, sc64), dy.double())
    assert (y.double() - y64).abs().max() <= 64 * U * y64.abs().max()
    for g, w in zip(got, want):
        assert g.shape == w.shape
        assert (g.double() - w).abs().max() <= 64 * U * w.abs().max() + 64 * U * 24


@pytest.mark.parametrize("have", ["none", "weight", "bias"])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_missing_vectors_and_wanted_gradients(dtype, have):
    rows, f = 50, 200
    x = randn((rows, f), dtype, 1).requires_grad_()
    w = (1 + randn((f,), dtype, 2, 0.2)).detach().requires_grad_() if have == "weight" else None
    b = randn((f,), dtype, 3).requires_grad_() if have == "bias" else None
    dy = randn((rows, f), dtype, 4)
    y = cr.layer_norm(x, w, b, EPS)
    w0 = torch.ones(f, device=dev()) if w is None else w.detach()
    b0 = torch.zeros(f, device=dev()) if b is None else b.detach()
    y64, slack, *_ = _norm64(x.detach(), w0, b0)
    assert_within(y.detach(), y64, slack)
    grads = torch.autograd.grad(y, [t for t in (x, w, b) if t is not None], dy, retain_graph=True)
    assert_within(grads[0], *_dx64(x.detach(), w0, b0, dy))
    dw64, sw, db64, sb = _sums64(x.detach(), w0, b0, dy, (0,))
    if w is not None:
        assert_within(grads[1], dw64, sw)
        assert torch.equal(torch.autograd.grad(y, w, dy)[0], grads[1])
    if b is not None:
        assert_within(grads[1], db64, sb)


def test_gradient_against_differences():
    rows, f, e = 6, 80, 1e-2
    x, w, b = (randn(s, torch.float32, i).requires_grad_() for i, s in enumerate(((rows, f), (f,), (f,))))
    dy = randn((rows, f), torch.float32, 9)
    grads = torch.autograd.grad(cr.layer_norm(x, w, b, EPS), (x, w, b), dy)
    v = [randn(t.shape, torch.float32, 20 + i) for i, t in enumerate((x, w, b))]
    at = lambda s: cr.layer_norm(*(t.detach() + s * e * d for t, d in zip((x, w, b), v)), EPS).double()  # noqa: E731
    got = ((at(1) - at(-1)) * dy.double()).sum() / (2 * e)
    want = sum((g.double() * d.double()).sum() for g, d in zip(grads, v))
    # the third derivative along a step of 1e-2 of values of order 1: about 1e-4 of the sum of magnitudes, and the
    # float32 rounding of y over the step: 2^-24 / 1e-2
    scale = (at(0).abs() * dy.double().abs()).sum()
    assert (got - want).abs() <= (1e-3 + 16 * U / e) * scale


def test_constant_large_and_not_finite_rows():
    f = 700
    x = torch.ones((5, f), device=dev())
    x[1] = 3e4
    x[2, ::2] = -1.0  # mean 0, variance 1
    x[3, 5], x[4, 6] = float("nan"), float("inf")
    w, b = randn((f,), torch.float32, 1), randn((f,), torch.float32, 2)
    y = cr.layer_norm(x, w, b, EPS)
    assert (y[0] - b).abs().max() == 0  # the mean of equal values is exact here: 700 times 1
    assert (y[2].double() - (x[2].double() * w.double() * (1 + EPS) ** -0.5 + b.double())).abs().max() <= 64 * U * 8
    assert torch.isnan(y[3:5]).all() and torch.isfinite(y[:3]).all()
    x.requires_grad_()
    (dx,) = torch.autograd.grad(cr.layer_norm(x, w, b, EPS), x, torch.ones_like(x))
    assert torch.isfinite(dx[:3]).all() and torch.isnan(dx[3:5]).all()


def test_empty_strided_and_expanded():
    w, b = torch.ones(8, device=dev(), requires_grad=True), torch.zeros(8, device=dev(), requires_grad=True)
    x = torch.empty((0, 8), device=dev(), requires_grad=True)
    y = cr.layer_norm(x, w, b)
    dx, dw, db = torch.autograd.grad(y.sum(), (x, w, b))
    assert y.shape == dx.shape == (0, 8) and dw.eq(0).all() and db.eq(0).all()
    s = torch.zeros((2, 1, 8), device=dev(), requires_grad=True)
    e = torch.empty((2, 0, 8), device=dev())
    (ds,) = torch.autograd.grad(cr.modulated_layer_norm(e, s, s.detach()).sum(), s)
    assert ds.shape == s.shape and ds.eq(0).all()
    big = randn((6, 10, 77), torch.bfloat16, 1)
    for v in (big[:, :, 3:64], big[::2], big.transpose(0, 1), big[:, 1:]):
        assert torch.equal(cr.layer_norm(v), cr.layer_norm(v.contiguous().clone()))
    x = randn((9, 77), torch.bfloat16, 2).requires_grad_()
    (a,) = torch.autograd.grad(cr.layer_norm(x).sum(), x)
    (c,) = torch.autograd.grad(cr.layer_norm(x), x, torch.ones_like(x))
    assert torch.equal(a, c)


def test_sums_do_not_depend_on_what_ran_before():
    x, w, b = randn((4000, 513), torch.bfloat16, 1), torch.ones(513, device=dev()), torch.zeros(513, device=dev())
    w.requires_grad_(), b.requires_grad_()
    dy = randn(x.shape, torch.bfloat16, 2)
    first = torch.autograd.grad(cr.layer_norm(x, w, b), (w, b), dy)
    for _ in range(3):
        again = torch.autograd.grad(cr.layer_norm(x, w, b), (w, b), dy)
        assert all(torch.equal(p, q) for p, q in zip(first, again))


def test_offsets_past_32_bits():
    rows, f = 280000, 8192
    x = randn((rows, f), torch.bfloat16, 1)
    y = cr.layer_norm(x)
    dx = torch.autograd.grad(cr.layer_norm(x.requires_grad_()), x, y)[0]
    for part in (slice(0, 2), slice(rows - 2, rows)):
        part_x = x.detach()[part].clone()
        assert torch.equal(y[part], cr.layer_norm(part_x))
        part_x.requires_grad_()
        assert torch.equal(dx[part], torch.autograd.grad(cr.layer_norm(part_x), part_x, y[part].clone())[0])


def test_other_stream():
    x, w, b = randn((640, 1024), torch.bfloat16, 1), randn((1024,), torch.bfloat16, 2), randn((1024,), torch.bfloat16, 3)
    w.requires_grad_()
    want = torch.autograd.grad(cr.layer_norm(x, w, b), w, x)[0]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = torch.autograd.grad(cr.layer_norm(x, w, b), w, x)[0]
    side.synchronize()
    assert torch.equal(got, want)


def test_refusals():
    x = randn((4, 64), torch.bfloat16, 1)
    w = torch.ones(64, device=dev())
    with pytest.raises(ValueError, match="weight must have shape"):
        cr.layer_norm(x, w[:32])
    with pytest.raises(ValueError, match="bias must have shape"):
        cr.layer_norm(x, w, w[:32])
    with pytest.raises(ValueError, match="eps"):
        cr.layer_norm(x, eps=-1.0)
    with pytest.raises(ValueError, match="CUDA"):
        cr.layer_norm(x.cpu())
    with pytest.raises(ValueError, match="float32, float16 or bfloat16"):
        cr.layer_norm(x.double())
    with pytest.raises(ValueError, match="features"):
        cr.layer_norm(torch.empty((4, 0), device=dev()))
    with pytest.raises(ValueError, match="modulation vector"):
        cr.modulated_layer_norm(x.view(2, 2, 64), w.view(1, 64), w.expand(3, 64))
    with pytest.raises(ValueError, match="modulation vector"):
        cr.modulated_layer_norm(x.view(2, 2, 64), w.view(1, 64), w[:32].view(1, 32))
    lib = _lib.load()
    p = _lib.ptr(x)
    assert lib.convrot_layer_norm(p, 2, 4, 64, None, None, 2, 3, 64, 0, 1e-6, p, None, None, None) == -1
    assert lib.convrot_layer_norm(p, 2, 4, 64, None, None, 1, 4, 64, 0, 1e-6, p, None, None, None) == -1
    assert lib.convrot_layer_norm_backward(p, p, 2, 4, 64, None, 2, 4, 64, 0, p, p, p, p, None, p, 16, None) == -1
    assert "workspace" in lib.convrot_last_error().decode()
