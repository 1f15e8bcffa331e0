"""The AdamW step over many tensors (convrot_adamw, adamw_step, AdamW) and the gradient norm (convrot_square_sums,
grad_norm) against 64-bit arithmetic.

Bounds, in float32 half steps U.  m: two products and a sum, and the two factors' own rounding: 4 U of what is added; v: one
product more, 5 U.  The update: the error of m, and half of v's, the root, the two factors, the sum with eps and a
quotient of two units in the last place: 16 U in all beside m's.  The parameter: its decay and the difference, 4 U."""

from __future__ import annotations

import copy
import io
import math

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.fp8_64 import e4m3
from tests.gpu_util import dev
from tests.ops64 import DTYPES, U, assert_within, randn

pytestmark = pytest.mark.gpu

E4M3 = torch.float8_e4m3fn
HOW = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)
SHAPES = [(1,), (7,), (8,), (255,), (256,), (257,), (33, 65), (512, 16), (3, 5, 7), (4096,), (0,), (1000, 130)]


def _blocks(t):
    """The values of t in memory order in rows of 256, zeros behind the last."""

    flat = t.reshape(-1).double()
    return torch.nn.functional.pad(flat, (0, -flat.numel() % 256)).view(-1, 256)


def _decoded(codes, scales, column):
    flat = _blocks(codes) * scales[:, column, None].double()
    return flat.reshape(-1)[:codes.numel()].view(codes.shape)


def _moments(shape, seed, first):
    g = randn(shape, torch.float32, seed)
    size = torch.exp(randn(shape, torch.float32, seed + 1))
    return (g * 0 if first else 0.1 * g * size), (g * 0 if first else size * size)


def _as_8_bits(m, v):
    """Moments as the operator keeps them, made in 64 bits."""

    out, scales = [], []
    for x in (m.double(), v.double().sqrt()):
        rows = _blocks(x)
        scale = (rows.abs().amax(1, keepdim=True) / 448).float()
        codes = e4m3(torch.where(scale > 0, rows / scale.double(), rows * 0))
        out.append(codes.reshape(-1)[:x.numel()].view(x.shape).to(E4M3))
        scales.append(scale[:, 0])
    return out[0], out[1], torch.stack(scales, 1).contiguous()


def _state(shapes, dtype, bits, seed, first=False):
    params = [randn(s, dtype, seed + 10 * i) for i, s in enumerate(shapes)]
    grads = [randn(s, dtype, seed + 10 * i + 1) for i, s in enumerate(shapes)]
    pairs = [_moments(s, seed + 10 * i + 2, first) for i, s in enumerate(shapes)]
    if bits == 32:
        return params, grads, [m for m, _ in pairs], [v for _, v in pairs], None
    kept = [_as_8_bits(m, v) for m, v in pairs]
    return params, grads, [k[0] for k in kept], [k[1] for k in kept], [k[2] for k in kept]


def _check_codes(codes, scale, want, slack, root=False):
    """codes * scale is want (rows of 256, 64 bits) to half a step of the code, which `slack` may move past a border."""

    top = want.abs().amax(1)
    assert ((scale.double() - top / 448).abs() <= slack.amax(1) / 448 + U * top / 448).all()
    q = torch.where(scale[:, None] > 0, want / scale[:, None].double(), want * 0)
    half = torch.exp2(torch.floor(torch.log2(q.abs().clamp(min=2.0 ** -6))) - 4)
    allowed = half * 1.0001 + torch.where(scale[:, None] > 0, slack / scale[:, None].double(), want * 0)
    off = (codes - q).abs()
    if root:  # what is above 0 stays so
        assert ((codes > 0) == (want > 0)).all()
        allowed = torch.where(codes == 2.0 ** -9, allowed.clamp(min=2.0 ** -9), allowed)
    assert (off <= allowed).all()


def _check_step(before, after, grads, bits, step, how=HOW, factor=1.0):
    """One step of one tensor against 64 bits; before and after: (p, m, v or codes, scales)."""

    b1, b2 = how["betas"]
    p, g = before[0].double(), grads.double() * factor
    if bits == 32:
        m0, v0 = before[1].double(), before[2].double()
    else:
        m0, v0 = _decoded(before[1], before[3], 0), _decoded(before[2], before[3], 1) ** 2
    m, v = b1 * m0 + (1 - b1) * g, b2 * v0 + (1 - b2) * g * g
    m_slack = 4 * U * (b1 * m0.abs() + (1 - b1) * g.abs()) + (2 * U * g.abs() if factor != 1.0 else 0.0)
    v_slack = 5 * U * v + (4 * U * v if factor != 1.0 else 0.0) + 2.0 ** -149
    if bits == 32:
        assert_within(after[1], m, m_slack)
        assert_within(after[2], v, v_slack)
    elif p.numel():
        _check_codes(_blocks(after[1]), after[3][:, 0], _blocks(m), _blocks(m_slack) + 2 * U * _blocks(m).abs())
        _check_codes(_blocks(after[2]), after[3][:, 1], _blocks(v.sqrt()), 5 * U * _blocks(v.sqrt()) + 2.0 ** -75, root=True)
    den = v.sqrt() / math.sqrt(1 - b2 ** step) + how["eps"]
    size = how["lr"] / (1 - b1 ** step)
    update = size * m / den
    want = p * (1 - how["lr"] * how["weight_decay"]) - update
    # a root of a square below float32's range is lost: at most 2^-74 in the denominator
    slack = 4 * U * p.abs() + 16 * U * update.abs() + size / den * m_slack + update.abs() * 2.0 ** -74 / den
    assert_within(after[0], want, slack)


@pytest.mark.parametrize("first", [False, True])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", DTYPES)
def test_step(dtype, bits, first):
    params, grads, ms, vs, scales = _state(SHAPES, dtype, bits, 100, first)
    before = copy.deepcopy((params, ms, vs, scales))
    step = 1 if first else 57
    kept = [g.clone() for g in grads]
    assert cr.adamw_step(params, grads, ms, vs, scales, step, **HOW) is None
    for i in range(len(SHAPES)):
        column = lambda lists: tuple(x[i] if x is not None else None for x in lists)  # noqa: E731
        _check_step(column(before), column((params, ms, vs, scales)), grads[i], bits, step)
        assert torch.equal(grads[i], kept[i])
    # the same bits again
    again = copy.deepcopy(before)
    cr.adamw_step(again[0], grads, again[1], again[2], again[3], step, **HOW)
    assert all(torch.equal(a, b) for a, b in zip(again[0], params))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_start_anywhere(bits):
    # views at offsets that no vector access fits, next to one another: their neighbours keep their values
    n = 1000
    for offset in (1, 2, 3, 5, 8):
        params, grads, ms, vs, scales = _state([(n,)], torch.bfloat16, bits, 300)
        want = copy.deepcopy((params, ms, vs, scales))
        cr.adamw_step(want[0], grads, want[1], want[2], want[3], 9, **HOW)
        bases = [torch.zeros(n + 16, dtype=t.dtype, device=dev()) for t in (params[0], grads[0], ms[0], vs[0])]
        views = [b[offset:offset + n] for b in bases]
        for view, t in zip(views, (params[0], grads[0], ms[0], vs[0])):
            view.copy_(t)
        cr.adamw_step([views[0]], [views[1]], [views[2]], [views[3]], scales, 9, **HOW)
        for view, t in zip((views[0], views[2], views[3]), (want[0][0], want[1][0], want[2][0])):
            assert torch.equal(view.float(), t.float())
        for b in bases:
            assert b[:offset].float().eq(0).all() and b[offset + n:].float().eq(0).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [31, 32, 33, 511, 512, 513, 1200])
def test_many_tensors(count, bits):
    shapes = [((i * 37) % 700 + (i % 3 > 0),) for i in range(count)]
    params, grads, ms, vs, scales = _state(shapes, torch.float32, bits, 17)
    one = copy.deepcopy((params, ms, vs, scales))
    cr.adamw_step(params, grads, ms, vs, scales, 3, **HOW)
    for i in range(0, count, 29):  # as tensors alone
        each = [[x[i]] if x is not None else None for x in one]
        cr.adamw_step(each[0], [grads[i]], each[1], each[2], each[3], 3, **HOW)
        assert torch.equal(each[0][0], params[i]) and torch.equal(each[1][0].float(), ms[i].float())
    start = _state(shapes, torch.float32, bits, 17)[0]
    assert not any(torch.equal(a, b) for a, b in zip(params, start) if a.numel())  # every one has moved


def test_mixed_types_missing_gradients_and_layouts():
    shapes = [(300,), (40, 50), (2, 6, 5, 5), (77,)]
    params, grads, ms, vs, _ = _state(shapes, torch.float32, 32, 400)
    params[1], grads[1] = params[1].bfloat16(), grads[1].bfloat16()
    # dense in another order, the gradient packed
    params[2] = params[2].to(memory_format=torch.channels_last)
    ms[2], vs[2] = (t.to(memory_format=torch.channels_last) for t in (ms[2], vs[2]))
    before = copy.deepcopy((params, ms, vs))
    grads[3] = None
    version = params[0]._version
    cr.adamw_step(params, grads, ms, vs, None, 4, **HOW)
    for i in range(3):
        _check_step((before[0][i], before[1][i], before[2][i], None), (params[i], ms[i], vs[i], None), grads[i], 32, 4)
    assert torch.equal(params[3], before[0][3]) and torch.equal(ms[3], before[1][3])
    assert params[0]._version > version  # autograd sees that it was written


@pytest.mark.parametrize("bits", [32, 8])
def test_clipping(bits):
    params, grads, ms, vs, scales = _state([(1000,), (33, 65)], torch.float32, bits, 500)
    exact = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    for limit in (exact / 3, exact * 2):
        now = copy.deepcopy((params, ms, vs, scales))
        norm = cr.adamw_step(now[0], grads, now[1], now[2], now[3], 5, max_norm=limit, **HOW)
        assert abs(norm.item() - exact) <= 2 * U * exact
        for i in range(2):
            column = lambda lists: tuple(x[i] if x is not None else None for x in lists)  # noqa: E731
            _check_step(column((params, ms, vs, scales)), column(now), grads[i], bits, 5, factor=min(1.0, limit / (exact + 1e-6)))


@pytest.mark.parametrize("bits", [32, 8])
def test_zero_gradients_and_zero_moments(bits):
    params, grads, ms, vs, scales = _state([(700,)], torch.float32, bits, 600, first=True)
    before = params[0].clone()
    grads[0][:300] = 0
    cr.adamw_step(params, grads, ms, vs, scales, 1, **HOW)
    still = before[:300].double() * (1 - HOW["lr"] * HOW["weight_decay"])
    assert_within(params[0][:300], still, 2 * U * still.abs())
    assert ms[0][:300].float().eq(0).all() and vs[0][:300].float().eq(0).all()
    if bits == 8:
        assert scales[0][0].eq(0).all() and scales[0][2].gt(0).all()


def test_gradients_that_are_not_finite():
    for bad in (float("inf"), float("nan")):
        params, grads, ms, vs, _ = _state([(600,)], torch.float32, 32, 700)
        grads[0][300] = bad
        cr.adamw_step(params, grads, ms, vs, None, 2, **HOW)
        fine = torch.ones(600, dtype=torch.bool, device=dev())
        fine[300] = False
        assert torch.isfinite(params[0][fine]).all() and not torch.isfinite(ms[0][300])
        params, grads, ms, vs, scales = _state([(600,)], torch.float32, 8, 700)
        grads[0][300] = bad
        cr.adamw_step(params, grads, ms, vs, scales, 2, **HOW)
        assert torch.isfinite(params[0][fine]).all()
        assert torch.isnan(scales[0][1]).all() and torch.isfinite(scales[0][0]).all() and torch.isfinite(scales[0][2]).all()
        assert ms[0][256:512].float().eq(0).all() and vs[0][256:512].float().eq(0).all()
        params, grads, ms, vs, _ = _state([(600,)], torch.float32, 32, 700)
        grads[0][300] = bad
        norm = cr.adamw_step(params, grads, ms, vs, None, 2, max_norm=1.0, **HOW)
        assert not math.isfinite(norm.item())
        assert torch.isnan(params[0][300])
        if math.isnan(bad):
            assert torch.isnan(params[0]).all()


def test_values_of_all_sizes_in_one_block():
    # roots far below their block's largest keep a code above 0, so that no later step divides by eps alone
    params, grads, ms, vs, scales = _state([(256,)], torch.float32, 8, 800, first=True)
    grads[0] = torch.exp2(-torch.arange(256, device=dev()).float() / 4)
    before = copy.deepcopy((params, ms, vs, scales))
    cr.adamw_step(params, grads, ms, vs, scales, 1, **HOW)
    _check_step(tuple(x[0] for x in before), (params[0], ms[0], vs[0], scales[0]), grads[0], 8, 1)
    assert vs[0].float().min() == 2.0 ** -9


def test_step_and_rate_on_the_device():
    for bits in (32, 8):
        a, b = (_state(SHAPES, torch.float32, bits, 900) for _ in range(2))
        cr.adamw_step(*a, 123, **HOW)
        how = dict(HOW, lr=torch.tensor(HOW["lr"], device=dev()))
        cr.adamw_step(*b, torch.tensor(123.0, device=dev()), **how)
        for x, y, old in zip(a[0], b[0], _state(SHAPES, torch.float32, bits, 900)[0]):
            # the factors of the step, rounded once each on either side: 2 U of the update and of the parameter
            assert ((x.double() - y.double()).abs() <= 4 * U * (x.double().abs() + (x - old).double().abs())).all()
        assert all(torch.equal(x.float(), y.float()) for x, y in zip(a[2], b[2]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shapes", [[(1,)], [(5,), (0,), (256,)], [(1000, 1000)], [(i,) for i in range(1100)], [(3_000_001,)],
                                    [(2048 * 4 * n + 1,) for n in (0, 1, 2)], [(2048 * 128,)], [(2048 * 127 + 1,), (0,)],
                                    [(2048 * 128 + 1,)], [(9, 100)] * 64, [(9, 100)] * 65, [(3,)] * 128, [(3,)] * 129])
def test_grad_norm(dtype, shapes):
    grads = [randn(s, dtype, 31 + i) for i, s in enumerate(shapes)]
    exact = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    norm = cr.grad_norm(grads)
    assert norm.shape == () and norm.dtype == torch.float32
    # eight squares and their sums in float32 at 9 U at most, halved by the root, and the result's rounding
    assert abs(norm.item() - exact) <= 6 * U * exact
    assert torch.equal(norm, cr.grad_norm(tuple(grads) + (None,)))


def test_grad_norm_of_mixed_types_layouts_and_ranges():
    grads = [randn((50, 60), torch.float32, 1).t(), randn((333,), torch.bfloat16, 2)[1:], randn((64, 64), torch.float16, 3)[::2],
             randn((1, 40), torch.float32, 4).expand(30, 40)]
    exact = math.sqrt(sum(g.double().square().sum().item() for g in grads))
    assert abs(cr.grad_norm(grads).item() - exact) <= 6 * U * exact
    for size in (1e30, 1e-30, 1e-42):
        g = randn((1000,), torch.float32, 5) * size
        exact = g.double().norm().item()
        assert abs(cr.grad_norm([g]).item() - exact) <= 6 * U * exact + 2.0 ** -149
    assert cr.grad_norm([torch.zeros(100, device=dev())]).item() == 0
    assert cr.grad_norm([torch.zeros(0, device=dev())]).item() == 0
    huge = torch.full((10,), 3e38, device=dev())
    assert math.isinf(cr.grad_norm([huge]).item())
    assert math.isnan(cr.grad_norm([torch.tensor([1.0, float("nan")], device=dev())]).item())
    assert math.isinf(cr.grad_norm([torch.tensor([1.0, float("-inf")], device=dev())]).item())


def test_offsets_past_32_bits():
    n = 2 ** 31 + 12345
    tail = 5000
    p = torch.zeros(n, dtype=torch.bfloat16, device=dev())
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev())
    m, v = (torch.zeros(n, dtype=torch.uint8, device=dev()).view(E4M3) for _ in range(2))
    scales = torch.zeros((-(-n // 256), 2), device=dev())
    start = (n - tail) // 256 * 256  # whole blocks
    g[start:] = randn((n - start,), torch.bfloat16, 6)
    norm = cr.adamw_step([p], [g], [m], [v], [scales], 1, max_norm=1.0, **HOW)
    q, w = torch.zeros(n - start, dtype=torch.bfloat16, device=dev()), g[start:].clone()
    small = [torch.zeros(n - start, dtype=torch.uint8, device=dev()).view(E4M3) for _ in range(2)]
    some = torch.zeros((-(-(n - start) // 256), 2), device=dev())
    want = cr.adamw_step([q], [w], [small[0]], [small[1]], [some], 1, max_norm=1.0, **HOW)
    assert abs(norm.item() - want.item()) <= 2 * U * want.item()
    assert (p[start:].float() - q.float()).abs().max() <= 2.0 ** -7 * q.float().abs().max() and p[:start].eq(0).all()
    assert ((scales[start // 256:] - some).abs() <= 8 * U * some).all() and scales[:start // 256].eq(0).all()


def test_other_stream():
    a, b = (_state(SHAPES, torch.float32, 8, 1100) for _ in range(2))
    cr.adamw_step(*a, 7, max_norm=1.0, **HOW)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cr.adamw_step(*b, 7, max_norm=1.0, **HOW)
    side.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(a[0], b[0]))


# --- the optimizer ------------------------------------------------------------


def _parameters(dtype=torch.float32, seed=1):
    return [torch.nn.Parameter(randn(s, dtype, seed + i)) for i, s in enumerate([(40, 30), (300,), (7, 9, 11)])]


def _set_grads(params, seed):
    for i, p in enumerate(params):
        p.grad = randn(p.shape, p.dtype, seed + i)


def test_optimizer_against_torch():
    # six steps: each within the bounds above, which a later step only shrinks; the updates are at most lr * 10 each
    ours, theirs = _parameters(), _parameters()
    how = dict(lr=1e-2, betas=(0.9, 0.95), eps=1e-8, weight_decay=0.1)
    a = cr.AdamW([dict(params=ours[:2]), dict(params=ours[2:], lr=2e-2)], **how)
    b = torch.optim.AdamW([dict(params=theirs[:2]), dict(params=theirs[2:], lr=2e-2)], **how)
    for step in range(6):
        for params, optimizer in ((ours, a), (theirs, b)):
            _set_grads(params, 50 + 10 * step)
            if step == 2:
                params[0].grad = None  # its count falls behind
            optimizer.step()
        for p, q in zip(ours, theirs):
            assert ((p - q).abs() <= (step + 1) * (8 * U * q.abs() + 64 * U * 0.2)).all()
    loaded = cr.AdamW([dict(params=ours[:2]), dict(params=ours[2:])], **how)
    loaded.load_state_dict(b.state_dict())
    assert loaded.param_groups[1]["lr"] == 2e-2 and loaded.state[ours[0]]["step"] == 5
    with torch.no_grad():
        for p, q in zip(ours, theirs):
            p.copy_(q)
    for params, optimizer in ((ours, loaded), (theirs, b)):
        _set_grads(params, 200)
        optimizer.step()
    for p, q in zip(ours, theirs):
        assert ((p - q).abs() <= 8 * U * q.abs() + 64 * U * 0.2).all()


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_optimizer_state_dict(dtype, bits):
    params = _parameters(dtype)
    a = cr.AdamW(params, state_bits=bits, max_norm=1.0)
    for step in range(3):
        _set_grads(params, 300 + step)
        a.step()
    assert a.last_norm.shape == ()
    saved, values = copy.deepcopy(a.state_dict()), [p.detach().clone() for p in params]
    _set_grads(params, 400)
    a.step()
    others = [torch.nn.Parameter(v) for v in values]
    b = cr.AdamW(others, state_bits=bits, max_norm=1.0)
    b.load_state_dict(saved)
    state = b.state[others[0]]
    assert state["exp_avg"].dtype == (torch.float32 if bits == 32 else E4M3)
    _set_grads(others, 400)
    b.step()
    assert all(torch.equal(p, q) for p, q in zip(params, others))
    with pytest.raises(ValueError, match="not kept in"):
        cr.AdamW(others, state_bits=40 - bits).load_state_dict(saved)
    if bits == 8:
        turned = [torch.nn.Parameter(v.t().contiguous().t() if v.dim() == 2 else v) for v in values]
        other = cr.AdamW(turned, state_bits=8)
        with pytest.raises(ValueError, match="memory layout"):
            other.load_state_dict(saved)
        assert not other.state  # nothing is loaded by halves


def test_copies_and_saves_of_the_optimizer():
    params = _parameters()
    a = cr.AdamW(params, state_bits=8, max_norm=1.0)
    _set_grads(params, 450)
    a.step()
    file = io.BytesIO()  # pickle alone does not take torch's 8-bit floats
    torch.save(a, file)
    file.seek(0)
    for b in (copy.deepcopy(a), torch.load(file, weights_only=False)):
        others = b.param_groups[0]["params"]
        assert (b.state_bits, b.max_norm) == (8, 1.0) and all(torch.equal(p, q) for p, q in zip(params, others))
        _set_grads(others, 460)
        b.step()
    _set_grads(params, 460)
    a.step()
    assert all(torch.equal(p, q) for p, q in zip(params, others))
    assert all(torch.equal(a.state[p]["scales"], b.state[q]["scales"]) for p, q in zip(params, others))


def test_two_steps_at_once():
    # two streams, each with tensors of its own, one after the other without waiting
    states = [_state([(100_000,), (333, 77)], torch.bfloat16, 8, 1200 + i) for i in range(2)]
    want = copy.deepcopy(states)
    for s in want:
        cr.adamw_step(*s, 7, max_norm=1.0, **HOW)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for stream in streams:
        stream.wait_stream(torch.cuda.current_stream())
    for s, stream in zip(states, streams):
        with torch.cuda.stream(stream):
            cr.adamw_step(*s, 7, max_norm=1.0, **HOW)
    torch.cuda.synchronize()
    for s, w in zip(states, want):
        assert all(torch.equal(a, b) for a, b in zip(s[0], w[0])) and all(torch.equal(a, b) for a, b in zip(s[4], w[4]))


def test_clipping_over_groups():
    params = _parameters()
    _set_grads(params, 500)
    exact = math.sqrt(sum(p.grad.double().square().sum().item() for p in params))
    others = _parameters()
    for p, q in zip(params, others):
        q.grad = p.grad * (1.0 / (exact + 1e-6))
    a = cr.AdamW([dict(params=params[:1]), dict(params=params[1:])], max_norm=1.0)
    a.step()
    assert abs(a.last_norm.item() - exact) <= 2 * U * exact
    cr.AdamW(others).step()
    for p, q in zip(params, others):  # the first update is lr * g / |g|: the factor's rounding is lost in it
        assert ((p - q).abs() <= 8 * U * (q.abs() + 1e-3)).all()


def test_captured_step():
    params, eager = _parameters(), _parameters()
    a, b = cr.AdamW(params, state_bits=8, max_norm=1.0, capturable=True), cr.AdamW(eager, state_bits=8, max_norm=1.0)
    _set_grads(params, 600)
    _set_grads(eager, 600)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a.step()
    torch.cuda.current_stream().wait_stream(side)
    b.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        a.step()
    for step in range(4):
        for i, (p, q) in enumerate(zip(params, eager)):
            g = randn(p.shape, p.dtype, 700 + 10 * step + i)
            p.grad.copy_(g)
            q.grad = g
        graph.replay()
        b.step()
        for p, q in zip(params, eager):
            assert ((p - q).abs() <= (step + 2) * 16 * U * (q.abs() + 1e-2)).all()
    assert a.param_groups[0]["step"].item() == 5
    fresh = cr.AdamW(_parameters(), capturable=True)
    _set_grads(fresh.param_groups[0]["params"], 1)
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="before the capture"):
        with torch.cuda.graph(graph):
            fresh.step()


def test_refusals():
    params, grads, ms, vs, scales = _state([(300,), (20,)], torch.float32, 8, 1)
    run = lambda p=params, g=grads, m=ms, v=vs, s=scales, step=1, **how: cr.adamw_step(p, g, m, v, s, step, **{**HOW, **how})  # noqa: E731
    with pytest.raises(ValueError, match="equally many"):
        run(g=grads[:1])
    with pytest.raises(ValueError, match="twice"):
        run(p=[params[0]] * 2, g=[grads[0]] * 2, m=[ms[0]] * 2, v=[vs[0]] * 2, s=[scales[0]] * 2)
    with pytest.raises(ValueError, match="gradient 1"):
        run(g=[grads[0], grads[1].half()])
    with pytest.raises(ValueError, match="moments of parameter 0"):
        run(m=[ms[0].float(), ms[1]])
    with pytest.raises(ValueError, match="moments of parameter 0"):
        run(s=None)
    with pytest.raises(ValueError, match="scales of parameter 0"):
        run(s=[scales[0][:1], scales[1]])
    with pytest.raises(ValueError, match="counts from 1"):
        run(step=0)
    with pytest.raises(ValueError, match="betas"):
        run(betas=(1.0, 0.9))
    with pytest.raises(ValueError, match="CUDA"):
        run(g=[grads[0].cpu(), grads[1]])
    with pytest.raises(ValueError, match="unsupported dtype"):
        cr.grad_norm([grads[0].double()])
    with pytest.raises(ValueError, match="at least one"):
        cr.grad_norm([None])
    with pytest.raises(ValueError, match="must be tensors"):
        cr.grad_norm([3.0])
    base = torch.zeros((20, 20), device=dev())
    with pytest.raises(ValueError, match="dense in memory"):
        cr.adamw_step([base[:, :5]], [base[:, 5:10]], [base[:, 10:15]], [base[:, 15:]], None, 1, **HOW)
    with pytest.raises(ValueError, match="one float32"):
        run(step=torch.tensor(1, device=dev()))
    with pytest.raises(ValueError, match="twice"):
        run(m=[ms[0], ms[1]], v=[ms[0], vs[1]])
    p = [torch.nn.Parameter(torch.zeros(4, device=dev()))]
    for other in (torch.optim.AdamW(p, amsgrad=True), torch.optim.AdamW(p, maximize=True), torch.optim.Adam(p, weight_decay=0.1)):
        p[0].grad = torch.ones(4, device=dev())
        other.step()
        with pytest.raises(ValueError, match="this AdamW"):
            cr.AdamW(p).load_state_dict(other.state_dict())


def test_dimensions_of_one_may_have_any_stride():
    p, g, m, v = (randn((40,), torch.float32, i).as_strided((1, 40), (s, 1)) for i, s in enumerate((7, 1, 40, 3)))
    v = v.square()
    q = [t.clone().reshape(40) for t in (p, g, m, v)]
    g2 = torch.stack((g[0], g[0]), 1)[:, 0].reshape(1, 40)  # not contiguous: copied
    cr.adamw_step([p], [g2], [m], [v], None, 3, **HOW)
    cr.adamw_step([q[0]], [q[1]], [q[2]], [q[3]], None, 3, **HOW)
    assert torch.equal(p[0], q[0]) and torch.equal(m[0], q[2])
