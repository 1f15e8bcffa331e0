"""Tensors of one AdamW step that overlap: refused before anything is launched where one of them is written."""

from __future__ import annotations

import pytest
import torch

import convrot_mlx_b200 as cr
from tests.gpu_util import dev
from tests.ops64 import randn

pytestmark = pytest.mark.gpu

HOW = dict(lr=3e-3, betas=(0.9, 0.99), eps=1e-8, weight_decay=0.02)
E4M3 = torch.float8_e4m3fn


def _tensors(sizes, bits, seed=1):
    """A step's five lists, every tensor with a storage of its own."""

    kind = torch.float32 if bits == 32 else E4M3
    moments = [[torch.zeros(n, dtype=torch.float32, device=dev()).to(kind) for n in sizes] for _ in range(2)]
    scales = [torch.zeros((-(-n // 256), 2), device=dev()) for n in sizes] if bits == 8 else None
    return ([randn((n,), torch.float32, seed + i) for i, n in enumerate(sizes)],
            [randn((n,), torch.float32, seed + 50 + i) for i, n in enumerate(sizes)], *moments, scales)


def _refused(lists):
    kept = [[t.clone() for t in x] for x in lists if x is not None]
    with pytest.raises(ValueError, match="overlaps another tensor"):
        cr.adamw_step(*lists, 1, **HOW)
    for x, y in zip((x for x in lists if x is not None), kept):
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(x, y))


@pytest.mark.parametrize("bits", [32, 8])
def test_a_tensor_given_twice(bits):
    for which in range(5 if bits == 8 else 4):
        if which == 1:  # a gradient may be shared
            continue
        lists = _tensors([300, 300, 300], bits)
        lists[which][2] = lists[which][0]
        _refused(lists)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("which", [0, 2, 3])
def test_views_that_overlap_in_part(bits, which):
    for first, second in (((0, 300), (299, 599)), ((0, 600), (100, 400)), ((100, 400), (0, 101)), ((0, 300), (0, 200))):
        sizes = [b - a for a, b in (first, second)]
        lists = _tensors(sizes + [77], bits)
        base = torch.zeros(700, dtype=torch.float32, device=dev()).to(lists[which][0].dtype)
        lists[which][0], lists[which][1] = base[slice(*first)], base[slice(*second)]
        _refused(lists)


def test_scales_that_overlap_in_part():
    lists = _tensors([600, 600], 8)
    base = torch.zeros((5, 2), device=dev())
    lists[4][0], lists[4][1] = base[:3], base[2:]
    _refused(lists)


def test_tensors_of_different_kinds_that_overlap():
    lists = _tensors([300, 300], 32)
    lists[2][0] = lists[0][1]  # a moment that is another parameter
    _refused(lists)
    lists = _tensors([300, 300], 32)
    base = torch.zeros(700, device=dev())
    lists[0][0], lists[3][1] = base[:300], base[200:500]
    _refused(lists)
    lists = _tensors([300, 300], 32)  # a gradient that is another parameter, or shifted against its own
    lists[1][0] = lists[0][1]
    _refused(lists)
    lists = _tensors([300, 300], 32)
    base = torch.zeros(700, device=dev())
    lists[0][1], lists[1][1] = base[1:301], base[:300]
    _refused(lists)


@pytest.mark.parametrize("bits", [32, 8])
def test_views_side_by_side(bits):
    # packed buffers in any order, the gradient one of a parameter's own tensors, one gradient for two parameters
    sizes = [300, 1, 2048, 77, 300]
    want = _tensors(sizes, bits)
    want[1][4] = want[1][0]
    want[1][1] = want[0][1]
    lists = [list(x) if x is not None else None for x in want]
    order = [3, 0, 4, 2, 1]
    for which, x in enumerate(lists):
        if x is None:
            continue
        base = torch.zeros(sum(t.numel() for t in x), dtype=torch.float32, device=dev()).to(x[0].dtype)
        at = 0
        for i in order:
            view = base[at:at + x[i].numel()].view(x[i].shape)
            view.copy_(x[i])
            x[i] = view
            at += view.numel()
    lists[1][4] = lists[1][0]
    lists[1][1] = lists[0][1]
    want = tuple([t.clone() for t in x] if x is not None else None for x in want)
    kept = want[0][1].clone()
    want[1][1] = kept  # the same value, apart
    cr.adamw_step(*want, 1, **HOW)
    cr.adamw_step(*lists, 1, **HOW)
    for which in (0, 2, 3, 4) if bits == 8 else (0, 2, 3):
        assert all(torch.equal(a.float(), b.float()) for a, b in zip(want[which], lists[which]))
