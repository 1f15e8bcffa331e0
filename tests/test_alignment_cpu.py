"""Pointers off their elements' alignment are refused on the host (no GPU needed): a kernel would fault on them."""

from __future__ import annotations

import ctypes

import pytest

from convrot_mlx_b200 import _lib
from tests.test_more_ops_cpu import _AdamWOptions, _AdamWTensor, _GradTensor

FAKE = ctypes.c_void_p(4096)  # never dereferenced: every call below ends in its checks


@pytest.mark.parametrize("name", ["convrot_gelu_saved8", "convrot_gelu_saved8_backward"])
@pytest.mark.parametrize("dtype,size", [(0, 4), (1, 2), (2, 2)])
def test_gelu(name, dtype, size):
    lib = _lib.load()

    def run(x=4096, y=4096, scales=4096):
        x, y, scales = (ctypes.c_void_p(v) for v in (x, y, scales))
        args = (x, dtype, 4, 300, y, FAKE, scales) if name == "convrot_gelu_saved8" else (x, dtype, 4, 300, FAKE, scales, y)
        return getattr(lib, name)(*args, None)

    for bad in (dict(x=4096 + size // 2), dict(y=4096 + size // 2), dict(scales=4098)):
        assert run(**bad) == -1 and "aligned" in lib.convrot_last_error().decode()


def _aligned(status):
    return status == 0 or "aligned" not in _lib.load().convrot_last_error().decode()


def test_fp8_bias():
    run = lambda bias: _lib.load().convrot_fp8_gemm(FAKE, 400, FAKE, 4, FAKE, 400, 0, FAKE, 4, ctypes.c_void_p(bias), FAKE, 2,  # noqa: E731
                                                    4, 300, 400, None)
    assert run(4098) == -1 and not _aligned(-1)


@pytest.mark.parametrize("name,at", [("step_device", 4098), ("lr_device", 4098), ("norm", 4098), ("sums", 4100)])
def test_adamw_options(name, at):
    options = dict(step=1.0, lr=1e-3, beta1=0.9, beta2=0.99, eps=1e-8, weight_decay=0.0, sums_count=1, max_norm=1.0)
    tensors = (_AdamWTensor * 1)(_AdamWTensor(4096, 4096, 4096, 4096, 4096, 0))  # no values: nothing is launched
    run = lambda value: _lib.load().convrot_adamw(1, tensors, 0, 8, ctypes.byref(_AdamWOptions(**options, **{name: value})), None)  # noqa: E731
    assert run(4096) == 0
    assert run(at) == -1 and not _aligned(-1)


def test_norm():
    lib, one = _lib.load(), (_GradTensor * 1)(_GradTensor(4096, 10))
    assert lib.convrot_square_sums(1, one, 0, None, 1, ctypes.c_void_p(4098), None) == -1
    assert lib.convrot_norm_of_sums(ctypes.c_void_p(4100), 1, FAKE, None) == -1
    assert lib.convrot_norm_of_sums(FAKE, 1, ctypes.c_void_p(4098), None) == -1
