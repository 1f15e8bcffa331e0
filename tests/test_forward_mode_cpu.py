"""Forward-mode derivatives of the 8-bit and training operators are refused, whichever input carries the tangent (host
checks, before any device work)."""

from __future__ import annotations

import pytest
import torch
from torch.autograd import forward_ad

import convrot_mlx_b200 as cr

X, V, S = torch.randn(2, 3, 8), torch.randn(8), torch.randn(2, 8)
Q, POS = torch.randn(1, 2, 4, 8), torch.zeros(4, 2)
W8 = torch.zeros((5, 8), dtype=torch.int8)

CALLS = {  # the call, and its floating inputs
    "int8_linear": (lambda x, s, b: cr.int8_linear(x, W8, s, b), (X, torch.ones(5), torch.zeros(5))),
    "axial_rotary": (lambda q, k, p: cr.axial_rotary(q, k, p, (4, 4)), (Q, Q, POS)),
    "layer_norm": (lambda x, w, b: cr.layer_norm(x, w, b), (X, V, V)),
    "modulated_layer_norm": (lambda x, a, b: cr.modulated_layer_norm(x, a, b), (X, S, S)),
    "gelu_tanh_saved8": (cr.gelu_tanh_saved8, (X,)),
}


@pytest.mark.parametrize("name,which", [(n, i) for n, (_, args) in CALLS.items() for i in range(len(args))])
def test_tangents_are_refused(name, which):
    call, args = CALLS[name]
    with forward_ad.dual_level():
        args = [forward_ad.make_dual(a, torch.ones_like(a)) if i == which else a for i, a in enumerate(args)]
        with pytest.raises(NotImplementedError, match=f"forward-mode derivative of {name} "):
            call(*args)
        with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
            call(*args)
        with torch.inference_mode(), pytest.raises(ValueError, match="CUDA"):  # no derivative is formed there
            call(*args)


@pytest.mark.parametrize("name", CALLS)
def test_plain_inputs_are_not(name):
    call, args = CALLS[name]
    with forward_ad.dual_level(), pytest.raises(ValueError, match="CUDA"):
        call(*args)
