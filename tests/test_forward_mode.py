"""The operators have no forward-mode derivatives: a tangent of any input raises, of the operator itself and of its backward (it must not be left
out of the result). Shapes only, on the meta device."""

import pytest
import torch
from test_second_derivative import CALLS, _meta

forward_ad = torch.autograd.forward_ad


@pytest.mark.parametrize("recorded", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_tangents_raise(name, recorded):
    call, shapes = CALLS[name]
    with forward_ad.dual_level():
        for i in range(len(shapes)):
            x = [_meta(*s).requires_grad_(recorded) for s in shapes]
            x[i] = forward_ad.make_dual(x[i], _meta(*shapes[i]))
            with pytest.raises(RuntimeError, match="no forward-mode derivative"):
                call(*x)


@pytest.mark.parametrize("create_graph", [False, True])
@pytest.mark.parametrize("name", CALLS)
def test_tangents_of_a_gradient_raise(name, create_graph):
    call, shapes = CALLS[name]
    with forward_ad.dual_level():
        x = [_meta(*s).requires_grad_() for s in shapes]
        out = call(*x)
        outs = [out] if torch.is_tensor(out) else list(out)
        douts = [forward_ad.make_dual(torch.empty_like(o), torch.empty_like(o)) for o in outs]
        with pytest.raises(RuntimeError, match="no forward-mode derivative"):
            torch.autograd.grad(outs, x, douts, create_graph=create_graph)
