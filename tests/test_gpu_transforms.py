"""Transforms that group norm and dropout do not go through are refused on the
GPU: nothing is computed that would pass for their result."""

import pytest
import torch
import torch.autograd.forward_ad as fwd

from deepof_amd import ops

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
CALLS = {
    "group_norm": lambda x: ops.group_norm(x, 2),
    "dropout": lambda x: ops.dropout(x, 0.5, (1, 2)),
    "dropout of 0": lambda x: ops.dropout(x, 0.0, act="elu"),
}


@pytest.mark.parametrize("grad", [False, True])
@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_forward_mode_derivatives_are_refused(call, grad):
    x = torch.randn(1, 4, 3, 3, device=DEV, requires_grad=grad)
    with fwd.dual_level():
        dual = fwd.make_dual(x, torch.ones_like(x))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            call(dual)
    call(x)


@pytest.mark.parametrize("which", ["weight", "bias"])
def test_forward_mode_derivatives_of_parameters_are_refused(which):
    x = torch.randn(1, 4, 3, 3, device=DEV)
    p = {"weight": torch.ones(4, device=DEV), "bias": torch.ones(4, device=DEV)}
    with fwd.dual_level():
        p[which] = fwd.make_dual(p[which], torch.ones(4, device=DEV))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            ops.group_norm(x, 2, **p)


@pytest.mark.parametrize("call", CALLS.values(), ids=CALLS)
def test_tracing_is_refused(call):
    from torch.fx.experimental.proxy_tensor import make_fx

    x = torch.randn(1, 4, 3, 3, device=DEV)
    with pytest.raises(NotImplementedError, match="cannot be traced"):
        torch.jit.trace(call, x)
    with pytest.raises(NotImplementedError, match="cannot be traced"):
        make_fx(call)(x)
    call(x)
