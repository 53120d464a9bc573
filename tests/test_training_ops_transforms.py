"""The training step's operators where something other than autograd watches the calls.  They fill their outputs through pointers, which
a recording does not see: they refuse, and the sub-networks' norms take torch's operators.  CPU: the checks come before the device's."""
import pytest
import torch
from torch.utils.flop_counter import FlopCounterMode

from categoricalnf_amd import functional as Fn
from categoricalnf_amd import ops

X, W, T = torch.randn(3, 4), torch.randn(5, 4), torch.tensor([0, 1, 2])

CALLS = {
    "layer_norm": lambda x: Fn.layer_norm(x),
    "ops.layer_norm": lambda x: ops.layer_norm(x),
    "ops.layer_norm_bwd": lambda x: ops.layer_norm_bwd(x, x, None, x[:, 0], x[:, 0])[0],
    "ops.linear_cross_entropy_bwd": lambda x: ops.linear_cross_entropy_bwd(x, W, T, None, x[:2, :3], x[0, :3])[0],
    "ops.adamw_step": lambda x: ops.adamw_step([x], [x], [x], [x], step=1, lr=0.1) or x,
}


@pytest.mark.parametrize("name", CALLS)
def test_recordings_are_refused(name):
    with pytest.raises(RuntimeError, match="cannot record"):
        torch.jit.trace(CALLS[name], X, check_trace=False)
    with pytest.raises(RuntimeError, match="cannot record"):
        torch.fx.experimental.proxy_tensor.make_fx(CALLS[name])(X)
    with pytest.raises(ops.HipOnlyError):
        CALLS[name](X)


def test_modules_see_a_recording():
    seen = []

    def f(x):
        seen.append(Fn.recorded())
        return x + 1
    f(X)
    torch.jit.trace(f, X, check_trace=False)
    torch.fx.experimental.proxy_tensor.make_fx(f)(X)
    with FlopCounterMode(display=False):
        f(X)
    f(X)
    assert seen == [False, True, True, True, False]
