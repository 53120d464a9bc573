"""The training step's operators where something other than autograd watches the calls.  They fill their outputs through pointers, which
a recording does not see: they refuse, and the sub-networks' norms take torch's operators.  CPU: the checks come before the device's."""
import pytest
import torch
import torch.autograd.forward_ad as fwad
from torch.utils.flop_counter import FlopCounterMode

from categoricalnf_amd import functional as Fn
from categoricalnf_amd import ops

X, W, T = torch.randn(3, 4), torch.randn(5, 4), torch.tensor([0, 1, 2])

CALLS = {
    "layer_norm": lambda x: Fn.layer_norm(x),
    "ops.layer_norm": lambda x: ops.layer_norm(x),
    "ops.layer_norm_bwd": lambda x: ops.layer_norm_bwd(x, x, None, x[:, 0], x[:, 0])[0],
    "ops.linear_cross_entropy_bwd": lambda x: ops.linear_cross_entropy_bwd(x, W, T, None, x[:2, :3], x[0, :3])[0],
    "ops.adamw_moments": lambda x: ops.adamw_moments(x, x, x, x)[0],
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
        seen.append(Fn.transformed())
        return x + 1
    f(X)
    torch.jit.trace(f, X, check_trace=False)
    torch.fx.experimental.proxy_tensor.make_fx(f)(X)
    with FlopCounterMode(display=False):
        f(X)
    f(X)
    assert seen == [False, True, True, True, False]


CE = lambda x, w, b: ops.native().linear_ce(x, w, T, b, -100, 1, torch.zeros(1, dtype=torch.int32))
TANGENTS = {**{k: (f, X) for k, f in CALLS.items() if not k.startswith("ops.adamw")}, "layer_norm, bias": (lambda b: Fn.layer_norm(X, None, b), X[0]),
            "linear_cross_entropy": (lambda x: CE(x, W, None), X), "linear_cross_entropy, weight": (lambda w: CE(X, w, None), W),
            "linear_cross_entropy, bias": (lambda b: CE(X, W, b), W[:, 0].contiguous())}


@pytest.mark.parametrize("name", TANGENTS)
def test_tangents_are_refused(name):
    """With frozen operands, and under no_grad, where no autograd node would notice."""
    call, x = TANGENTS[name]
    with fwad.dual_level():
        for grad in (True, False):
            for leaf in (x.clone(), x.clone().requires_grad_()):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError, match="forward-mode"):
                    call(fwad.make_dual(leaf, torch.ones_like(x)))


def test_modules_see_tangents():
    assert not Fn.transformed()
    with fwad.dual_level():
        assert Fn.transformed()
    assert not Fn.transformed()


def test_modules_see_function_transforms():
    seen = []

    def f(x):
        seen.append(Fn.transformed())
        return (x * x).sum()
    torch.func.vmap(f)(X), torch.func.grad(f)(X), torch.func.jvp(f, (X,), (X,)), torch.func.vjp(f, X), torch.func.hessian(f)(X)
    assert len(seen) >= 5 and all(seen) and not Fn.transformed()


@pytest.mark.parametrize("name", [k for k in TANGENTS])
def test_function_transforms_are_refused(name):
    call, x = TANGENTS[name]
    for transform in (lambda f: lambda v: torch.func.vmap(f)(v[None]), torch.func.grad, lambda f: lambda v: torch.func.jvp(f, (v,), (v,))):
        with pytest.raises(NotImplementedError, match="torch.func|forward-mode"):
            transform(call)(x.clone())
    with pytest.raises(NotImplementedError, match="torch.func"):
        torch.func.vmap(lambda v: ops.adamw_step([v], [v], [v], [v], step=1, lr=0.1) or v)(X)


def test_modules_see_a_compilation():
    def f(x):
        return x + 1 if Fn.transformed() else x - 1
    torch._dynamo.reset()
    assert torch.equal(torch.compile(f, backend="eager", fullgraph=True)(X), X + 1) and torch.equal(f(X), X - 1)
