"""Host side of the training step's operators: refusals of the C entry points (before anything is launched), of CPU tensors, and
the optimiser's bookkeeping without a GPU."""
import ctypes

import pytest
import torch

from categoricalnf_amd import _lib, functional as Fn, ops
from categoricalnf_amd.layers.networks.help_layers import LayerNorm
from categoricalnf_amd.optim import AdamW

P = ctypes.c_void_p(16)          # a pointer that no refused call may follow


@pytest.fixture(scope="module")
def lib():
    from categoricalnf_amd import build
    build.build()
    return _lib.load()


def test_layer_norm_refuses_before_launching(lib):
    ok = [P, 8, None, None, P, None, None, 4, 8, 1e-5, 0, 0, None]
    for i, bad in ((0, None), (4, None), (5, P), (7, -1), (8, 0), (1, -8), (10, 3), (11, -1)):
        args = list(ok)
        args[i] = bad
        assert lib.cnf_layer_norm(*args) == 1 and b"cnf_layer_norm" in lib.cnf_last_error(), i
    assert lib.cnf_layer_norm(*(ok[:7] + [0] + ok[8:])) == 0          # no rows: nothing to do
    need = lib.cnf_layer_norm_bwd_workspace_floats(1000, 40)
    assert need >= 2 * 40
    ok = [P, 40, P, 40, None, P, P, P, P, None, P, need, 1000, 40, 0, 0, None]
    for i, bad in ((0, None), (2, None), (5, None), (6, None), (7, None), (10, None), (11, need - 1), (13, 0), (14, 7), (3, -1)):
        args = list(ok)
        args[i] = bad
        assert lib.cnf_layer_norm_bwd(*args) == 1 and b"cnf_layer_norm_bwd" in lib.cnf_last_error(), i


def test_layer_norm_workspace_covers_every_layout(lib):
    """Never less than one partial row, never more than 1024 of them, monotone enough to be bounded by the rows."""
    for cols in (1, 3, 8, 64, 100, 1024, 1025, 5000, 16384, 16385, 40000):
        for rows in (1, 2, 7, 300, 5000, 10 ** 6, 10 ** 9):
            n = lib.cnf_layer_norm_bwd_workspace_floats(rows, cols)
            assert n % (2 * cols) == 0 and 1 <= n // (2 * cols) <= min(rows, 1024)
    assert lib.cnf_layer_norm_bwd_workspace_floats(0, 8) == 0


def test_adamw_refuses_before_launching(lib):
    ptrs = (ctypes.c_void_p * 2)(16, 16)
    nulls = (ctypes.c_void_p * 2)(16, None)
    sizes = (ctypes.c_int64 * 2)(4, 4)
    neg = (ctypes.c_int64 * 2)(4, -1)
    ok = [2, ptrs, ptrs, ptrs, ptrs, None, None, sizes, 0, 0, 32, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1.0, None, None, None]
    for i, bad in ((0, -1), (1, None), (2, nulls), (3, None), (7, neg), (8, 5), (9, 1), (10, 16), (10, 8), (12, 1.0), (13, -0.1), (16, 0.0)):
        args = list(ok)
        args[i] = bad
        assert lib.cnf_adamw_step(*args) == 1 and b"cnf_adamw_step" in lib.cnf_last_error(), i
    assert lib.cnf_adamw_step(*([0] + ok[1:])) == 0
    assert lib.cnf_adamw_moments(None, P, P, P, P, P, 4, None) == 1 and lib.cnf_adamw_moments(P, P, P, P, P, P, 0, None) == 0


def test_cpu_tensors_are_refused():
    x = torch.randn(3, 4)
    with pytest.raises(ops.HipOnlyError):
        ops.layer_norm(x)
    with pytest.raises(ops.HipOnlyError):
        Fn.layer_norm(x.requires_grad_())
    with pytest.raises(ops.HipOnlyError):
        ops.adamw_step([torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], [torch.zeros(3)], step=1, lr=1e-3)


def test_layer_norm_module_on_the_host_is_torchs():
    m, ref = LayerNorm(6), torch.nn.LayerNorm(6)
    x = torch.randn(2, 5, 6)
    assert torch.equal(m(x), ref(x)) and set(m.state_dict()) == set(ref.state_dict())
    assert LayerNorm((5, 6))(x).shape == x.shape


def test_optimiser_arguments():
    p = [torch.nn.Parameter(torch.zeros(3))]
    for kw in (dict(lr=-1.0), dict(betas=(0.9, 1.0)), dict(betas=(-0.1, 0.9)), dict(eps=-1e-8), dict(weight_decay=-1.0), dict(state_bits=16),
               dict(lr=torch.tensor(1e-3))):
        with pytest.raises(ValueError):
            AdamW(p, **kw)
    opt = AdamW(p, lr=0.5)
    assert opt.moments(p[0]) is None and opt.step() is None           # no gradients: nothing happens
    p[0].grad = torch.ones(3)
    with pytest.raises(ops.HipOnlyError):
        opt.step()


def test_drivers_offer_the_optimisers():
    from categoricalnf_amd.experiments import run_graph_coloring, run_language_modeling, run_set_modeling
    for mod in (run_graph_coloring, run_language_modeling, run_set_modeling):
        args = mod.parse([])
        p = [torch.nn.Parameter(torch.zeros(3))]
        assert type(mod.make_optimizer(args, p)) is torch.optim.RAdam
        for name, bits in (("adamw", 32), ("adamw8", 8)):
            opt = mod.make_optimizer(mod.parse(["--optimizer", name, "--weight_decay", "0.5"]), p)
            assert type(opt) is AdamW and opt.param_groups[0]["state_bits"] == bits and opt.param_groups[0]["weight_decay"] == 0.5
