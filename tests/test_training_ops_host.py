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


def test_linear_ce_refuses_before_launching(lib):
    need = lib.cnf_linear_ce_workspace_bytes(100, 50, 16, 0, 0)
    assert need > 0 and lib.cnf_linear_ce_workspace_bytes(0, 50, 16, 0, 0) == 0 and lib.cnf_linear_ce_workspace_bytes(10, 50, 16, 9, 0) == 0
    #     x  xs  w  ws  b     t  ign   loss max sum red   exp   ws bytes R    V   H   dt bdt flags stream
    ok = [P, 16, P, 16, None, P, -100, P, P, P, None, None, P, need, 100, 50, 16, 0, 0, None, None]
    for i, bad in ((0, None), (2, None), (5, None), (7, None), (8, None), (9, None), (12, None), (13, need - 1), (14, -1), (15, 0), (16, 0), (17, 3),
                   (18, -1), (1, -16), (12, ctypes.c_void_p(24))):
        args = list(ok)
        args[i] = bad
        assert lib.cnf_linear_ce(*args) == 1 and b"cnf_linear_ce" in lib.cnf_last_error(), i
    assert lib.cnf_linear_ce(*(ok[:14] + [0] + ok[15:])) == 0                     # no rows and nothing to reduce
    need = lib.cnf_linear_ce_workspace_bytes(100, 50, 16, 0, 1)
    #     x  xs  w  ws  b     t  ign   max sum exp   g  per count dx dw db   ws bytes R    V   H   dt bdt stream
    ok = [P, 16, P, 16, None, P, -100, P, P, None, P, 1, None, P, P, None, P, need, 100, 50, 16, 0, 0, None]
    for i, bad in ((0, None), (2, None), (5, None), (7, None), (8, None), (10, None), (11, 0), (16, None), (17, need - 1), (18, 0), (19, 0), (21, 4),
                   (16, ctypes.c_void_p(20))):
        args = list(ok)
        args[i] = bad
        assert lib.cnf_linear_ce_bwd(*args) == 1 and b"cnf_linear_ce_bwd" in lib.cnf_last_error(), i
    for none in ((13, 14), (14,)):                                               # nothing asked for; dbias without dweight
        args = list(ok)
        args[15] = P if none == (14,) else None
        for i in none:
            args[i] = None
        assert lib.cnf_linear_ce_bwd(*args) == 1


def test_sizes_beyond_the_loop_counters_are_refused(lib):
    """Rows, classes or features that a kernel's 32-bit counters and offsets do not reach: an error before anything is launched."""
    for R, V, H in ((4, 2 ** 30 + 1, 8), (4, 50, 2 ** 21 + 8), (2 ** 31 - 1, 50, 16)):
        assert lib.cnf_linear_ce_workspace_bytes(R, V, H, 1, 1) == 0
        args = [P, H, P, H, None, P, -100, P, P, P, None, None, P, 2 ** 62, R, V, H, 1, 1, None, None]
        assert lib.cnf_linear_ce(*args) == 1 and b"bad size" in lib.cnf_last_error()
        args = [P, H, P, H, None, P, -100, P, P, None, P, 1, None, P, P, None, P, 2 ** 62, R, V, H, 1, 1, None]
        assert lib.cnf_linear_ce_bwd(*args) == 1 and b"bad size" in lib.cnf_last_error()
    C = 2 ** 30 + 1
    assert lib.cnf_layer_norm(P, C, None, None, P, None, None, 1, C, 1e-5, 0, 0, None) == 1 and b"bad size" in lib.cnf_last_error()
    assert lib.cnf_layer_norm_bwd(P, C, P, C, None, P, P, P, None, None, None, 0, 1, C, 0, 0, None) == 1 and b"bad size" in lib.cnf_last_error()
    assert lib.cnf_layer_norm_bwd_workspace_floats(1, C) == 0


def test_linear_ce_workspace_is_bounded(lib):
    """The gradient of the logits never takes more than 512 MiB beyond what one strip of 256 classes needs, however large the
    vocabulary: nothing of size rows x vocabulary is kept."""
    for rows, vocab, hidden in ((8192, 200_000, 1024), (100_000, 50_000, 512), (1, 10 ** 6, 4096)):
        for dtype, parts in ((0, 2), (1, 1), (2, 1)):
            n = lib.cnf_linear_ce_workspace_bytes(rows, vocab, hidden, dtype, 1)
            copies = parts * 2 * (rows + vocab) * (hidden + 8)
            partial = 64 * rows * (hidden + 8) * 4 + 64 * vocab * (hidden + 8) * 4 if rows < 1000 else 3 * (rows + vocab) * (hidden + 8) * 4
            assert n <= copies + partial + max(512 << 20, (rows + 256) * 256 * 2 * parts) + (rows + 256) * 16 + (1 << 20), (rows, vocab, n)


def test_cpu_tensors_are_refused():
    x = torch.randn(3, 4)
    with pytest.raises(ops.HipOnlyError):
        Fn.linear_cross_entropy(x, torch.randn(5, 4), torch.tensor([0, 1, 2]))
    with pytest.raises(ops.HipOnlyError):
        ops.linear_cross_entropy(x, torch.randn(5, 4), torch.tensor([0, 1, 2]))
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
