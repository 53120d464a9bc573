"""Calls of the raw gradients that reach past a tensor: an error, and nothing is launched."""
import pytest
import torch

from categoricalnf_amd import ops

pytestmark = pytest.mark.gpu


def test_count_is_one_value():
    x, w, t = torch.randn(6, 8, device="cuda"), torch.randn(5, 8, device="cuda"), torch.arange(6, device="cuda") % 5
    _, stats, reduced, exps = ops.linear_cross_entropy(x, w, t, want_reduced=True)
    g = torch.ones(1, device="cuda")
    want = ops.linear_cross_entropy_bwd(x, w, t, None, stats, g, count=reduced[2:], exponents=exps)
    for count in (reduced[:0], reduced, reduced[2:].double(), reduced[2:].cpu()):
        with pytest.raises(ValueError):
            ops.linear_cross_entropy_bwd(x, w, t, None, stats, g, count=count, exponents=exps)
    assert all(a is b or torch.equal(a, b) for a, b in zip(want, ops.linear_cross_entropy_bwd(x, w, t, None, stats, g, count=reduced[2:], exponents=exps)))


def test_layer_norm_bwd_needs_a_last_axis():
    x = torch.zeros(3, 0, device="cuda")
    s = torch.zeros(3, device="cuda")
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x, x, None, s, s)
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x.sum(), x.sum(), None, s, s)
