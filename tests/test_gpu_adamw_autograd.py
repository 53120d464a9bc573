"""AdamW writes through pointers: what autograd and the optimiser's own bookkeeping have to notice of it."""
import pytest
import torch

from categoricalnf_amd import ops
from categoricalnf_amd.optim import AdamW

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("bits", [32, 8])
def test_a_step_counts_as_a_change_in_place(bits):
    net = torch.nn.Sequential(torch.nn.Linear(20, 30), torch.nn.Linear(30, 2)).cuda()
    opt = AdamW(net.parameters(), lr=1e-2, state_bits=bits, min_8bit_size=100)
    x = torch.randn(4, 20, device="cuda")
    net(x).sum().backward()
    opt.step()
    kept = [p for p in net.parameters()] + [v for p in net.parameters() for k, v in opt.state[p].items() if k != "step"]
    before, grads = [t._version for t in kept], [p.grad._version for p in net.parameters()]
    loss = net(x).square().sum()                        # saves the second layer's weight
    opt.step()
    assert [t._version for t in kept] == [v + 1 for v in before] and [p.grad._version for p in net.parameters()] == grads
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        loss.backward()


def test_inference_tensors_have_no_version():
    with torch.inference_mode():
        p, g, m, v = (torch.ones(5, device="cuda") for _ in range(4))
    ops.adamw_step([p], [g], [m], [v], step=1, lr=0.5, weight_decay=0.0)
    assert bool((p != 1).all())


def test_idle_parameters_of_a_captured_step_keep_their_count():
    """Replays after an eager step with the same gradients present: the idle parameter's counter stands, and is right when it is active again."""
    ps = [torch.nn.Parameter(torch.randn(300, device="cuda")) for _ in range(3)]
    opt = AdamW(ps, lr=torch.tensor(1e-2, device="cuda"), capturable=True)
    for p in ps:
        p.grad = torch.randn(300, device="cuda")
    opt.step()
    ps[1].grad = None
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    idle = ps[1].detach().clone()
    with torch.cuda.graph(graph):
        opt.step()
    for k in range(1, 5):
        graph.replay()
        torch.cuda.synchronize()
        assert [float(opt.state[p]["step"]) for p in ps] == [2 + k, 1, 2 + k] and torch.equal(ps[1], idle)
    ps[1].grad = torch.ones(300, device="cuda")
    opt.step()
    assert [float(opt.state[p]["step"]) for p in ps] == [7, 2, 7]
