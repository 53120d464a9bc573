"""The sub-networks' norm where something other than autograd watches the calls: what torch's norm gives there."""
import pytest
import torch
import torch.autograd.forward_ad as fwad

from categoricalnf_amd import functional as Fn
from categoricalnf_amd.layers.networks.help_layers import LayerNorm

pytestmark = pytest.mark.gpu


def pair(cols=24, dtype=torch.float32, seed=0):
    """This package's norm and torch's with the same parameters, and an input."""
    torch.manual_seed(seed)
    mine, ref = LayerNorm(cols).cuda().to(dtype), torch.nn.LayerNorm(cols).cuda().to(dtype)
    with torch.no_grad():
        ref.weight.normal_(), ref.bias.normal_()
    mine.load_state_dict(ref.state_dict())
    return mine, ref, torch.randn(5, cols, device="cuda", dtype=dtype)


def test_traced_norm_gives_what_the_eager_one_gives():
    mine, ref, x = pair()
    for check in (True, False):
        traced = torch.jit.trace(mine, x, check_trace=check)
        for seed in range(3):
            y = torch.randn(5, 24, device="cuda", generator=torch.Generator("cuda").manual_seed(seed))
            assert torch.equal(traced(y), ref(y))
    graph = torch.fx.experimental.proxy_tensor.make_fx(mine)(x)
    assert torch.equal(graph(x * 2), ref(x * 2))
    with pytest.raises(RuntimeError, match="cannot record"):
        torch.jit.trace(lambda v: Fn.layer_norm(v), x)
    with pytest.raises(RuntimeError, match="cannot record"):
        torch.jit.trace(lambda v: Fn.linear_cross_entropy(v, x, torch.arange(5, device="cuda")), x)
    assert torch.equal(mine(x), Fn.layer_norm(x, mine.weight, mine.bias))


def test_tangents_pass_the_norm():
    mine, ref, x = pair()
    for m in (mine, ref):
        m.requires_grad_(False)
    t = torch.randn_like(x)
    for grad in (True, False):
        with torch.set_grad_enabled(grad), fwad.dual_level():
            got, want = (fwad.unpack_dual(m(fwad.make_dual(x, t))) for m in (mine, ref))
            assert torch.equal(got.primal, want.primal) and torch.equal(got.tangent, want.tangent)
            with pytest.raises(NotImplementedError):
                Fn.layer_norm(fwad.make_dual(x, t))
            with pytest.raises(NotImplementedError):
                Fn.linear_cross_entropy(fwad.make_dual(x, t), x, torch.arange(5, device="cuda"))


def test_function_transforms_pass_the_norm():
    mine, ref, x = pair()
    params = {k: v.detach() for k, v in mine.named_parameters()}
    for make in (lambda m: torch.func.vmap(m)(x[None].expand(3, -1, -1) * torch.arange(1, 4, device="cuda")[:, None, None]),
                 lambda m: torch.func.grad(lambda v: m(v).square().sum())(x),
                 lambda m: torch.func.jvp(m, (x,), (x.flip(0),))[1],
                 lambda m: torch.func.grad(lambda q: torch.func.functional_call(m, q, (x,)).square().sum())(params)["weight"],
                 lambda m: torch.func.vmap(torch.func.grad(lambda q, v: torch.func.functional_call(m, q, (v,)).square().sum()), in_dims=(None, 0))(params, x)["bias"]):
        got, want = make(mine), make(ref)
        assert torch.equal(got, want)
    # the function itself takes no transform
    for call in (lambda: torch.func.vmap(Fn.layer_norm)(x), lambda: torch.func.grad(lambda v: Fn.layer_norm(v).sum())(x)):
        with pytest.raises(NotImplementedError, match="torch.func"):
            call()


@pytest.mark.parametrize("affine", ["both", "weight", "none"])
def test_second_derivatives_of_the_norm(affine):
    """A penalty on the gradient's square, its own gradients in the input, the parameters and the upstream gradient against 64 bits.  The
    longest chain: four sums over 24 columns, one over 5 rows, some 40 products: 150 roundings of 2^-24, of sums of absolute values
    that exceed a tensor's largest element by less than a factor of 16; those of the first gradient enter the second squared: twice."""
    torch.manual_seed(1)
    mine = LayerNorm(24, elementwise_affine=affine != "none", bias=affine == "both").cuda()
    with torch.no_grad():
        for p in mine.parameters():
            p.normal_()
    ref = torch.nn.LayerNorm(24, elementwise_affine=affine != "none", bias=affine == "both").double()
    ref.load_state_dict({k: v.double().cpu() for k, v in mine.state_dict().items()})
    x, u = torch.randn(5, 24), torch.randn(5, 24)

    def second(m, x, u):
        x, u = x.clone().requires_grad_(), u.clone().requires_grad_()
        wrt = [x] + list(m.parameters())
        first = torch.autograd.grad(m(x), wrt, u, create_graph=True)
        return first, torch.autograd.grad(sum(g.square().sum() for g in first), wrt[:2] + [u])
    first, got = second(mine, x.cuda(), u.cuda())
    want_first, want = second(ref, x.double(), u.double())
    for a, b in zip(first + got, want_first + want):
        assert float((a.detach().cpu().double() - b).abs().max()) <= 2 * 150 * 2.0 ** -24 * 16 * float(b.detach().abs().max())
    # the gradient alone still comes from the kernel
    xg = x.cuda().requires_grad_()
    (a,), (b,) = (torch.autograd.grad(f(xg), xg, u.cuda()) for f in (mine, lambda v: Fn.layer_norm(v, mine.weight, mine.bias)))
    assert torch.equal(a, b)


def test_second_derivatives_in_16_bits_keep_the_types():
    m = LayerNorm(16).cuda().bfloat16()
    x = torch.randn(3, 2, 16, device="cuda", dtype=torch.bfloat16, requires_grad=True)
    g = torch.autograd.grad(m(x).square().sum(), [x, m.weight, m.bias], create_graph=True)
    assert all(a.dtype == torch.bfloat16 for a in g)
    h = torch.autograd.grad(sum(a.float().square().sum() for a in g), [x, m.weight])
    assert all(a.dtype == torch.bfloat16 and bool(torch.isfinite(a).all()) for a in h)


@pytest.mark.parametrize("backend", ["eager", "aot_eager"])
def test_compiled_norm_is_one_graph(backend):
    mine, ref, x = pair()
    torch._dynamo.reset()
    compiled = torch.compile(mine, backend=backend, fullgraph=True)
    xs = [x.clone().requires_grad_() for _ in range(2)]
    got, want = compiled(xs[0]), ref(xs[1])
    assert torch.equal(got, want)
    got.square().sum().backward(), want.square().sum().backward()
    assert torch.equal(xs[0].grad, xs[1].grad) and torch.equal(mine.weight.grad, ref.weight.grad)


def test_batched_gradients_of_the_norm():
    """Several upstream gradients at once: each one's gradients as they come alone from torch's norm (the operators of the composed
    backward: the bound of test_second_derivatives_of_the_norm for one derivative)."""
    mine, ref, x = pair()
    u = torch.randn(3, 5, 24, device="cuda")
    ref.double()
    wrt = lambda m, v: [v] + list(m.parameters())
    xg, xr = x.clone().requires_grad_(), x.double().requires_grad_()
    got = torch.autograd.grad(mine(xg), wrt(mine, xg), u, is_grads_batched=True)
    for k in range(3):
        want = torch.autograd.grad(ref(xr), wrt(ref, xr), u[k].double())
        for a, b in zip(got, want):
            assert float((a[k].double() - b).abs().max()) <= 150 * 2.0 ** -24 * 16 * float(b.abs().max())
    j = torch.autograd.functional.jacobian(lambda v: mine(v).sum(0), x, vectorize=True)
    r = torch.autograd.functional.jacobian(lambda v: ref(v).sum(0), x.double())
    assert float((j.double() - r).abs().max()) <= 150 * 2.0 ** -24 * 16 * float(r.abs().max())
    with pytest.raises(RuntimeError):
        torch.autograd.grad(Fn.layer_norm(xg), xg, u, is_grads_batched=True)


def test_tangents_of_the_upstream_gradient():
    mine, ref, x = pair()
    u, t = torch.randn(2, 5, 24, device="cuda")
    out = []
    for m in (mine, ref):
        xg = x.clone().requires_grad_()
        y = m(xg)
        with fwad.dual_level():
            (d,) = torch.autograd.grad(y, xg, fwad.make_dual(u, t))
            out.append(fwad.unpack_dual(d))
    for a, b in ((out[0].primal, out[1].primal), (out[0].tangent, out[1].tangent)):
        assert float((a - b).abs().max()) <= 2 * 150 * 2.0 ** -24 * 16 * float(b.abs().max())
