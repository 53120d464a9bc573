"""Layer norm (ops.layer_norm, functional.layer_norm, layers.networks.help_layers.LayerNorm) against the definition in 64 bits.

Tolerances, u = 2^-24 (half a step of fp32), h = half a step of the output's type:
  * a row's mean is a sum of C values: at most C / 1024 + 16 additions in a lane and 11 levels of a tree, so it is off by at most
    n u mean|x| with n = C / 1024 + 32; the centred values, the variance (half its relative error reaches rstd) and the product with
    rstd add fewer than n more of u each.  d_xhat = 2 n u (|xhat| + rstd max|x|) bounds the normalised value;
  * y = xhat w + b: |w| d_xhat + 2 u (|xhat w| + |b|), plus h |y|;
  * dx = rstd (gw - A - xhat B), A = mean gw, B = mean gw xhat: two sums of C terms (n u each relative to the sums of magnitudes),
    the error of xhat in B and beside it, and three roundings;
  * dweight: a sum over R rows in any order: at most (R + 64) u sum|g xhat| + sum |g| d_xhat, plus h; dbias without the second."""
import pytest
import torch

from categoricalnf_amd import functional as Fn
from categoricalnf_amd import ops
from categoricalnf_amd.layers.networks.help_layers import LayerNorm

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(x, g, w, b, eps=1e-5):
    """(values, tolerances) of y, dx, dw, db in float64 on the CPU; a tolerance without the output type's rounding."""
    x, g = x.detach().double().cpu(), g.double().cpu()
    C, R = x.shape[-1], x.numel() // x.shape[-1]
    x, g = x.reshape(R, C), g.reshape(R, C)
    w = torch.ones(C, dtype=torch.float64) if w is None else w.detach().double().cpu()
    b = torch.zeros(C, dtype=torch.float64) if b is None else b.detach().double().cpu()
    n = C / 1024 + 32
    mean = x.mean(1, keepdim=True)
    rstd = 1 / torch.sqrt(((x - mean) ** 2).mean(1, keepdim=True) + eps)
    xh = (x - mean) * rstd
    d_xh = 2 * n * U * (xh.abs() + rstd * x.abs().amax(1, keepdim=True))
    gw = g * w
    A, B = gw.mean(1, keepdim=True), (gw * xh).mean(1, keepdim=True)
    mA, mB = gw.abs().mean(1, keepdim=True), (gw * xh).abs().mean(1, keepdim=True)
    d_rstd = 2 * n * U * (1 + (rstd * x.abs().amax(1, keepdim=True)))        # relative
    val = {"y": xh * w + b, "dx": rstd * (gw - A - xh * B), "dw": (g * xh).sum(0), "db": g.sum(0)}
    tol = {"y": w.abs() * d_xh + 2 * U * ((xh * w).abs() + b.abs()),
           "dx": rstd * (n * U * (gw.abs() + mA + xh.abs() * mB) + d_xh * mB + xh.abs() * (gw.abs() * d_xh).mean(1, keepdim=True))
           + d_rstd * rstd * (gw.abs() + A.abs() + (xh * B).abs()),
           "dw": (R + 64) * U * (g * xh).abs().sum(0) + (g.abs() * d_xh).sum(0), "db": (R + 64) * U * g.abs().sum(0)}
    return val, tol


def check(name, got, val, tol):
    got = got.detach()
    ref = val[name].reshape(got.shape)
    bound = tol[name].reshape(got.shape) + half_step(got.dtype) * ref.abs() + torch.finfo(got.dtype).smallest_normal * half_step(got.dtype) * 2
    err = (got.double().cpu() - ref).abs()
    bad = err > bound
    assert not bad.any(), "%s: %d of %d off, worst %g of %g" % (name, int(bad.sum()), bad.numel(), float(err[bad].max()),
                                                                float((err / bound)[bad].max()))


def run_and_check(x, w, b, g):
    leaves = [t for t in (x, w, b) if t is not None]
    for t in leaves:
        t.requires_grad_()
    y = Fn.layer_norm(x, w, b)
    grads = dict(zip([k for k, t in (("dx", x), ("dw", w), ("db", b)) if t is not None], torch.autograd.grad(y, leaves, g)))
    assert y.dtype == x.dtype and y.shape == x.shape and y.is_contiguous()
    val, tol = reference(x, g, w, b)
    check("y", y, val, tol)
    for k, t in grads.items():
        check(k, t, val, tol)
    with torch.no_grad():
        assert torch.equal(ops.layer_norm(x, w, b), y)
    return y, grads


def make(shape, dtype, seed=0, pdtype=None, affine=True):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    C = shape[-1]
    x = (torch.randn(shape, generator=gen, device="cuda") * 2 + 0.7).to(dtype)
    g = torch.randn(shape, generator=gen, device="cuda").to(dtype)
    if not affine:
        return x, None, None, g
    w = (1 + 0.3 * torch.randn(C, generator=gen, device="cuda")).to(pdtype or dtype)
    b = (0.3 * torch.randn(C, generator=gen, device="cuda")).to(pdtype or dtype)
    return x, w, b, g


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("cols", [1, 2, 3, 7, 8, 16, 17, 63, 64, 65, 100, 128, 200, 256, 777, 1000, 1024, 1025, 1032, 2048, 4096, 5001,
                                  8192, 16384, 16385, 20000])
def test_values_and_gradients(cols, dtype):
    rows = 300 if cols <= 1100 else 7
    run_and_check(*make((rows, cols), dtype, seed=cols))


@pytest.mark.parametrize("rows", [1, 2, 3, 5, 63, 257, 4999, 70001])
@pytest.mark.parametrize("cols", [1, 8, 24, 130])
def test_row_counts(rows, cols):
    run_and_check(*make((rows, cols), F32, seed=rows))


@pytest.mark.parametrize("rows,cols", [(3000, 1500), (1300, 20001)])
def test_wide_rows_on_many_workgroups(rows, cols):
    run_and_check(*make((rows, cols), BF16, seed=3))


def test_no_parameters_or_one_of_them():
    x, w, b, g = make((50, 96), F32)
    run_and_check(x, None, None, g)
    x, w, b, g = make((50, 96), BF16)
    run_and_check(x, w, None, g)
    x, w, b, g = make((50, 96), F16)
    run_and_check(x, None, b, g)


@pytest.mark.parametrize("dtype", [BF16, F16])
def test_fp32_parameters_of_a_16_bit_input(dtype):
    y, grads = run_and_check(*make((77, 120), dtype, pdtype=F32))
    assert grads["dw"].dtype == F32 and grads["db"].dtype == F32 and grads["dx"].dtype == dtype


@pytest.mark.parametrize("dtype", [F32, F16])
@pytest.mark.parametrize("layout", ["slice", "unaligned", "transposed", "columns_apart", "three_axes"])
def test_strided_inputs(layout, dtype):
    wide, w, b, _ = make((40, 80), dtype)
    w, b = w[:64].clone(), b[:64].clone()
    x = {"slice": lambda: wide[:, :64], "unaligned": lambda: wide[:, 1:65],
         "transposed": lambda: torch.randn(64, 40, device="cuda").to(dtype).t(),
         "columns_apart": lambda: torch.randn(40, 128, device="cuda").to(dtype)[:, ::2],
         "three_axes": lambda: torch.randn(5, 8, 64, device="cuda").to(dtype).transpose(0, 1)}[layout]().detach()
    g = torch.randn(x.shape, device="cuda").to(dtype)
    if layout == "slice":
        g = torch.randn(40, 72, device="cuda").to(dtype)[:, 8:]
    run_and_check(x, w, b, g)


def test_expanded_gradient_and_no_gradient_for_the_input():
    x, w, b, _ = make((33, 48), F32)
    run_and_check(x, w, b, torch.randn(48, device="cuda").expand(33, 48))
    x, w, b, g = make((33, 48), F32)
    w.requires_grad_(), b.requires_grad_()
    y = Fn.layer_norm(x, w, b)
    val, tol = reference(x, g, w, b)
    for k, t in zip(("dw", "db"), torch.autograd.grad(y, (w, b), g)):
        check(k, t, val, tol)


def test_no_rows():
    x = torch.zeros(0, 16, device="cuda", requires_grad=True)
    w = torch.ones(16, device="cuda", requires_grad=True)
    y = Fn.layer_norm(x, w, None)
    gx, gw = torch.autograd.grad(y, (x, w), torch.zeros(0, 16, device="cuda"))
    assert y.shape == (0, 16) and gx.shape == (0, 16) and torch.equal(gw, torch.zeros_like(gw))


def test_common_offset_and_constant_rows():
    """A common offset of 4096 leaves the spread of a row to the last 11 bits of its values: the centred sum of squares keeps it."""
    x, w, b, g = make((64, 500), F32)
    run_and_check((x + 4096).detach(), w, b, g)
    c = torch.full((3, 64), 2.5, device="cuda")
    assert torch.equal(ops.layer_norm(c), torch.zeros_like(c))


def test_nonfinite_rows_stay_alone():
    x, w, b, g = make((20, 100), F32)
    clean = ops.layer_norm(x, w, b)
    x[3, 7], x[11, 0], x[12, 99] = float("nan"), float("inf"), float("-inf")
    y = ops.layer_norm(x, w, b)
    bad = torch.zeros(20, dtype=torch.bool, device="cuda")
    bad[[3, 11, 12]] = True
    assert torch.isnan(y[bad]).all() and torch.equal(y[~bad], clean[~bad])


def test_gradients_against_differences():
    """d/dt sum(g * f(x + t d)) by central differences of the 64-bit definition, at the kernel's gradient."""
    x, w, b, g = make((6, 40), F32, seed=9)
    _, grads = run_and_check(x, w, b, g)
    d = torch.randn(6, 40).double()

    def f(t):
        xx = x.detach().double().cpu() + t * d
        xc = xx - xx.mean(1, keepdim=True)
        y = xc / torch.sqrt((xc ** 2).mean(1, keepdim=True) + 1e-5) * w.detach().double().cpu() + b.detach().double().cpu()
        return float((y * g.double().cpu()).sum())
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    mine = float((grads["dx"].double().cpu() * d).sum())
    # the difference quotient is off by t^2 / 6 f''' + f eps / t: below 1e-8 |f| here; the kernel's sum by its own bound
    _, tol = reference(x, g, w, b)
    assert abs(slope - mine) <= 1e-7 * (1 + abs(f(0.0))) + float(((tol["dx"] + U * grads["dx"].double().cpu().abs()) * d.abs()).sum())


def test_same_bits_on_every_run_and_on_another_stream():
    x, w, b, g = make((5000, 264), BF16)
    _, first = run_and_check(x, w, b, g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = Fn.layer_norm(x, w, b)
        second = torch.autograd.grad(y, (x, w, b), g)
    torch.cuda.synchronize()
    for p, q in zip(first.values(), second):
        assert torch.equal(p, q)


def test_captured_step_replays():
    """Forward and backward in one HIP graph; replays on new inputs equal the eager result."""
    x, w, b, g = make((513, 96), F32)
    w2, b2 = w.clone().requires_grad_(), b.clone().requires_grad_()
    xs, gs = x.clone().requires_grad_(), g.clone()

    def step():
        y = Fn.layer_norm(xs, w2, b2)
        return (y.detach(),) + torch.autograd.grad(y, (xs, w2, b2), gs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 5):
        x1, _, _, g1 = make((513, 96), F32, seed=seed)
        with torch.no_grad():
            xs.copy_(x1), gs.copy_(g1)
        graph.replay()
        torch.cuda.synchronize()
        x1.requires_grad_()
        y = Fn.layer_norm(x1, w2, b2)
        for p, q in zip(out, (y.detach(),) + torch.autograd.grad(y, (x1, w2, b2), g1)):
            assert torch.equal(p, q)
        del y


def test_more_elements_than_2_to_the_31():
    """Rows whose elements lie beyond 2^31 give what they give at the front."""
    C, n = 512, 300
    R = 2 ** 31 // C + n
    x, g = torch.zeros(R, C, dtype=BF16, device="cuda"), torch.zeros(R, C, dtype=BF16, device="cuda")
    x[-n:].normal_(), g[-n:].normal_()
    w, b = torch.randn(C, device="cuda").to(BF16), torch.randn(C, device="cuda").to(BF16)
    front_x, front_g = x[-n:].clone(), g[-n:].clone()
    x.requires_grad_(), front_x.requires_grad_()
    y, front_y = Fn.layer_norm(x, w, b), Fn.layer_norm(front_x, w, b)
    assert torch.equal(y[-n:], front_y) and torch.equal(y[:2], b.expand(2, C))
    (dx,), (front_dx,) = torch.autograd.grad(y, x, g), torch.autograd.grad(front_y, front_x, front_g)
    assert torch.equal(dx[-n:], front_dx) and not dx[:-n].any()


def test_module_is_the_kernel_on_the_gpu_and_torch_elsewhere():
    torch.manual_seed(0)
    mine, ref = LayerNorm(72).cuda(), torch.nn.LayerNorm(72)
    with torch.no_grad():
        mine.weight.normal_(), mine.bias.normal_()
    ref.load_state_dict({k: v.cpu() for k, v in mine.state_dict().items()})
    x = torch.randn(4, 9, 72)
    y = mine(x.cuda())
    assert torch.equal(y, ops.layer_norm(x.cuda(), mine.weight, mine.bias))
    val, tol = reference(x, x, ref.weight, ref.bias)
    check("y", y, val, tol)
    assert torch.equal(mine.cpu()(x), ref(x))
    x64 = torch.randn(3, 72, dtype=torch.float64, device="cuda")
    torch.testing.assert_close(mine.cuda().double()(x64).cpu(), ref.double()(x64.cpu()))


def test_refusals_on_the_gpu():
    x = torch.randn(4, 8, device="cuda")
    with pytest.raises(ValueError):
        ops.layer_norm(x, torch.ones(7, device="cuda"))
    with pytest.raises(TypeError):
        ops.layer_norm(x, torch.ones(8, device="cuda"), torch.ones(8, device="cuda", dtype=F16))
    with pytest.raises(TypeError):
        ops.layer_norm(x.double())
    with pytest.raises(ValueError):
        ops.layer_norm(torch.zeros(4, 0, device="cuda"))
    with pytest.raises(ops.HipOnlyError):
        ops.layer_norm(x, torch.ones(8))
    y, mean, rstd = ops.layer_norm(x, want_stats=True)
    with pytest.raises(ValueError):
        ops.layer_norm_bwd(x, x[:2], None, mean, rstd)
    xg = x.clone().requires_grad_()
    s = Fn.layer_norm(xg).square().sum()
    (g,) = torch.autograd.grad(s, xg, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()
