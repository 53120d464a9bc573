"""Linear cross entropy (ops.linear_cross_entropy, functional.linear_cross_entropy) against the definition in 64 bits.

Tolerances, u = 2^-24, h = half a step of the operands' type, P = 6 roundings per term for fp32 operands (three products of fp16
parts; the part left out, below 2^-22 = 4 u of |x w|, counts less than the other three) and 1 otherwise:
  * a logit is a sum of P H exact products, at most 2 u lost per addition (the matrix unit may cut where it aligns):
    e_l = 2 (P H + 16) u sum_k |x w| + 2 u |b|;
  * exp2 of a rounded argument: relative (2 |l - m| + 4) u per term; the sum of V terms: at most V / 8 + 64 additions in a lane and
    the tree; the logarithm and the two differences add 4 u of their magnitudes.  The loss is off by at most e_l of its target
    plus the p-weighted error of the others;
  * d = g (p - [v = t]): |g| p (e_l + e_lse + relative error of p) + 2 u |d|, and its rounding to the operands' type, h |d| (fp32:
    2^-24; fp16 below its normal range: 2^-38 of the largest |g|);
  * dx, dweight: these errors times |w|, |x|, 2 (P n + 16) u of the sum of magnitudes over n terms, and h of the result."""
import math

import pytest
import torch

from categoricalnf_amd import functional as Fn
from categoricalnf_amd import ops
from categoricalnf_amd.layers.categorical_encoding.decoder import DecoderLinear

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def reference(x, w, t, b, g, ignore=-100):
    """Values and tolerances (without the results' own rounding) in float64 on the GPU; g: [R] gradients of the row losses."""
    P, h = (6, U) if x.dtype == F32 else (1, half_step(x.dtype))
    x, w = x.detach().double().reshape(-1, x.shape[-1]), w.detach().double()
    t, g = t.reshape(-1).long(), g.detach().double().reshape(-1)
    R, H, V = x.shape[0], x.shape[1], w.shape[0]
    keep = t != ignore
    b = torch.zeros(V, dtype=torch.float64, device=x.device) if b is None else b.detach().double()
    l = x @ w.t().contiguous() + b
    mag = x.abs() @ w.abs().t().contiguous()
    e_l = 2 * (P * H + 16) * U * mag + 2 * U * b.abs()
    m = l.max(1, keepdim=True)[0]
    lse = torch.logsumexp(l, 1, keepdim=True)
    p = torch.exp(l - lse)
    rel = (2 * (l - m).abs() + 4) * U
    e_lse = (p * (e_l + rel)).sum(1, keepdim=True) + (V / 8 + 64) * U
    tt = t.clamp(min=0)[:, None]
    own = l.gather(1, tt)
    val = {"loss": torch.where(keep, (lse - own)[:, 0], 0.0)}
    tol = {"loss": torch.where(keep, (e_lse + e_l.gather(1, tt) + 4 * U * ((lse - m).abs() + (m - own).abs()))[:, 0], 0.0)}
    gk = torch.where(keep, g, 0.0)[:, None]
    d = p.scatter_add(1, tt, torch.full_like(own, -1.0)) * gk
    e_d = gk.abs() * p * (e_l + e_lse + rel + 4 * U) + (2 * U + h) * d.abs() + gk.abs() * 2 * U * torch.zeros_like(p).scatter_(1, tt, 1.0)
    if x.dtype and h == half_step(F16):
        e_d = e_d + 2.0 ** -38 * gk.abs().max()
    val.update(dx=d @ w, dw=d.t().contiguous() @ x, db=d.sum(0))
    tol.update(dx=e_d @ w.abs() + 2 * (P * V + 16) * U * (d.abs() @ w.abs()),
               dw=e_d.t().contiguous() @ x.abs() + 2 * (P * R + 16) * U * (d.abs().t().contiguous() @ x.abs()),
               db=e_d.sum(0) + 2 * (P * R + 16) * U * d.abs().sum(0))
    return val, tol


def check(name, got, val, tol):
    got = got.detach()
    ref = val[name].reshape(got.shape)
    bound = tol[name].reshape(got.shape) + half_step(got.dtype) * ref.abs() + torch.finfo(got.dtype).smallest_normal * half_step(got.dtype) * 2
    err = (got.double() - ref).abs()
    # a value that rounds to the type's infinity: from half a step above its largest number on; within `bound` of there either is right
    edge = torch.finfo(got.dtype).max * (1 + half_step(got.dtype) / 2)
    right_inf = torch.isinf(got) & (got.sign() == ref.sign()) & (ref.abs() + bound >= edge)
    bad = ~((err <= bound) | right_inf)
    assert not bad.any(), "%s: %d of %d off, worst error %g, worst ratio %g" % (name, int(bad.sum()), bad.numel(), float(err[bad].max()),
                                                                                 float((err / bound)[bad].max()))


def make(R, V, H, dtype, seed=0, bias=True, ignored=0.2, bias_dtype=None):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, generator=gen, device="cuda")
    x, w = rnd(R, H).to(dtype), (rnd(V, H) * (2 / math.sqrt(H))).to(dtype)
    b = rnd(V).to(bias_dtype or dtype) if bias else None
    t = torch.randint(0, V, (R,), generator=gen, device="cuda")
    t[torch.rand(R, generator=gen, device="cuda") < ignored] = -100
    return x, w, b, t, torch.rand(R, generator=gen, device="cuda") + 0.1


def run_and_check(x, w, b, t, g, ignore=-100):
    leaves = [s.requires_grad_() for s in (x, w, b) if s is not None]
    names = ["dx", "dw"] + (["db"] if b is not None else [])
    loss = Fn.linear_cross_entropy(x, w, t, b, ignore_index=ignore, reduction="none")
    grads = dict(zip(names, torch.autograd.grad(loss, leaves, g.reshape(loss.shape))))
    assert loss.dtype == F32 and loss.shape == t.shape
    val, tol = reference(x, w, t, b, g, ignore)
    check("loss", loss, val, tol)
    for k, v in grads.items():
        assert v.dtype == {"dx": x, "dw": w, "db": b}[k].dtype and v.is_contiguous()
        check(k, v, val, tol)
    ops.check_flags(x.device)
    return loss.detach(), grads


SHAPES = [(1, 1, 1), (1, 2, 1), (2, 1, 3), (3, 5, 7), (1, 300, 40), (64, 51, 64), (100, 27, 64), (129, 257, 65), (127, 1000, 8), (255, 130, 500),
          (513, 700, 128), (300, 1300, 72), (2000, 300, 64), (4099, 51, 64), (40, 5000, 264), (70, 17, 1000), (700, 2, 12), (17, 10007, 33)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_values_and_gradients(shape, dtype):
    run_and_check(*make(*shape, dtype, seed=sum(shape)))


@pytest.mark.parametrize("dtype,shape", [(BF16, (8192, 4100, 64)), (F32, (8192, 4100, 64)), (F16, (8200, 9000, 40)), (BF16, (8192, 600, 1024)),
                                         (BF16, (600, 9000, 1024)), (F32, (3000, 9000, 100)), (F32, (520, 9000, 520))], ids=str)
def test_large_tiles_and_pieces_of_the_vocabulary(shape, dtype):
    run_and_check(*make(*shape, dtype, bias=dtype != BF16))


@pytest.mark.parametrize("dtype,rows", [(BF16, 16500), (F16, 16500), (F32, 8300)])
def test_two_pieces_of_the_vocabulary(dtype, rows):
    """More than 512 MiB of d: the second piece adds to dx and writes its own rows of dw and db."""
    x, w, b, t, g = make(rows, 17000, 136, dtype)
    run_and_check(x, w, b, t, g)


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_without_bias_and_with_an_fp32_bias(dtype):
    run_and_check(*make(150, 90, 48, dtype, bias=False))
    run_and_check(*make(150, 90, 48, dtype, bias_dtype=F32))


@pytest.mark.parametrize("reduction", ["mean", "sum"])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_reductions(reduction, dtype):
    x, w, b, t, _ = make(333, 120, 56, dtype)
    for s in (x, w, b):
        s.requires_grad_()
    loss = Fn.linear_cross_entropy(x, w, t, b, reduction=reduction)
    assert loss.dtype == F32 and loss.shape == ()
    up = torch.tensor(0.7, device="cuda")
    grads = torch.autograd.grad(loss, (x, w, b), up)
    n = int((t != -100).sum())
    share = 1.0 / n if reduction == "mean" else 1.0
    val, tol = reference(x, w, t, b, torch.full((333,), 0.7 * share, dtype=torch.float64, device="cuda"))
    # the sum is taken in 64 bits and rounded once, the mean's gradient is one quotient
    assert abs(loss.item() - float(val["loss"].sum()) * share) <= float(tol["loss"].sum()) * share + U * abs(loss.item()) * 2
    for k, v in zip(("dx", "dw", "db"), grads):
        tol[k] += 2 * U * val[k].abs() * 2
        check(k, v, val, tol)
    with torch.no_grad():
        assert torch.equal(Fn.linear_cross_entropy(x, w, t, b, reduction=reduction), loss)


def test_three_axes_strides_and_int32_targets():
    for dtype in (F32, BF16):
        wide = torch.randn(6, 10, 50, device="cuda").to(dtype)
        ww = torch.randn(40, 60, device="cuda").to(dtype)
        b = torch.randn(40, device="cuda").to(dtype)
        t = torch.randint(0, 40, (6, 10), device="cuda")
        g = torch.rand(60, device="cuda")
        for x, w in ((wide[:, :, :32], ww[:, :32]), (wide[:, :, 1:33], ww[:, 3:35]), (wide[:, :, :32].transpose(0, 1).contiguous().transpose(0, 1), ww[:, ::2][:, :30].repeat(1, 2)[:, :32]),
                     (wide[:, :, ::2][:, :, :24], ww[:, :24])):
            run_and_check(x.detach(), w.detach(), b.detach(), t, g)
        run_and_check(wide[:, :, :32].detach(), ww[:, :32].detach(), b.detach(), t.int(), g)


def test_other_ignore_index_and_all_ignored():
    x, w, b, t, g = make(50, 30, 16, F32, ignored=0.0)
    run_and_check(x, w, b, t, g, ignore=int(t[0]))
    x, w, b, t, g = make(50, 30, 16, F32, ignored=1.1)
    loss, grads = run_and_check(x, w, b, t, g)
    assert not loss.any() and not any(v.any() for v in grads.values())
    mean = Fn.linear_cross_entropy(x, w, t, b)
    assert torch.isnan(mean)
    assert float(Fn.linear_cross_entropy(x, w, t, b, reduction="sum")) == 0.0
    for v in torch.autograd.grad(mean, (x, w, b)):
        assert not v.any()


def test_category_outside_the_vocabulary():
    x, w, b, t, _ = make(20, 30, 16, F32, ignored=0.0)
    clean = Fn.linear_cross_entropy(x, w, t, b, reduction="none")
    for bad in (30, -1, 2 ** 40):
        t2 = t.clone()
        t2[3] = bad
        x.requires_grad_()
        loss = Fn.linear_cross_entropy(x, w, t2, b, reduction="none")
        (gx,) = torch.autograd.grad(loss, x, torch.ones_like(loss))
        with pytest.raises(AssertionError):
            ops.check_flags(x.device)
        ops.check_flags(x.device)
        rest = torch.arange(20, device="cuda") != 3
        assert torch.isnan(loss[3]) and torch.equal(loss[rest], clean[rest]) and not gx[3].any() and gx[rest].any(1).all()


def test_masked_entries_of_the_vocabulary():
    """Entries whose bias is -inf or the type's lowest value have probability 0, also where they fill whole tiles."""
    for low in (-math.inf, torch.finfo(F32).min):
        x, w, b, t, g = make(40, 600, 24, F32, ignored=0.0)
        b[100:420] = low
        t[:] = torch.randint(0, 100, (40,), device="cuda")
        loss, grads = run_and_check_masked(x, w, b, t, g, slice(100, 420))
        assert torch.isfinite(loss).all()


def run_and_check_masked(x, w, b, t, g, gone):
    keep = torch.ones(w.shape[0], dtype=torch.bool, device="cuda")
    keep[gone] = False
    new = torch.cumsum(keep, 0) - 1
    for s in (x, w, b):
        s.requires_grad_()
    loss = Fn.linear_cross_entropy(x, w, t, b, reduction="none")
    dx, dw, db = torch.autograd.grad(loss, (x, w, b), g)
    val, tol = reference(x, w[keep], new[t], b[keep], g)
    tol["loss"] = tol["loss"] + (w.shape[0] / 8) * U
    check("loss", loss, val, tol), check("dx", dx, val, tol), check("dw", dw[keep], val, tol), check("db", db[keep], val, tol)
    assert not dw[gone].any() and not db[gone].any()
    return loss, (dx, dw, db)


def test_rows_that_are_not_finite_stay_alone():
    x, w, b, t, g = make(30, 200, 40, F32, ignored=0.0)
    clean = Fn.linear_cross_entropy(x, w, t, b, reduction="none")
    x2 = x.clone()
    x2[4, 3], x2[9, 0] = float("nan"), float("inf")
    loss = Fn.linear_cross_entropy(x2, w, t, b, reduction="none")
    rest = torch.ones(30, dtype=torch.bool, device="cuda")
    rest[[4, 9]] = False
    assert not torch.isfinite(loss[~rest]).any() and torch.equal(loss[rest], clean[rest])


@pytest.mark.parametrize("shape", [(200, 300, 40), (150, 700, 200), (1100, 700, 64)], ids=str)
def test_rows_of_very_different_sizes(shape):
    """fp32 operands are split after a scaling: a row's loss and gradient do not suffer from larger rows beside it.  dweight adds rows
    of all sizes: each of them, and its d, is kept to 2^-39 of the largest, so that R products are off by 2^-38 max|g| max|x| each."""
    x, w, b, t, g = make(*shape, F32)
    x = x * 10.0 ** torch.linspace(-3, 12, shape[0], device="cuda")[torch.randperm(shape[0], device="cuda")][:, None]
    for v in (x, w, b):
        v.requires_grad_()
    loss = Fn.linear_cross_entropy(x, w, t, b, reduction="none")
    grads = torch.autograd.grad(loss, (x, w, b), g)
    val, tol = reference(x, w, t, b, g)
    tol["dw"] = tol["dw"] + shape[0] * 2.0 ** -38 * float(g.max()) * float(x.detach().abs().max())
    for name, got in zip(("loss", "dx", "dw", "db"), (loss,) + grads):
        check(name, got, val, tol)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("shape", [(70, 51, 64), (300, 300, 40), (300, 600, 200)], ids=str)
def test_what_ignored_rows_hold_does_not_matter(shape, dtype):
    """The bits of a call whose ignored rows are zeros; in fp32 (whose rows are laid out anew) also with infinities and NaN in them."""
    x, w, b, t, g = make(*shape, dtype)
    gone = (t == -100).nonzero()[:, 0]
    def run(fills):
        x2 = x.detach().clone()
        for i, r in enumerate(gone.tolist()):
            x2[r] = fills[i % len(fills)]
        x2.requires_grad_()
        leaves = (x2, w.detach().requires_grad_(), b.detach().requires_grad_())
        loss = Fn.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction="none")
        return (loss.detach(),) + torch.autograd.grad(loss, leaves, g)
    clean = run([0.0])
    fills = [1e30, -3e38, 0.0] + ([math.inf, math.nan] if dtype == F32 else [])
    for a, c in zip(run(fills), clean):
        assert torch.equal(a, c)


@pytest.mark.parametrize("reduction", ["mean", "sum", "none"])
def test_the_loss_may_be_changed_in_place(reduction):
    x, w, b, t, _ = make(30, 40, 16, F32)
    grads = []
    for inplace in (False, True):
        leaves = [v.detach().clone().requires_grad_() for v in (x, w, b)]
        loss = Fn.linear_cross_entropy(leaves[0], leaves[1], t, leaves[2], reduction=reduction)
        assert loss._base is None
        if inplace:
            loss /= 4
        else:
            loss = loss / 4
        loss.sum().backward()
        grads.append([v.grad for v in leaves])
    assert all(torch.equal(a, c) for a, c in zip(*grads))


@pytest.mark.parametrize("vocab", [2 ** 24 - 1, 2 ** 24 + 3])
def test_vocabularies_around_2_to_the_24(vocab):
    """The most classes whose index shares a word with a row's shift, and more; targets at both ends."""
    x, w, b, t, g = make(5, vocab, 8, BF16, ignored=0.0)
    t[0], t[1], t[2] = vocab - 1, 0, -100
    run_and_check(x, w, b, t, g)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_a_million_features(dtype):
    run_and_check(*make(3, 5, 2 ** 20 + 8, dtype, ignored=0.0))


def test_more_elements_than_2_to_the_31():
    """Rows whose elements lie beyond 2^31 give what they give at the front."""
    H, V, n = 64, 51, 3000
    R = 2 ** 31 // H + n
    small, w, b, t, _ = make(n, V, H, BF16)
    x = torch.zeros(R, H, dtype=BF16, device="cuda")
    x[-n:] = small
    target = torch.full((R,), -100, device="cuda")
    target[-n:] = t
    x.requires_grad_(), w.requires_grad_(), b.requires_grad_()
    loss = Fn.linear_cross_entropy(x, w, target, b, reduction="sum")
    (dx, dw, db) = torch.autograd.grad(loss, (x, w, b))
    val, tol = reference(small, w, t, b, torch.ones(n, device="cuda"))
    tol["dw"] = tol["dw"] * (1 + R / n)          # the reference's count of additions: n rows, here R
    tol["db"] = tol["db"] * (1 + R / n)
    assert abs(float(loss.detach()) - float(val["loss"].sum())) <= float(tol["loss"].sum()) + U * float(val["loss"].sum())
    check("dx", dx[-n:], val, tol), check("dw", dw, val, tol), check("db", db, val, tol)
    assert not dx[:-n].any()


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_large_logits(dtype):
    """Logits of some thousands: the maximum is taken out before the exponential; certain rows have loss 0 and gradient 0."""
    x, w, b, t, g = make(64, 100, 32, dtype)
    run_and_check((x * 300).detach(), (w * 3).detach(), b, t, g)
    w1 = torch.zeros(10, 16, device="cuda", dtype=dtype)
    w1[3] = 100
    x1 = torch.ones(5, 16, device="cuda", dtype=dtype)
    loss, grads = run_and_check(x1, w1, None, torch.full((5,), 3, device="cuda"), torch.ones(5, device="cuda"))
    assert not loss.any() and not grads["dx"].any()


def test_small_upstream_gradients_in_fp16():
    """The mean of many rows: gradients of 1e-7 per row would vanish in fp16 without the power of two."""
    x, w, b, t, g = make(300, 400, 64, F16)
    run_and_check(x, w, b, t, g * 1e-7)
    run_and_check(x, w, b, t, g * 1e6)


def test_fp32_at_the_ends_of_its_range():
    """The split into three bf16 parts at magnitudes where a part could overflow or vanish."""
    x, w, b, t, g = make(40, 50, 16, F32)
    run_and_check((x * 1e30).detach(), (w * 1e-30).detach(), b, t, g * 1e-3)
    big = torch.full((4, 8), torch.finfo(F32).max, device="cuda")
    small = torch.full((6, 8), 1e-38, device="cuda") * torch.arange(1, 7, device="cuda")[:, None]
    loss = Fn.linear_cross_entropy(big, small, torch.zeros(4, dtype=torch.long, device="cuda"), reduction="none")
    ref = torch.nn.functional.cross_entropy(big.double() @ small.double().t(), torch.zeros(4, dtype=torch.long, device="cuda"), reduction="none")
    # 1e-38 is below 2^-126: its lower parts may be cut at 2^-133, 2^-7 of the value and 2^-7 of logits of up to 163
    assert (loss.double() - ref).abs().max() <= 2.0 ** -7 * 2 * 163.4


def test_gradients_against_differences():
    x, w, b, t, g = make(12, 40, 20, F32, ignored=0.2)
    _, grads = run_and_check(x, w, b, t, g)
    gen = torch.Generator(device="cuda").manual_seed(5)
    dirs = [torch.randn(s.shape, generator=gen, device="cuda", dtype=torch.float64) for s in (x, w, b)]

    def f(s):
        l = torch.nn.functional.linear(*[(p.detach().double() + s * q) for p, q in zip((x, w, b), dirs)])
        each = torch.nn.functional.cross_entropy(l, t, ignore_index=-100, reduction="none")
        return float((each * g.double()).sum())
    slope = (f(1e-5) - f(-1e-5)) / 2e-5
    mine = sum(float((grads[k].double() * q).sum()) for k, q in zip(("dx", "dw", "db"), dirs))
    _, tol = reference(x, w, t, b, g)
    # the quotient: t^2 / 6 f''' (f''' is some hundreds here) + eps f / t, below 1e-7 |f| + 1e-7
    bound = sum(float(((tol[k] + U * grads[k].double().abs()) * q.abs()).sum()) for k, q in zip(("dx", "dw", "db"), dirs))
    assert abs(slope - mine) <= bound + 1e-7 * (1 + abs(f(0.0)))


def test_only_some_gradients():
    x, w, b, t, g = make(60, 70, 40, BF16)
    _, full = run_and_check(x, w, b, t, g)
    for want in ((True, False, False), (False, True, False), (False, False, True), (True, False, True)):
        ls = [s.detach().requires_grad_(q) for s, q in zip((x, w, b), want)]
        loss = Fn.linear_cross_entropy(ls[0], ls[1], t, ls[2], reduction="none")
        got = torch.autograd.grad(loss, [s for s, q in zip(ls, want) if q], g)
        for k, v in zip([k for k, q in zip(("dx", "dw", "db"), want) if q], got):
            assert torch.equal(v, full[k])


def test_no_rows():
    w, b = torch.randn(7, 4, device="cuda", requires_grad=True), torch.randn(7, device="cuda", requires_grad=True)
    x = torch.zeros(0, 4, device="cuda", requires_grad=True)
    t = torch.zeros(0, dtype=torch.long, device="cuda")
    loss = Fn.linear_cross_entropy(x, w, t, b, reduction="none")
    gx, gw, gb = torch.autograd.grad(loss, (x, w, b), torch.zeros(0, device="cuda"))
    assert loss.shape == (0,) and gx.shape == (0, 4) and not gw.any() and not gb.any()
    assert torch.isnan(Fn.linear_cross_entropy(x, w, t, b))


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_same_bits_on_every_run_and_on_another_stream(dtype):
    x, w, b, t, g = make(1500, 900, 96, dtype)
    loss, first = run_and_check(x, w, b, t, g)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        ls = [s.detach().requires_grad_() for s in (x, w, b)]
        again = Fn.linear_cross_entropy(ls[0], ls[1], t, ls[2], reduction="none")
        second = torch.autograd.grad(again, ls, g)
    torch.cuda.synchronize()
    assert torch.equal(loss, again)
    for p, q in zip(first.values(), second):
        assert torch.equal(p, q)


@pytest.mark.parametrize("dtype,shape", [(F32, (300, 51, 64)), (BF16, (257, 500, 72)), (F16, (130, 900, 30))])
def test_captured_step_replays(dtype, shape):
    x, w, b, t, _ = make(*shape, dtype)
    xs, ws, bs = (s.clone().requires_grad_() for s in (x, w, b))
    ts = t.clone()

    def step(x, w, b, t):
        loss = Fn.linear_cross_entropy(x, w, t, b)
        return (loss.detach(),) + torch.autograd.grad(loss, (x, w, b))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(xs, ws, bs, ts)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(xs, ws, bs, ts)
    for seed in range(1, 5):
        x1, w1, b1, t1, _ = make(*shape, dtype, seed=seed)
        with torch.no_grad():
            xs.copy_(x1), ws.copy_(w1), bs.copy_(b1), ts.copy_(t1)
        graph.replay()
        torch.cuda.synchronize()
        for p, q in zip(out, step(x1.requires_grad_(), w1.requires_grad_(), b1.requires_grad_(), t1)):
            assert torch.equal(p, q)


def test_refusals_on_the_gpu():
    x, w, b, t, _ = make(10, 20, 8, F32)
    ce = Fn.linear_cross_entropy
    for args, kind in (((x, w[:, :7], t, b), ValueError), ((x, w, t[:9], b), ValueError), ((x, w, t, b[:19]), ValueError), ((x, w.half(), t, b), TypeError),
                       ((x.double(), w.double(), t, None), TypeError), ((x, w, t.float(), b), TypeError), ((x, w.cpu(), t, b), ops.HipOnlyError),
                       ((x, w, t.cpu(), b), ops.HipOnlyError), ((x, w, t, b.half()), TypeError), ((x[:, :0], w[:, :0], t, b), ValueError),
                       ((x, w[:0], t, None), ValueError), ((x, w[0], t, None), ValueError)):
        with pytest.raises(kind):
            ce(*args)
    with pytest.raises(ValueError):
        ce(x, w, t, b, reduction="max")
    x.requires_grad_()
    (g,) = torch.autograd.grad(ce(x, w, t, b), x, create_graph=True)
    with pytest.raises(RuntimeError):
        g.sum().backward()


def test_decoder_under_autocast():
    torch.manual_seed(0)
    dec = DecoderLinear(num_categories=30, embed_dim=5, hidden_size=64, num_layers=1).cuda()
    z, c = torch.randn(200, 5, device="cuda"), torch.randint(0, 30, (200,), device="cuda")
    ref = dec.class_log_prob(z, c)
    with torch.autocast("cuda", dtype=BF16):
        out = dec.class_log_prob(z, c)
    grads = torch.autograd.grad(out.sum(), dec.parameters())
    # the products before the last are of bf16 operands with bf16 results: the features, two weights and two results round by 2^-8 of
    # what is summed, each; a feature of the hidden layer is at most a sum of such, and a log-probability moves by at most twice a logit
    with torch.no_grad():
        h = dec._features(z).abs()
        for m in list(dec.layers.inp_layer.modules()) + list(dec.layers.main_net.modules()):
            if isinstance(m, torch.nn.Linear):
                h = h @ m.weight.abs().t() + m.bias.abs()
    assert out.dtype == F32 and bool(((out - ref).abs() <= 2 * 6 * 2.0 ** -8 * h.max(-1)[0]).all())
    assert all(bool(torch.isfinite(g).all()) for g in grads)


def test_decoder_ignores_no_category():
    dec = DecoderLinear(num_categories=30, embed_dim=5, hidden_size=64, num_layers=1).cuda()
    z, c = torch.randn(8, 5, device="cuda"), torch.randint(0, 30, (8,), device="cuda")
    for bad in (-100, -1, 30):
        c[3] = bad
        with torch.no_grad():
            out = dec.class_log_prob(z, c)
        with pytest.raises(AssertionError):
            ops.check_flags(z.device)
        assert torch.isnan(out[3]) and torch.isfinite(out[:3]).all()


@pytest.mark.parametrize("num_layers", [0, 1, 2])
def test_decoder_scores_one_class_without_the_others(num_layers):
    """DecoderLinear.class_log_prob: the gathered entry of forward()'s log-softmax, and its gradients."""
    torch.manual_seed(0)
    dec = DecoderLinear(num_categories=300, embed_dim=5, hidden_size=64, num_layers=num_layers).cuda()
    z = torch.randn(40, 3, 5, device="cuda")
    c = torch.randint(0, 300, (40, 3), device="cuda")
    ref = dec(z).gather(-1, c[..., None])[..., 0]
    got = dec.class_log_prob(z, c)
    torch.testing.assert_close(got, ref, rtol=2e-6, atol=2e-5)
    ga = torch.autograd.grad(ref.sum(), dec.parameters())
    gb = torch.autograd.grad(got.sum(), dec.parameters())
    for p, q in zip(ga, gb):
        torch.testing.assert_close(q, p, rtol=1e-4, atol=1e-5 * float(p.abs().max()) + 1e-7)
