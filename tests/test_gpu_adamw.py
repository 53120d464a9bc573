"""AdamW over lists of tensors (ops.adamw_step, optim.AdamW), moments in 32 and in 8 bits.

The oracle of the arithmetic is the same chain of fp32 operations in numpy on the CPU (IEEE sums, products, quotients and square
roots: equal bits), which is itself held against the definition in 64 bits: with u = 2^-24 each of m and v is off by at most
3 u (|b m| + |(1 - b) g|), (4 u for v: the square), the step by the relative errors of m, v (half), and 6 roundings, p by two more."""
import math

import numpy as np
import pytest
import torch

from categoricalnf_amd import ops
from categoricalnf_amd.optim import AdamW

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
B1, B2, EPS = 0.9, 0.999, 1e-8
DT = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
f32 = np.float32


def blocks(a):
    return np.concatenate([a, np.zeros(-len(a) % 256, a.dtype)]).reshape(-1, 256)


def encode_m(m):
    b = blocks(m)
    with np.errstate(all="ignore"):
        s = np.abs(b).max(1) * f32(1.0 / 16129)
        s = np.where(np.isfinite(s), s, f32("nan")).astype(f32)
        q = np.minimum(np.rint(np.sqrt(np.abs(b) / s[:, None])), 127)
        q = np.where(s[:, None] > 0, q, 0) * np.sign(np.nan_to_num(b))
    return q.astype(np.int8).reshape(-1)[:len(m)], s


def encode_v(v):
    r = np.sqrt(blocks(v))
    with np.errstate(all="ignore"):
        s = r.max(1) * f32(1.0 / 65025)
        s = np.where(np.isfinite(s), s, f32("nan")).astype(f32)
        q = np.clip(np.rint(np.sqrt(r / s[:, None])), 1, 255)
        q = np.where((s[:, None] > 0) & (r > 0), q, 0)
    return q.astype(np.uint8).reshape(-1)[:len(v)], s


def decode_m(q, s):
    f = blocks(q).astype(f32)
    with np.errstate(all="ignore"):
        return ((f * np.abs(f)) * s[:, None]).reshape(-1)[:len(q)]


def decode_v(q, s):
    f = blocks(q).astype(f32)
    with np.errstate(all="ignore"):
        r = (f * f) * s[:, None]
        return (r * r).reshape(-1)[:len(q)]


def chain(p, g, m, v, step, lr, decay):
    """One step in fp32, each operation rounded once: (p, m, v)."""
    c = {k: f32(x) for k, x in (("b1", B1), ("c1", 1 - B1), ("b2", B2), ("c2", 1 - B2), ("eps", EPS), ("keep", 1 - lr * decay),
                                ("size", lr / (1 - B1 ** step)), ("root", 1 / math.sqrt(1 - B2 ** step)))}
    with np.errstate(all="ignore"):
        m = m * c["b1"] + g * c["c1"]
        v = v * c["b2"] + (g * g) * c["c2"]
        p = p * c["keep"] - m / (np.sqrt(v) * c["root"] + c["eps"]) * c["size"]
    assert p.dtype == m.dtype == v.dtype == f32
    return p, m, v


def flat(t):
    return t.detach().float().cpu().numpy().reshape(-1)


class Tensors:
    """Lists of tensors on the GPU and their numpy twins."""

    def __init__(self, sizes, pdtype="f32", gdtype=None, bits=32, seed=0, offset=0):
        gen = torch.Generator().manual_seed(seed)
        self.bits, self.pdtype, self.offset = bits, DT[pdtype], offset
        mk = lambda n, s, dt: self.place((torch.randn(n, generator=gen) * s).to(dt))
        self.p = [mk(n, 0.1, DT[pdtype]) for n in sizes]
        self.g = [mk(n, 10.0 ** (-i % 5 - 3), DT[gdtype or pdtype]) for i, n in enumerate(sizes)]
        m = [0.5 * flat(g) for g in self.g]
        v = [flat(g) ** 2 * f32(0.3) for g in self.g]
        if bits == 32:
            self.m, self.v = [self.place(torch.from_numpy(a)) for a in m], [self.place(torch.from_numpy(a)) for a in v]
            self.ms = self.vs = None
        else:
            em, ev = [encode_m(a) for a in m], [encode_v(a) for a in v]
            self.m, self.v = [self.place(torch.from_numpy(q)) for q, _ in em], [self.place(torch.from_numpy(q)) for q, _ in ev]
            self.ms, self.vs = [torch.from_numpy(s).cuda() for _, s in em], [torch.from_numpy(s).cuda() for _, s in ev]

    def place(self, t):
        """On the GPU, `offset` elements into a buffer of its own: offset 1 is an address that no vector access may take."""
        buf = torch.zeros(t.numel() + self.offset, dtype=t.dtype, device="cuda")
        buf[self.offset:].copy_(t)
        return buf[self.offset:]

    def host(self):
        if self.bits == 32:
            return [(flat(p), flat(g), flat(m), flat(v)) for p, g, m, v in zip(self.p, self.g, self.m, self.v)]
        return [(flat(p), flat(g), decode_m(m.cpu().numpy(), ms.cpu().numpy()), decode_v(v.cpu().numpy(), vs.cpu().numpy()))
                for p, g, m, v, ms, vs in zip(self.p, self.g, self.m, self.v, self.ms, self.vs)]

    def step(self, step=5, lr=1e-3, decay=0.02):
        ops.adamw_step(self.p, self.g, self.m, self.v, step=step, lr=lr, beta1=B1, beta2=B2, eps=EPS, weight_decay=decay,
                       exp_avg_scales=self.ms, exp_avg_sq_scales=self.vs)

    def check(self, before, step=5, lr=1e-3, decay=0.02):
        for i, (p, g, m, v) in enumerate(before):
            cp, cm, cv = chain(p, g, m, v, step, lr, decay)
            assert np.array_equal(flat(self.p[i]), torch.from_numpy(cp).to(self.pdtype).float().numpy(), equal_nan=True), i
            if self.bits == 32:
                assert np.array_equal(flat(self.m[i]), cm, equal_nan=True) and np.array_equal(flat(self.v[i]), cv, equal_nan=True), i
            else:
                (qm, sm), (qv, sv) = encode_m(cm), encode_v(cv)
                assert np.array_equal(self.m[i].cpu().numpy(), qm) and np.array_equal(self.ms[i].cpu().numpy(), sm, equal_nan=True), i
                assert np.array_equal(self.v[i].cpu().numpy(), qv) and np.array_equal(self.vs[i].cpu().numpy(), sv, equal_nan=True), i


SIZES = [1, 2, 3, 4, 5, 255, 256, 257, 1000, 4095, 4096, 4097, 8192, 100003]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("pdtype,gdtype", [("f32", None), ("bf16", None), ("f16", None), ("bf16", "f32"), ("f16", "f32")])
@pytest.mark.parametrize("offset", [0, 1])
def test_step_is_the_chain_of_operations(bits, pdtype, gdtype, offset):
    t = Tensors(SIZES, pdtype, gdtype, bits, offset=offset)
    before = t.host()
    t.step()
    t.check(before)
    before = t.host()
    t.step(step=6)
    t.check(before, step=6)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [69, 70, 71, 97, 98, 99, 140, 141, 196, 197])
def test_tensor_counts_around_a_launch(bits, count):
    t = Tensors([(37 * i) % 700 + 1 for i in range(count)], bits=bits, seed=count)
    before = t.host()
    t.step()
    t.check(before)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 55, 56, 57, 64, 65, 79, 80, 81, 500])
def test_tensor_counts(bits, count):
    t = Tensors([(37 * i) % 700 + 1 for i in range(count)], bits=bits, seed=count)
    before = t.host()
    t.step()
    t.check(before)


def test_empty_tensors_and_lists():
    ops.adamw_step([], [], [], [], step=1, lr=1e-3)
    t = Tensors([0, 5, 0, 300, 0])
    before = t.host()
    t.step()
    t.check(before)
    t = Tensors([0, 0])
    t.step()


def test_chain_against_64_bits():
    t = Tensors([5000], seed=3)
    (p, g, m, v), = [tuple(a.astype(np.float64) for a in h) for h in t.host()]
    step, lr, decay = 7, 2e-3, 0.05
    t.step(step=step, lr=lr, decay=decay)
    m64, v64 = B1 * m + (1 - B1) * g, B2 * v + (1 - B2) * g * g
    upd = lr / (1 - B1 ** step) * m64 / (np.sqrt(v64) / math.sqrt(1 - B2 ** step) + EPS)
    tm, tv = 3 * U * (np.abs(B1 * m) + np.abs((1 - B1) * g)), 4 * U * v64
    assert (np.abs(flat(t.m[0]) - m64) <= tm).all() and (np.abs(flat(t.v[0]) - v64) <= tv).all()
    rel = tm / np.maximum(np.abs(m64), 1e-300) + 0.5 * tv / v64 + 6 * U
    tp = np.abs(upd) * rel + 3 * U * (np.abs(p) + np.abs(upd))
    assert (np.abs(flat(t.p[0]) - (p * (1 - lr * decay) - upd)) <= tp).all()


def test_8_bit_grid():
    """Codes back to values: m to half a step of its grid, sqrt(v) too, and no positive second moment becomes zero.  A step of
    q^2 at value x of largest X is at most 2 sqrt(x X) / n + X / n^2 wide, n = 127 or 255."""
    t = Tensors([4096], bits=8, seed=5)
    with torch.no_grad():
        t.g[0].mul_(torch.exp(3 * torch.randn(4096, device="cuda")))
    (p, g, m, v), = t.host()
    t.step()
    _, cm, cv = chain(p, g, m, v, 5, 1e-3, 0.02)
    gm, gv = ops.adamw_moments(t.m[0], t.v[0], t.ms[0], t.vs[0])
    assert np.array_equal(flat(gm), decode_m(t.m[0].cpu().numpy(), t.ms[0].cpu().numpy()))
    assert np.array_equal(flat(gv), decode_v(t.v[0].cpu().numpy(), t.vs[0].cpu().numpy()))
    for got, want, n in ((np.abs(flat(gm)), np.abs(cm), 127), (np.sqrt(flat(gv)), np.sqrt(cv), 255)):
        top = blocks(want).max(1).repeat(256)
        half = (2 * np.sqrt(want * top) / n + top / n ** 2) / 2
        floor = top / n ** 2 if n == 255 else 0.0        # sqrt(v) below half the first step is raised to it
        assert (np.abs(got - want) <= half * (1 + 1e-5) + floor).all()
    assert (flat(gv)[cv > 0] > 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_nonfinite_gradients(bits):
    t = Tensors([1000, 1000], bits=bits)
    with torch.no_grad():
        t.g[0][3], t.g[0][300], t.g[0][700] = float("nan"), float("inf"), 3e19      # 3e19^2 overflows
    before = t.host()
    t.step()
    t.check(before)
    before = t.host()
    t.step(step=6)
    t.check(before, step=6)
    assert np.isfinite(flat(t.p[1])).all()


def test_zero_gradients_and_zero_state():
    for bits in (32, 8):
        t = Tensors([600], bits=bits)
        with torch.no_grad():
            for l in (t.g, t.m, t.v) + ((t.ms, t.vs) if bits == 8 else ()):
                l[0].zero_()
        before = t.host()
        t.step(step=1)
        t.check(before, step=1)
        assert np.isfinite(flat(t.p[0])).all()


def test_values_of_step_and_lr_on_the_device():
    """lr and the step count read from device scalars: the constants come from exp2 instead of pow, so size and root may differ by
    a step of fp32 (2 u relative each) from the host's."""
    for step in (1, 2, 1000, 200000):
        a, b = Tensors([5000], seed=step), Tensors([5000], seed=step)
        a.step(step=step)
        p0 = flat(b.p[0])
        b.step(step=torch.tensor(float(step), device="cuda"), lr=torch.tensor(1e-3, device="cuda"))
        # the device's lr is fp32(1e-3): relative 2^-24 on the step and on lr wd
        pa, pb = flat(a.p[0]).astype(np.float64), flat(b.p[0]).astype(np.float64)
        assert (np.abs(pa - pb) <= 8 * U * np.abs(pa - p0) + 3 * U * np.abs(pa) + 8 * U * 1e-3).all()
        assert torch.equal(a.m[0], b.m[0]) and torch.equal(a.v[0], b.v[0])


# ---- the optimiser -----------------------------------------------------------------------------------------------------------

def net(seed=0, dtype=torch.float32):
    torch.manual_seed(seed)
    return torch.nn.Sequential(torch.nn.Linear(70, 90), torch.nn.Tanh(), torch.nn.Linear(90, 3)).cuda().to(dtype)


def set_grads(model, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)
    for p in model.parameters():
        p.grad = torch.randn(p.shape, generator=gen, device="cuda").to(p.dtype) * 0.1


def test_optimiser_follows_torch():
    """30 steps next to torch.optim.AdamW: each step's update agrees to some 10 u of its size (lr at most), so the parameters do to
    30 * 16 u * lr plus 30 roundings of a value."""
    a, b = net(), net()
    mine, ref = AdamW(a.parameters(), lr=1e-2, weight_decay=0.1), torch.optim.AdamW(b.parameters(), lr=1e-2, weight_decay=0.1)
    for i in range(30):
        set_grads(a, i), set_grads(b, i)
        mine.step(), ref.step()
    for p, q in zip(a.parameters(), b.parameters()):
        d = (p - q).abs().double()
        assert (d <= 30 * 16 * U * 1e-2 * 4 + 30 * 2 * U * q.abs().double()).all()
        m, v = mine.moments(p)
        torch.testing.assert_close(m, ref.state[q]["exp_avg"], rtol=1e-5, atol=1e-7)
        torch.testing.assert_close(v, ref.state[q]["exp_avg_sq"], rtol=1e-5, atol=1e-9)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits, dtype):
    a = net(dtype=dtype)
    opt = AdamW(a.parameters(), lr=1e-2, state_bits=bits, min_8bit_size=256)
    for i in range(3):
        set_grads(a, i)
        opt.step()
    b = net(1, dtype)
    b.load_state_dict(a.state_dict())
    new = AdamW(b.parameters(), lr=5.0, state_bits=bits)
    new.load_state_dict(opt.state_dict())
    for p, q in zip(a.parameters(), b.parameters()):
        assert set(opt.state[p]) == set(new.state[q])
        for k, t in opt.state[p].items():
            assert t.dtype == new.state[q][k].dtype and torch.equal(t, new.state[q][k]), k
    for i in range(3, 6):
        set_grads(a, i), set_grads(b, i)
        opt.step(), new.step()
    for p, q in zip(a.parameters(), b.parameters()):
        assert torch.equal(p, q)
    if bits == 8:
        assert opt.state[a[0].weight]["exp_avg"].dtype == torch.int8 and opt.state[a[2].bias]["exp_avg"].dtype == torch.float32


def test_checkpoint_of_torch_adamw():
    a, b = net(), net()
    ref = torch.optim.AdamW(a.parameters(), lr=1e-2)
    for i in range(3):
        set_grads(a, i)
        ref.step()
    b.load_state_dict(a.state_dict())
    mine = AdamW(b.parameters(), lr=1e-2)
    mine.load_state_dict(ref.state_dict())
    set_grads(a, 9), set_grads(b, 9)
    ref.step(), mine.step()
    for p, q in zip(a.parameters(), b.parameters()):
        torch.testing.assert_close(p, q, rtol=4 * U, atol=64 * U * 1e-2)
        assert float(mine.state[q]["step"]) == 4


def test_parameters_without_gradients_do_not_count_steps():
    a = net()
    opt = AdamW(a.parameters(), lr=1e-2)
    set_grads(a, 0)
    opt.step()
    set_grads(a, 1)
    a[0].weight.grad = None
    w = a[0].weight.detach().clone()
    opt.step()
    assert torch.equal(w, a[0].weight) and float(opt.state[a[0].weight]["step"]) == 1 and float(opt.state[a[2].weight]["step"]) == 2
    set_grads(a, 2)
    opt.step()
    assert float(opt.state[a[0].weight]["step"]) == 2 and float(opt.state[a[2].weight]["step"]) == 3


def test_captured_step_replays_with_a_schedule():
    a, b = net(), net()
    lr = torch.tensor(1e-2, device="cuda")
    opt = AdamW(a.parameters(), lr=lr, capturable=True, state_bits=8, min_8bit_size=256)
    ref = AdamW(b.parameters(), lr=lr.clone(), capturable=True, state_bits=8, min_8bit_size=256)
    grads = [torch.zeros_like(p) for p in a.parameters()]
    for p, g in zip(a.parameters(), grads):
        p.grad = g
    set_b = lambda: [setattr(q, "grad", g.clone()) for q, g in zip(b.parameters(), grads)]
    fill = lambda i: [g.normal_(generator=torch.Generator(device="cuda").manual_seed(100 * i + k)) for k, g in enumerate(grads)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fill(0)
        opt.step()
    torch.cuda.current_stream().wait_stream(side)
    set_b()
    ref.step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    for i in range(1, 6):
        fill(i)
        lr.fill_(1e-2 / i)
        ref.param_groups[0]["lr"].fill_(1e-2 / i)
        graph.replay()
        set_b()
        ref.step()
        torch.cuda.synchronize()
        for p, q in zip(a.parameters(), b.parameters()):
            assert torch.equal(p, q), i
            assert all(torch.equal(t, ref.state[q][k]) for k, t in opt.state[p].items())
    assert float(opt.state[a[0].weight]["step"]) == 6


def test_on_another_stream():
    t, r = Tensors([100003]), Tensors([100003])
    r.step()
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        t.step()
    torch.cuda.synchronize()
    assert torch.equal(t.p[0], r.p[0]) and torch.equal(t.v[0], r.v[0])


@pytest.mark.parametrize("optimizer", ["adamw", "adamw8"])
@pytest.mark.parametrize("graph_step", [False, True])
def test_driver_trains_checkpoints_and_resumes(optimizer, graph_step, tmp_path):
    """--optimizer of the set-modelling driver: eager and captured steps, a checkpoint, a resumed run."""
    from categoricalnf_amd.experiments import run_set_modeling as rs
    common = ["--optimizer", optimizer, "--batch_size", "16", "--eval_freq", "6", "--coupling_num_flows", "2", "--coupling_hidden_size", "64",
              "--checkpoint_path", str(tmp_path)] + (["--graph_step"] if graph_step else [])
    first = rs.main(common + ["--max_iterations", "6"])
    second = rs.main(common + ["--max_iterations", "12"])
    assert math.isfinite(first["val_bpd"]) and math.isfinite(second["val_bpd"])


@pytest.mark.parametrize("bits", [32, 8])
def test_more_elements_than_2_to_the_31(bits):
    n, tail = 2 ** 31 + 5120, 7168           # whole blocks of 256, so that the tail alone has the same blocks
    p, g = torch.zeros(n, dtype=torch.bfloat16, device="cuda"), torch.zeros(n, dtype=torch.bfloat16, device="cuda")
    types = (torch.float32, torch.float32) if bits == 32 else (torch.int8, torch.uint8)
    m, v = (torch.zeros(n, dtype=t, device="cuda") for t in types)
    g[-tail:].normal_()
    scales = [torch.zeros(n // 256, device="cuda") for _ in range(2)] if bits == 8 else []
    small = [t[-tail:].clone() for t in (p, g, m, v)] + [s[-(tail // 256):].clone() for s in scales]
    def step(p, g, m, v, *s):
        ops.adamw_step([p], [g], [m], [v], step=1, lr=1e-2, exp_avg_scales=[s[0]] if s else None, exp_avg_sq_scales=[s[1]] if s else None)
    step(p, g, m, v, *scales)
    step(*small)
    for a, b in zip([p, m, v] + scales, [small[0]] + small[2:]):
        assert torch.equal(a[-b.numel():], b) and not a[:-b.numel()].any()


def test_refusals():
    t = Tensors([300, 40])
    call = lambda **kw: ops.adamw_step(kw.get("p", t.p), kw.get("g", t.g), kw.get("m", t.m), kw.get("v", t.v), step=kw.get("step", 1),
                                       lr=kw.get("lr", 1e-3), beta1=kw.get("beta1", 0.9), exp_avg_scales=kw.get("ms"), exp_avg_sq_scales=kw.get("vs"))
    before = [x.clone() for x in t.p]
    for bad, kind in ((dict(g=t.g[:1]), ValueError), (dict(p=[t.p[0], t.p[0]], g=[t.g[0]] * 2, m=[t.m[0]] * 2, v=[t.v[0]] * 2), ValueError),
                      (dict(p=[t.p[0], t.p[1].double()]), ValueError), (dict(m=[t.m[0], t.m[0]]), ValueError), (dict(step=0), ValueError),
                      (dict(beta1=1.0), ValueError), (dict(ms=[1]), ValueError), (dict(g=[g.half() for g in t.g]), TypeError),
                      (dict(p=[t.p[0].cpu(), t.p[1].cpu()]), ops.HipOnlyError), (dict(g=[t.g[0], t.g[1].cpu()]), ValueError),
                      (dict(lr=torch.tensor(1e-3)), ValueError), (dict(step=torch.tensor(1, device="cuda")), ValueError),
                      (dict(m=t.v), ValueError), (dict(p=t.m), ValueError), (dict(m=[t.p[0], t.m[1]]), ValueError),
                      (dict(v=[t.v[0].double(), t.v[1]]), ValueError), (dict(ms=[t.m[0], t.m[1]], vs=[t.v[0], t.v[1]]), ValueError)):
        with pytest.raises(kind):
            call(**bad)
    for x, y in zip(t.p, before):
        assert torch.equal(x, y)
    # 8-bit moments whose scales are shared: between two tensors, and between the two moments
    p, g = [torch.zeros(40, device="cuda") for _ in range(2)], [torch.ones(40, device="cuda") for _ in range(2)]
    m, v = [torch.zeros(40, dtype=torch.int8, device="cuda") for _ in range(2)], [torch.zeros(40, dtype=torch.uint8, device="cuda") for _ in range(2)]
    s = [torch.zeros(1, device="cuda") for _ in range(4)]
    for ms, vs in (([s[0], s[0]], s[2:]), (s[:2], [s[2], s[2]]), (s[:2], s[1:3])):
        with pytest.raises(ValueError):
            call(p=p, g=g, m=m, v=v, ms=ms, vs=vs)
    call(p=p, g=g, m=m, v=v, ms=s[:2], vs=s[2:])
    w = torch.nn.Parameter(torch.randn(6, 4, device="cuda").t())
    opt = AdamW([w])
    w.grad = torch.randn(4, 6, device="cuda")
    with pytest.raises(ValueError):
        opt.step()
    e = torch.nn.Embedding(5, 3, sparse=True).cuda()
    opt = AdamW(e.parameters())
    e(torch.tensor([1], device="cuda")).sum().backward()
    with pytest.raises(RuntimeError):
        opt.step()
