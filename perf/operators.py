"""Three operators of a training step, in their plain form and as this package's kernels: layer norm with its gradients, the
softmax cross entropy of a linear layer over a vocabulary with its gradients (without keeping the logits), and one AdamW step
over a list of tensors with moments in 32 or in 8 bits.

`run` computes the plain form with elementary torch operations in 32 bits where `own` is false, and calls the package where it
is true.  `exact` computes the same outputs from the definitions in 64 bits."""
import math

import torch

own = False

DEVICE = "cuda"
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK8 = 256                 # consecutive elements of a tensor that share the two scales of its 8-bit moments
BETA1, BETA2, EPS = 0.9, 0.999, 1e-8


# ---- cases -----------------------------------------------------------------------------------------------------------------

def listed():
    return [
        # layer norm in front of a sub-network's output layer, evaluated on one small set: latency
        {"name": "ln_eval_small", "op": "ln", "train": False, "rows": 16, "cols": 64, "dtype": "f32", "pad": 0, "affine": True},
        # the Edge-GNN's pair features: 64 graphs of 703 pairs, 128 features, a training step
        {"name": "ln_train_pairs", "op": "ln", "train": True, "rows": 64 * 703, "cols": 128, "dtype": "f32", "pad": 0, "affine": True},
        # an odd width whose rows lie apart (a slice of a wider tensor), half precision
        {"name": "ln_train_odd", "op": "ln", "train": True, "rows": 4999, "cols": 777, "dtype": "f16", "pad": 9, "affine": True},
        # a large Transformer batch in bf16
        {"name": "ln_train_large", "op": "ln", "train": True, "rows": 131072, "cols": 1024, "dtype": "bf16", "pad": 0, "affine": True},
        # a decoder's log-probability of the right class for a few tokens (hidden size 64, 51 classes), no gradient: latency
        {"name": "ce_eval_small", "op": "ce", "train": False, "rows": 64, "vocab": 51, "hidden": 64, "dtype": "f32", "bias": True, "ignored": 0.0, "mean": False},
        # the same decoder in training on 128 sentences of 288 characters
        {"name": "ce_train_chars", "op": "ce", "train": True, "rows": 128 * 288, "vocab": 51, "hidden": 64, "dtype": "f32", "bias": True, "ignored": 0.1, "mean": True},
        # ... and on a vocabulary of 10 000 words
        {"name": "ce_train_words", "op": "ce", "train": True, "rows": 128 * 288, "vocab": 10000, "hidden": 64, "dtype": "f32", "bias": True, "ignored": 0.1, "mean": True},
        # a word-level output layer of 1024 features in bf16
        {"name": "ce_train_large", "op": "ce", "train": True, "rows": 8192, "vocab": 32000, "hidden": 1024, "dtype": "bf16", "bias": False, "ignored": 0.05, "mean": True},
        # one flow step's parameters: a handful of small tensors, latency
        {"name": "adamw_small", "op": "adamw", "layers": 2, "hidden": 64, "dtype": "f32", "bits": 32},
        # a set-modelling flow: 820 tensors
        {"name": "adamw_many", "op": "adamw", "layers": 82, "hidden": 256, "dtype": "f32", "bits": 32},
        # a language model's few large matrices, moments in 8 bits
        {"name": "adamw_8bit", "op": "adamw", "layers": 4, "hidden": 2048, "dtype": "f32", "bits": 8},
        # bf16 parameters, moments in 32 bits
        {"name": "adamw_large", "op": "adamw", "layers": 5, "hidden": 4096, "dtype": "bf16", "bits": 32},
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["ln", "ce", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    if op == "ln":
        cols = _log_int(rng, 1, 20000)
        if rng.random() < 0.5:
            cols = max(8, cols // 8 * 8)
        rows = _log_int(rng, 1, max(1, min(200000, 100_000_000 // cols)))
        return {"op": "ln", "train": rng.random() < 0.7, "rows": rows, "cols": cols, "dtype": dtype,
                "pad": rng.choice([0, 0, 0, 8, 64, rng.randint(1, 40)]), "affine": rng.random() < 0.85}
    if op == "ce":
        hidden = _log_int(rng, 1, 2048)
        if rng.random() < 0.5:
            hidden = max(8, hidden // 8 * 8)
        vocab = _log_int(rng, 1, 60000)
        most = 2e11 / (vocab * hidden)
        rows = _log_int(rng, 1, max(1, int(min(40000, most, 1e9 / vocab))))
        return {"op": "ce", "train": rng.random() < 0.7, "rows": rows, "vocab": vocab, "hidden": hidden, "dtype": dtype,
                "bias": rng.random() < 0.6, "ignored": rng.choice([0.0, 0.1, 0.5]), "mean": rng.random() < 0.6}
    layers = _log_int(rng, 1, 90)
    hidden = _log_int(rng, 3, max(4, min(4096, int(math.sqrt(80e6 / (5 * layers))))))
    return {"op": "adamw", "layers": layers, "hidden": hidden, "dtype": dtype, "bits": rng.choice([32, 8])}


def _shapes(case):
    """The tensors of `layers` equal blocks: two feed-forward matrices, a square one, their biases, a norm, two tiny ones."""
    h = case["hidden"]
    return [(2 * h, h), (2 * h,), (h, 2 * h), (h,), (h, h), (h,), (h,), (h,), (6, 6), (6,)] * case["layers"]


# ---- inputs ----------------------------------------------------------------------------------------------------------------

def prepare(case, seed):
    gen = torch.Generator(device=DEVICE).manual_seed(int(seed))

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device=DEVICE)

    state = {"case": case}
    if case["op"] == "ln":
        dt, rows, cols = DTYPES[case["dtype"]], case["rows"], case["cols"]
        # activations of a residual stream: a mean of their own per row, a spread that differs between the columns
        wide = normal(rows, cols + case["pad"])
        wide.mul_(0.5 + torch.rand(cols + case["pad"], generator=gen, device=DEVICE)).add_(normal(rows, 1))
        wide = wide.to(dt)
        state["x"] = wide[:, :cols]
        state["weight"] = (1 + 0.2 * normal(cols)).to(dt) if case["affine"] else None
        state["bias"] = (0.2 * normal(cols)).to(dt) if case["affine"] else None
        if case["train"]:
            state["grad"] = normal(rows, cols).to(dt)
            for k in ("x", "weight", "bias"):
                if state[k] is not None:
                    state[k].requires_grad_()
    elif case["op"] == "ce":
        dt, rows, vocab, hidden = DTYPES[case["dtype"]], case["rows"], case["vocab"], case["hidden"]
        state["x"] = normal(rows, hidden).to(dt)
        state["weight"] = (normal(vocab, hidden) * (2.0 / math.sqrt(hidden))).to(dt)
        state["bias"] = (0.5 * normal(vocab)).to(dt) if case["bias"] else None
        # frequent classes first, as in a vocabulary sorted by frequency; padding at the end of the token list
        u = torch.rand(rows, generator=gen, device=DEVICE, dtype=torch.float64)
        target = (torch.exp(u * math.log(vocab + 1.0)) - 1).long().clamp_(0, vocab - 1)
        keep = rows - int(rows * case["ignored"])
        target[keep:] = -100
        state["target"] = target
        if case["train"]:
            state["grad"] = torch.ones((), device=DEVICE) if case["mean"] else torch.rand(rows, generator=gen, device=DEVICE)
            for k in ("x", "weight", "bias"):
                if state[k] is not None:
                    state[k].requires_grad_()
    else:
        dt, shapes = DTYPES[case["dtype"]], _shapes(case)
        sizes = [math.prod(s) for s in shapes]
        # the tensors lie in one buffer, each at a multiple of BLOCK8 elements: the step sees the list, the outputs come whole
        starts, total = [], 0
        for n in sizes:
            starts.append(total)
            total += -(-n // BLOCK8) * BLOCK8
        used = torch.zeros(total, dtype=torch.bool, device=DEVICE)
        for a, n in zip(starts, sizes):
            used[a:a + n] = True
        scale = torch.exp(2 * normal(total // BLOCK8)).repeat_interleave(BLOCK8)      # gradients differ by tensor and region

        def cut(flat):
            return [flat[a:a + n].view(s) for a, n, s in zip(starts, sizes, shapes)]
        grad = normal(total) * 1e-3 * scale * used
        # moments as they are after some steps: means of earlier gradients and of their squares
        m = (0.3 * normal(total) * 1e-3 * scale) * used
        v = ((0.3 + torch.rand(total, generator=gen, device=DEVICE)) * (1e-3 * scale) ** 2) * used
        state["p"], state["g"] = (0.05 * normal(total) * used).to(dt), grad.to(dt)
        if case["bits"] == 32:
            state["m"], state["v"] = m, v
            state["exp_avg"], state["exp_avg_sq"] = cut(m), cut(v)
            state["exp_avg_scale"] = state["exp_avg_sq_scale"] = None
        else:
            state["m"], state["ms"] = _encode_m(m)
            state["v"], state["vs"] = _encode_v(v)
            state["exp_avg"], state["exp_avg_sq"] = cut(state["m"]), cut(state["v"])
            blocks = [(a // BLOCK8, -(-n // BLOCK8)) for a, n in zip(starts, sizes)]
            state["exp_avg_scale"] = [state["ms"][a:a + n] for a, n in blocks]
            state["exp_avg_sq_scale"] = [state["vs"][a:a + n] for a, n in blocks]
        state["params"], state["grads"] = cut(state["p"]), cut(state["g"])
        state["step"] = 10
    return state


# ---- 8-bit moments: m = s q |q| with q in -127..127, v = (s q^2)^2 with q in 0..255, one s for each block -----------------------

def _blocks(flat):
    n = flat.numel()
    return torch.cat([flat.reshape(-1), flat.new_zeros(-n % BLOCK8)]).view(-1, BLOCK8)


def _encode_m(m):
    b = _blocks(m)
    s = b.abs().amax(1) * torch.tensor(1.0 / 16129, dtype=m.dtype, device=m.device)
    q = torch.sqrt(b.abs() / s[:, None]).round().clamp(max=127)
    q = torch.where(torch.isfinite(s[:, None]) & (s[:, None] > 0), q, torch.zeros_like(q)) * torch.sign(b)
    s = torch.where(torch.isfinite(s), s, torch.full_like(s, float("nan")))
    return q.nan_to_num(0).to(torch.int8).reshape(-1)[:m.numel()].view(m.shape), s


def _encode_v(v):
    b = _blocks(v)
    r = torch.sqrt(b)
    s = r.amax(1) * torch.tensor(1.0 / 65025, dtype=v.dtype, device=v.device)
    q = torch.sqrt(r / s[:, None]).round().clamp(min=1, max=255)
    q = torch.where(torch.isfinite(s[:, None]) & (s[:, None] > 0) & (r > 0), q, torch.zeros_like(q))
    s = torch.where(torch.isfinite(s), s, torch.full_like(s, float("nan")))
    return q.to(torch.uint8).reshape(-1)[:v.numel()].view(v.shape), s


def _decode_m(q, s):
    f = _blocks(q).to(s.dtype)
    return (f * f.abs() * s[:, None]).reshape(-1)[:q.numel()].view(q.shape)


def _decode_v(q, s):
    f = _blocks(q).to(s.dtype)
    r = f * f * s[:, None]
    return (r * r).reshape(-1)[:q.numel()].view(q.shape)


# ---- one pass --------------------------------------------------------------------------------------------------------------

def run(state):
    return {"ln": _layer_norm, "ce": _cross_entropy, "adamw": _adamw}[state["case"]["op"]](state)


def _layer_norm(state):
    x, weight, bias, train = state["x"], state["weight"], state["bias"], state["case"]["train"]
    if own:
        from categoricalnf_amd import functional as Fn
        y = Fn.layer_norm(x, weight, bias)
        if not train:
            return {"y": y}
        wrt = [t for t in (x, weight, bias) if t is not None]
        g = torch.autograd.grad(y, wrt, state["grad"])
        return dict(zip(("y", "dx", "dweight", "dbias"), (y,) + tuple(g)))
    with torch.no_grad():
        dt = x.dtype
        xf = x.float()
        mean = xf.mean(1, keepdim=True)
        xc = xf - mean
        rstd = 1 / torch.sqrt((xc * xc).mean(1, keepdim=True) + 1e-5)
        xhat = xc * rstd
        y = xhat if weight is None else xhat * weight.float() + bias.float()
        if not train:
            return {"y": y.to(dt)}
        g = state["grad"].float()
        gw = g if weight is None else g * weight.float()
        dx = rstd * (gw - gw.mean(1, keepdim=True) - xhat * (gw * xhat).mean(1, keepdim=True))
        out = {"y": y.to(dt), "dx": dx.to(dt)}
        if weight is not None:
            out["dweight"], out["dbias"] = (g * xhat).sum(0).to(dt), g.sum(0).to(dt)
        return out


def _cross_entropy(state):
    x, weight, bias, target, case = state["x"], state["weight"], state["bias"], state["target"], state["case"]
    if own:
        from categoricalnf_amd import functional as Fn
        loss = Fn.linear_cross_entropy(x, weight, target, bias, reduction="mean" if case["mean"] else "none")
        if not case["train"]:
            return {"loss": loss}
        wrt = [t for t in (x, weight, bias) if t is not None]
        g = torch.autograd.grad(loss, wrt, state["grad"])
        return dict(zip(("loss", "dx", "dweight", "dbias"), (loss.detach(),) + tuple(g)))
    with torch.no_grad():
        dt = x.dtype
        xf, wf = x.float(), weight.float()
        logits = xf @ wf.t()
        if bias is not None:
            logits += bias.float()
        top = logits.amax(1, keepdim=True)
        e = torch.exp(logits - top)
        total = e.sum(1, keepdim=True)
        keep = target >= 0
        index = target.clamp(min=0)[:, None]
        loss = (torch.log(total) + top - logits.gather(1, index))[:, 0] * keep
        count = keep.sum()
        value = loss.sum() / count if case["mean"] else loss
        if not case["train"]:
            return {"loss": value}
        scale = (state["grad"] / count if case["mean"] else state["grad"]) * keep
        d = e.div_(total)
        d.scatter_add_(1, index, torch.full_like(total, -1.0))
        d.mul_(scale[:, None])
        out = {"loss": value, "dx": (d @ wf).to(dt), "dweight": (d.t() @ xf).to(dt)}
        if bias is not None:
            out["dbias"] = d.sum(0).to(dt)
        return out


def _adamw(state):
    lr, decay = 1e-3, 0.01
    bits8 = state["case"]["bits"] == 8
    state["step"] += 1
    if own:
        from categoricalnf_amd import ops
        ops.adamw_step(state["params"], state["grads"], state["exp_avg"], state["exp_avg_sq"], step=state["step"], lr=lr, beta1=BETA1,
                       beta2=BETA2, eps=EPS, weight_decay=decay, exp_avg_scales=state["exp_avg_scale"], exp_avg_sq_scales=state["exp_avg_sq_scale"])
        if bits8:
            m, v = ops.adamw_moments(state["m"], state["v"], state["ms"], state["vs"])
            return {"p": state["p"], "m": m, "v": v}
        return {"p": state["p"], "m": state["m"], "v": state["v"]}
    c = _constants(state["step"], lr, decay)
    params, grads = state["params"], state["grads"]
    narrow = params[0].dtype != torch.float32
    p = [t.float() for t in params] if narrow else params
    g = [t.float() for t in grads] if narrow else grads
    if bits8:
        m = [_decode_m(q, s) for q, s in zip(state["exp_avg"], state["exp_avg_scale"])]
        v = [_decode_v(q, s) for q, s in zip(state["exp_avg_sq"], state["exp_avg_sq_scale"])]
    else:
        m, v = state["exp_avg"], state["exp_avg_sq"]
    torch._foreach_mul_(m, c["beta1"])
    torch._foreach_add_(m, torch._foreach_mul(g, c["one_beta1"]))
    g2 = torch._foreach_mul(g, g)
    torch._foreach_mul_(g2, c["one_beta2"])
    torch._foreach_mul_(v, c["beta2"])
    torch._foreach_add_(v, g2)
    denom = torch._foreach_sqrt(v)
    torch._foreach_mul_(denom, c["root"])
    torch._foreach_add_(denom, c["eps"])
    update = torch._foreach_div(m, denom)
    torch._foreach_mul_(update, c["size"])
    torch._foreach_mul_(p, c["keep"])
    torch._foreach_sub_(p, update)
    if narrow:
        torch._foreach_copy_(params, p)
    if bits8:
        coded_m, coded_v = [_encode_m(t) for t in m], [_encode_v(t) for t in v]
        torch._foreach_copy_(state["exp_avg"] + state["exp_avg_scale"], [q for q, _ in coded_m] + [s for _, s in coded_m])
        torch._foreach_copy_(state["exp_avg_sq"] + state["exp_avg_sq_scale"], [q for q, _ in coded_v] + [s for _, s in coded_v])
        return {"p": state["p"], "m": _decode_m(state["m"], state["ms"]), "v": _decode_v(state["v"], state["vs"])}
    return {"p": state["p"], "m": state["m"], "v": state["v"]}


def _constants(step, lr, decay):
    """The step's numbers, each rounded to 32 bits once."""
    full = {"beta1": BETA1, "one_beta1": 1 - BETA1, "beta2": BETA2, "one_beta2": 1 - BETA2, "eps": EPS, "keep": 1 - lr * decay,
            "size": lr / (1 - BETA1 ** step), "root": 1 / math.sqrt(1 - BETA2 ** step)}
    return {k: float(torch.tensor(v, dtype=torch.float32)) for k, v in full.items()}


# ---- work and the 64-bit results -----------------------------------------------------------------------------------------------

def work(case):
    size = 4 if case.get("dtype") == "f32" else 2
    if case["op"] == "ln":
        n = case["rows"] * case["cols"]
        vec = 2 * case["cols"] * size if case["affine"] else 0
        if not case["train"]:
            return {"bytes": 2 * n * size + vec, "flops": 8 * n}
        # forward: x in, y out; backward: x and dy in, dx out
        return {"bytes": 5 * n * size + 3 * vec, "flops": 20 * n}
    if case["op"] == "ce":
        r, v, h = case["rows"], case["vocab"], case["hidden"]
        reads = (r * h + v * h + (v if case["bias"] else 0)) * size + 8 * r
        if not case["train"]:
            return {"bytes": reads + 4 * r, "flops": 2 * r * v * h}
        return {"bytes": 2 * reads + 4 * r, "flops": 6 * r * v * h}
    n = sum(math.prod(s) for s in _shapes(case))
    if case["bits"] == 32:
        return {"bytes": n * (3 * size + 16), "flops": 14 * n}
    # codes in and out, the decoded values out
    return {"bytes": n * (3 * size + 4 + 8) + 16 * (n // BLOCK8), "flops": 30 * n}


def exact(case, seed):
    state = prepare(case, seed)
    with torch.no_grad():
        if case["op"] == "ln":
            return _exact_layer_norm(state, case)
        if case["op"] == "ce":
            return _exact_cross_entropy(state, case)
        return _exact_adamw(state, case)


def _exact_layer_norm(state, case):
    x = state["x"].double()
    w = state["weight"].double() if case["affine"] else torch.ones(x.shape[1], dtype=torch.float64, device=x.device)
    b = state["bias"].double() if case["affine"] else torch.zeros_like(w)
    mu = x.sum(1, keepdim=True) / x.shape[1]
    x = x.sub_(mu)
    inv = torch.rsqrt(x.square().sum(1, keepdim=True) / x.shape[1] + 1e-5)
    n = x.mul_(inv)                                       # normalised rows
    out = {"y": torch.addcmul(b, n, w)}
    if case["train"]:
        gy = state["grad"].double()
        if case["affine"]:
            out["dweight"], out["dbias"] = torch.einsum("rc,rc->c", gy, n), gy.sum(0)
        gn = gy * w
        # the projection of the gradient on the space orthogonal to (1, ..., 1) and to the normalised row
        along = torch.einsum("rc,rc->r", gn, n)[:, None] / x.shape[1]
        out["dx"] = (gn - gn.sum(1, keepdim=True) / x.shape[1] - n * along) * inv
    return out


def _exact_cross_entropy(state, case):
    if case["rows"] * case["vocab"] > 1_500_000_000:
        return None
    x, w, t = state["x"].double(), state["weight"].double(), state["target"]
    b = state["bias"].double() if case["bias"] else None
    rows = torch.nonzero(t >= 0)[:, 0]
    lp = torch.nn.functional.linear(x[rows], w, b).log_softmax(1)
    each = -lp[torch.arange(len(rows), device=x.device), t[rows]]
    if case["mean"]:
        loss = each.mean()
        scale = torch.full_like(each, 1.0 / max(len(rows), 1))
    else:
        loss = torch.zeros(case["rows"], dtype=torch.float64, device=x.device)
        loss[rows] = each
        scale = state["grad"].double()[rows] if case["train"] else None
    out = {"loss": loss}
    if case["train"]:
        p = lp.exp_()
        p[torch.arange(len(rows), device=x.device), t[rows]] -= 1
        p *= scale[:, None]
        out["dx"] = torch.zeros_like(x)
        out["dx"][rows] = torch.mm(p, w)
        out["dweight"] = torch.mm(p.t(), x[rows])
        if case["bias"]:
            out["dbias"] = p.sum(0)
    return out


def _exact_adamw(state, case):
    lr, decay, t = 1e-3, 0.01, state["step"] + 1
    p, g = state["p"].double(), state["g"].double()
    if case["bits"] == 8:
        qm, qv = state["m"].double().view(-1, BLOCK8), state["v"].double().view(-1, BLOCK8)
        m = (qm * qm.abs() * state["ms"].double()[:, None]).view(-1)
        v = (qv.square() * state["vs"].double()[:, None]).square().view(-1)
    else:
        m, v = state["m"].double(), state["v"].double()
    m = torch.lerp(g, m, BETA1)
    v = torch.lerp(g * g, v, BETA2)
    p = p * (1 - lr * decay) - lr * (m / (1 - BETA1 ** t)) / (torch.sqrt(v / (1 - BETA2 ** t)) + EPS)
    if case["bits"] == 8:
        # the nearest code of the block's grid; a second moment above zero keeps a code above zero
        top = m.abs().view(-1, BLOCK8).amax(1, keepdim=True)
        unit = top.clamp(min=1e-300) / 127 ** 2
        q = (m.abs().view(-1, BLOCK8) / unit).sqrt().round()
        m = (torch.sign(m).view(-1, BLOCK8) * q * q * unit).view(-1)
        r = v.sqrt().view(-1, BLOCK8)
        unit = r.amax(1, keepdim=True).clamp(min=1e-300) / 255 ** 2
        q = torch.maximum((r / unit).sqrt().round(), (r > 0).double())
        v = (q * q * unit).square().view(-1)
    return {"p": p, "m": m, "v": v}
