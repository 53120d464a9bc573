"""AdamW over all parameters of a model in a few kernel launches, moments in fp32 or in 8 bits (cnf_adamw_step).

The reference trains with RAdam / Adam from torch.optim (general/train.py:331-358, general/mutils.py:142-170); this is the
decoupled-weight-decay member of that family for the drivers' `--optimizer` and for `graphs.GraphedTraining(optimizer_cls=AdamW)`."""
import torch

from . import ops

_CPU = torch.device("cpu")
# what a capture records runs again in every replay: only the step itself may be in it
_IN_CAPTURE = "AdamW.step() inside a stream capture: %s, in every replay again; run one step with the same gradients present before the capture"


class AdamW(torch.optim.Optimizer):
    """p = p (1 - lr weight_decay) - lr m_hat / (sqrt(v_hat) + eps), as torch.optim.AdamW.

    state_bits=8 keeps the moments of every tensor of at least `min_8bit_size` elements in 8 bits (2 + 8 / 256 bytes per element
    instead of 8: int8 / uint8 codes on a quadratic grid, one scale for 256 elements); smaller tensors, whose moments weigh
    nothing, keep fp32.  Moments are fp32 (or codes) whatever the parameters' type; a parameter in 16 bits is rounded to nearest
    at every step, so steps below half its spacing are lost — train 16-bit models with fp32 parameters where that matters.

    capturable=True: the step counter is a device tensor and `lr` may be one (float32), so that a captured `step()` can be
    replayed.  A step with the same gradients present has to run before the capture.  Parameters, gradients and moments must be dense (contiguous); sparse gradients are refused."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=1e-2, *, state_bits=32, min_8bit_size=4096,
                 capturable=False):
        if not isinstance(lr, torch.Tensor) and not lr >= 0.0:
            raise ValueError("Invalid learning rate: %r" % (lr,))
        if isinstance(lr, torch.Tensor) and not capturable:
            raise ValueError("lr as a tensor needs capturable=True")
        if len(betas) != 2 or not all(0.0 <= b < 1.0 for b in betas):
            raise ValueError("Invalid betas: %r" % (betas,))
        if not eps >= 0.0 or not weight_decay >= 0.0:
            raise ValueError("Invalid eps / weight_decay: %r / %r" % (eps, weight_decay))
        if state_bits not in (32, 8):
            raise ValueError("state_bits is 32 or 8, got %r" % (state_bits,))
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      min_8bit_size=int(min_8bit_size), capturable=bool(capturable)))

    # ---- state -------------------------------------------------------------------------------------------------------------
    def _init_state(self, p, group, step):
        state = self.state[p]
        state["step"] = step
        if group["state_bits"] == 8 and p.numel() >= group["min_8bit_size"]:
            blocks = -(-p.numel() // ops.ADAMW_BLOCK)
            state["exp_avg"] = torch.zeros(p.shape, dtype=torch.int8, device=p.device)
            state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.uint8, device=p.device)
            state["exp_avg_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
            state["exp_avg_sq_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        else:
            state["exp_avg"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
            state["exp_avg_sq"] = torch.zeros(p.shape, dtype=torch.float32, device=p.device)
        return state

    def moments(self, p):
        """(m, v) of a parameter in fp32, whatever its state's bits; None before its first step."""
        state = self.state.get(p)
        if not state:
            return None
        if "exp_avg_scale" in state:
            return ops.adamw_moments(state["exp_avg"], state["exp_avg_sq"], state["exp_avg_scale"], state["exp_avg_sq_scale"])
        return state["exp_avg"], state["exp_avg_sq"]

    def load_state_dict(self, state_dict):
        """As torch's, but the moments keep the types they were saved with (torch casts a state to its parameter's type, which
        would destroy codes, and fp32 moments of 16-bit parameters).  A checkpoint whose steps this class does not compute (amsgrad,
        maximize, another rule than decoupled weight decay) is refused."""
        for group in state_dict["param_groups"]:
            for option in ("amsgrad", "maximize"):
                if group.get(option):
                    raise ValueError("the checkpoint's optimiser has %s, which this AdamW does not compute" % option)
            if "decoupled_weight_decay" in group and not group["decoupled_weight_decay"] and group.get("weight_decay"):
                raise ValueError("the checkpoint's optimiser adds its weight decay to the gradients, which this AdamW does not")
        super().load_state_dict(state_dict)
        for group in self.param_groups:                   # a checkpoint of torch.optim.AdamW lacks this class's options
            for k, v in self.defaults.items():
                group.setdefault(k, v)
        ids = [i for g in state_dict["param_groups"] for i in g["params"]]
        mine = [p for g in self.param_groups for p in g["params"]]
        group_of = {p: g for g in self.param_groups for p in g["params"]}
        for i, p in zip(ids, mine):
            saved = state_dict["state"].get(i)
            if saved is None:
                continue
            for k in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
                if k in saved:
                    self.state[p][k] = saved[k].detach().to(device=p.device, copy=True).contiguous()
            step = saved["step"]
            step = step.detach().float().reshape(()) if isinstance(step, torch.Tensor) else torch.tensor(float(step))
            self.state[p]["step"] = step.to(device=p.device if group_of[p]["capturable"] else "cpu", copy=True)
        self._share_steps()

    def _share_steps(self):
        """Parameters that have taken the same number of steps share one counter tensor."""
        shared = {}
        for group in self.param_groups:
            for p in group["params"]:
                state = self.state.get(p)
                if state:
                    key = (state["step"].device, float(state["step"]), group["capturable"])
                    state["step"] = shared.setdefault(key, state["step"])

    # ---- one step ----------------------------------------------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        capturing = torch.cuda.is_available() and torch.cuda.is_current_stream_capturing()
        fresh, moved, calls, idle = {}, {}, {}, []
        for group in self.param_groups:
            capturable = group["capturable"]
            if capturing and not capturable:
                raise RuntimeError("AdamW.step() inside a stream capture needs capturable=True")
            for p in group["params"]:
                g = p.grad
                state = self.state.get(p)
                if g is None:
                    if state:
                        idle.append(state)
                    continue
                if g.is_sparse:
                    raise RuntimeError("AdamW does not take sparse gradients")
                home = p.device if capturable else _CPU
                if not state:
                    if capturing:
                        raise RuntimeError(_IN_CAPTURE % "a parameter's state would be created")
                    if home not in fresh:
                        fresh[home] = torch.zeros((), dtype=torch.float32, device=home)
                    state = self._init_state(p, group, fresh[home])
                step = state["step"]
                if step.is_cuda != capturable and step.device != home:        # the group's flag was switched (a checkpoint of a captured run, and back)
                    if capturing:
                        raise RuntimeError(_IN_CAPTURE % "a step counter would be moved to the device")
                    if (id(step), home) not in moved:
                        moved[id(step), home] = (step, step.to(home))
                    step = state["step"] = moved[id(step), home][1]
                bits8 = "exp_avg_scale" in state
                key = (id(group), p.device, p.dtype, g.dtype, bits8, id(step))
                call = calls.get(key)
                if call is None:
                    call = calls[key] = (group, step, bits8, [], [], [], [], [], [])
                call[3].append(p)
                call[4].append(g)
                call[5].append(state["exp_avg"])
                call[6].append(state["exp_avg_sq"])
                if bits8:
                    call[7].append(state["exp_avg_scale"])
                    call[8].append(state["exp_avg_sq_scale"])
        steps = {id(call[1]): call[1] for call in calls.values()}
        stay = {}
        for state in idle:                                # no gradient this time: the parameter's own count does not advance
            step = state["step"]
            if id(step) in steps:
                if capturing:
                    raise RuntimeError(_IN_CAPTURE % "the step counter of a parameter without a gradient would be split from the others'")
                if id(step) not in stay:
                    stay[id(step)] = step.clone()
                state["step"] = stay[id(step)]
        for step in steps.values():
            step += 1
        for group, step, bits8, ps, gs, ms, vs, mss, vss in calls.values():
            beta1, beta2 = group["betas"]
            ops.adamw_step(ps, gs, ms, vs, step=step if group["capturable"] else float(step), lr=group["lr"], beta1=beta1, beta2=beta2,
                           eps=group["eps"], weight_decay=group["weight_decay"], exp_avg_scales=mss if bits8 else None,
                           exp_avg_sq_scales=vss if bits8 else None)
        return loss
