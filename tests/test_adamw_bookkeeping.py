"""optim.AdamW: state, counters and checkpoints around the step.  CPU: the kernel call is replaced, or never reached."""
import pytest
import torch

from categoricalnf_amd import ops
from categoricalnf_amd.optim import AdamW


@pytest.fixture
def steps(monkeypatch):
    """Calls of the kernel, as lists of parameters; the stream is being captured while `steps.capturing`."""
    class Calls(list):
        capturing = False
    calls = Calls()
    monkeypatch.setattr(ops, "adamw_step", lambda ps, *a, **kw: calls.append([id(p) for p in ps]))
    monkeypatch.setattr(torch.cuda, "is_available", lambda: True)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: calls.capturing)
    return calls


def params(n=3):
    ps = [torch.nn.Parameter(torch.zeros(4)) for _ in range(n)]
    for p in ps:
        p.grad = torch.ones(4)
    return ps


def test_a_capture_creates_no_state(steps):
    ps = params()
    opt = AdamW(ps, capturable=True)
    steps.capturing = True
    with pytest.raises(RuntimeError, match="before the capture"):
        opt.step()
    assert not steps and not opt.state
    steps.capturing = False
    opt.step()
    steps.capturing = True
    opt.step()
    assert len(steps) == 2


def test_a_capture_splits_no_counter(steps):
    """A clone in the captured graph would take the shared counter's value anew in every replay."""
    ps = params()
    opt = AdamW(ps, capturable=True)
    opt.step()
    ps[1].grad = None
    steps.capturing = True
    with pytest.raises(RuntimeError, match="before the capture"):
        opt.step()
    assert len(steps) == 1 and all(float(opt.state[p]["step"]) == 1 for p in ps)
    steps.capturing = False
    opt.step()                                     # eagerly: the idle parameter keeps its count from here on
    steps.capturing = True
    opt.step()
    assert [float(opt.state[p]["step"]) for p in ps] == [3, 1, 3]


def test_a_capture_moves_no_counter(steps):
    ps = params(1)
    opt = AdamW(ps, capturable=True)
    opt.step()
    opt.state[ps[0]]["step"] = torch.ones((), device="meta")
    steps.capturing = True
    with pytest.raises(RuntimeError, match="before the capture"):
        opt.step()
    assert len(steps) == 1


def state_of(cls, steps=1, **kw):
    p = torch.nn.Parameter(torch.zeros(4))
    opt = cls([p], **kw)
    for _ in range(steps):
        p.grad = torch.ones(4)
        opt.step()
    return opt.state_dict()


@pytest.mark.parametrize("kw", [dict(amsgrad=True), dict(maximize=True)])
def test_checkpoints_of_other_rules_are_refused(kw):
    opt = AdamW(params(1))
    with pytest.raises(ValueError, match=list(kw)[0]):
        opt.load_state_dict(state_of(torch.optim.AdamW, **kw))
    assert not opt.state and "amsgrad" not in opt.param_groups[0]
    with pytest.raises(ValueError, match="weight decay"):
        opt.load_state_dict(state_of(torch.optim.Adam, weight_decay=0.1))
    opt.load_state_dict(state_of(torch.optim.AdamW, lr=0.25))
    opt.load_state_dict(state_of(torch.optim.Adam))
    assert opt.param_groups[0]["lr"] == 1e-3


def test_drivers_resume_with_the_optimiser_that_wrote_the_checkpoint(tmp_path, steps):
    from categoricalnf_amd.experiments.run_set_modeling import load_checkpoint
    made = {"radam": torch.optim.RAdam, "adamw": AdamW, "adamw8": lambda ps: AdamW(ps, state_bits=8, min_8bit_size=1)}
    for a, write in made.items():
        file = str(tmp_path / (a + ".tar"))
        opt = write(params(1))
        opt.step()
        torch.save({"optimizer_state_dict": opt.state_dict(), "iteration": 1}, file)
        for b, read in made.items():
            other = read(params(1))
            if (a == "radam") == (b == "radam"):
                load_checkpoint(file, optimizer=other)
                assert other.state
            else:
                with pytest.raises(ValueError, match="--optimizer"):
                    load_checkpoint(file, optimizer=other)
                assert not other.state
