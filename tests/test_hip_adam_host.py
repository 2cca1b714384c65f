"""CPU tests of HipAdam's host side: what it does with its state around deferred updates, loading and changes of width (the update itself needs the GPU)."""
import pytest
import torch


class _Stream:
    def __init__(self):
        self.waited = []

    def wait_event(self, event):
        self.waited.append(event)


@pytest.mark.parametrize("call", ["moments", "state_dict", "load_state_dict"])
def test_readers_of_state_wait_for_deferred_updates(monkeypatch, call):
    from med_ts_llm_amd.hip.optim import HipAdam
    p = torch.nn.Parameter(torch.zeros(5))
    opt = HipAdam([p])
    opt.state[p].update(step=1, exp_avg=torch.ones(5), exp_avg_sq=torch.ones(5))
    sd = torch.optim.Optimizer.state_dict(opt)
    stream = _Stream()
    monkeypatch.setattr(torch.cuda, "current_stream", lambda *a: stream)
    getattr(opt, call)(*([sd] if call == "load_state_dict" else []))
    assert stream.waited == []
    opt._late_done = "the last step's"
    getattr(opt, call)(*([sd] if call == "load_state_dict" else []))
    assert stream.waited == ["the last step's"] and opt._late_done == "the last step's"


def test_moments_are_copies():
    from med_ts_llm_amd.hip.optim import HipAdam
    p = torch.nn.Parameter(torch.zeros(5))
    opt = HipAdam([p])
    opt.state[p].update(step=1, exp_avg=torch.ones(5), exp_avg_sq=torch.ones(5))
    m, v = opt.moments()[p]
    opt.state[p]["exp_avg"].zero_()
    opt.state[p]["exp_avg_sq"].zero_()
    assert bool((m == 1).all()) and bool((v == 1).all())
