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


def test_a_failed_change_of_width_keeps_the_state():
    """(here: for want of a GPU) the moments are still there afterwards"""
    from med_ts_llm_amd.hip import _native as N
    from med_ts_llm_amd.hip.optim import HipAdam, adam8_state
    p = torch.nn.Parameter(torch.zeros(5))
    narrow, wide = HipAdam([p], state_bits=8), HipAdam([p])
    narrow.state[p].update(step=1, exp_avg=torch.ones(5), exp_avg_sq=torch.ones(5))
    wide.state[p].update(step=1, **dict(zip(("exp_avg_q", "exp_avg_sq_q", "q_exp"), adam8_state(p))))
    for opt in (narrow, wide):
        held = dict(opt.state[p])
        with pytest.raises(N.MtlError):
            opt._to_width(opt.state[p], p)
        assert opt.state[p].keys() == held.keys() and all(opt.state[p][k] is held[k] for k in held)


@pytest.mark.parametrize("bits,optimizer,device,fine", [(8, "sgd", "cuda", False), (8, "adam", "cpu", False), (8, "adamw", "cpu", False), (16, "adam", "cuda", False), (16, "sgd", "cpu", False),
                                                        (32, "sgd", "cuda", True), (32, "adam", "cpu", True), (None, "adamw", "cpu", True)])
def test_the_trainer_does_not_ignore_the_width_of_its_state(bits, optimizer, device, fine):
    from types import SimpleNamespace

    from med_ts_llm_amd.tasks.base import BaseTask
    from med_ts_llm_amd.utils import dict_to_object
    setup = {} if bits is None else {"optimizer_state_bits": bits}
    task = SimpleNamespace(finetuning=False, model=torch.nn.Linear(2, 2), device=torch.device(device),
                           config=dict_to_object({"setup": setup, "training": {"learning_rate": 1e-3, "optimizer": optimizer}}))
    if fine:
        assert BaseTask.build_optimizer(task) is not None
    else:
        with pytest.raises(ValueError, match="optimizer_state_bits"):
            BaseTask.build_optimizer(task)


def test_a_part_of_a_state_twice_is_refused():
    """codes of the first moment given as the root's too, one exponent tensor for two parameters"""
    from med_ts_llm_amd.hip import _native as N
    from med_ts_llm_amd.hip.optim import Adam8State, adam8_state, adam8_step
    p, q, g = torch.zeros(70), torch.zeros(70), torch.zeros(70)
    a, b, empty = adam8_state(p), adam8_state(q), torch.zeros(0)
    for states in ([Adam8State(a.exp_avg, a.exp_avg, a.exponents), b], [a, Adam8State(b.exp_avg, b.exp_avg_sq, a.exponents)], [a, Adam8State(b.exp_avg, a.exp_avg, b.exponents)]):
        with pytest.raises(ValueError, match="twice"):
            adam8_step([p, q], [g, g], states, 1)
    with pytest.raises(N.MtlError):                               # (sound, but on the CPU)
        adam8_step([p, q, empty, empty], [g, g, empty, empty], [a, b, adam8_state(empty), adam8_state(empty)], 1)


def test_a_bf16_copy_that_does_not_hold_its_parameter_is_refused():
    """(the step writes [rows, cols] into it)"""
    from med_ts_llm_amd.hip import _native as N
    from med_ts_llm_amd.hip.optim import Bf16Shadow, adam8_state, adam8_step
    small, wide, flat, cube = torch.zeros(3, 8), torch.zeros(6, 8), torch.zeros(24), torch.zeros(3, 4, 2)
    copy = Bf16Shadow(small, torch.zeros(3, 16, dtype=torch.bfloat16))
    for p in (wide, flat, cube, torch.zeros(1, 24)):
        with pytest.raises(ValueError, match="copy"):
            adam8_step([p], [torch.zeros_like(p)], [adam8_state(p)], 1, shadows=[copy], first_moment="threshold")
    with pytest.raises(N.MtlError):                               # (sound, but on the CPU)
        adam8_step([small], [torch.zeros_like(small)], [adam8_state(small)], 1, shadows=[copy], first_moment="threshold")
