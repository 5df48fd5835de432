"""Filters under temperatures at which logits that differ have equal probabilities stay with the host sampler, on the CPU."""
import numpy as np
import pytest

from kapel_b200.engine.scheduler import EngineOptions, Request, Scheduler
from kapel_b200.sampling import Sampler, Sampling
from test_scheduler import FakeEngine


class _DeviceLogits:
    is_cuda = True
    shape = (1, 50)


@pytest.mark.parametrize("temperature", [float("inf"), 1e300, 1e17, 1e9])
@pytest.mark.parametrize("filters", [dict(top_k=3), dict(top_p=0.5), dict(min_p=0.2)])
def test_a_hot_request_with_filters_is_not_chosen_on_the_device(temperature, filters):
    sched = Scheduler(FakeEngine(), EngineOptions())
    rid = sched.add(Request([1, 2, 3], sampling=Sampling(temperature=temperature, **filters)))
    assert not sched.entries[rid].request.sampling.filtered_on_device()
    assert sched._choose_on_device(_DeviceLogits(), [rid], [0]) is None


def test_others_are():
    for temperature in (0.0, -1.0, 1e-9, 0.7, 100.0):
        assert Sampling(temperature=temperature, top_k=5, top_p=0.9, min_p=0.1).filtered_on_device()
    assert not Sampling(temperature=0.7, top_k=5, repetition_penalty=1.1).filtered_on_device()


def test_what_the_host_does_there():
    """The largest logit is the last; its probability is that of all others, so the nucleus is the lower half by index and top_k cuts nothing."""
    row = np.linspace(-1.0, 1.0, 8)
    for temperature in (1e17, float("inf")):
        assert np.flatnonzero(Sampler(Sampling(temperature=temperature, top_p=0.5)).distribution(row, (), 0)[1]).tolist() == [0, 1, 2, 3]
    assert (Sampler(Sampling(temperature=float("inf"), top_k=2)).distribution(row, (), 0)[1] == 0.125).all()
