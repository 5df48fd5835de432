"""Requests whose settings decide whatever the logits: the device path takes no number from their generators, as the host does not."""
import numpy as np
import pytest
import torch

from kapel_b200.engine.scheduler import EngineOptions, Request, Scheduler
from kapel_b200.sampling import Sampler, Sampling
from test_scheduler import FakeEngine

SETTINGS = [dict(temperature=0.0, top_k=5), dict(temperature=0.8, top_p=0.0), dict(temperature=0.8, top_p=-1.0, top_k=3), dict(temperature=0.8, min_p=1.5),
            dict(temperature=float("nan"), top_k=5), dict(temperature=0.8, top_k=5), dict(temperature=0.8, top_p=0.9, min_p=1.0), dict(temperature=1.2)]


@pytest.mark.gpu
def test_the_generators_move_as_on_the_host():
    rng = np.random.default_rng(3)
    sched = Scheduler(FakeEngine(pages=40, max_sequences=len(SETTINGS)), EngineOptions())
    ids = [sched.add(Request([1, 2, 3], sampling=Sampling(seed=i, **s))) for i, s in enumerate(SETTINGS)]
    host = [Sampler(Sampling(seed=i, **s)) for i, s in enumerate(SETTINGS)]
    for _ in range(4):
        logits = rng.normal(0.0, 2.0, (len(ids), 50)).astype(np.float32)
        got = sched._choose_on_device(torch.from_numpy(logits).cuda(), ids, list(range(len(ids)))).cpu().tolist()
        assert got == [h.choose(row) for h, row in zip(host, logits)]
        assert [sched.entries[r].sampler.rng.s for r in ids] == [h.rng.s for h in host]
