"""Answers to one prompt keep their place among those that wait, on the CPU."""
import pytest

from kapel_b200.engine.scheduler import EngineOptions, Request, Scheduler
from test_fork import ForkingEngine, alone, run


def test_a_group_whose_first_answer_is_cancelled_keeps_its_place():
    eng = ForkingEngine(pages=60)
    sched = Scheduler(eng, EngineOptions(max_sequences=1))
    before = [sched.add(Request([i + 1, 2, 3], max_tokens=3)) for i in range(2)]
    ids = sched.add_samples(Request([4, 5, 6, 7], max_tokens=3), 3)
    behind = sched.add(Request([9, 9], max_tokens=3))
    sched.cancel(ids[0])
    assert list(sched.waiting) == [*before, ids[1], behind] and sched.answers == {ids[1]: [ids[2]]}
    order = []
    while sched.has_work():
        for ev in sched.step():
            if ev.id not in order:
                order.append(ev.id)
    assert order == [*before, ids[1], ids[2], behind]        # one at a time: an answer that finds no slot waits ahead of everybody
    assert eng.cache.free_pages() == eng.cache.total_pages()


def test_the_last_two_of_a_waiting_group():
    eng = ForkingEngine(pages=60)
    sched = Scheduler(eng, EngineOptions())
    ids = sched.add_samples(Request([4, 5, 6, 7], max_tokens=3), 2)
    other = sched.add(Request([1, 2], max_tokens=3))
    sched.cancel(ids[0])
    assert list(sched.waiting) == [ids[1], other] and not sched.answers
    out = run(sched)
    assert out[ids[1]] == alone([4, 5, 6, 7], 3) and out[other] == alone([1, 2], 3)


@pytest.mark.parametrize("steps", [1, 2])
def test_a_running_group_s_next_answer_comes_ahead_of_everybody(steps):
    eng = ForkingEngine(pages=60)
    sched = Scheduler(eng, EngineOptions(max_sequences=1, max_pass_tokens=2))
    ids = sched.add_samples(Request([4, 5, 6, 7, 8, 9, 10], max_tokens=3), 3)
    other = sched.add(Request([1, 2], max_tokens=3))
    for _ in range(steps):
        sched.step()
    sched.cancel(ids[0])
    assert list(sched.waiting) == [ids[1], other]
    out = run(sched)
    assert all(out[i] == alone([4, 5, 6, 7, 8, 9, 10], 3) for i in ids[1:]) and out[other] == alone([1, 2], 3)
