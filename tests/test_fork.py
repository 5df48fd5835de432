"""Forked sequences: pages held together, their bookkeeping, and the scheduler's answers to one prompt, on the CPU."""
import random

import numpy as np
import pytest

from kapel_b200.cache import CacheFull, CacheManager, CacheNeeds, PagedKV, StateSpec
from kapel_b200.engine.batch import SHARED_BYTES, SHARED_POSITIONS_32, sharing_of
from kapel_b200.engine.scheduler import EngineOptions, Request, Scheduler
from kapel_b200.sampling import Sampling
from test_scheduler import FakeEngine, StagingEngine


def manager(pages=20, window=24, max_sequences=4):
    return CacheManager({0: CacheNeeds(PagedKV(2, 16, window)), 1: CacheNeeds(PagedKV(2, 16, None))}, 16, pages, max_sequences)


def feed(m, seq, n):
    p = m.plan([(seq, n)])
    m.commit(p)
    return p


def test_whole_pages_are_held_together_and_the_last_one_is_copied():
    m = manager(window=64)
    m.add_sequence("a")
    feed(m, "a", 37)
    before = m.free_pages()
    copies = m.fork("a", "b")
    a, b = [m.page_list("a", g) for g in (0, 1)], [m.page_list("b", g) for g in (0, 1)]
    for g in (0, 1):
        assert a[g][:2] == b[g][:2] and a[g][2] != b[g][2]
    assert copies == [(0, a[0][2], b[0][2]), (1, a[1][2], b[1][2])]
    assert m.length("b") == 37 and m.free_pages() == [n - 1 for n in before]
    m.check()
    pa, pb = feed(m, "a", 1), feed(m, "b", 1)
    assert pa.groups[0].lines[0] != pb.groups[0].lines[0] and pb.positions.tolist() == [37] and pb.fresh.tolist() == [False]
    m.remove_sequence("a")
    m.check()
    assert m.page_list("b", 1)[:2] == a[1][:2]
    m.remove_sequence("b")
    assert m.free_pages() == [20, 20]
    m.check()


def test_a_full_last_page_needs_no_copy():
    m = manager()
    m.add_sequence("a")
    feed(m, "a", 32)
    assert m.fork("a", "b") == []
    feed(m, "a", 1), feed(m, "b", 1)
    assert m.page_list("a", 1)[2] != m.page_list("b", 1)[2]
    m.check()


def test_a_window_s_pages_go_back_when_the_last_holder_has_passed_them():
    m = manager(window=24)
    m.add_sequence("a")
    feed(m, "a", 40)
    assert m.page_list("a", 0)[0] == -1
    m.fork("a", "b")
    free = m.free_pages()[0]
    feed(m, "a", 20)
    assert m.page_list("a", 0)[1] == -1 and m.page_list("b", 0)[1] >= 0
    m.check()
    taken = len(m.page_list("a", 0)) - 3
    assert m.free_pages()[0] == free - taken                 # page 1 is still b's; both still need their own page 2
    feed(m, "b", 20)
    assert m.page_list("b", 0)[1] == -1 and m.free_pages()[0] == free - 2 * taken + 1
    m.check()


def test_what_cannot_be_forked_takes_nothing():
    m = manager(pages=3, max_sequences=3)
    m.add_sequence("a")
    with pytest.raises(ValueError, match="holds nothing"):
        m.fork("a", "b")
    with pytest.raises(KeyError):
        m.fork("x", "b")
    feed(m, "a", 20)
    m.fork("a", "b")
    with pytest.raises(ValueError, match="already"):
        m.fork("a", "b")
    with pytest.raises(CacheFull):                           # the third copy of the last page finds none
        m.fork("a", "c")
    assert "c" not in m and m.free_slots() == 1
    m.check()
    m.remove_sequence("b")
    m.fork("a", "c")
    m2 = manager(max_sequences=1)
    m2.add_sequence("a")
    feed(m2, "a", 3)
    with pytest.raises(CacheFull):
        m2.fork("a", "b")
    m2.check()


def test_a_step_planned_before_the_fork_may_still_go_or_be_taken_back():
    for commit in (True, False):
        m = manager()
        m.add_sequence("a")
        feed(m, "a", 16)
        p = m.plan([("a", 1)])
        m.fork("a", "b")
        assert m.length("b") == 16 and len(m.page_list("b", 1)) == 1
        m.commit(p) if commit else m.abort(p)
        feed(m, "b", 1)
        feed(m, "a", 1)
        m.check()


def test_rows_that_share_are_told():
    m = manager(pages=200, max_sequences=8)
    for s in "ax":
        m.add_sequence(s)
        feed(m, s, 40)
    assert m.shared_runs(["a", "x"]) is None
    m.fork("a", "b"), m.fork("a", "c")
    ids, lengths = m.shared_runs(["x", "a", "b", "c"])
    assert lengths.tolist() == [0, 32, 32, 32] and len(set(ids[1:].tolist())) == 1 and ids[0] != ids[1]
    ids, lengths = m.shared_runs(["a", "x", "b", "c"])       # "a" stands alone
    assert lengths.tolist() == [0, 0, 32, 32]
    p = m.plan([(s, 1) for s in "abc"])
    assert p.share is not None and p.share[1].tolist() == [32, 32, 32]
    p.line_bytes = SHARED_BYTES // 64                        # the three rows need 64 positions less
    assert sharing_of(p) is p.share
    p.line_bytes = SHARED_BYTES // 64 - 1
    assert sharing_of(p) is None
    p.item_bytes = 4
    assert (sharing_of(p) is not None) == (64 >= SHARED_POSITIONS_32 * 9)
    m.abort(p)
    assert m.plan([("a", 2), ("b", 1)]).share is None        # not a step of single tokens
    m2 = manager(pages=200, max_sequences=8)
    m2.add_sequence("a")
    feed(m2, "a", 4 * SHARED_POSITIONS_32 + 5)
    m2.fork("a", "b")
    p = m2.plan([("a", 1), ("b", 1)])
    p.item_bytes = 4
    assert sharing_of(p) is p.share
    m2.abort(p)
    m2.remove_sequence("a")
    assert m2.shared_runs(["b"]) is None
    short = manager()
    short.add_sequence("a")
    feed(short, "a", 9)
    short.fork("a", "b")
    assert short.shared_runs(["a", "b"]) is None             # no whole page


def test_random_orders_lose_no_page():
    rng = random.Random(3)
    for _ in range(60):
        m = manager(pages=rng.randint(6, 40), window=rng.choice([8, 24, 60]), max_sequences=rng.randint(2, 6))
        live, names = [], 0
        for _ in range(80):
            what = rng.random()
            try:
                if what < 0.2 or not live:
                    m.add_sequence(names)
                    live.append(names)
                    names += 1
                elif what < 0.45:
                    m.fork(rng.choice(live), names)
                    live.append(names)
                    names += 1
                elif what < 0.6:
                    m.remove_sequence(live.pop(rng.randrange(len(live))))
                else:
                    p = m.plan([(s, rng.randint(1, 20)) for s in rng.sample(live, rng.randint(1, len(live)))])
                    m.commit(p) if rng.random() < 0.8 else m.abort(p)
            except (CacheFull, ValueError):
                pass
            m.check()
        for s in live:
            m.remove_sequence(s)
        assert m.free_pages() == m.total_pages()


class ForkingEngine(FakeEngine):
    forks = 0

    def fork(self, seq_id, new_ids):
        made = []
        try:
            for n in new_ids:
                self.cache.fork(seq_id, n)
                made.append(n)
        except CacheFull:
            for n in made:
                self.cache.remove_sequence(n)
            raise
        for n in new_ids:
            self.fed[n] = list(self.fed[seq_id])
        self.forks += len(new_ids)


class ForkingStagingEngine(ForkingEngine, StagingEngine):
    pass


def alone(prompt, n):
    seq = list(prompt)
    for _ in range(n):
        seq.append(FakeEngine.next_token(seq))
    return seq[len(prompt):]


def run(sched, limit=2000):
    out = {}
    for _ in range(limit):
        if not sched.has_work():
            return out
        for ev in sched.step():
            assert ev.finish != "error", ev.error
            out.setdefault(ev.id, []).append(ev.token)
        sched.cache.check()
    raise AssertionError("the scheduler does not come to an end")


@pytest.mark.parametrize("kind", [ForkingEngine, ForkingStagingEngine])
@pytest.mark.parametrize("prompt_len,n,budget", [(1, 3, 64), (2, 3, 64), (17, 1, 64), (17, 4, 64), (33, 4, 5), (100, 5, 32)])
def test_every_answer_is_the_one_given_alone(kind, prompt_len, n, budget):
    eng = kind(pages=60, window=24, max_sequences=8)
    sched = Scheduler(eng, EngineOptions(max_pass_tokens=budget))
    prompt = [(3 * i + 1) % 50 for i in range(prompt_len)]
    other = sched.add(Request([4, 5, 6], max_tokens=20))
    ids = sched.add_samples(Request(prompt, max_tokens=12), n)
    assert len(set(ids)) == n
    out = run(sched)
    assert out[other] == alone([4, 5, 6], 20)
    for rid in ids:
        assert out[rid] == alone(prompt, 12)
    assert eng.cache.free_pages() == eng.cache.total_pages() and not sched.answers
    if prompt_len > 1 and n > 1:
        assert eng.forks == n - 1
        assert sum(c for p in eng.passes for r, c in p if r in ids) == prompt_len - 1 + n * 12       # the prompt once, then a token a step


def test_answers_draw_with_seeds_of_their_own():
    eng = ForkingEngine(pages=40)
    sched = Scheduler(eng, EngineOptions())
    ids = sched.add_samples(Request([1, 2, 3], sampling=Sampling(temperature=1.0, seed=7)), 3)
    assert [sched.entries[r].request.sampling.seed for r in ids] == [7, 8, 9]


def test_answers_beyond_the_slots_and_pages_wait_and_come():
    prompt = [(7 * i) % 50 for i in range(40)]
    for pages, slots in ((60, 3), (9, 8), (7, 8)):
        eng = ForkingEngine(pages=pages, max_sequences=slots)
        sched = Scheduler(eng, EngineOptions())
        ids = sched.add_samples(Request(prompt, max_tokens=25), 7)
        out = run(sched)
        assert all(out[r] == alone(prompt, 25) for r in ids)
        assert eng.cache.free_pages() == eng.cache.total_pages()
        if pages == 60:                                      # three at a time: the prompt for each group once
            assert sum(c for p in eng.passes for r, c in p) == 3 * 39 + 7 * 25


def test_an_engine_without_fork_computes_each():
    eng = FakeEngine(pages=60)
    sched = Scheduler(eng, EngineOptions())
    ids = sched.add_samples(Request([1, 2, 3], max_tokens=4), 3)
    out = run(sched)
    assert all(out[r] == alone([1, 2, 3], 4) for r in ids)
    with pytest.raises(ValueError):
        sched.add_samples(Request([1, 2, 3]), 0)


def test_cancelled_answers():
    prompt = [(7 * i) % 50 for i in range(40)]
    for when in (0, 1, 3):
        for which in (0, 1, 3):
            eng = ForkingEngine(pages=60)
            sched = Scheduler(eng, EngineOptions(max_pass_tokens=16))
            ids = sched.add_samples(Request(prompt, max_tokens=6), 4)
            for _ in range(when):
                sched.step()
            sched.cancel(ids[which])
            out = run(sched)
            assert all(out[r] == alone(prompt, 6) for r in ids if r != ids[which])
            assert eng.cache.free_pages() == eng.cache.total_pages()
    eng = ForkingEngine(pages=60)
    sched = Scheduler(eng, EngineOptions(max_pass_tokens=16))
    ids = sched.add_samples(Request(prompt, max_tokens=6), 4)
    sched.step()
    for r in ids:
        sched.cancel(r)
    assert not sched.has_work() and not sched.answers and eng.cache.free_pages() == eng.cache.total_pages()


def test_a_prompt_that_can_never_run_ends_all_its_answers():
    eng = ForkingEngine(pages=2)
    sched = Scheduler(eng, EngineOptions())
    ids = sched.add_samples(Request(list(range(50)), max_tokens=6), 3)
    events = sched.step()
    assert [e.id for e in events] == ids and all(e.finish == "error" for e in events) and not sched.has_work()


def test_a_fork_that_fails_ends_what_runs_and_loses_no_answer():
    class Broken(ForkingEngine):
        def fork(self, seq_id, new_ids):
            if not self.forks:
                self.forks = 1
                raise MemoryError("injected")
            super().fork(seq_id, new_ids)

    eng = Broken(pages=60)
    sched = Scheduler(eng, EngineOptions())
    ids = sched.add_samples(Request([1, 2, 3, 4], max_tokens=4), 3)
    out = {}
    while sched.has_work():
        for ev in sched.step():
            out.setdefault(ev.id, []).append(ev.finish if ev.finish == "error" else ev.token)
    assert out[ids[0]] == ["error"] and all(out[r] == alone([1, 2, 3, 4], 4) for r in ids[1:])
    assert eng.cache.free_pages() == eng.cache.total_pages()


def test_the_command_line_refuses_no_answers():
    from kapel_b200.cli import main

    assert main(["run", "somewhere", "--tokens", "1,2", "--samples", "0"]) == 2
