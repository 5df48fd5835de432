"""Which groups of layers read shared pages once, by what their windows leave of them, on the CPU."""
import numpy as np
import pytest

from kapel_b200.cache import CacheManager, CacheNeeds, PagedKV
from kapel_b200.engine.batch import SHARED_BYTES, SHARED_POSITIONS_32, sharing_groups, sharing_of


def plan_of(prompt, forks, window, own=1):
    """Requests forked behind `prompt` positions that have fed `own` tokens each, and the step after it; a request of its own at the end."""
    m = CacheManager({0: CacheNeeds(PagedKV(2, 16, window)), 1: CacheNeeds(PagedKV(2, 16, None))}, 16, 4000, forks + 2)
    m.add_sequence(0)
    m.commit(m.plan([(0, prompt)]))
    for i in range(1, forks):
        m.fork(0, i)
    m.add_sequence("own")
    entries = [*range(forks), "own"]
    for _ in range(own):
        m.commit(m.plan([(i, 1) for i in entries]))
    return m.plan([(i, 1) for i in entries])


def bytes_for(positions):
    return -(-SHARED_BYTES // positions)


def test_a_window_counts_what_it_leaves():
    p = plan_of(160, 4, 24)
    assert p.windows == (24, None) and p.row_count.tolist() == [162] * 4 + [2]
    # the windowed layers see 160 - (162 - 24) = 22 of the 160 shared positions a row
    for positions, groups in ((3 * 160, (False, True)), (3 * 22 + 1, (False, True)), (3 * 22, (True, True)), (3 * 160 + 1, None)):
        p.line_bytes = bytes_for(positions)
        assert sharing_groups(p) == groups
        assert sharing_of(p) is (p.share if groups else None)


def test_a_window_that_has_passed_what_is_shared():
    p = plan_of(32, 4, 24, own=30)
    p.line_bytes = SHARED_BYTES
    assert sharing_groups(p) == (False, True)
    p = plan_of(16, 3, 24, own=40)
    p.item_bytes, p.share = 4, (p.share[0], p.share[1])
    assert sharing_groups(p) is None                         # 32 positions saved of 4 requests, and none in the windowed layers


def test_two_requests_are_read_by_themselves_in_bfloat16():
    for forks, pays in ((2, False), (3, True), (8, True)):
        p = plan_of(64, forks, 4096)
        p.line_bytes = SHARED_BYTES
        assert sharing_groups(p) == ((True, True) if pays else None)
    p = plan_of(16 * SHARED_POSITIONS_32, 2, 4096)
    p.item_bytes = 4
    assert sharing_groups(p) == (True, True)


@pytest.mark.parametrize("window", [8, 50, 200, None])
def test_against_counting_position_by_position(window):
    rng = np.random.default_rng(3)
    for _ in range(40):
        lengths, ids, counts = [], [], []
        for run in range(rng.integers(1, 5)):
            shared = 16 * int(rng.integers(0, 12))
            for _ in range(rng.integers(1, 6)):
                lengths.append(shared)
                ids.append(run)
                counts.append(shared + int(rng.integers(1, 90)))
        p = plan_of(20, 2, window)
        p.share = np.asarray(ids, np.int32), np.asarray(lengths, np.int32)
        p.row_count, p.positions = np.asarray(counts, np.int32), np.asarray(counts, np.int32) - 1
        sees = [set(range(max(0, c - window) if window else 0, c)) & set(range(n)) for c, n in zip(counts, lengths)]
        once = sum(len(set().union(*[s for s, i in zip(sees, ids) if i == run])) for run in set(ids))
        saved = sum(map(len, sees)) - once
        for p.line_bytes in (1, bytes_for(max(1, saved)), bytes_for(saved + 1)):
            want = saved > 0 and saved * p.line_bytes >= SHARED_BYTES and saved >= 2 * once
            groups = sharing_groups(p)
            assert (groups is not None and groups[p.windows.index(window)]) == want
