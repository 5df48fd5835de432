"""The filtered draw on the device against the host sampler, which chooses in 64 bits by the same rules."""
import ctypes

import numpy as np
import pytest
import torch

from kapel_b200.sampling import Sampler, Sampling


class _Given(Sampler):
    """The host's chooser with a given uniform number: its distribution, walked as its draw walks it."""

    def pick(self, row, u):
        token, p = self.distribution(row, (), 0)
        if token is not None:
            return token
        total = np.cumsum(p)
        over = np.flatnonzero((total > u) & (p > 0))
        return int(over[0]) if over.size else int(np.flatnonzero(p > 0)[-1])


def host_tokens(logits, settings):
    return [_Given(Sampling(temperature=t, top_k=k, top_p=p, min_p=m)).pick(row, u) for row, (t, k, p, m, u) in zip(logits, settings)]


def device_tokens(logits, settings):
    from kapel_b200 import kernels as K

    f = lambda j: torch.tensor([s[j] for s in settings], dtype=torch.float64, device="cuda")
    k = torch.tensor([s[1] for s in settings], dtype=torch.int32, device="cuda")
    return K.sample_filtered(torch.from_numpy(np.ascontiguousarray(logits, np.float32)).cuda(), f(0), k, f(2), f(3), f(4)).cpu().tolist()


def exact_token(row, temperature, top_k, top_p, min_p, u):
    """The definition for rows of few distinct values, where a share of the whole may be reached exactly: 5,000 equal tokens hold 0.37 after
    1,850 of them, but 1,850 roundings of 1 / 5,000 added up one after the other (as the host does) come to less. Weights of the
    64-bit type, sums and products with 64 bits of mantissa: whole numbers of equal weights stay whole."""
    x = row.astype(np.float64) / temperature
    alive = np.arange(x.size)
    if 0 < top_k < x.size:
        alive = alive[x >= np.sort(x)[::-1][top_k - 1]]
    w = np.exp(x - x.max()).astype(np.longdouble)
    if top_p < 1.0:
        order = alive[np.argsort(-x[alive], kind="stable")]
        before = np.cumsum(w[order]) - w[order]
        alive = np.sort(order[before < np.longdouble(top_p) * w[order].sum()])
    alive = alive[w[alive] >= np.longdouble(min_p) * w[alive].max()]
    total = np.cumsum(w[alive])
    return int(alive[np.flatnonzero(total > np.longdouble(u) * total[-1])[0]])


def check(logits, settings):
    got, want = device_tokens(logits, settings), host_tokens(np.asarray(logits, np.float32), settings)
    assert got == want, [(i, g, w, settings[i]) for i, (g, w) in enumerate(zip(got, want)) if g != w]


ALL = [(t, k, p, m) for t in (0.3, 1.0, 2.5) for k in (0, 1, 7, 100000) for p in (1.0, 0.9, 0.3) for m in (0.0, 0.1)]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [1, 2, 31, 257, 1000, 8191, 8193, 16385, 50257, 256000])
def test_every_combination_of_filters(vocab):
    rng = np.random.default_rng(vocab)
    logits = rng.normal(0.0, 2.0, (len(ALL), vocab))
    check(logits, [(*s, float(u)) for s, u in zip(ALL, rng.random(len(ALL)))])


@pytest.mark.gpu
@pytest.mark.parametrize("spread", [1e-3, 0.5, 8.0, 200.0])
@pytest.mark.parametrize("vocab", [3000, 70001])
def test_flat_and_peaked_rows(spread, vocab):
    rng = np.random.default_rng(int(spread * 1000))
    logits = rng.normal(0.0, spread, (len(ALL), vocab))
    check(logits, [(*s, float(u)) for s, u in zip(ALL, rng.random(len(ALL)))])


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [64, 5000, 40000])
def test_ties(vocab):
    """Few distinct values: the k-th's ties stay, the nucleus takes the lower index first. More equal tokens than the list holds."""
    rng = np.random.default_rng(5)
    logits = np.concatenate([rng.integers(-2, 3, (24, vocab)), np.zeros((12, vocab)), np.where(rng.random((12, vocab)) < 0.5, 0.0, -0.0),
                             np.full((12, vocab), 7.25)]).astype(np.float32)
    kinds = [(1.0, 0, 0.37, 0.0), (0.7, 5, 1.0, 0.0), (1.0, 3000, 0.61, 0.0), (1.3, 0, 0.9, 0.5), (1.0, 0, 1.0, 1.0), (0.5, 0, 0.02, 0.0)]
    settings = [(*kinds[i % 6], float(u)) for i, u in enumerate(rng.random(len(logits)))]
    got, want = device_tokens(logits, settings), [exact_token(row, *s) for row, s in zip(logits, settings)]
    assert got == want, [(i, g, w, settings[i]) for i, (g, w) in enumerate(zip(got, want)) if g != w]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [50257, 256000])
@pytest.mark.parametrize("rows", [1, 9, 20, 45, 150])
def test_rows_by_themselves_and_many(rows, vocab):
    """How many blocks a row has depends on the number of rows."""
    rng = np.random.default_rng(rows)
    logits = rng.normal(0.0, 2.0, (rows, vocab)) + rng.choice([0.0, 20.0, -1000.0], (rows, 1))
    kinds = [(0.8, 0, 0.99, 0.0), (1.0, 5000, 1.0, 0.0), (1.5, 0, 0.9999, 0.0), (0.7, 0, 1.0, 0.001), (1.0, 30000, 0.97, 0.0), (2.0, 0, 0.5, 0.0), (0.3, 0, 1.0, 0.0), (0.0, 7, 0.5, 0.0)]
    check(logits, [(*kinds[(i + rows) % len(kinds)], float(u)) for i, u in enumerate(rng.random(rows))])


@pytest.mark.gpu
@pytest.mark.parametrize("rows", [6, 60])
def test_ties_in_large_rows(rows):
    """81 values, some 3,000 tokens of each."""
    rng = np.random.default_rng(rows + 2)
    logits = (rng.integers(-40, 41, (rows, 256000)) / 8.0).astype(np.float32)
    kinds = [(1.0, 0, 0.37, 0.0), (2.0, 0, 0.999, 0.0), (1.0, 3000, 0.61, 0.0), (30.0, 0, 0.9, 0.5), (1.0, 70000, 1.0, 0.0), (10.0, 0, 0.02, 0.0)]
    settings = [(*kinds[i % 6], float(u)) for i, u in enumerate(rng.random(rows))]
    got, want = device_tokens(logits, settings), [exact_token(row, *s) for row, s in zip(logits, settings)]
    assert got == want, [(i, g, w, settings[i]) for i, (g, w) in enumerate(zip(got, want)) if g != w]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [20000, 256000])
def test_values_far_apart(vocab):
    """Of both signs, from 1e-40 to 1e4 in size: neither equal steps of the value nor of its bits part them evenly."""
    rng = np.random.default_rng(21)
    logits = (rng.choice([-1.0, 1.0], (24, vocab)) * 10.0 ** rng.uniform(-40.0, 4.0, (24, vocab))).astype(np.float32)
    logits[12:] = -np.abs(logits[12:])                       # the largest is next to nothing, and half of all lie within 1e-18 of it
    kinds = [(2000.0, 0, 0.9, 0.0), (1.0, 0, 0.9999999, 0.0), (1e4, 0, 0.3, 0.0), (100.0, vocab // 2, 0.8, 0.0), (1e30, 0, 0.7, 0.0), (1e-20, 0, 0.6, 0.0)]
    settings = [(*kinds[i % 6], float(u)) for i, u in enumerate(rng.random(24))]
    got, want = device_tokens(logits, settings), [exact_token(row, *s) for row, s in zip(logits, settings)]
    assert got == want, [(i, g, w, settings[i]) for i, (g, w) in enumerate(zip(got, want)) if g != w]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [500, 30000, 256000])
def test_a_token_far_above_the_rest(vocab):
    """The k-th largest lies where no weight counts any more, among masked tokens or not; the nucleus is one token, or a temperature brings the rest back."""
    rng = np.random.default_rng(vocab)
    logits = rng.normal(0.0, 2.0, (36, vocab)).astype(np.float32)
    logits[:, vocab // 3] = np.repeat([30.0, 300.0, 1e30], 12)
    logits[6:12][rng.random((6, vocab)) < 0.97] = np.finfo(np.float32).min
    logits[18:24][rng.random((6, vocab)) < 0.97] = -np.inf
    kinds = [(0.5, 64, 0.9, 0.0), (0.5, 300, 1.0, 0.0), (50.0, 64, 0.95, 0.0), (50.0, 5000, 0.8, 0.0), (0.3, 1000, 0.999999, 0.01), (400.0, 20, 1.0, 0.0)]
    check(logits, [(*kinds[i % 6], float(u)) for i, u in enumerate(rng.random(36))])


@pytest.mark.gpu
def test_ends_of_the_uniform_number_and_of_the_settings():
    rng = np.random.default_rng(9)
    logits = rng.normal(0.0, 2.0, (40, 9001))
    us = [0.0, 1e-300, np.nextafter(1.0, 0.0), 0.5]
    kinds = [(1.0, 0, 1.0, 0.0), (1.0, 50, 0.9, 0.0), (1.0, 0, 0.9999999, 0.0), (1.0, 0, 1e-12, 0.0), (1e-3, 0, 0.9, 0.0), (100.0, 0, 0.9, 0.0),
             (1.0, 9001, 0.5, 0.0), (1.0, 9000, 1.0, 0.0), (0.0, 5, 0.5, 0.1), (1.0, 0, 1.0, 1.0)]
    check(logits, [(*k, u) for k in kinds for u in us])


@pytest.mark.gpu
def test_masked_tokens_are_never_chosen():
    """Tokens at -inf or at the type's lowest value, and rows that leave one token or none."""
    rng = np.random.default_rng(11)
    for vocab in (40, 20000):
        logits = rng.normal(0.0, 2.0, (36, vocab)).astype(np.float32)
        logits[:12][rng.random((12, vocab)) < 0.9] = -np.inf
        logits[12:24][rng.random((12, vocab)) < 0.9] = np.finfo(np.float32).min
        logits[24:30] = -np.inf
        logits[24:27, 17] = 1.0
        logits[27:30] = np.finfo(np.float32).min
        logits[30:33] = -np.inf
        logits[30:33, vocab - 1] = -5.0
        logits[33:36] = -np.inf
        kinds = [(1.0, 0, 1.0, 0.0), (1.0, 10, 0.9, 0.0), (0.8, 0, 0.8, 0.05)]
        check(logits, [(*kinds[i % 3], float(u)) for i, u in enumerate(rng.random(36))])


@pytest.mark.gpu
def test_logits_that_are_no_numbers():
    rng = np.random.default_rng(12)
    for vocab in (40, 20000):
        logits = rng.normal(0.0, 2.0, (12, vocab)).astype(np.float32)
        logits[:6, 3] = np.nan
        logits[3:6] = np.nan
        logits[5, 8] = -1.0
        logits[6:9, vocab // 2 :] = np.inf
        logits[9:, 0] = np.nan
        logits[9:, 9] = np.inf
        kinds = [(1.0, 0, 1.0, 0.0), (1.0, 10, 0.9, 0.0), (0.8, 0, 0.8, 0.05)]
        check(logits, [(*kinds[i % 3], 0.4) for i in range(12)])


@pytest.mark.gpu
def test_settings_that_leave_nothing_give_token_0():
    logits = np.random.default_rng(13).normal(0.0, 1.0, (6, 5000))
    settings = [(1.0, 0, 0.0, 0.0, 0.5), (1.0, 0, -1.0, 0.0, 0.5), (1.0, 0, 1.0, 1.5, 0.5), (1.0, 5, 0.0, 0.0, 0.5), (float("nan"), 0, 1.0, 0.0, 0.5),
                (1.0, 3, 0.9, 2.0, 0.5)]
    assert device_tokens(logits, settings) == [0] * 6
    assert device_tokens(logits, [(0.0, 0, 0.0, 2.0, 0.5)] * 6) == np.argmax(logits.astype(np.float32), axis=1).tolist()     # greedy comes first


@pytest.mark.gpu
def test_a_vocabulary_beyond_the_cluster_s_shared_memory():
    from kapel_b200 import kernels as K

    rng = np.random.default_rng(14)
    logits = rng.normal(0.0, 1.0, (12, K.SAMPLE_FILTERED_VOCAB))
    kinds = [(1.0, 0, 1.0, 0.0), (1.0, 40, 0.9, 0.0), (0.8, 0, 0.95, 0.0), (1.0, 100000, 0.7, 0.01)]
    check(logits, [(*kinds[i % 4], float(u)) for i, u in enumerate(rng.random(12))])


@pytest.mark.gpu
def test_the_draws_follow_the_probabilities():
    """4,096 equidistant numbers over one row: every token is drawn as often as its share of the total, to within the two ends of its interval."""
    rng = np.random.default_rng(15)
    row = rng.normal(0.0, 1.5, 60)
    n = 4096
    settings = [(0.9, 20, 0.9, 0.0, (i + 0.5) / n) for i in range(n)]
    got = np.bincount(device_tokens(np.tile(row, (n, 1)), settings), minlength=60)
    _, p = Sampler(Sampling(temperature=0.9, top_k=20, top_p=0.9)).distribution(row.astype(np.float32), (), 0)
    assert np.abs(got - n * p).max() <= 1.0 + 1e-6


@pytest.mark.gpu
def test_a_recorded_choice_and_another_stream():
    from kapel_b200 import kernels as K

    rng = np.random.default_rng(16)
    logits = torch.zeros((3, 30000), dtype=torch.float32, device="cuda")
    f = lambda *v: torch.tensor(v, dtype=torch.float64, device="cuda")
    t, k, p, m, u = f(1.0, 0.7, 1.2), torch.tensor([0, 40, 0], dtype=torch.int32, device="cuda"), f(0.9, 1.0, 1.0), f(0.0, 0.0, 0.1), f(0.2, 0.5, 0.8)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.stream(side):
        K.sample_filtered(logits, t, k, p, m, u)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = K.sample_filtered(logits, t, k, p, m, u)
    for _ in range(3):
        fresh = rng.normal(0.0, 2.0, (3, 30000)).astype(np.float32)
        logits.copy_(torch.from_numpy(fresh))
        graph.replay()
        assert out.cpu().tolist() == host_tokens(fresh, [(1.0, 0, 0.9, 0.0, 0.2), (0.7, 40, 1.0, 0.0, 0.5), (1.2, 0, 1.0, 0.1, 0.8)])


@pytest.mark.gpu
def test_two_streams_at_once():
    from kapel_b200 import kernels as K

    rng = np.random.default_rng(9)
    f = lambda a: torch.tensor(a, dtype=torch.float64, device="cuda")
    cases = []
    for rows, vocab in ((24, 256000), (5, 3001)):
        cases.append((torch.from_numpy(rng.normal(0.0, 2.0, (rows, vocab)).astype(np.float32)).cuda(), f([0.9] * rows), torch.tensor([i % 3 * 40 for i in range(rows)], dtype=torch.int32, device="cuda"),
                      f([0.95] * rows), f([0.01] * rows), f(rng.random(rows))))
    want = [K.sample_filtered(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for j, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[j].append(K.sample_filtered(*cases[j]))
    torch.cuda.synchronize()
    for j in range(2):
        for x in got[j]:
            assert torch.equal(x, want[j])


@pytest.mark.gpu
def test_no_rows():
    from kapel_b200 import kernels as K

    e = torch.empty((0,), dtype=torch.float64, device="cuda")
    assert K.sample_filtered(torch.empty((0, 10), device="cuda"), e, e.int(), e, e, e).shape == (0,)


@pytest.mark.gpu
def test_what_is_refused():
    from kapel_b200 import kernels as K

    logits = torch.zeros((2, 100), device="cuda")
    f = torch.ones((2,), dtype=torch.float64, device="cuda")
    k = torch.zeros((2,), dtype=torch.int32, device="cuda")
    good = dict(logits=logits, temperature=f, top_k=k, top_p=f, min_p=f, uniform=f)
    K.sample_filtered(**good)
    for bad in (dict(logits=logits.double()), dict(logits=logits.t().contiguous().t()), dict(logits=logits[0]), dict(temperature=f.float()), dict(top_k=f),
                dict(top_k=k.long()), dict(top_p=f[:1]), dict(min_p=f.cpu()), dict(uniform=f.view(2, 1)),
                dict(logits=torch.zeros((2, K.SAMPLE_FILTERED_VOCAB + 1), device="cuda"))):
        with pytest.raises(K.KernelError):
            K.sample_filtered(**{**good, **bad})


def test_the_launcher_refuses_without_a_gpu():
    try:
        from kapel_b200 import kernels as K

        lib = K.library()
    except Exception as err:
        pytest.skip(f"the CUDA library cannot be built or loaded here: {err}")
    vp, i32 = ctypes.c_void_p, ctypes.c_int
    call = lib.kb_sample_filtered
    for args, word in (((4096, 4096, 4096, 4096, 4096, 4096, 4096, -1, 100), "rows -1"), ((4096, 4096, 4096, 4096, 4096, 4096, 4096, 1, 0), "vocab 0"),
                       ((4096, 4096, 4096, 4096, 4096, 4096, 4096, 1, (1 << 19) + 1), "vocabulary"), ((4096, 4096, None, 4096, 4096, 4096, 4096, 1, 100), "null"),
                       ((4096, 4096, 4096, 4096, 4096, 4096, 4096, 1 << 29, 100), "too many")):
        assert call(*[vp(a) for a in args[:7]], *[i32(a) for a in args[7:]], vp(None)) != 0
        assert word in lib.kb_last_error().decode()


@pytest.mark.gpu
def test_a_model_with_filters_runs_ahead_and_gives_the_host_s_tokens():
    """Requests with filters are chosen on the device, ahead of the host; the tokens are those of the host's chooser on the same logits."""
    from kapel_b200 import Model
    from kapel_b200.engine.scheduler import Request
    from helpers import TINY_A

    def tokens(on_device):
        model = Model.random(TINY_A, seed=3, dtype="bf16", max_tokens_cached=4096, max_sequences=8)
        sched = model.scheduler(max_sequences=8)
        if not on_device:
            sched._choose_on_device = lambda *a: None
        kinds = [dict(temperature=0.8, top_k=50), dict(temperature=1.0, top_p=0.9, min_p=0.02), dict(temperature=0.9), dict(), dict(temperature=1.2, min_p=0.1, top_k=9)]
        out = {sched.add(Request([5 + i, 7, 11], Sampling(seed=i, **kinds[i % 5]), max_tokens=20, ignore_eos=True)): [] for i in range(5)}
        while sched.has_work():
            for ev in sched.step():
                assert ev.error is None, ev.error
                out[ev.id].append(ev.token)
        return list(out.values()), sched.ahead_passes

    device, ahead = tokens(True)
    host, none_ahead = tokens(False)
    assert device == host and ahead > 10 and none_ahead == 0
