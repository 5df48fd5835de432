"""Filtered draws of rows so cold, or of logits so large, that the neighbouring floats of the largest logit are far apart in weight: against the
definition with 64 bits of mantissa, the logits' differences taken before the division."""
import numpy as np
import pytest
import torch

from kapel_b200.sampling import Sampling
from test_gpu_sample_filtered import _Given, device_tokens


def exact_token(row, temperature, top_k, top_p, min_p, u):
    x = (row.astype(np.longdouble) - np.longdouble(row.max())) / np.longdouble(temperature)
    alive = np.arange(x.size)
    if 0 < top_k < x.size:
        alive = alive[x >= np.sort(x)[::-1][top_k - 1]]
    w = np.exp(x)
    if top_p < 1.0:
        order = alive[np.argsort(-x[alive], kind="stable")]
        before = np.cumsum(w[order]) - w[order]
        alive = np.sort(order[before < np.longdouble(top_p) * w[order].sum()])
    alive = alive[w[alive] >= np.longdouble(min_p) * w[alive].max()]
    total = np.cumsum(w[alive])
    return int(alive[np.flatnonzero(total > np.longdouble(u) * total[-1])[0]])


FILTERS = [(0, 1.0, 0.0), (0, 0.9, 0.0), (5000, 1.0, 0.0), (0, 1.0, 0.01), (5000, 0.7, 0.0), (20, 0.8, 0.0)]


@pytest.mark.gpu
@pytest.mark.parametrize("vocab", [40, 7000, 30000])
@pytest.mark.parametrize("top", [20.0, 1e3, 3e6])
def test_tokens_a_few_float_steps_below_the_largest(top, vocab):
    """0 to 21 steps of a float below the largest, the rest far below: some of the weights lie around 2^-1022, where an exponent put together out of bits would
    leave its field."""
    rng = np.random.default_rng(int(top) + vocab)
    temperatures = [10.0 ** -k for k in range(2, 10)] + [2e-9, 5e-6]
    rows, settings = [], []
    for i, t in enumerate(temperatures):
        for j, (k, p, m) in enumerate(FILTERS):
            row = rng.normal(-top, 1.0, vocab).astype(np.float32)
            at = rng.choice(vocab, 22, replace=False)
            row[at] = (np.float32(top).view(np.int32) - np.arange(22)).astype(np.int32).view(np.float32)
            rows.append(row)
            settings.append((t, k, p, m, float(rng.random())))
    got, want = device_tokens(np.stack(rows), settings), [exact_token(r, *s) for r, s in zip(rows, settings)]
    assert got == want, [(i, g, w, settings[i]) for i, (g, w) in enumerate(zip(got, want)) if g != w]


@pytest.mark.gpu
def test_weights_down_to_the_smallest_the_type_has():
    """A uniform number of 0 takes the first token that has a weight at all: e^-740 is one in 64 bits, e^-747 is none."""
    below = np.float32([-800.0, -747.0, -740.0, -720.0, -709.0, -700.0, -3e38, np.finfo(np.float32).min])
    logits = np.zeros((below.size, 9), np.float32)
    logits[:, 0] = below
    for filters in ((0, 1.0, 0.0), (8, 1.0, 0.0)):
        settings = [(1.0, *filters, 0.0)] * below.size
        assert device_tokens(logits, settings) == [0 if (-745.0 < b and filters[0] == 0) else 1 for b in below]
        assert device_tokens(logits, settings) == [_Given(Sampling(temperature=1.0, top_k=filters[0])).pick(r, 0.0) for r in logits]


@pytest.mark.gpu
@pytest.mark.parametrize("temperature", [1e-30, 1e-36, 1e-38, 1e-40, 5e-324])
def test_the_smallest_temperatures(temperature):
    """Only what ties with the largest is left, whatever the filters."""
    rng = np.random.default_rng(4)
    logits = rng.integers(-3, 4, (12, 5000)).astype(np.float32)
    logits[6:] *= 1e30
    for k, p, m in ((0, 1.0, 0.0), (0, 0.6, 0.0), (3000, 1.0, 0.0), (0, 1.0, 0.5)):
        us = rng.random(12)
        got = device_tokens(logits, [(temperature, k, p, m, float(u)) for u in us])
        for row, token, u in zip(logits, got, us):
            ties = np.flatnonzero(row == row.max())
            kept = ties[: int(np.ceil(p * ties.size))] if p < 1.0 else ties
            assert token == kept[int(u * kept.size)]


@pytest.mark.gpu
def test_the_largest_logits_under_the_highest_temperatures():
    """Differences that 32 bits do not hold, quotients next to nothing: all weights alike."""
    logits = np.full((4, 3000), 3e38, np.float32)
    logits[:, ::2] = -3e38
    us = [0.0, 0.2, 0.6, np.nextafter(1.0, 0.0)]
    assert device_tokens(logits, [(float("inf"), 0, 1.0, 0.0, u) for u in us]) == [int(u * 3000) for u in us]
    # At u = 0.6 the target is the running total of 900 of the 1,500 pairs itself: 0.6 in 64 bits is 2.2e-17 below 3/5, and u times the whole, rounded to 53 bits
    # (up to 2^-54 of it, 5.6e-17), may or may not reach that total, itself a sum of 1,800 roundings. Either side of a border within 1e-12 of u is right.
    for row, u, token in zip(logits, us, device_tokens(logits, [(1e38, 0, 1.0, 0.0, u) for u in us])):
        assert exact_token(row, 1e38, 0, 1.0, 0.0, max(0.0, u - 1e-12)) <= token <= exact_token(row, 1e38, 0, 1.0, 0.0, min(u + 1e-12, np.nextafter(1.0, 0.0)))
