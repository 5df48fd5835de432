"""Nuclei whose border lies within 1e-10 of top_p, where the roundings of hundreds of thousands of small weights would show, against the definition with 64 bits
of mantissa.

On the device a weight that decides the cut is off by at most 2^-53 of the likeliest token's, and by some 1e-14 of itself: 256,000 of them by 2.9e-11 of the
likeliest at the worst, which is less than that of the whole. So a top_p 1e-10 of itself beyond a border is on the right side of it."""
import numpy as np
import pytest

from test_gpu_sample_cold import exact_token
from test_gpu_sample_filtered import device_tokens

VOCAB = 256000


def compare(rows, settings):
    got, want = device_tokens(np.stack(rows), settings), [exact_token(r, *s) for r, s in zip(rows, settings)]
    assert got == want, [(i, g, w, settings[i]) for i, (g, w) in enumerate(zip(got, want)) if g != w]


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1e-10, -1e-10])
@pytest.mark.parametrize("tail,rows", [(-31.4, 2), (-31.4, 20), (-31.4, 70), (-34.9, 2), (-36.3, 2), (-36.9, 20)])      # eight blocks a row and four
def test_many_weights_next_to_nothing(tail, rows, off):
    """Weights of 1 and 0.5 and 255,998 of about 2^-45.3, 2^-50.4, 2^-52.4 (more than half a unit) or 2^-53.2 (less): whether the second token is left depends on all of them."""
    rng = np.random.default_rng(int(-10 * tail))
    logits, settings = [], []
    for i in range(rows):
        row = np.full(VOCAB, tail, np.float32)
        a, b = np.sort(rng.choice(VOCAB, 2, replace=False))
        row[a], row[b] = 0.0, np.log(0.5)
        logits.append(row)
        w = np.exp(row.astype(np.longdouble))
        share = w[a] / w.sum()
        settings.append((1.0, 0, float(share * (1 + np.longdouble(off))), 0.0, 0.99))
    compare(logits, settings)


@pytest.mark.gpu
@pytest.mark.parametrize("off", [1e-10, -1e-10])
@pytest.mark.parametrize("temperature", [0.05, 0.3, 1.0])
@pytest.mark.parametrize("top_k", [0, 100000])
def test_borders_of_rows_as_models_give_them(top_k, temperature, off):
    """The draw lands on the token at the border where that is left."""
    rng = np.random.default_rng(int(100 * temperature) + top_k)
    logits, settings = [], []
    for share in (0.5, 0.9, 0.95, 0.99, 0.9999):
        for _ in range(4):
            row = rng.normal(0.0, 2.0, VOCAB).astype(np.float32)
            w = np.exp((row.astype(np.longdouble) - np.longdouble(row.max())) / np.longdouble(temperature))
            order = np.argsort(-row, kind="stable")[: top_k or VOCAB]
            upto = np.cumsum(w[order])
            j = int(np.searchsorted(upto, share * upto[-1]))
            kept = np.sort(order[: j + 2])                   # with the token behind the border
            before = np.cumsum(w[kept]) - w[kept]
            at = int(np.searchsorted(kept, order[j + 1]))
            logits.append(row)
            settings.append((temperature, top_k, float(upto[j] / upto[-1] * (1 + np.longdouble(off))), 0.0, float((before[at] + w[order[j + 1]] / 2) / w[kept].sum())))
    compare(logits, settings)
