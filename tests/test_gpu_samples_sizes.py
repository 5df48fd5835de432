"""Which head sizes a step of forked requests takes through the attention over shared pages."""
import numpy as np
import pytest
import torch

from helpers import TOL, random_tokens, rel_err
from test_gpu_mixed_attention import config
from test_gpu_samples import engine_of, step


def test_sizes_that_gain():
    try:
        from kapel_b200 import kernels as K

        K.library()
    except Exception as err:
        pytest.skip(f"the CUDA library cannot be built or loaded here: {err}")
    bf, f32 = torch.bfloat16, torch.float32
    for (dtype, *sizes), takes, pays in (((bf, 8, 4, 256, 256, 16), 1, 1), ((bf, 16, 4, 128, 128, 32), 1, 1), ((bf, 4, 4, 64, 64, 16), 1, 1), ((bf, 12, 4, 96, 96, 16), 1, 0),
                                         ((bf, 16, 1, 32, 32, 16), 1, 0), ((bf, 8, 4, 128, 128, 10), 1, 0), ((bf, 8, 2, 128, 64, 16), 1, 1), ((bf, 32, 1, 64, 64, 16), 1, 1),
                                         ((bf, 6, 2, 20, 20, 16), 1, 1), ((f32, 12, 4, 96, 96, 16), 1, 1), ((f32, 8, 4, 256, 256, 16), 1, 1), ((torch.half, 8, 4, 128, 128, 16), 0, 0),
                                         ((bf, 33, 1, 64, 64, 16), 0, 0), ((bf, 9, 4, 64, 64, 16), 0, 0), ((bf, 8, 4, 257, 257, 16), 0, 0)):
        assert K.shared_prefix_takes(dtype, *sizes) == bool(takes) and K.shared_prefix_pays(dtype, *sizes) == bool(pays), (dtype, sizes)


@pytest.mark.gpu
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("head_dim,shared", [(64, True), (128, True), (256, True), (96, False), (32, False)])
def test_a_step_in_bfloat16(head_dim, shared, graphs, monkeypatch):
    from kapel_b200 import kernels as K
    from kapel_b200.engine import batch

    calls, attention = [], K.shared_prefix_attention
    monkeypatch.setattr(K, "shared_prefix_attention", lambda *a, **kw: calls.append(1) or attention(*a, **kw))
    monkeypatch.setattr(batch, "SHARED_BYTES", 1)
    eng = engine_of(config(head_dim, 2, 50.0), "bfloat16", graphs=graphs)
    rng = np.random.default_rng(2)
    prompt = random_tokens(rng, 50, eng.vocab_size)
    tails = {i: random_tokens(rng, 5, eng.vocab_size) for i in "abc"}
    step(eng, ("a", prompt, []))
    eng.fork("a", "bc")
    got = np.array([step(eng, *[(i, [tails[i][t]], [0]) for i in "abc"]) for t in range(5)])
    eng.check()
    assert (len(calls) > 0) == shared
    for at, i in enumerate("abc"):
        step(eng, (f"own {i}", prompt, []))
        want = np.concatenate([step(eng, (f"own {i}", [t], [0])) for t in tails[i]])
        assert rel_err(got[:, at], want) < 2 * TOL["bfloat16"], i            # both sides are off by up to the bound
