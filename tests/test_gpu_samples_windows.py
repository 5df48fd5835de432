"""A step of forked requests in which only the layers without a window read shared pages once."""
import numpy as np
import pytest

from helpers import TOL, random_tokens, rel_err
from test_gpu_mixed_attention import config
from test_gpu_samples import engine_of, step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("head_dim", [64, 256])
def test_layer_groups_go_by_themselves(head_dim, graphs, monkeypatch):
    """Windows of 48: behind 100 positions the windowed layers see 45 or fewer of the 96 shared ones. Three requests save 192 positions there without a window."""
    from kapel_b200 import kernels as K
    from kapel_b200.engine import batch

    windows, attention = [], K.shared_prefix_attention
    monkeypatch.setattr(K, "shared_prefix_attention", lambda *a, **kw: windows.append(a[8]) or attention(*a, **kw))
    eng = engine_of(config(head_dim, 2, 50.0), "bfloat16", graphs=graphs)
    rng = np.random.default_rng(2)
    prompt = random_tokens(rng, 100, eng.vocab_size)
    tails = {i: random_tokens(rng, 5, eng.vocab_size) for i in "abc"}
    step(eng, ("a", prompt, []))
    eng.fork("a", "bc")
    got = []
    for t, least in enumerate((192, 192, 80, 80, 1 << 40)):  # positions saved from which it pays: the layers without a window, twice, all, twice, none
        monkeypatch.setattr(batch, "SHARED_BYTES", least * eng.cache.line_bytes)
        windows.clear()
        got.append(step(eng, *[(i, [tails[i][t]], [0]) for i in "abc"]))
        if t in (0, 2):
            assert set(windows) == ({None} if t == 0 else {None, 48})
        if t == 4:
            assert not windows
    eng.check()
    if graphs:
        assert {k[2:] for k in eng.graphs.graphs} == {((False, True),), ((True, True),), ()}
    got = np.array(got)
    for at, i in enumerate("abc"):
        step(eng, (f"own {i}", prompt, []))
        want = np.concatenate([step(eng, (f"own {i}", [t], [0])) for t in tails[i]])
        assert rel_err(got[:, at], want) < 2 * TOL["bfloat16"], i            # both sides are off by up to the bound
