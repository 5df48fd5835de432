"""Forked requests and several answers to one prompt on the GPU: every family's layers go on from a fork as if each request had computed its prompt
itself, with shared pages read once where the layer's attention takes them."""
import importlib

import numpy as np
import pytest
import torch

from helpers import TINY, TOL, random_tokens, rel_err

pytestmark = pytest.mark.gpu

FAMILIES = [("gemma2", "A"), ("gemma2", "B")] + [(f, n) for f in ("fusitar", "kofutar", "teluzen", "lokedra", "mukunex", "sopalorn") for n in "ABC"]


def config_of(family, name):
    configs = TINY if family == "gemma2" else importlib.import_module(f"test_gpu_{family}").CONFIGS
    if name not in configs:
        pytest.skip(f"{family} has no configuration {name}")
    return configs[name][0]


def engine_of(config, dtype, **kw):
    from kapel_b200.engine import Engine

    return Engine.random(config, seed=5, dtype=dtype, max_tokens=2048, max_sequences=12, **kw)


def step(eng, *entries):
    from kapel_b200.engine import StepEntry

    return eng.step([StepEntry(i, t, w) for i, t, w in entries]).float().cpu().numpy()


@pytest.mark.parametrize("prompt_len", [16, 41])
@pytest.mark.parametrize("graphs", [True, False])
@pytest.mark.parametrize("shared", [True, False])
@pytest.mark.parametrize("family,name", FAMILIES)
def test_forked_requests_go_on_as_if_alone(family, name, shared, graphs, prompt_len, monkeypatch):
    """32-bit: logits of three forked requests beside one of its own against the same tokens computed without a fork."""
    from kapel_b200.engine import batch

    monkeypatch.setattr(batch, "SHARED_POSITIONS_32", 0 if shared else 1 << 30)
    eng = engine_of(config_of(family, name), "float32", graphs=graphs)
    rng = np.random.default_rng(1)
    prompt = random_tokens(rng, prompt_len, eng.vocab_size)
    tails = {i: random_tokens(rng, 6, eng.vocab_size) for i in ("a", "b", "c", "d")}
    step(eng, ("a", prompt, []))
    step(eng, ("d", prompt[:9], []))
    eng.fork("a", ["b", "c"])
    eng.cache.check()
    got = {i: [] for i in tails}
    for t in range(6):
        for i, row in zip("abcd", step(eng, *[(i, [tails[i][t]], [0]) for i in "abcd"])):
            got[i].append(row)
    eng.check()
    for i in tails:
        want = step(eng, (f"own {i}", (prompt if i != "d" else prompt[:9]) + tails[i], list(range(prompt_len if i != "d" else 9, (prompt_len if i != "d" else 9) + 6))))
        assert rel_err(np.array(got[i]), want) < TOL["float32"], i
        eng.end(f"own {i}")
        eng.end(i)
    eng.cache.check()
    assert eng.cache.free_pages() == eng.cache.total_pages()


@pytest.mark.parametrize("family,name", [("gemma2", "A"), ("gemma2", "B"), ("mukunex", "C"), ("sopalorn", "A"), ("kofutar", "A")])
def test_forked_requests_in_bfloat16(family, name, monkeypatch):
    from kapel_b200.engine import batch

    monkeypatch.setattr(batch, "SHARED_BYTES", 1)
    monkeypatch.setattr(batch, "SHARED_POSITIONS_32", 0)
    eng = engine_of(config_of(family, name), "bfloat16")
    rng = np.random.default_rng(2)
    prompt = random_tokens(rng, 50, eng.vocab_size)
    tails = {i: random_tokens(rng, 5, eng.vocab_size) for i in "abc"}
    step(eng, ("a", prompt, []))
    eng.fork("a", "bc")
    got = np.array([step(eng, *[(i, [tails[i][t]], [0]) for i in "abc"]) for t in range(5)])
    eng.check()
    for at, i in enumerate("abc"):
        step(eng, (f"own {i}", prompt, []))
        want = np.concatenate([step(eng, (f"own {i}", [t], [0])) for t in tails[i]])
        assert rel_err(got[:, at], want) < 2 * TOL["bfloat16"], i            # both sides are off by up to the bound


def test_a_fork_that_finds_no_room_leaves_the_engine_as_it_was(monkeypatch):
    from kapel_b200 import kernels as K
    from kapel_b200.cache import CacheFull

    eng = engine_of(config_of("mukunex", "A"), "float32", pages=8)
    step(eng, ("a", [1] * 20, []))
    before = eng.cache.free_pages()
    with pytest.raises(CacheFull):
        eng.fork("a", [f"n{i}" for i in range(9)])
    assert eng.cache.free_pages() == before and eng.cache.sequences() == ["a"]
    monkeypatch.setattr(K, "copy_rows", lambda *a: (_ for _ in ()).throw(K.KernelError("injected")))
    with pytest.raises(K.KernelError):
        eng.fork("a", ["b"])
    assert eng.cache.free_pages() == before and eng.cache.sequences() == ["a"]
    eng.cache.check()


def test_copied_rows():
    from kapel_b200 import kernels as K

    for shape, dtype in (((7, 3, 16, 32), torch.bfloat16), ((9, 5), torch.float32), ((4, 2, 16, 20), torch.bfloat16), ((3, 1), torch.float32), ((6, 100003), torch.float32)):
        t = torch.randn(shape, device="cuda").to(dtype)
        want = t.clone()
        a, b = torch.tensor([0, 0, 2, -1, 99], dtype=torch.int32, device="cuda"), torch.tensor([1, shape[0] - 1 if shape[0] > 3 else 1, 99, 1, 1], dtype=torch.int32, device="cuda")
        K.copy_rows(t, a, b)
        want[1] = want[0]
        if shape[0] > 3:
            want[-1] = want[0]
        assert torch.equal(t, want)                          # rows that are none are left out
    with pytest.raises(K.KernelError):
        K.copy_rows(t, a, b[:2])
    with pytest.raises(K.KernelError):
        K.copy_rows(t, a.long(), b.long())


@pytest.mark.parametrize("family,name", [("gemma2", "A"), ("mukunex", "A"), ("sopalorn", "B")])
def test_greedy_answers_are_the_one_answer(family, name, monkeypatch):
    from kapel_b200 import Model
    from kapel_b200.engine import batch

    monkeypatch.setattr(batch, "SHARED_BYTES", 1)
    monkeypatch.setattr(batch, "SHARED_POSITIONS_32", 0)
    model = Model(None, dtype="f32", max_sequences=12, _engine=engine_of(config_of(family, name), "float32"))
    prompt = random_tokens(np.random.default_rng(3), 37, model.engine.vocab_size)
    want = model.generate(prompt, max_tokens=16, temperature=0.0, ignore_eos=True)
    for n, slots in ((1, None), (5, None), (5, 3)):
        assert model.generate_samples(prompt, n, max_tokens=16, temperature=0.0, ignore_eos=True, max_sequences=slots) == [want] * n
    assert model.engine.cache.free_pages() == model.engine.cache.total_pages()


def test_drawn_answers_are_those_of_their_seeds(monkeypatch):
    """In 32-bit: answer i is what a request alone draws with seed + i, under filters that are applied on the device."""
    from kapel_b200 import Model
    from kapel_b200.engine import batch

    monkeypatch.setattr(batch, "SHARED_BYTES", 1)
    monkeypatch.setattr(batch, "SHARED_POSITIONS_32", 0)
    model = Model(None, dtype="f32", max_sequences=12, _engine=engine_of(config_of("gemma2", "A"), "float32"))
    prompt = random_tokens(np.random.default_rng(4), 50, model.engine.vocab_size)
    kw = dict(max_tokens=24, temperature=1.1, top_k=60, top_p=0.95, ignore_eos=True)
    answers = model.generate_samples(prompt, 6, seed=100, **kw)
    assert answers == [model.generate(prompt, seed=100 + i, **kw) for i in range(6)]
    assert len({tuple(a) for a in answers}) == 6
    assert model.last_scheduler.staged_passes >= 0
    with pytest.raises(ValueError):
        model.generate_samples(prompt, 0)


def test_shared_steps_are_recorded_and_run_ahead(monkeypatch):
    from kapel_b200 import Model
    from kapel_b200.engine import batch

    monkeypatch.setattr(batch, "SHARED_BYTES", 1)
    monkeypatch.setattr(batch, "SHARED_POSITIONS_32", 0)
    eng = engine_of(config_of("gemma2", "A"), "bfloat16")
    model = Model(None, dtype="bf16", max_sequences=12, _engine=eng)
    model.generate_samples([3, 4, 5] * 12, 4, max_tokens=40, temperature=0.9, top_p=0.9, ignore_eos=True)
    assert any(len(k) > 2 for k in eng.graphs.graphs) and model.last_scheduler.ahead_passes > 20
    eng.check()


def test_the_command_line_gives_a_line_an_answer(tmp_path, capsys):
    import json

    from kapel_b200.cli import main

    path = tmp_path / "config.json"
    path.write_text(json.dumps(config_of("gemma2", "A")))
    assert main(["run", "--random", str(path), "--tokens", "1,2,3,4", "--samples", "3", "--max-tokens", "5", "--temperature", "1.0", "--top-p", "0.9", "--ignore-eos",
                 "--dtype", "f32", "--stats"]) == 0
    out = capsys.readouterr()
    assert len(out.out.split()) == 3 and all(len(l.split(",")) == 5 for l in out.out.split()) and "3 answers" in out.err
