"""Requests of the ragged-step engine beside one another: names, slots, adapters and rows of a step that other requests have or had."""
import pytest
import torch

from oracle import mapedra_oracle as O
from test_engine_operators_gpu import ATTENTION, TOL, engine, rel_err
from test_mapedra_gpu import run_cut, toks
from test_requests_of_their_own_gpu import adapter, build, merged, run_cut_live, shapes

pytestmark = pytest.mark.gpu


def adapted(slots=4):
    """(engine with one adapter loaded, engine of the model that it makes, engine of the plain one)"""
    from paligemma_multimodal_system_b200.adapters import AdapterSet
    from paligemma_multimodal_system_b200.engine import SequenceEngine
    weights, g = O.random_weights(ATTENTION, seed=3), torch.Generator().manual_seed(4)
    model = build(ATTENTION, weights, torch.float32)
    sets = AdapterSet(model, 2, 8)
    own = adapter(sets, shapes(sets), g, 8, sorted(shapes(sets)))
    sets.load("one", own)
    return SequenceEngine(model, 2048, slots, adapters=sets), SequenceEngine(build(ATTENTION, merged(weights, own, 1.0), torch.float32), 2048, slots), SequenceEngine(model, 2048, slots)


def test_forks_named_by_an_iterator_keep_the_adapter():
    eng, ref, _ = adapted()
    prompt, later = toks(70, 80, 1), toks(5, 80, 2)
    eng.step([("a", prompt, [])], adapters={"a": "one"})
    eng.fork("a", (n for n in ("b", "c")))
    want = run_cut(ref, "x", prompt + later, [70, 4, 1])[70:]
    for rid in "abc":
        assert rel_err(run_cut_live(eng, rid, later, [4, 1]), want) < TOL[torch.float32], rid


def test_a_name_that_is_taken_again_has_no_adapter_of_before():
    eng, _, plain = adapted()
    prompt = toks(30, 80, 1)
    eng.step([("a", toks(9, 80, 3), [])], adapters={"a": "one"})
    eng.store.release("a")
    eng.remove_adapter("one")  # nobody has it
    got = eng.step([("a", prompt, range(30))])
    assert rel_err(got, run_cut(plain, "a", prompt, [30])) < TOL[torch.float32]


def test_generation_leaves_requests_of_any_name_alone():
    eng, ref = engine(ATTENTION, torch.float32), engine(ATTENTION, torch.float32)
    prompt, mine, later = toks(20, 80, 1), toks(33, 80, 2), toks(4, 80, 3)
    want = ref.generate([prompt, prompt[:7]], 6)
    eng.step([(("gen", 0), mine, [])])
    assert eng.generate([prompt, prompt[:7]], 6) == want
    with pytest.raises(OSError):
        eng.generate([prompt], 6, draft=_fails)
    assert list(eng.store.live) == [("gen", 0)]
    assert rel_err(run_cut_live(eng, ("gen", 0), later, [3, 1]), run_cut(ref, "x", mine + later, [33, 3, 1])[33:]) < TOL[torch.float32]
    inner = []

    def asks(history):  # a draft that is made by the same engine
        inner.append(eng.generate([history], 2)[0])
        return inner[-1], [-1, 0]

    assert eng.generate([prompt, prompt[:7]], 6, draft=asks) == want and inner


def _fails(history):
    raise OSError("no guess")


def test_generation_where_nothing_is_free():
    eng = engine(ATTENTION, torch.float32, slots=2)
    eng.step([("a", toks(9, 80, 1), []), ("b", toks(9, 80, 2), [])])
    assert eng.generate([], 4) == [] and eng.generate([], 4, logprobs=1) == ([], [])
    with pytest.raises(MemoryError, match="slots"):
        eng.generate([[1, 2]], 4)
    eng.release("a")
    assert len(eng.generate([[1, 2]], 4)[0]) == 4
    eng = engine(ATTENTION, torch.float32, max_tokens=128)
    eng.step([("a", toks(100, 80, 1), [])])
    with pytest.raises(MemoryError, match="pages"):
        eng.generate([[1, 2]], 4)
    assert list(eng.store.live) == ["a"]


@pytest.mark.parametrize("step_tokens,most", [(512, 4 * 9), (16, 16), (7, 7), (4, 4)])
def test_steps_of_drafts_have_no_more_rows_than_other_steps(step_tokens, most, monkeypatch):
    eng = engine(ATTENTION, torch.float32)
    prompts = [toks(n, 80, n) for n in (3, 4, 2, 1)]
    want, rows, run = eng.generate(prompts, 12), [], type(eng)._draft_step

    def counted(self, entries):
        rows.append(sum(len(t) for _, t, _ in entries))
        return run(self, entries)

    monkeypatch.setattr(type(eng), "_draft_step", counted)
    assert eng.generate(prompts, 12, step_tokens=step_tokens, draft=lambda h: ([h[-1]] * 8, range(-1, 7))) == want
    assert (not rows or max(rows) <= most) and (step_tokens < 5 or max(rows) > 4)


def test_an_adapter_that_nobody_loaded_is_refused_before_anything_runs(monkeypatch):
    eng, _, _ = adapted(slots=1)
    monkeypatch.setattr(eng.model, "step", lambda *a, **k: pytest.fail("a step ran"))
    with pytest.raises(KeyError, match="prompt 1"):
        eng.generate([[1, 2], [3]], 4, adapters=["one", "two"])
    with pytest.raises(KeyError, match="prompt 0"):
        engine(ATTENTION, torch.float32).generate([[1, 2]], 4, adapters=["one"])
