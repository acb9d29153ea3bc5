"""Scoring takes slots of its own: whatever name a live request has, it is neither read, continued nor released."""
import pytest
import torch

from test_engine_operators_gpu import ATTENTION, engine
from test_mapedra_gpu import toks

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("name", [("score", 0), ("score", 1), 0, None, "score"])
def test_a_live_request_of_any_name(name):
    eng, alone = engine(ATTENTION, torch.float32), engine(ATTENTION, torch.float32)
    mine, prompts = toks(30, 80, 1), [toks(9, 80, 2), toks(70, 80, 3)]
    eng.step([(name, mine, [])])
    got, want = eng.score(prompts, top=2), alone.score(prompts, top=2)
    assert [len(r) for r in got] == [8, 69] and got == want
    assert eng.store.live[name].length == 30 and list(eng.store.live) == [name]
    alone.step([("a", mine, [])])
    assert torch.equal(eng.step([(name, [5], [0])]), alone.step([("a", [5], [0])]))
