"""A step that is captured while Python has an older graph to collect: destroying one inside a capture would end it."""
import gc

import pytest
import torch

from test_engine_operators_gpu import ATTENTION, engine
from test_mapedra_gpu import toks

pytestmark = pytest.mark.gpu


class _Held:
    def __init__(self):
        self.graph, self.itself, x = torch.cuda.CUDAGraph(), self, torch.zeros(4, device="cuda")
        torch.cuda.synchronize()
        with torch.cuda.graph(self.graph):
            x += 1


def test_a_graph_that_is_garbage_waits_until_the_capture_is_over(monkeypatch):
    eng, ref = engine(ATTENTION, torch.float32), engine(ATTENTION, torch.float32)
    want = ref.generate([toks(9, 80, 1)], 6)
    held, step, captures = [_Held()], type(eng.model).step, []

    def collects(self, *args, **kwargs):
        if torch.cuda.is_current_stream_capturing():
            held.clear()
            captures.append([[i] for i in range(200000)])
        return step(self, *args, **kwargs)

    monkeypatch.setattr(type(eng.model), "step", collects)
    assert gc.isenabled()
    assert eng.generate([toks(9, 80, 1)], 6) == want
    assert captures and gc.isenabled()
