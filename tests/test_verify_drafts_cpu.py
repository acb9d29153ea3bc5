"""Calls of verify_drafts that are refused before anything runs, and the reference that its GPU tests go by."""
import numpy as np
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops
from verify_reference import distribution, judge, pick


class _OnDevice(torch.Tensor):  # (refusals come before anything touches the device)
    is_cuda = True


def step(rows=3, parents=True):
    z = torch.zeros(rows, dtype=torch.int32)
    one = torch.zeros(1, dtype=torch.int32)
    return seq_ops.RequestBatch(T=rows, E=1, max_n=rows, tokens=z, pos=z, row_entry=z, row0=one, n=one + rows, ctx=one, slot=one, page_table=one.view(1, 1), max_pages=1,
                                parents=torch.tensor([-1] + list(range(rows - 1)), dtype=torch.int32) if parents is True else parents)


def logits(rows=3, V=40, dtype=torch.float32):
    return torch.zeros(rows, V, dtype=dtype).as_subclass(_OnDevice)


@pytest.mark.parametrize("call", [
    lambda: (logits(), step(parents=None)),
    lambda: (logits(), step(parents=torch.zeros(3, dtype=torch.int64))),
    lambda: (logits(), step(parents=torch.zeros(2, dtype=torch.int32))),
    lambda: (logits(4), step()),
    lambda: (logits(dtype=torch.bfloat16), step()),
    lambda: (torch.zeros(3, 40), step()),
    lambda: (logits().t().contiguous().t(), step()),
    lambda: (logits()[0], step()),
    lambda: (logits(1).expand(3, 40), step()),
    lambda: (logits(), step(), torch.zeros(3, 2), logits(1).expand(3, 40)),
    lambda: (logits(V=0), step()),
    lambda: (logits(), step(), torch.zeros(3)),
    lambda: (logits(), step(), torch.zeros(3, 2, dtype=torch.float64)),
    lambda: (logits(), step(), torch.zeros(2, 3).t()),
    lambda: (logits(), step(), None, logits()),
    lambda: (logits(), step(), torch.zeros(3, 2), logits(V=41)),
    lambda: (logits(), step(), torch.zeros(3, 2), logits(2)),
    lambda: (logits(), step(), torch.zeros(3, 2), None, 0.0),
    lambda: (logits(), step(), torch.zeros(3, 2), None, float("nan")),
    lambda: (logits(), step(), torch.zeros(3, 2), None, float("inf")),
    lambda: (logits(), step(), torch.zeros(3, 2), None, 1.0, -0.1),
    lambda: (logits(), step(), torch.zeros(3, 2), None, 1.0, 1.1),
    lambda: (logits(), step(), torch.zeros(3, 2), logits(), 1.0, 1.0, -1.0),
    lambda: (logits(), step(), torch.zeros(3, 2), logits(), 1.0, 1.0, 1.0, float("nan")),
])
def test_what_is_refused(call):
    with pytest.raises(ValueError):
        seq_ops.verify_drafts(*call())


def test_a_step_of_drafts_keeps_what_requests_have_of_their_own():
    import dataclasses
    b = step()
    again = dataclasses.replace(b, shared={})
    assert type(again) is seq_ops.RequestBatch and again.parents is b.parents and again.adapters is None
    assert seq_ops.StepBatch.parents is None and seq_ops.StepBatch.adapters is None


def test_the_reference_gives_the_targets_distribution():
    """Two drafted children of one row and a token behind: the first token of the answer is distributed as the target's, whatever the draft's distribution is."""
    g = torch.Generator().manual_seed(5)
    V, N = 4, 4000
    target, draft = torch.randn(V, generator=g), torch.randn(V, generator=g)
    p, q = distribution(target, 1.0, 1.0), distribution(draft, 1.0, 1.0)
    rows = torch.stack([target, target, target])
    drafts = torch.stack([draft, draft, draft])
    seen = np.zeros(V)
    for _ in range(N):
        kids = [pick(q, float(torch.rand((), generator=g))) for _ in range(2)]
        tokens, parents = [0] + kids, [-1, 0, 0]
        walk, nxt = judge(rows, tokens, parents, 0, 3, torch.rand(3, 2, generator=g), drafts, 1.0, 1.0, 1.0, 1.0)
        seen[tokens[walk[1]] if len(walk) > 1 else nxt] += 1
    # each count is binomial: five standard deviations
    assert (np.abs(seen - N * p.numpy()) < 5 * np.sqrt(N * (p * (1 - p)).numpy())).all()
