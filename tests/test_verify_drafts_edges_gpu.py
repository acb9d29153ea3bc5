"""Verified drafts at the ends of their ranges, against 64 bits: random numbers of 0, entries that are masked in front of the first one with any mass."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops
from test_verify_drafts_gpu import batch, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,masked", [(3001, 1200), (70001, 30000), (257216, 257000), (257216, 129)])
@pytest.mark.parametrize("mask", [float("-inf"), torch.finfo(torch.float32).min])
@pytest.mark.parametrize("top_p", [1.0, 0.9])
def test_a_random_number_of_zero_draws_the_first_token_with_any_mass(V, masked, mask, top_p):
    ns = [2, 1]
    logits, draft, parents, tokens, u = make(ns, V, 1, 5)
    logits[:, :masked] = mask
    logits[2, masked] = 30.0  # nearly everything
    u[:, 1] = 0
    for d in (None, draft):
        got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), None if d is None else d.cuda(), 1.0, top_p)
        assert all(int(t) >= masked for t in got[2])
        check(got, ns, logits, parents, tokens, u, d, 1.0, top_p)
