"""Verified drafts at the ends of their ranges, against 64 bits: temperatures that leave nothing but the largest entries or make all of them alike, random numbers of 0, entries that are masked
in front of the first one with any mass."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops
from test_verify_drafts_gpu import batch, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V,most", [(70001, 69000), (70001, 31), (5000, 4321)])
@pytest.mark.parametrize("temperature", [1e-12, 1e-20, 1e-29])
@pytest.mark.parametrize("top_p", [1.0, 0.9])
def test_temperatures_that_leave_the_largest_entries(V, most, temperature, top_p):
    """The largest entry, at any share of a row, has all of the mass: guesses of it stay, a draft's other token does not."""
    ns = [3, 2, 3]
    logits, draft, parents, tokens, u = make(ns, V, 1, 5, agree=0.0)
    logits[:, most], draft[:, (most + V // 2) % V] = 40.0, 40.0
    logits[7, most] = logits[7, most // 2] = 41.0  # two largest ones share it
    tokens[1:3], tokens[4], tokens[6:8] = [most, most], (most + V // 2) % V, [(most + V // 2) % V, most]
    for d in (None, draft, logits.clone()):
        got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), None if d is None else d.cuda(), temperature, top_p)
        check(got, ns, logits, parents, tokens, u, d, temperature, top_p)


@pytest.mark.parametrize("V", [5001, 70001])
@pytest.mark.parametrize("temperature", [4e36, 5e36, 1e37, 3e37, 4e37])
@pytest.mark.parametrize("top_p", [1.0, 0.5])
def test_temperatures_that_make_all_alike(V, temperature, top_p):
    """Logits over a temperature near the end of fp32, masked entries among them."""
    ns = [2, 3, 1]
    logits, draft, parents, tokens, u = make(ns, V, 2, 5, spread=1e36, temperature=temperature, top_p=top_p)
    logits[:, V // 3:V // 2], draft[:, V // 2:V // 2 + 40] = float("-inf"), float("-inf")
    for d in (None, draft):
        got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), None if d is None else d.cuda(), temperature, top_p)
        check(got, ns, logits, parents, tokens, u, d, temperature, top_p)


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


@pytest.mark.parametrize("V", [1, 40, 129, 700, 2049])
def test_rows_that_leave_most_of_a_cta_without_entries(V):
    """Warps without entries are through with a row at once; what they go by next is their own, whenever the others come.  The same answer every time, on three streams at once."""
    ns = [3, 2, 4, 1] * 40
    logits, draft, parents, tokens, u = make(ns, V, 2, 5, temperature=0.8, top_p=0.7)
    dev = (logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda(), 0.8, 0.7)
    first = seq_ops.verify_drafts(*dev)
    check(first, ns, logits, parents, tokens, u, draft, 0.8, 0.7)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams * 40:
        with torch.cuda.stream(s):
            outs.append(seq_ops.verify_drafts(*dev))
    torch.cuda.synchronize()
    for o in outs:
        assert all(torch.equal(a, b) for a, b in zip(o, first))
