"""Gates of attention of a few rows that are no numbers or infinite: a NaN stays one and reaches its own outputs only, as in the framework's other attention; -inf closes, +inf opens.

Tolerance: test_attn_rows_gpu's; the gate of fp32 rows is an exponential within two half steps, a sum and a division within half a step each: the logistic is off by less than
2^-22 of its value, inside the 2^-21 that is allowed there."""
import math

import pytest
import torch

from test_attn_rows_gpu import FORMS, Case, random_tree, same
from test_cache8_gpu import PAGE

pytestmark = pytest.mark.gpu
SHAPES = [([(1, 40), (1, 1500)], None), ([(1, 9000)], None), ([(6, 200), (3, 20)], True), ([(20, 700)], True)]


@pytest.mark.parametrize("dtype,cache", FORMS)
@pytest.mark.parametrize("lens,drafted", SHAPES)
@pytest.mark.parametrize("per_head", [False, True])
def test_gates_that_are_no_numbers(dtype, cache, lens, drafted, per_head):
    c = Case(dtype, cache, lens, 4, 2, 64, 64, [random_tree(n, 60) for n, _ in lens] if drafted else None, seed=50)
    g = torch.Generator(device="cuda").manual_seed(5)
    gate = (torch.randn(c.b.T, 4 if per_head else 256, generator=g, device="cuda") * 4).to(dtype)
    flat = gate.view(-1)
    some = torch.randperm(flat.numel(), generator=g, device="cuda")
    n = max(1, flat.numel() // 8)
    flat[some[:n]], flat[some[n:2 * n]], flat[some[2 * n:3 * n]] = math.nan, math.inf, -math.inf
    got = c.check(gate=gate, per_head=per_head)
    wide = (gate[..., None].expand(-1, -1, 64) if per_head else gate.view(-1, 4, 64)).double().cpu()
    assert torch.equal(got.isnan(), wide.isnan()) and not got[wide == -math.inf].any()


def test_the_two_parts_of_a_mixed_step_agree_on_a_gate_that_is_no_number():
    """A prompt portion and a decoded token of one step over 8-bit pages."""
    from paligemma_multimodal_system_b200 import seq_ops
    c = Case(torch.bfloat16, "e4m3", [(1, 77), (40, 30)], 4, 2, 64, 64, seed=51)
    gate = torch.randn(c.b.T, 256, device="cuda").to(torch.bfloat16)
    gate[:, ::3] = math.nan
    seq_ops.attn_ragged(c.q, *c.kv, gate, c.out, c.b, 4, 2, 64, 64, 0.125, 0.0, PAGE)
    assert torch.equal(c.out.isnan(), gate.isnan())
    want, tol = c.want(0.125, gate=gate)
    same(c.out.double().cpu().view(want.shape), want, tol)
