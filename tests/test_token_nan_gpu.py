"""Scored tokens whose own logit is a NaN have no rank; beside a NaN, other tokens' ranks count the numbers above them."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("V", [5, 4099, 257216])
@pytest.mark.parametrize("rows", [1, 4, 500])
@pytest.mark.parametrize("sign", [-1.0, 1.0, 0.0])
def test_a_token_that_is_no_number(V, rows, sign):
    from paligemma_multimodal_system_b200 import seq_ops
    if rows * V > 5_000_000:
        rows = 150
    g = torch.Generator(device="cuda").manual_seed(V + rows)
    x = torch.randn(rows, V + 1, generator=g, device="cuda")[:, :V] if sign == 0.0 else sign * (1 + torch.rand(rows, V, generator=g, device="cuda"))
    at = torch.tensor([(0, V // 2, V - 1, V // 3)[i % 4] for i in range(rows)], device="cuda", dtype=torch.int32)
    x[torch.arange(rows, device="cuda"), at.long()] = math.nan
    lp, entropy, rank, ids, top = seq_ops.token_logprobs(x, at, top=3)
    assert (rank == -1).all() and lp.isnan().all() and entropy.isnan().all() and top.isnan().all()
    order = torch.sort(torch.where(x.isnan(), -math.inf, x), dim=-1, descending=True, stable=True).indices
    assert torch.equal(ids, order[:, :3].int())  # (a NaN is behind every number)
    other = order[:, 2].int().contiguous()
    assert (seq_ops.token_logprobs(x, other, top=0)[2] == 2).all()


def test_nothing_but_nans():
    from paligemma_multimodal_system_b200 import seq_ops
    x = torch.full((2, 3000), math.nan, device="cuda")
    lp, _, rank, ids, _ = seq_ops.token_logprobs(x, torch.tensor([0, 2999], device="cuda", dtype=torch.int32), top=4)
    assert rank.tolist() == [-1, -1] and lp.isnan().all() and ids.tolist() == [[0, 1, 2, 3]] * 2
