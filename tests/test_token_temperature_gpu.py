"""The smallest temperatures that are taken: all of the mass is on the largest logit."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("temperature", [4.3e-39, 1.2e-38, 1e-30])
def test_the_smallest_temperatures(temperature):
    from paligemma_multimodal_system_b200 import seq_ops
    x = torch.randn(3, 5000, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    best = x.argmax(-1).int()
    lp, entropy, rank, ids, top = seq_ops.token_logprobs(x, best, top=2, temperature=temperature)
    assert not lp.any() and not entropy.any() and not rank.any() and torch.equal(ids[:, 0], best) and not top[:, 0].any() and (top[:, 1] < -1e20).all()
    lp, entropy, rank, _, _ = seq_ops.token_logprobs(x, ids[:, 1].contiguous(), temperature=temperature)
    assert (lp < -1e20).all() and not entropy.any() and (rank == 1).all()


def test_smaller_ones_are_refused():
    from paligemma_multimodal_system_b200 import seq_ops
    x, t = torch.randn(2, 100, device="cuda"), torch.zeros(2, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="PG_ERR_ARG"):
        seq_ops.token_logprobs(x, t, temperature=3.5e-39)
