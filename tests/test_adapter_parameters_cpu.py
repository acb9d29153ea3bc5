"""Banks that are filled from a training program's parameters."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops


class _OnDevice(torch.Tensor):
    is_cuda = True


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_bank_takes_the_numbers_of_parameters_and_nothing_else(dtype):
    a, b = torch.randn(2, 8, 24).to(dtype), torch.randn(2, 24, 4).to(dtype)
    made = seq_ops.AdapterBank(*(x.as_subclass(_OnDevice).requires_grad_() for x in (a, b, torch.ones(2))), (16, 8))
    same = seq_ops.AdapterBank(*(x.as_subclass(_OnDevice) for x in (a, b, torch.ones(2))), (16, 8))
    for bank in (made, same):
        bank.put(1, 1, torch.nn.Parameter(a[0, :3].clone()), torch.nn.Parameter(b[0, :8, :3].clone()))
        assert not bank.a.requires_grad and not bank.b.requires_grad and not bank.scale.requires_grad
        bank.clear(0)
    assert torch.equal(made.a, same.a) and torch.equal(made.b, same.b)
