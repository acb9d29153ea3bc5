"""Outputs and gates of attention of a few rows whose rows do not lie where the kernel writes and reads are refused before anything is launched."""
import types

import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops

T, H, VDIM = 3, 2, 32
Z = torch.bfloat16


def _call(out, gate=None, per_head=False, score=None):
    b = types.SimpleNamespace(T=T, E=1, max_n=T, singles=0, max_single_ctx=0, dense_max_len=T, max_pages=1, tree=None, at=None)
    pages = torch.zeros(1, 64, 32, dtype=Z)
    seq_ops.attn_tree(torch.zeros(T, 64, dtype=Z), pages, pages, gate, out, b, H, 1, 32, VDIM, 0.1, 0.0, 64, gate_per_head=per_head, score=score)


@pytest.mark.parametrize("out", [torch.zeros(T, 128, dtype=Z)[:, :64], torch.zeros(T - 1, 64, dtype=Z), torch.zeros(T, 60, dtype=Z), torch.zeros(T * 60, dtype=Z), torch.zeros(2 * T, 64, dtype=Z)[::2],
                                 torch.zeros(T, H, 64, dtype=Z)[:, :, :32]])
def test_outputs(out):
    with pytest.raises(ValueError, match="output"):
        _call(out)


def test_outputs_with_a_pitch_of_their_own():
    score = types.SimpleNamespace(out_ld=128)
    for out in (torch.zeros(T, 64, dtype=Z), torch.zeros(T, 256, dtype=Z)[:, :64]):
        with pytest.raises(ValueError, match="output"):
            _call(out, score=score)


@pytest.mark.parametrize("gate,per_head", [(torch.zeros(T, 63, dtype=Z), False), (torch.zeros(T - 1, 64, dtype=Z), False), (torch.zeros(T, 1, dtype=Z), True), (torch.zeros(64, dtype=Z), False),
                                           (torch.zeros(T, 2, dtype=Z), False)])
def test_gates(gate, per_head):
    with pytest.raises(ValueError, match="gate"):
        _call(torch.zeros(T, 64, dtype=Z), gate, per_head)
