"""A layer's description of what it keeps is copied and stored like the tuple that it is."""
import copy
import pickle

import pytest
import torch

from paligemma_multimodal_system_b200.cache import KvSpec, SequenceStore

WAYS = dict(copy=copy.copy, deepcopy=copy.deepcopy, **{f"pickle-{p}": lambda x, p=p: pickle.loads(pickle.dumps(x, p)) for p in range(pickle.HIGHEST_PROTOCOL + 1)})


@pytest.mark.parametrize("way", WAYS)
def test_a_spec_is_copied(way):
    spec = KvSpec(128, 64, 2)
    again = WAYS[way](spec)
    assert type(again) is KvSpec and again == spec == ("kv", 128, 64) and again.heads == 2


@pytest.mark.parametrize("way", WAYS)
def test_a_layout_and_a_store_are_copied(way):
    layout = [KvSpec(128, 64, 2), ("state", (3,)), None, ("latent", 40)]
    assert WAYS[way](layout) == layout
    store = WAYS[way](SequenceStore(layout, 200, 2, torch.bfloat16, device="cpu"))
    assert store.layout == layout and store.layout[0].heads == 2 and store.k_pages[0].shape == (4, 64, 128)
    if way == "deepcopy":
        eight = copy.deepcopy(SequenceStore(layout, 200, 2, torch.bfloat16, device="cpu", kv_format="e4m3"))
        assert eight.k_pages[0].codes.shape == (4, 64, 128) and eight.k_pages[0].heads == 2
