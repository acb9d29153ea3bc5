"""The descriptor of a ragged step: how it is made by name, by place and again."""
import dataclasses
import inspect

import pytest

from paligemma_multimodal_system_b200 import seq_ops

FIRST = ["T", "E", "max_n", "tokens", "pos", "row_entry", "row0", "n", "ctx", "slot", "page_table", "max_pages", "singles", "max_single_ctx", "single_rows", "dense_row0", "dense_pages",
         "dense_max_pages", "dense_rows", "dense_max_len", "shared", "min_n"]


@pytest.mark.parametrize("kind", ["StepBatch", "TreeBatch"])
def test_a_step_takes_rows_and_masks_of_drafted_trees(kind):
    made = getattr(seq_ops, kind)
    b = made(**dict.fromkeys(FIRST[:12], 1), at="rows", tree="masks")
    assert isinstance(b, seq_ops.StepBatch) and (b.at, b.tree) == ("rows", "masks")
    again = dataclasses.replace(b, shared={})
    assert type(again) is type(b) and (again.at, again.tree) == ("rows", "masks")
    plain = made(**dict.fromkeys(FIRST[:12], 1))
    assert plain.at is None and plain.tree is None


def test_they_stand_behind_what_a_caller_may_give_by_position():
    assert list(inspect.signature(seq_ops.StepBatch).parameters) == FIRST + ["at", "tree"]
