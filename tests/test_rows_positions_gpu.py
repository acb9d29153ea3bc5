"""Windows go by positions: rows whose positions lie behind their entry's last cache row, or that skip some, see what the window leaves them."""
import pytest
import torch

from test_attn_rows_gpu import FORMS, Case, random_tree
from test_cache8_gpu import PAGE

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,cache", FORMS)
@pytest.mark.parametrize("lens", [[(6, 300), (2, 40)], [(3, 1500)], [(40, 200)], [(2, 9000)]])
@pytest.mark.parametrize("window,keep,further", [(100, 0, 40), (100, 5, 70), (64, 0, 90), (33, 70, 500)])
def test_positions_behind_the_last_row(dtype, cache, lens, window, keep, further):
    from paligemma_multimodal_system_b200 import seq_ops
    c = Case(dtype, cache, lens, 4, 2, 64, 64, [random_tree(n, 90 + i) for i, (n, _) in enumerate(lens)], seed=90)
    c.b.pos += torch.arange(c.b.T, device="cuda", dtype=torch.int32) % 3 * further  # (some rows stay where they are)
    c.check(score=seq_ops.ScoreOptions(4, window, keep), window=window, keep=keep)


@pytest.mark.parametrize("dtype,cache", FORMS)
def test_a_value_that_is_no_number_behind_such_a_window(dtype, cache):
    from paligemma_multimodal_system_b200 import seq_ops
    c = Case(dtype, cache, [(6, 300)], 4, 2, 64, 64, [[-1, 0, 0, 1, 2, 4]], seed=91)
    c.b.pos += torch.tensor([0, 40, 0, 40, 0, 40], device="cuda", dtype=torch.int32)
    j = 230  # rows at 300 .. 303 see 201 ..; those at 341 and further 242 ..
    p, slot = c.entries[0]["pages"][j // PAGE], j % PAGE
    if cache == "e4m3":
        c.kv[1].codes[p, slot] = 0x7f
    else:
        c.kv[1][p, slot] = float("nan")
    got = c.check(score=seq_ops.ScoreOptions(4, 100), window=100)
    assert got[[0, 2, 4]].isnan().all() and got[[1, 3, 5]].isfinite().all()
