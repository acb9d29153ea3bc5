"""Rows past max_n are left out: what stood in `out` stays, in every form, and the rows in front are what they are without it."""
import pytest
import torch

from test_attn_rows_gpu import FORMS, Case, random_tree, same
from test_cache8_gpu import PAGE

pytestmark = pytest.mark.gpu
# (entries, max_n, query heads, k/v heads): at most eight rows a k/v head, up to sixteen, more; one walk, shared in a cluster, shared through scratch; many entries
SHAPES = [([(12, 40), (3, 9)], 8, 2, 2), ([(12, 40), (3, 9)], 5, 2, 1), ([(20, 40), (3, 9)], 6, 8, 2), ([(12, 1500)], 8, 2, 2), ([(20, 1500)], 6, 8, 2), ([(12, 9000)], 4, 1, 1),
          ([(40, 100)] * 24, 9, 16, 4)]


@pytest.mark.parametrize("dtype,cache", FORMS)
@pytest.mark.parametrize("lens,max_n,H,G", SHAPES)
@pytest.mark.parametrize("drafted", [False, True])
def test_rows_past_the_largest_entry(dtype, cache, lens, max_n, H, G, drafted):
    from paligemma_multimodal_system_b200 import seq_ops
    c = Case(dtype, cache, lens, H, G, 64, 64, [random_tree(n, 80 + i) for i, (n, _) in enumerate(lens)] if drafted else None, seed=80)
    c.b.max_n = max_n
    seq_ops.attn_tree(c.q, *c.kv, None, c.out, c.b, H, G, 64, 64, 0.125, 0.0, PAGE)
    want, tol = c.want(0.125)
    got = c.out.double().cpu().view(want.shape)
    kept = torch.cat([torch.arange(n) >= max_n for n, _ in lens])
    assert kept.any() and (got[kept] == 7.0).all()
    same(got[~kept], want[~kept], tol[~kept])
