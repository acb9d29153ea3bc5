"""8-bit caches whose pages hold 32 or 128 rows: a mixed step gives what it gives over pages of 64 (whose results are tested against the formula), bit by bit -- the same tiles of
keys are walked in the same order, wherever they lie."""
import dataclasses

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def _step(page, lens, seed):
    """(batch, pages of every entry, pages in all): pages in any order.  The engine's pages hold 64 rows: the table of others takes the place of its own."""
    from paligemma_multimodal_system_b200 import seq_ops
    need = [-(-(n + c) // page) for n, c in lens]
    order = np.random.RandomState(seed).permutation(sum(need) + 2).tolist()
    pages = [[order.pop() for _ in range(k)] for k in need]
    b = seq_ops.make_step_batch([dict(tokens=[1] * n, ctx=c, slot=i, pages=range(-(-(n + c) // 64))) for i, (n, c) in enumerate(lens)])
    table = torch.tensor([own + [0] * (max(need) - len(own)) for own in pages], dtype=torch.int32, device="cuda")
    return dataclasses.replace(b, page_table=table, max_pages=max(need)), pages, sum(need) + 2


def _paged(codes, powers, page, pages, pool):
    """Rows of every entry into pages of `page` rows."""
    from paligemma_multimodal_system_b200.seq_ops import QuantizedPages
    heads = powers[0].shape[1]
    kept = QuantizedPages.empty(pool, page, heads, codes[0].shape[1] // heads)
    kept.codes.fill_(0x7f)  # whatever is nobody's is no number
    kept.powers.fill_(200)
    for c, p, own in zip(codes, powers, pages):
        for j in range(0, len(c), page):
            m = min(page, len(c) - j)
            kept.codes[own[j // page], :m], kept.powers[own[j // page], :, :m] = c[j:j + m], p[j:j + m].t()
    return kept


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("G,dim", [(2, 64), (1, 128)])
@pytest.mark.parametrize("page", [32, 128])
def test_a_mixed_step_over_pages_of_other_sizes(page, G, dim, dtype):
    from paligemma_multimodal_system_b200 import seq_ops
    lens, H = [(1, 77), (40, 30), (1, 0), (130, 0), (2, 600), (1, 300), (5, 128), (64, 64)], 4 * G
    g = torch.Generator(device="cuda").manual_seed(page + dim)
    kv = [([torch.randint(0, 0x78, (n + c, G * dim), generator=g, device="cuda", dtype=torch.uint8) for n, c in lens],
           [torch.randint(117, 123, (n + c, G), generator=g, device="cuda", dtype=torch.uint8) for n, c in lens]) for _ in "kv"]
    q = torch.randn(sum(n for n, _ in lens), H * dim, generator=g, device="cuda").to(dtype)
    got = []
    for size in (64, page):
        b, pages, pool = _step(size, lens, size)
        k, v = (_paged(*x, size, pages, pool) for x in kv)
        out = torch.full_like(q, 7.0)
        seq_ops.attn_ragged(q, k, v, None, out, b, H, G, dim, dim, dim ** -0.5, 0.0, size)
        got.append([out, *seq_ops.kv_read(k, v, b, dtype)])
    for a, c in zip(*got):
        assert torch.isfinite(c).all() and torch.equal(a, c)
