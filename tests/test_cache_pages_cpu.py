"""Moves of cache pages that are refused before anything runs."""
import copy

import numpy as np
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops


class _OnDevice(torch.Tensor):
    is_cuda = True

    def __deepcopy__(self, memo):
        return self.clone().as_subclass(_OnDevice)


def pages(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnDevice)


def cache(n=6):
    return seq_ops.CachePages([pages(n, 64, 32), pages(n, 64, 16, dtype=torch.float32)], 64)


@pytest.mark.parametrize("operands,page", [([], 64), ([torch.zeros(4, 64, 8)], 64), ([pages(4, 64, 8), pages(5, 64, 8)], 64), ([pages(4, 64, 8)], 32), ([pages(4, 64)], 64),
                                           ([pages(4, 64, 8)[:, :, :4]], 64), ([pages(4, 64, 0)], 64)])
def test_operands_that_are_no_cache(operands, page):
    with pytest.raises(ValueError):
        seq_ops.CachePages(operands, page)


@pytest.mark.parametrize("moves,error", [([[0, 1]], ValueError), ([0, 1, 2], ValueError), ([[0.0, 1.0, 2.0]], ValueError), ([[0, 6, 3]], IndexError), ([[6, 0, 3]], IndexError),
                                         ([[-1, 0, 3]], IndexError), ([[0, 1, 65]], IndexError), ([[0, 1, -1]], IndexError), ([[0, 1, 2], [3, 1, 2]], ValueError),
                                         ([[0, 1, 2], [1, 2, 2]], ValueError), ([[2, 2, 4]], ValueError), (5, ValueError), ([[True, False, True]], ValueError)])
def test_moves_that_are_refused(moves, error):
    with pytest.raises(error):
        seq_ops.copy_pages(cache(), moves)


def test_more_moves_are_looked_over_alike():
    c = cache(100)
    good = [[i, 50 + i, 3] for i in range(40)]
    for at, bad, error in ((7, [7, 49, 65], IndexError), (7, [100, 57, 3], IndexError), (39, [39, 57, 3], ValueError), (3, [60, 53, 3], ValueError), (3, [3, -1, 3], IndexError)):
        with pytest.raises(error):
            seq_ops.copy_pages(c, good[:at] + [bad] + good[at + 1:])


def test_an_operand_that_is_named_twice():
    p = pages(4, 64, 8)
    with pytest.raises(ValueError, match="twice"):
        seq_ops.CachePages([p, p], 64)


def test_nothing_to_move_is_no_call():
    seq_ops.copy_pages(cache(), [])
    seq_ops.copy_pages(cache(), np.zeros((0, 3), np.int32))


@pytest.mark.parametrize("path,kept", [(torch.zeros(2, 3), torch.zeros(2, dtype=torch.int32)), (torch.zeros(3, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)),
                                       (torch.zeros(2, 0, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)), (torch.zeros(2, 3, dtype=torch.int32), torch.zeros(3, dtype=torch.int32)),
                                       (torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2)), (torch.zeros(3, 2, dtype=torch.int32).t(), torch.zeros(2, dtype=torch.int32))])
def test_paths_that_are_refused(path, kept):
    z = torch.zeros(2, dtype=torch.int32)
    b = seq_ops.StepBatch(T=2, E=2, max_n=1, tokens=z, pos=z, row_entry=z, row0=z, n=z, ctx=z, slot=z, page_table=z.view(2, 1), max_pages=1)
    with pytest.raises(ValueError):
        seq_ops.keep_rows(cache(), b, path, kept)


def test_a_copy_says_where_the_copies_lie():
    c = cache()
    d = copy.deepcopy(c)
    assert d.operands[0].data_ptr() != c.operands[0].data_ptr() and bytes(d.table.numpy().tobytes())[:8] == int(d.operands[0].data_ptr()).to_bytes(8, "little")


def test_every_operand_is_in_the_table():
    q = seq_ops.QuantizedPages(torch.zeros(6, 64, 48, dtype=torch.uint8).as_subclass(_OnDevice), torch.zeros(6, 3, 64, dtype=torch.uint8).as_subclass(_OnDevice))
    c = seq_ops.CachePages([pages(6, 64, 33), q], 64)
    assert c.count == 3 and c.table.numel() == 32 * 3 and c.most_page_bytes == 64 * 66 and c.most_columns == 33


def test_shared_pages_are_free_when_all_owners_have_given_them_back():
    from paligemma_multimodal_system_b200.cache import PagePool, SequenceStore
    pool = PagePool(6)
    mine = pool.take(3)
    pool.share(mine[:2])
    pool.share(mine[:1])
    pool.give(mine)
    assert sorted(pool.free) == [2, 3, 4, 5]
    pool.give(mine[:2])
    assert sorted(pool.free) == [1, 2, 3, 4, 5]
    pool.give(mine[:1])
    assert sorted(pool.free) == list(range(6)) and not pool.shared
    with pytest.raises(RuntimeError):
        pool.give(mine[:1])
    store = SequenceStore([("kv", 8, 8)], 64 * 10, 4, torch.float32, allocate=False)
    store.admit("a")
    store.reserve("a", 150)
    store.commit("a", 150)
    b, c = store.fork("a", ["b", "c"])
    assert b.pages[:2] == c.pages[:2] == store.live["a"].pages[:2] and len({*store.live["a"].pages, *b.pages, *c.pages}) == 5 and b.length == c.length == 150
    (d,) = store.fork("b", ["d"], length=128)
    assert d.pages == b.pages[:2] and d.length == 128 and store.pool.shared == {p: 4 for p in d.pages}
    for rid in ("a", "d", "b"):
        store.release(rid)
    assert len(store.pool.free) == 7
    store.release("c")
    assert len(store.pool.free) == 10 and not store.pool.shared and len(store.free_slots) == 4


@pytest.mark.parametrize("history,most,match,tokens", [([], 4, 3, []), ([5], 4, 3, []), ([5, 5], 4, 3, [5]), ([1, 2, 3, 9, 1, 2, 3], 2, 3, [9, 1]), ([1, 2, 8, 7, 2], 4, 3, [8, 7, 2]),
                                                       ([4, 1, 2, 7, 3, 2, 6, 1, 2], 3, 2, [7, 3, 2]), ([1, 2, 3, 4], 4, 3, []), ([6, 6, 6, 6], 4, 2, [6])])
def test_guesses_from_the_text(history, most, match, tokens):
    from paligemma_multimodal_system_b200.engine import LookupDrafter
    assert LookupDrafter(most, match)(history) == (tokens, list(range(-1, len(tokens) - 1)))


def test_guesses_need_something_to_go_by():
    from paligemma_multimodal_system_b200.engine import LookupDrafter
    for bad in ((0, 3), (4, 0), (-1, 3)):
        with pytest.raises(ValueError):
            LookupDrafter(*bad)
