"""Adapter banks, plans and calls that are refused before anything runs; the rows of a plan."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops


class _OnDevice(torch.Tensor):
    is_cuda = True


def t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype).as_subclass(_OnDevice)


def bank(slots=2, rank=4, K=24, parts=(16, 8), dtype=torch.bfloat16):
    return seq_ops.AdapterBank(t(slots, len(parts) * rank, K, dtype=dtype), t(slots, sum(parts), rank, dtype=dtype), t(slots, dtype=torch.float32), parts)


@pytest.mark.parametrize("a,b,scale,parts", [
    (t(2, 8, 24), t(2, 24, 4), t(2, dtype=torch.float32), (16, 9)), (t(2, 8, 24), t(2, 24, 4), t(2, dtype=torch.float32), ()), (t(2, 8, 24), t(2, 24, 4), t(2), (16, 8)),
    (t(2, 8, 24), t(2, 24, 4), t(3, dtype=torch.float32), (16, 8)), (t(2, 7, 24), t(2, 24, 4), t(2, dtype=torch.float32), (16, 8)), (t(2, 8, 24), t(3, 24, 4), t(2, dtype=torch.float32), (16, 8)),
    (t(2, 8, 24), t(2, 24, 4, dtype=torch.float32), t(2, dtype=torch.float32), (16, 8)), (t(2, 8, 24, dtype=torch.float16), t(2, 24, 4, dtype=torch.float16), t(2, dtype=torch.float32), (16, 8)),
    (t(2, 129, 24), t(2, 24, 129), t(2, dtype=torch.float32), (24,)), (t(2, 0, 24), t(2, 24, 0), t(2, dtype=torch.float32), (24,)), (t(2, 36, 24), t(2, 9, 4), t(2, dtype=torch.float32), (1,) * 9),
    (torch.zeros(2, 8, 24), torch.zeros(2, 24, 4), torch.zeros(2), (16, 8)), (t(2, 8, 24), t(2, 24, 4), t(2, dtype=torch.float32), (24, 0)), (t(8, 24), t(24, 4), t(2, dtype=torch.float32), (16, 8))])
def test_banks_that_are_refused(a, b, scale, parts):
    with pytest.raises(ValueError):
        seq_ops.AdapterBank(a, b, scale, parts)


def test_a_bank_pads_ranks_and_depths_with_zeros():
    a, b = torch.randn(2, 6, 21).as_subclass(_OnDevice), torch.randn(2, 24, 3).as_subclass(_OnDevice)
    k = seq_ops.AdapterBank(a, b, t(2, dtype=torch.float32), (16, 8))
    assert k.a.shape == (2, 16, 24) and k.b.shape == (2, 24, 8)
    assert torch.equal(k.a[:, 8:11, :21], a[:, 3:]) and not k.a[:, 3:8].any() and not k.a[:, :, 21:].any() and torch.equal(k.b[..., :3], b) and not k.b[..., 3:].any()


@pytest.mark.parametrize("slot,part,a,b,error", [(2, 0, (4, 24), (16, 4), IndexError), (-1, 0, (4, 24), (16, 4), IndexError), (0, 2, (4, 24), (16, 4), IndexError), (0, 0, (5, 24), (16, 5), ValueError),
                                                 (0, 0, (4, 23), (16, 4), ValueError), (0, 1, (4, 24), (16, 4), ValueError), (0, 0, (4, 24), (16, 3), ValueError)])
def test_matrices_that_do_not_belong_into_a_bank(slot, part, a, b, error):
    with pytest.raises(error):
        bank().put(slot, part, torch.zeros(a), torch.zeros(b))


@pytest.mark.parametrize("ns,who,error", [([], [], ValueError), ([1, 2], [0], ValueError), ([1, 0], [0, 0], ValueError), ([1, 2], [0, -2], IndexError)])
def test_plans_that_are_refused(ns, who, error):
    with pytest.raises(error):
        seq_ops.AdapterPlan(ns, who, device="cpu")


@pytest.mark.parametrize("ns,who,tiles", [([1, 1, 1], [2, -1, 2], None), ([100, 1, 70, 1], [1, 0, 1, -1], None), ([1] * 40, [i % 3 for i in range(40)], 40), ([5, 130], [0, 0], None)])
def test_every_row_of_a_plan_stands_in_one_tile_of_its_adapter(ns, who, tiles):
    plan = seq_ops.AdapterPlan(ns, who, device="cpu", tiles=tiles)
    of = [w for n, w in zip(ns, who) for _ in range(n)]
    seen = []
    for a, first, count in plan.tiles.view(-1, 3).tolist():
        rows = plan.rows[first:first + count].tolist()
        assert count <= plan.tile_rows and all(of[r] == a for r in rows)
        seen += rows
    assert sorted(seen) == list(range(sum(ns))) and plan.most == max(who)


def test_a_plan_with_room_for_fewer_tiles_is_refused():
    with pytest.raises(ValueError):
        seq_ops.AdapterPlan([1, 1, 1], [0, 1, 2], device="cpu", tiles=2)
    with pytest.raises(ValueError):
        seq_ops.AdapterPlan([1], [0], device="cpu").fill([1], [0])


@pytest.mark.parametrize("x,y,out,error", [((3, 24), (3, 24), None, None), ((3, 23), (3, 24), None, ValueError), ((2, 24), (2, 24), None, ValueError), ((3, 24), (3, 25), None, ValueError),
                                           ((3, 24), (3, 24), (3, 23), ValueError), ((24,), (3, 24), None, ValueError)])
def test_calls_that_are_refused(x, y, out, error):
    if error is None:
        return
    with pytest.raises(error):
        seq_ops.adapter_add(t(*x), t(*y), bank(), seq_ops.AdapterPlan([1, 2], [0, 1], device="cpu"), out=None if out is None else t(*out))


def test_types_strides_and_adapters_that_are_refused():
    plan = seq_ops.AdapterPlan([1, 2], [0, 1], device="cpu")
    for x, y, k in ((t(3, 24, dtype=torch.float32), t(3, 24), bank()), (t(3, 24), t(3, 24, dtype=torch.float16), bank()), (t(3, 24, dtype=torch.float32), t(3, 24), bank(dtype=torch.float32)),
                    (t(24, 3).t(), t(3, 24), bank()), (t(3, 24), t(24, 3).t(), bank()), (t(1, 24).expand(3, 24), t(3, 24), bank())):
        with pytest.raises(ValueError):
            seq_ops.adapter_add(x, y, k, plan)
    with pytest.raises(IndexError):
        seq_ops.adapter_add(t(3, 24), t(3, 24), bank(), seq_ops.AdapterPlan([1, 2], [0, 2], device="cpu"))
    y = t(3, 24)
    with pytest.raises(ValueError):
        seq_ops.adapter_add(t(3, 24), t(3, 24), bank(), plan, out=t(3, 24, dtype=torch.float32))


def test_outputs_that_lie_in_their_inputs_are_refused():
    plan, both = seq_ops.AdapterPlan([1, 2], [0, 1], device="cpu"), t(4, 100)
    for out in (both[1:], both[:3, 3:27], both[:3, 40:64]):
        with pytest.raises(ValueError):
            seq_ops.adapter_add(both[:3, 24:48], both[:3, :24], bank(), plan, out=out[:, :24])

    def overlap(a, b):
        size = a.element_size()
        return seq_ops._rows_overlap(a.data_ptr(), 100 * size, a.shape[1] * size, b.data_ptr(), 100 * size, b.shape[1] * size, len(a))

    assert not overlap(both[:3, :24], both[:3, 24:48]) and not overlap(both[:2], both[2:])
    assert overlap(both[:3, 76:], both[:3, :25]) is False and overlap(both[:3, :25], both[:3, 24:48])


@pytest.mark.parametrize("ns,who,rows", [([1] * 40, [0, 1] * 20, 16), ([2368], [0], 16), ([2369], [0], 128), ([1024, 1, 1344], [0, 1, -1], 128), ([64] * 40, list(range(40)), 128), ([63] * 40, list(range(40)), 16)])
def test_tiles_by_the_rows(ns, who, rows):
    plan = seq_ops.AdapterPlan(ns, who, device="cpu")
    assert plan.tile_rows == rows and seq_ops.AdapterPlan(ns, who, device="cpu", tile_rows=144 - rows).tile_rows == 144 - rows
    tiles = plan.tiles.view(-1, 3).tolist()
    assert sum(n for _, _, n in tiles) == sum(ns) and all(0 < n <= rows for _, _, n in tiles)
    with pytest.raises(ValueError):
        seq_ops.AdapterPlan(ns, who, device="cpu", tile_rows=64)
