"""Long sums of one sign through low-rank adapters, against 64 bits.

Tiles of 16 rows: groups of up to 64 products are added up in fp32, eps32 = 2^-24 a group, and a group is cut off by 8 eps32 at most.  Tiles of 128 rows: the matrix unit adds 16 products at a
time to the sum that it holds and cuts off what does not fit; the sum never is larger than the whole, so each addition loses a step of fp32 (2^-23) of it at most, and what the 16 products lose
as they are lined up with it is counted as another.  Behind v = A x: three terms keep 2^-24, B has one rank here, out is rounded once."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("K", [2048, 8192, 16384])
def test_long_sums_of_one_sign(K, tile_rows):
    T, F, g = 400, 40, torch.Generator().manual_seed(K)
    x, a = (0.5 + torch.rand(T, K, generator=g)).bfloat16(), (0.5 + torch.rand(1, 1, K, generator=g)).bfloat16()
    b, y = torch.ones(1, F, 1).bfloat16(), torch.zeros(T, F)
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), torch.ones(1, device="cuda"), [F]), seq_ops.AdapterPlan([T], [0], tile_rows=tile_rows)
    got = seq_ops.adapter_add(x.cuda(), y.cuda(), bank, plan).double().cpu()
    want = (x.double() @ a[0].double().T).expand(T, F)
    bound = (K / 64 + 8) * 2.0 ** -24 if tile_rows == 16 else 2 * (K / 16) * 2.0 ** -23
    assert ((got - want).abs() <= (bound + 4 * 2.0 ** -24) * want).all(), float(((got - want).abs() / want).max())
