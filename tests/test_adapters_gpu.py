"""Low-rank adapters against 64 bits.

Tolerances, per output row: v = A x is a sum of K products in fp32 with terms of at most |A| |x|: error eps32 (K / 64 + 8) sum |A||x| at most, since groups of up to 64 products are added
up in fp32 and inside a group the instruction cuts off (four times 2^-24 of the group's largest partial sum, counted as a whole 8 eps32); handing v on in two terms loses 2^-17 of it, in
three 2^-24; the second sum adds (rank / 4) eps32 of sum |B||v|; y is added and the result rounded once, half a step of the type."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops

pytestmark = pytest.mark.gpu


def make(ns, who, K, parts, rank, slots, dtype, out, seed=0):
    g = torch.Generator().manual_seed(seed)
    T, F = sum(ns), sum(parts)
    x = torch.randn(T, K, generator=g).to(dtype)
    y = torch.randn(T, F, generator=g).to(out)
    a = (torch.randn(slots, len(parts) * rank, K, generator=g) * K ** -0.5).to(dtype)
    b = (torch.randn(slots, F, rank, generator=g) * rank ** -0.5).to(dtype)
    scale = 0.25 + torch.rand(slots, generator=g)
    return x, y, a, b, scale


def expected(x, y, a, b, scale, ns, who, parts, rank, gain=1.0):
    """(value, bound) in fp64."""
    eps = 2.0 ** -24
    value, bound = y.double(), torch.zeros(y.shape, dtype=torch.float64)
    K, t = x.shape[1], 0
    fp32 = y.dtype == torch.float32
    for n, s in zip(ns, who):
        if s >= 0:
            col = 0
            for i, w in enumerate(parts):
                A, B, X = a[s, i * rank:(i + 1) * rank].double(), b[s, col:col + w].double(), x[t:t + n].double()
                v, most = X @ A.T, X.abs() @ A.abs().T
                dv = eps * (K / 64 + 8) * most + v.abs() * (2.0 ** -24 if fp32 else 2.0 ** -17)
                f = gain * float(scale[s])
                value[t:t + n, col:col + w] += f * (v @ B.T)
                bound[t:t + n, col:col + w] = abs(f) * (dv @ B.abs().T + eps * (rank / 4 + 8) * (v.abs() @ B.abs().T))
                col += w
        t += n
    bound += value.abs() * torch.finfo(y.dtype).eps / 2 + eps * y.double().abs()
    bound[(torch.tensor(who).repeat_interleave(torch.tensor(ns)) < 0)] = 0  # (copied)
    return value, bound


def compare(got, value, bound):
    off = (got.double().cpu() - value).abs()
    worst = (off - bound).max()
    assert worst <= 0, f"off by {off.flatten()[(off - bound).argmax()]:.3g} where {bound.flatten()[(off - bound).argmax()]:.3g} is allowed"


FORMS = [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32), (torch.float32, torch.float32)]
STEPS = [([1], [0], 1), ([1] * 64, [i * 7 % 20 - (i % 9 == 0) for i in range(64)], 20), ([3, 1, 70, 1, 129, 1], [2, 0, 0, -1, 2, 1], 3), ([200], [0], 2), ([17, 5, 5], [-1, -1, -1], 1),
         ([400, 1, 1, 1], [1, 1, 0, -1], 2)]


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("dtype,out", FORMS)
@pytest.mark.parametrize("ns,who,slots", STEPS)
@pytest.mark.parametrize("K,parts,rank", [(256, [128], 16), (1000, [96, 40, 8], 8), (77, [33, 5], 3), (2048, [512, 64, 64], 64)])
def test_adapters(dtype, out, ns, who, slots, K, parts, rank, tile_rows):
    x, y, a, b, scale = make(ns, who, K, parts, rank, slots, dtype, out)
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan(ns, who, tile_rows=tile_rows)
    value, bound = expected(x, y, a, b, scale, ns, who, parts, rank)
    apart = seq_ops.adapter_add(x.cuda(), y.cuda(), bank, plan, out=torch.full_like(y, float("nan"), device="cuda"))
    compare(apart, value, bound)
    z = y.cuda()
    assert seq_ops.adapter_add(x.cuda(), z, bank, plan) is z and torch.equal(z, apart)


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("rank,parts", [(128, [64] * 8), (100, [320, 200]), (1, [8]), (40, [24, 24, 24, 24, 24])])
@pytest.mark.parametrize("dtype,out", FORMS)
def test_ranks_and_runs(rank, parts, dtype, out, tile_rows):
    ns, who = [90, 1, 30], [1, 0, 1]
    x, y, a, b, scale = make(ns, who, 136, parts, rank, 2, dtype, out, seed=rank)
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan(ns, who, tile_rows=tile_rows)
    value, bound = expected(x, y, a, b, scale, ns, who, parts, rank, gain=-1.5)
    compare(seq_ops.adapter_add(x.cuda(), y.cuda(), bank, plan, gain=-1.5), value, bound)


@pytest.mark.parametrize("tile_rows", [16, 128])
@pytest.mark.parametrize("dtype,out", FORMS)
@pytest.mark.parametrize("pitch,off", [(264, 8), (261, 3), (272, 1)])
def test_rows_at_any_pitch_and_columns_beside(dtype, out, pitch, off, tile_rows):
    ns, who, parts, K, rank = [40, 1, 1, 30], [0, 1, -1, 1], [100, 28], 200, 16
    x, y, a, b, scale = make(ns, who, K, parts, rank, 2, dtype, out)
    X, Y = torch.full((72, pitch), float("nan"), dtype=dtype, device="cuda"), torch.full((72, pitch), float("nan"), dtype=out, device="cuda")
    X[:, off:off + K], Y[:, off:off + 128] = x.cuda(), y.cuda()
    before = Y.clone()
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan(ns, who, tile_rows=tile_rows)
    seq_ops.adapter_add(X[:, off:off + K], Y[:, off:off + 128], bank, plan)
    value, bound = expected(x, y, a, b, scale, ns, who, parts, rank)
    compare(Y[:, off:off + 128], value, bound)
    Y[:, off:off + 128] = before[:, off:off + 128]
    assert torch.equal(Y.view(torch.uint8), before.view(torch.uint8))


@pytest.mark.parametrize("tile_rows", [16, 128])
def test_what_is_not_finite_stays_in_its_row(tile_rows):
    ns, who = [20, 3], [0, -1]
    x, y, a, b, scale = make(ns, who, 64, [32], 8, 1, torch.bfloat16, torch.float32)
    x[5, 3], x[21, 0], y[22, 1] = float("nan"), float("inf"), float("-inf")
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), [32]), seq_ops.AdapterPlan(ns, who, tile_rows=tile_rows)
    got = seq_ops.adapter_add(x.cuda(), y.cuda(), bank, plan, out=torch.empty(23, 32, device="cuda")).cpu()
    assert got[5].isnan().all() and torch.equal(got[20:], y[20:])
    x[5] = 0
    value, bound = expected(x, y, a, b, scale, ns, who, [32], 8)
    keep = [i for i in range(20) if i != 5]
    compare(got[keep], value[keep], bound[keep])


def test_a_bank_is_filled_part_by_part():
    bank = seq_ops.AdapterBank.empty(3, 16, 96, [40, 24], torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    a, b = torch.randn(5, 96, generator=g).bfloat16(), torch.randn(24, 5, generator=g).bfloat16()
    bank.put(1, 1, a, b)
    bank.scale[1] = 2.0
    x, y = torch.randn(4, 96, generator=g).bfloat16(), torch.randn(4, 64, generator=g).bfloat16()
    got = seq_ops.adapter_add(x.cuda(), y.cuda(), bank, seq_ops.AdapterPlan([4], [1])).cpu()
    assert torch.equal(got[:, :40], y[:, :40])
    value, bound = expected(x, y[:, 40:], a[None], b[None], torch.tensor([2.0]), [4], [0], [24], 5)
    compare(got[:, 40:], value, bound)
    bank.clear(1)
    assert torch.equal(seq_ops.adapter_add(x.cuda(), y.cuda(), bank, seq_ops.AdapterPlan([4], [1])).cpu(), y)


def test_a_plan_that_is_filled_again_under_a_graph():
    E, K, parts = 9, 128, [64]
    x, y, a, b, scale = make([1] * E, [0] * E, K, parts, 8, 4, torch.bfloat16, torch.float32)
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan([1] * E, [0] * E, tiles=E)
    X, Y, Z = x.cuda(), y.cuda(), torch.empty_like(y, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        seq_ops.adapter_add(X, Y, bank, plan, out=Z)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            seq_ops.adapter_add(X, Y, bank, plan, out=Z)
    torch.cuda.current_stream().wait_stream(side)
    for who in ([3, -1, 2, 2, 0, 1, 3, 3, -1], [0] * 9, [-1] * 9, [0, 1, 2, 3, 0, 1, 2, 3, 0]):
        plan.fill([1] * E, who)
        g.replay()
        value, bound = expected(x, y, a, b, scale, [1] * E, who, parts, 8)
        compare(Z, value, bound)


@pytest.mark.parametrize("rank,parts", [(100, [320, 200]), (128, [264]), (8, [16, 130, 8, 300, 24, 128, 129, 40]), (64, [128, 640, 72]), (72, [1000]), (16, [3]), (128, [64, 40, 24]), (128, [24] * 8)])
@pytest.mark.parametrize("dtype,out", FORMS[:2])
@pytest.mark.parametrize("ns,who,slots", [([300], [0], 1), ([150, 1, 260, 128, 1], [1, 0, -1, 1, 1], 2)])
def test_tiles_of_many_rows(rank, parts, dtype, out, ns, who, slots):
    """Blocks of 64 ranks and 128 columns that are not full, several parts, shares of K that differ, rows without an adapter beside."""
    K = 1096
    x, y, a, b, scale = make(ns, who, K, parts, rank, slots, dtype, out, seed=rank)
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan(ns, who, tile_rows=128)
    value, bound = expected(x, y, a, b, scale, ns, who, parts, rank)
    z = y.cuda()
    apart = seq_ops.adapter_add(x.cuda(), z, bank, plan, out=torch.full_like(z, float("nan")))
    compare(apart, value, bound)
    assert torch.equal(seq_ops.adapter_add(x.cuda(), z, bank, plan), apart)
    assert torch.equal(seq_ops.adapter_add(x.cuda(), y.cuda(), bank, plan), apart)  # the same sums every time


@pytest.mark.parametrize("dtype,out", FORMS[:2])
@pytest.mark.parametrize("K", [64, 200, 8])
def test_more_tiles_than_processors(dtype, out, K):
    ns, who, parts, rank = [20100, 300], [0, 1], [40, 136], 24
    x, y, a, b, scale = make(ns, who, K, parts, rank, 2, dtype, out)
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan(ns, who, tile_rows=128)
    value, bound = expected(x, y, a, b, scale, ns, who, parts, rank)
    compare(seq_ops.adapter_add(x.cuda(), y.cuda(), bank, plan), value, bound)


@pytest.mark.parametrize("pitch,off", [(1104, 8), (1101, 3)])
def test_tiles_of_many_rows_at_any_pitch(pitch, off):
    ns, who, parts, K, rank = [270], [0], [1000, 20], 1000, 32
    x, y, a, b, scale = make(ns, who, K, parts, rank, 1, torch.bfloat16, torch.bfloat16)
    X, Y = torch.full((270, pitch), float("nan"), dtype=torch.bfloat16, device="cuda"), torch.full((270, pitch), float("nan"), dtype=torch.bfloat16, device="cuda")
    X[:, off:off + K], Y[:, off:off + 1020] = x.cuda(), y.cuda()
    before = Y.clone()
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan(ns, who, tile_rows=128)
    seq_ops.adapter_add(X[:, off:off + K], Y[:, off:off + 1020], bank, plan)
    value, bound = expected(x, y, a, b, scale, ns, who, parts, rank)
    compare(Y[:, off:off + 1020], value, bound)
    Y[:, off:off + 1020] = before[:, off:off + 1020]
    assert torch.equal(Y.view(torch.uint8), before.view(torch.uint8))


def test_two_streams_and_a_captured_call():
    """Calls that run at the same time have scratch of their own."""
    ns, who, parts, K, rank = [700], [0], [512, 256], 1024, 64
    x, y, a, b, scale = make(ns, who, K, parts, rank, 1, torch.bfloat16, torch.float32)
    bank, plan = seq_ops.AdapterBank(a.cuda(), b.cuda(), scale.cuda(), parts), seq_ops.AdapterPlan(ns, who, tile_rows=128)
    X, Y = x.cuda(), y.cuda()
    want = seq_ops.adapter_add(X, Y, bank, plan, out=torch.empty_like(Y))
    value, bound = expected(x, y, a, b, scale, ns, who, parts, rank)
    compare(want, value, bound)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams * 4:
        with torch.cuda.stream(s):
            outs.append(seq_ops.adapter_add(X, Y, bank, plan, out=torch.empty_like(Y)))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)
    with torch.cuda.stream(streams[0]):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=streams[0]):
            o = seq_ops.adapter_add(X, Y, bank, plan, out=torch.empty_like(Y))
    torch.cuda.synchronize()
    for _ in range(2):
        o.zero_()
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(o, want)
