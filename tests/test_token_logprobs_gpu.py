"""pg_token_logprobs against the definition in 64 bits: log probability, entropy, rank and top alternatives of logits rows.

Tolerances: d = (x - m) / T is formed in fp32 from an exact or once rounded difference (2^-24 relative) times a rounded factor (2^-23): |d| < 2^7 here, so e^d is off by less
than 2^7 * 2^-22 = 2^-15 relative where d is that large, and such terms weigh e^-128; where terms weigh (|d| < 16) it is 2^-18.  The hardware exponential adds 2^-22, sums of up to
2^18 terms over 512 threads 2^-14 in the worst case and 2^-19 in practice.  ln S <= 13 is then off by 2^-13 at most, and d_t by 2^-22 |d_t|: 2e-4 absolute, 2^-20 relative."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu


def _call(x, t, top=0, temperature=1.0):
    from paligemma_multimodal_system_b200 import seq_ops
    return [o.cpu() for o in seq_ops.token_logprobs(x, torch.as_tensor(t, dtype=torch.int32, device="cuda"), top=top, temperature=temperature)]


def _want(x, t, top, temperature):
    z = x.double().cpu() / temperature
    logs = torch.log_softmax(z, -1)
    p = logs.exp()
    entropy = -torch.where(p == 0, torch.zeros_like(p), p * logs).sum(-1)
    ids = torch.sort(x.cpu(), dim=-1, descending=True, stable=True).indices
    t = torch.as_tensor(t).long()
    lp = logs.gather(1, t[:, None])[:, 0]
    rank = (ids == t[:, None]).int().argmax(-1)
    return lp, entropy, rank.int(), ids[:, :top].int(), logs.gather(1, ids[:, :top])


def _check(x, t, top=0, temperature=1.0):
    got, want = _call(x, t, top, temperature), _want(x, t, top, temperature)
    for k in (2, 3):
        assert torch.equal(got[k], want[k]), (k, got[k], want[k])
    for k in (0, 1, 4):
        g, w = got[k].double(), want[k]
        fine = torch.isfinite(w)
        assert torch.equal(g[~fine].isnan(), w[~fine].isnan()) and torch.equal(g[~fine & ~w.isnan()], w[~fine & ~w.isnan()])
        assert torch.all((g - w).abs()[fine] <= 2e-4 + 2.0 ** -20 * w.abs()[fine]), (k, (g - w).abs()[fine].max())


def _logits(rows, V, seed, spread=3.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(rows, V, generator=g, device="cuda") * spread


@pytest.mark.parametrize("V,top", [(1, 0), (1, 1), (2, 2), (3, 1), (31, 31), (33, 32), (1000, 5), (4095, 32), (4099, 20), (8193, 1), (32000, 20), (65537, 32), (257216, 0), (257216, 32)])
@pytest.mark.parametrize("rows", [1, 3, 40])
def test_sizes(V, top, rows):
    x = _logits(rows, V, V + rows)
    t = [(7 * i * i + V // 2) % V for i in range(rows)]
    _check(x, t, top, 0.7 if rows == 3 else 1.0)


@pytest.mark.parametrize("rows", [150, 400])
def test_many_rows(rows):
    x = _logits(rows, 5003, rows)
    _check(x, [(i * 37) % 5003 for i in range(rows)], 7)


@pytest.mark.parametrize("first,pitch", [(0, 5000), (1, 5001), (2, 5003), (3, 5002)])
def test_rows_on_any_address(first, pitch):
    x = _logits(6, pitch, pitch)[:, first:first + 4801]
    _check(x, [0, 1, 4800, 2400, 3, 4799], 9)


def test_ties_go_to_the_lower_index():
    x = torch.full((4, 70000), 1.25, device="cuda")
    x[1, ::3] = 2.0
    x[2] = torch.randint(0, 7, (70000,), device="cuda").float()
    x[3, 69999] = 3.0
    x[0, 5] = -0.0
    x[0, 4] = 0.0
    _check(x, [69999, 69998, 12345, 0], 32)


@pytest.mark.parametrize("order", ["rising", "falling", "steps"])
def test_ordered_rows_fill_the_list(order):
    v = torch.arange(100000, device="cuda", dtype=torch.float32) / 5000
    x = torch.stack([v, v + 0.5]) if order == "rising" else torch.stack([v.flip(0), v.flip(0)]) if order == "falling" else torch.stack([v.floor(), v.floor()])
    _check(x.contiguous(), [99999, 17], 32)


def test_masked_entries():
    x = _logits(5, 40000, 3)
    x[0, 100:] = -math.inf
    x[1, :39990] = -math.inf
    x[2, ::2] = -math.inf
    x[3, 1:] = -math.inf
    x[4, 5] = 1000.0
    _check(x, [99, 39995, 1, 0, 5], 32)
    _check(x, [200, 0, 0, 39999, 6], 4)  # masked tokens: -inf, ranks among them by index


def test_rows_without_numbers():
    x = _logits(5, 9001, 4)
    x[0, 17] = math.nan
    x[1, 9000] = math.inf
    x[2] = -math.inf
    x[3] = math.nan
    lp, entropy, rank, ids, top = _call(x, [1, 2, 3, 4, 5], 3)
    assert lp[:4].isnan().all() and entropy[:4].isnan().all() and top[:4].isnan().all()
    assert ids[1, 0] == 9000 and ids[2].tolist() == [0, 1, 2] and ids[3].tolist() == [0, 1, 2] and 17 not in ids[0].tolist()
    _check(x[4:], [5], 3)  # a neighbour's row is its own


def test_tokens_outside_the_vocabulary():
    x = _logits(3, 500, 5)
    lp, entropy, rank, ids, _ = _call(x, [-1, 500, 20], 2)
    assert lp[:2].isnan().all() and rank[:2].tolist() == [-1, -1] and entropy.isfinite().all() and lp[2].isfinite()


@pytest.mark.parametrize("temperature", [0.01, 0.6, 1.0, 100.0])
def test_temperatures(temperature):
    _check(_logits(4, 33000, 6, 0.5), [1, 2, 3, 4], 5, temperature)


def test_captured_and_replayed():
    from paligemma_multimodal_system_b200 import seq_ops
    x, t = _logits(8, 30000, 7), torch.arange(8, dtype=torch.int32, device="cuda")
    seq_ops.token_logprobs(x, t, top=4)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = seq_ops.token_logprobs(x, t, top=4)
    x.copy_(_logits(8, 30000, 8))
    g.replay()
    torch.cuda.synchronize()
    for a, b in zip(out, seq_ops.token_logprobs(x, t, top=4)):
        assert torch.equal(a, b)


def test_no_rows():
    from paligemma_multimodal_system_b200 import seq_ops
    out = seq_ops.token_logprobs(torch.empty(0, 10, device="cuda"), torch.empty(0, dtype=torch.int32, device="cuda"), top=2)
    assert [tuple(o.shape) for o in out] == [(0,), (0,), (0,), (0, 2), (0, 2)]


@pytest.mark.parametrize("first,pitch,V", [(0, 3001, 3001), (3, 9007, 9001), (1, 2050, 2049)])
def test_more_rows_than_blocks(first, pitch, V):
    """Blocks that take several rows in turn, on all alignments; some rows need the careful way (masked, equal, rising) between others that do not."""
    rows = 1000
    x = _logits(rows, pitch, pitch)[:, first:first + V]
    x[5::50, 20:] = -math.inf
    x[6::50] = 1.0
    x[7::50] = torch.arange(V, device="cuda").float()
    x[8::50, 1::2] = x[8::50, 0::2][:, :x[8::50, 1::2].shape[1]]
    _check(x, [(i * 37) % V for i in range(rows)], 25)
    _check(x, [(i * 31) % V for i in range(rows)], 0)
    _check(x, [0] * rows, 1)


@pytest.mark.parametrize("mask", [-math.inf, -1e9, torch.finfo(torch.float32).min])
@pytest.mark.parametrize("rows,V", [(1, 257216), (40, 70001), (500, 5003)])
def test_masks_that_leave_fewer_than_asked_for(mask, rows, V):
    """The rest of the alternatives are masked entries, the lowest ids first, wherever those that are left lie: in front, behind, in one thread's tiles, among the first masked ones."""
    x = torch.full((rows, V), mask, device="cuda")
    some = torch.randn(rows, 12, generator=torch.Generator(device="cuda").manual_seed(V), device="cuda")
    for r in range(rows):
        at = [torch.arange(12), V - 12 + torch.arange(12), 1024 * torch.arange(4), 3 * torch.arange(12) + 1, torch.arange(1) + V // 2][r % 5]
        x[r, at.cuda()] = some[r, :len(at)]
    for top in (1, 4, 13, 32):
        _check(x, [(i * 37) % V for i in range(rows)], top)
    x[:, :V - 40] = 3.0 * mask if mask == -1e9 else -math.inf  # the equal ones that count lie behind
    _check(x, [V - 1] * rows, 32)


@pytest.mark.parametrize("rows,V", [(1, 257216), (70, 65536), (500, 32000)])
def test_large_entries_in_few_threads_tiles(rows, V):
    """More than the list holds, all of them above the rest: the row is read again by keys."""
    x = _logits(rows, V, 5 * V)
    x[:, torch.arange(V, device="cuda") // 4 % 256 < 12] += 100.0
    _check(x, [(i * 37) % V for i in range(rows)], 32)
    _check(x, [0] * rows, 5)
