"""Rows of paged caches that move: bits are compared, and what no move names stays."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops

pytestmark = pytest.mark.gpu


def pools(n, widths, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, (n, 64, w * dt.itemsize), generator=g, dtype=torch.uint8).view(dt).cuda() for w, dt in widths]


def quantized(n, heads, size, seed=1):
    g = torch.Generator().manual_seed(seed)
    return seq_ops.QuantizedPages(torch.randint(0, 256, (n, 64, heads * size), generator=g, dtype=torch.uint8).cuda(),
                                  torch.randint(0, 256, (n, heads, 64), generator=g, dtype=torch.uint8).cuda())


def bits(ops):
    out = []
    for o in ops:
        out += [o.codes.cpu(), o.powers.transpose(1, 2).contiguous().cpu()] if isinstance(o, seq_ops.QuantizedPages) else [o.view(torch.uint8).cpu()]
    return [x.clone() for x in out]  # [pages, 64, bytes of a row]


WIDTHS = [(512, torch.bfloat16), (8, torch.float32), (33, torch.bfloat16), (7, torch.uint8), (2, torch.float32), (2048, torch.float32)]


@pytest.mark.parametrize("moves", [[(0, 1, 64)], [(3, 0, 1)], [(5, 2, 21), (5, 4, 64), (1, 0, 0), (3, 6, 63)]])
def test_pages_are_copied(moves):
    ops = pools(9, WIDTHS) + [quantized(9, 3, 16), quantized(9, 130, 16)]
    want = bits(ops)
    seq_ops.copy_pages(seq_ops.CachePages(ops, 64), moves)
    for a, b, n in moves:
        for x in want:
            x[b, :n] = x[a, :n].clone()
    assert all(torch.equal(x, y) for x, y in zip(want, bits(ops)))


def test_more_moves_than_one_launch_takes():
    ops = pools(1200, [(16, torch.bfloat16), (3, torch.bfloat16)])
    want = bits(ops)
    moves = [(i, 600 + (i * 7) % 600, i % 65) for i in range(600)]
    seq_ops.copy_pages(seq_ops.CachePages(ops, 64), moves)
    for a, b, n in moves:
        for x in want:
            x[b, :n] = x[a, :n]
    assert all(torch.equal(x, y) for x, y in zip(want, bits(ops)))


def test_pages_of_one_row_are_slots():
    state = torch.randn(5, 1, 777, device="cuda")
    want = state.clone()
    want[4], want[0] = want[2], want[2]
    seq_ops.copy_pages(seq_ops.CachePages([state], 1), [(2, 4, 1), (2, 0, 1)])
    assert torch.equal(state, want)


def test_an_operand_past_two_to_the_31_bytes():
    big = torch.zeros(40000, 64, 512, device="cuda", dtype=torch.bfloat16)  # 2.6 GB
    big[3] = torch.randn(64, 512, device="cuda").bfloat16()
    seq_ops.copy_pages(seq_ops.CachePages([big], 64), [(3, 39999, 64)])
    assert torch.equal(big[39999], big[3]) and not big[39998].any()


def step(ns, ctx, seed=0, spare=2):
    g = torch.Generator().manual_seed(seed)
    need = [(n + c + 63) // 64 for n, c in zip(ns, ctx)]
    order = torch.randperm(sum(need) + spare, generator=g).tolist()
    entries = []
    for n, c, k in zip(ns, ctx, need):
        entries.append(dict(tokens=[1] * n, ctx=c, slot=0, pages=order[:k]))
        order = order[k:]
    return seq_ops.make_step_batch(entries), entries, sum(need) + spare


def run_keep(ns, ctx, paths, ops_of, width=None):
    b, entries, n_pages = step(ns, ctx)
    ops = ops_of(n_pages)
    want = bits(ops)
    width = width or max(max(len(p) for p in paths), 1)
    path = torch.tensor([p + [-1] * (width - len(p)) for p in paths], dtype=torch.int32, device="cuda")
    kept = torch.tensor([len(p) for p in paths], dtype=torch.int32, device="cuda")
    seq_ops.keep_rows(seq_ops.CachePages(ops, 64), b, path, kept)
    for x in want:
        for e, p in enumerate(paths):
            at = lambda r: (entries[e]["pages"][(ctx[e] + r) // 64], (ctx[e] + r) % 64)
            rows = [x[at(r)].clone() for r in p]
            for i, row in enumerate(rows):
                x[at(i)] = row
    assert all(torch.equal(x, y) for x, y in zip(want, bits(ops)))


def test_accepted_rows_move_together():
    ns, ctx = [8, 1, 40, 200, 5, 31], [60, 3, 0, 127, 64, 33]
    paths = [[0, 2, 5, 7], [0], [0, 1, 2, 30, 39], list(range(0, 200, 2)), [], [1, 3, 4, 5, 6, 7, 8, 9, 10, 11, 12, 13, 14, 15, 16, 17, 18, 30]]
    run_keep(ns, ctx, paths, lambda n: pools(n, WIDTHS) + [quantized(n, 3, 16), quantized(n, 130, 16)])


def test_every_row_moves_by_one():
    run_keep([150], [30], [list(range(1, 150))], lambda n: pools(n, WIDTHS) + [quantized(n, 8, 64)])


def test_counts_and_rows_outside_the_entry_move_nothing_else():
    b, entries, n_pages = step([4, 4], [62, 10])
    ops = pools(n_pages, WIDTHS) + [quantized(n_pages, 3, 16)]
    want = bits(ops)
    path = torch.tensor([[0, 4, -7, 1 << 30], [0, 1, 2, 3]], dtype=torch.int32, device="cuda")
    seq_ops.keep_rows(seq_ops.CachePages(ops, 64), b, path, torch.tensor([9, -2], dtype=torch.int32, device="cuda"))
    assert all(torch.equal(x, y) for x, y in zip(want, bits(ops)))


def test_captured_and_replayed():
    b, entries, n_pages = step([6], [61])
    ops = pools(n_pages, [(64, torch.bfloat16)])
    cache = seq_ops.CachePages(ops, 64)
    path, kept = torch.tensor([[0, 2, 4]], dtype=torch.int32, device="cuda"), torch.tensor([3], dtype=torch.int32, device="cuda")
    free = [p for p in range(n_pages) if p not in entries[0]["pages"]]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    start = ops[0].clone()
    with torch.cuda.stream(side):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            seq_ops.copy_pages(cache, [(entries[0]["pages"][0], free[0], 64)])
            seq_ops.keep_rows(cache, b, path, kept)
    torch.cuda.current_stream().wait_stream(side)
    same = lambda x, y: torch.equal(x.view(torch.uint8), y.view(torch.uint8))  # (bits: some are NaN)
    assert same(ops[0], start)  # (captured, not run)
    for p in ([0, 2, 4], [0, 1, 5]):
        ops[0].copy_(start)
        path.copy_(torch.tensor([p], dtype=torch.int32))
        g.replay()
        want = start.clone()
        want[free[0]] = start[entries[0]["pages"][0]]
        for i, r in enumerate(p):
            want[entries[0]["pages"][(61 + i) // 64], (61 + i) % 64] = start[entries[0]["pages"][(61 + r) // 64], (61 + r) % 64]
        assert same(ops[0], want)
