"""Attention of a few rows over the 8-bit cache where value rows differ much in size: neither a row that a query does not see nor one of hardly any weight takes the others' values away.

Tolerance: as test_attn_rows_gpu (a weight's relative rounding, scores, sums), and what is left of small weights: a row's weights are halves, scaled so that its largest product of
weight and power, T, lies in 2^14 .. 2^15; below 2^-14 halves are 2^-24 apart, so a weight is off by at most 2^-25 of them, 2^-39 T in products."""
import pytest
import torch

from test_attn_rows_gpu import Case, same
from test_cache8_gpu import PAGE

pytestmark = pytest.mark.gpu
DTYPES = [torch.bfloat16, torch.float32]


def _place(c, e, j):
    return c.entries[e]["pages"][j // PAGE], j % PAGE


def _check(c, window=0, logistic=None):
    from paligemma_multimodal_system_b200 import seq_ops
    H, G, scale = c.H, c.G, c.dim ** -0.5
    score = seq_ops.ScoreOptions(H, window) if window else seq_ops.ScoreOptions(H, logistic=True, head_bias=logistic) if logistic is not None else None
    fn = seq_ops.attn_ragged if c.b.tree is None and c.b.singles == c.b.E else seq_ops.attn_tree
    fn(c.q, *c.kv, None, c.out, c.b, H, G, c.dim, c.vdim, scale, 0.0, PAGE, score=score)
    want, tol = c.want(scale, window=window, logistic=logistic)
    pos = c.b.pos.cpu().long()
    for i, (n, ctx) in enumerate(c.lens):
        a = int(c.b.row0[i])
        k, v, seen = c.rows(0, i), c.rows(1, i), c.mask(i)
        keys = torch.cat([torch.arange(ctx), pos[a:a + n]])
        if window:
            seen = seen & (pos[a:a + n, None] - keys < window)
        at = [_place(c, i, j) for j in range(n + ctx)]
        powers = 2.0 ** (torch.stack([c.kv[1].powers[p, :, s] for p, s in at]).double().cpu() - 127)  # [keys, G]
        for h in range(H):
            s = c.q[a:a + n, h * c.dim:(h + 1) * c.dim].double().cpu() @ k[:, h // (H // G)].T * scale
            if logistic is not None:
                w = torch.sigmoid(s + float(logistic[h])) * seen
                den = torch.ones(n, 1, dtype=torch.float64)
            else:
                s = s.masked_fill(~seen, -1e300)
                w = torch.exp(s - s.max(-1, keepdim=True).values) * seen
                den = w.sum(-1, keepdim=True)
            T = (w * powers[:, h // (H // G)]).max(-1, keepdim=True).values
            codes = v[:, h // (H // G)].abs() / powers[:, h // (H // G)][:, None]
            tol[a:a + n, h] += 2.0 ** -39 * T * (seen[..., None] * codes[None]).sum(1) / den
    got = c.out.double().cpu().view(want.shape)
    same(got, want, tol)
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("above", [30, 60, 100])
def test_a_branch_that_is_not_seen(dtype, above):
    """0 -> {1 -> 3, 2 -> 4 -> 5}: node 2's value is 2^above times the others'; 0, 1 and 3 do not see it."""
    c = Case(dtype, "e4m3", [(6, 35), (2, 3)], 4, 2, 64, 64, [[-1, 0, 0, 1, 2, 4], [-1, 0]], seed=40)
    p, slot = _place(c, 0, 37)
    c.kv[1].powers[p, :, slot] += above
    got = _check(c)
    assert got[[0, 1, 3]].abs().max() < 2.0 ** 9 and got[[0, 1, 3]].abs().amax(-1).min() > 2.0 ** -8


@pytest.mark.parametrize("dtype", DTYPES)
def test_keys_behind_the_window(dtype):
    c = Case(dtype, "e4m3", [(1, 900), (1, 333), (1, 100)], 4, 2, 64, 64, seed=41)
    for i, (n, ctx) in enumerate(c.lens):
        for j in range(max(0, ctx - 99)):  # (a row at ctx sees ctx - 99 ..)
            p, slot = _place(c, i, j)
            c.kv[1].powers[p, :, slot] += 70
    got = _check(c, window=100)
    assert got.abs().max() < 2.0 ** 9


def _quiet(c, i, keys, score, above):
    """Entry i: every key's score is nearly 0, those of `keys` have `score` (nats) and values 2^above times the others'.  Queries are ones."""
    n, ctx = c.lens[i]
    c.q.fill_(1.0)
    for j in range(n + ctx):
        p, slot = _place(c, i, j)
        c.kv[0].powers[p, :, slot] -= 20
    code = {-40.0: 0xca, -20.0: 0xc2, 20.0: 0x42}[score]  # +-5, +-2.5: score = 64 / 8 * code
    for j in keys:
        p, slot = _place(c, i, j)
        c.kv[0].codes[p, slot] = code
        c.kv[0].powers[p, :, slot] = 127
        c.kv[1].powers[p, :, slot] += above


SHAPES = [("decoded", [(1, 1500)], 4, 2, None), ("tree", [(6, 200)], 8, 2, [[-1, 0, 0, 1, 2, 4]]), ("rows of many trees", [(9, 150)] * 24, 16, 4, [[-1, 0, 1, 2, 3, 4, 5, 6, 7]] * 24),
          ("scratch", [(1, 9000)], 2, 1, None)]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("name,lens,H,G,parents", SHAPES, ids=[s[0] for s in SHAPES])
@pytest.mark.parametrize("above", [20, 40, 55, 75])
def test_a_large_value_of_hardly_any_weight(dtype, name, lens, H, G, parents, above):
    """Score -40 is a weight of 2^-57.7: products from 2^-38 to 2^17 of the others'.  In the first, a middle and the last of the keys that all rows see."""
    for at in (0, 0.4, 1):
        c = Case(dtype, "e4m3", lens, H, G, 64, 64, parents, seed=42)
        for i in range(len(lens) if name != "rows of many trees" else 3):
            _quiet(c, i, [int(at * (lens[i][1] - 1))], -40.0, above)
        _check(c)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("above", [-45, 45])
@pytest.mark.parametrize("score", [-20.0, 20.0])
@pytest.mark.parametrize("first", [True, False])
def test_halves_of_a_walk_45_powers_apart(dtype, above, score, first):
    """Half of the keys are 2^45 larger or smaller and weigh e^20 more or less: the reference rises and falls along the walk."""
    for lens, parents in (([(1, 1500)], None), ([(6, 700)], [[-1, 0, 0, 1, 2, 4]])):
        c = Case(dtype, "e4m3", lens, 4, 2, 64, 64, parents, seed=43)
        half = lens[0][1] // 2
        _quiet(c, 0, range(half) if first else range(half, lens[0][1]), score, above)
        _check(c)


@pytest.mark.parametrize("dtype", DTYPES)
def test_logistic_weights(dtype):
    bias = torch.linspace(-3, 0, 4, device="cuda")
    c = Case(dtype, "e4m3", [(6, 300), (2, 3)], 4, 2, 64, 64, [[-1, 0, 0, 1, 2, 4], [-1, 0]], seed=44)
    _quiet(c, 0, [17], -40.0, 45)
    p, slot = _place(c, 0, 302)
    c.kv[1].powers[p, :, slot] += 60
    _check(c, logistic=bias)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("low,high", [(60, 60), (60, 72), (0, 200), (60, 200), (190, 200)])
def test_small_and_large_powers(dtype, low, high):
    c = Case(dtype, "e4m3", [(1, 300), (1, 1500), (1, 40)], 4, 2, 64, 64, seed=45)
    g = torch.Generator(device="cuda").manual_seed(low + high)
    c.kv[1].powers.copy_(torch.where(torch.rand(c.kv[1].powers.shape, generator=g, device="cuda") < 0.5, low, high).to(torch.uint8))
    _check(c)
