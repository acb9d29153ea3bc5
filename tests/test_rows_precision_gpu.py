"""How many bits weights and scores of attention of a few rows have, seen through the rounding of bf16 outputs: few keys, whose scores are small whole numbers over eight, so that
products and their sums are exact.

What is left, relative to A = sum_j w_ij |v_j| / sum_j w_ij (u = 2^-24, half a step of fp32; s: scores, m: their largest):
  weights    log2(e) as a number, its product with a score, the difference to the maximum: (2 |s| + 2 |m| + |s - m|) u, the exponential 2^-22; a weight and the sum: twice
  rounding   a weight as two halves 2^-22, as two bf16 terms 2^-17 (2^-18 in each of two operations)
  sums       L u for the weights', at most eight instructions or joins of 2 u each for the outputs', four roundings behind them
  a cap      three roundings in front of the tangent, a polynomial 2^-22 of its value off, two behind it: 2^-20 |s|; where a score is 0.625 caps or more, 2^-20 of the cap
and of the output at most half a step of its binade."""
import pytest
import torch

from test_attn_rows_gpu import Case, random_tree
from test_cache8_gpu import PAGE

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SHAPES = [([(1, n) for n in range(2, 12)] * 7, None), ([(6, n) for n in range(2, 12)], "tree"), ([(9, 5)] * 24, "tree")]


def _half_step(x):
    """Half a step of bf16 at x."""
    return 2.0 ** (torch.floor(torch.log2(x.abs().clamp(min=2.0 ** -100))) - 8)


def _off(cache, lens, kind, cap, H=16, G=4):
    """The largest |output - exact| - allowed."""
    from paligemma_multimodal_system_b200 import seq_ops
    c = Case(torch.bfloat16, cache, lens, H, G, 64, 64, [random_tree(n, 70 + i) for i, (n, _) in enumerate(lens)] if kind else None, seed=70)
    g = torch.Generator(device="cuda").manual_seed(7)
    c.q.copy_(torch.randint(-1, 2, c.q.shape, generator=g, device="cuda"))
    k = torch.randint(-2, 3, (c.pool, PAGE, G * 64), generator=g, device="cuda")
    if cache == "e4m3":
        c.kv[0].codes.copy_(torch.tensor([0xc0, 0xb8, 0, 0x38, 0x40], device="cuda", dtype=torch.uint8)[k + 2])
        c.kv[0].powers.fill_(127)
    else:
        c.kv[0].copy_(torch.where(c.kv[0].isnan(), c.kv[0], k.to(torch.bfloat16)))
    (seq_ops.attn_tree if kind else seq_ops.attn_ragged)(c.q, *c.kv, None, c.out, c.b, H, G, 64, 64, 0.125, cap, PAGE)
    got, worst = c.out.double().cpu().view(c.b.T, H, 64), -1.0
    for i, (n, ctx) in enumerate(c.lens):
        a, k, v, seen = int(c.b.row0[i]), c.rows(0, i), c.rows(1, i), c.mask(i)
        for h in range(H):
            s = c.q[a:a + n, h * 64:(h + 1) * 64].double().cpu() @ k[:, h // (H // G)].T * 0.125
            far = cap and bool((s.abs() >= 0.6 * cap).any())
            if cap:
                s = cap * torch.tanh(s / cap)
            s = s.masked_fill(~seen, -1e300)
            m = s.max(-1, keepdim=True).values
            w = torch.exp(s - m) * seen
            p = w / w.sum(-1, keepdim=True)
            values = v[:, h // (H // G)]
            want, A = p @ values, p @ values.abs()
            big = s[seen].abs().max()
            e = 6 * big * U + 2.0 ** -22 + (2.0 ** -20 * (cap if far else big) if cap else 0.0)
            t = A * (2 * e + (2.0 ** -22 if cache == "e4m3" else 2.0 ** -17) + (n + ctx) * U + 16 * U + 4 * U)
            half = torch.maximum(_half_step(want), _half_step(want.abs() + t))
            worst = max(worst, float(((got[a:a + n, h] - want).abs() - half - t).max()))
    return worst


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("lens,kind", SHAPES)
def test_weights(cache, lens, kind):
    if cache == "e4m3" or kind:
        assert _off(cache, lens, kind, 0.0) <= 0


@pytest.mark.parametrize("cache", ["e4m3", "same"])
@pytest.mark.parametrize("lens,kind", SHAPES)
@pytest.mark.parametrize("cap", [2.0, 30.0, 500.0, 2000.0])
def test_capped_scores(cache, lens, kind, cap):
    if cache == "e4m3" or kind:
        assert _off(cache, lens, kind, cap) <= 0
