"""Attention of a few rows an entry (pg_attn_rows): decoded tokens over the 8-bit cache and drafted trees over a cache of any type, against the formula in 64 bits on the
same cached values.

Tolerance per element, with A = sum_j w_ij |v_j| / sum_j w_ij and Z = max_j scale sum_d |q_d k_jd|: scores are sums of fp32 products whose partial sums may be cut
(2^-23 an addition, at most 24 additions): delta = 2^-18 Z, plus 2^-20 for the exponential and what bends the score; weights are then off by 2 delta A.  The sum over L keys adds
(L / 16 * terms + 8) 2^-23 A.  A weight's own rounding: 2^-11 (one half: 8-bit cache under bf16 rows), else 2^-15 (two bf16 terms) or less.  The output: half a step."""
import math

import numpy as np
import pytest
import torch

from test_cache8_gpu import PAGE, batch_of, fresh, stored, values_of

pytestmark = pytest.mark.gpu


class Case:
    def __init__(self, dtype, cache, lens, H, G, dim, vdim, parents=None, seed=0, spread=1.0):
        self.dtype, self.cache, self.lens, self.H, self.G, self.dim, self.vdim = dtype, cache, lens, H, G, dim, vdim
        self.b, self.entries, self.pool = batch_of(lens, seed, parents)
        g = torch.Generator(device="cuda").manual_seed(seed * 31 + dim + H)
        T = self.b.T
        self.q = (torch.randn(T, H * dim, generator=g, device="cuda") * spread).to(dtype)
        self.kv, self.keep = [], []
        for size in (dim, vdim):
            if cache == "e4m3":
                pages = fresh(self.pool, G, size)
                new = torch.randint(0, 256, pages.codes.shape, generator=g, device="cuda", dtype=torch.uint8)
                new = torch.where((new & 0x7f) == 0x7f, new ^ 0x10, new)
                powers = torch.randint(117, 123, pages.powers.shape, generator=g, device="cuda", dtype=torch.uint8)
            else:
                pages = torch.full((self.pool, PAGE, G * size), math.nan, device="cuda", dtype=dtype)
                new = torch.randn(pages.shape, generator=g, device="cuda").to(dtype)
                powers = None
            for e, (n, ctx) in zip(self.entries, lens):  # rows that nobody owns stay NaN
                for j0 in range(0, n + ctx, PAGE):
                    p, m = e["pages"][j0 // PAGE], min(PAGE, n + ctx - j0)
                    if powers is None:
                        pages[p, :m] = new[p, :m]
                    else:
                        pages.codes[p, :m], pages.powers[p, :, :m] = new[p, :m], powers[p, :, :m]
            self.kv.append(pages)
        self.out = torch.full((T, H * vdim), 7.0, device="cuda", dtype=dtype)

    def rows(self, which, i):
        """float64 [ctx + n, G, size] of one entry."""
        pages, (n, ctx) = self.kv[which], self.lens[i]
        if self.cache == "e4m3":
            return torch.from_numpy(values_of(*stored(pages, self.entries[i], n + ctx, self.G)))
        p = torch.tensor(self.entries[i]["pages"], device="cuda")
        return pages[p].flatten(0, 1)[:n + ctx].double().cpu().unflatten(-1, (self.G, -1))

    def mask(self, i):
        n, ctx = self.lens[i]
        a = int(self.b.row0[i])
        seen = torch.ones(n, n + ctx, dtype=torch.bool)
        if self.b.tree is None:
            seen[:, ctx:] = torch.tril(torch.ones(n, n, dtype=torch.bool))
        else:
            words = self.b.tree[a:a + n].cpu().long() & 0xFFFFFFFF
            seen[:, ctx:] = ((words[:, :, None] >> torch.arange(32)) & 1).flatten(1)[:, :n].bool()
        return seen

    def want(self, scale, softcap=0.0, gate=None, per_head=False, window=0, keep=0, sink=None, dist=None, head_scale=None, logistic=None, out_scale=1.0):
        """(exact [T, H, vdim], allowed difference) in float64."""
        T, H, G, vdim = self.b.T, self.H, self.G, self.vdim
        out, tol = torch.zeros(T, H, vdim, dtype=torch.float64), torch.zeros(T, H, vdim, dtype=torch.float64)
        pos = self.b.pos.cpu().long()
        weight_step = (2.0 ** -11 if self.dtype == torch.bfloat16 else 2.0 ** -21) if self.cache == "e4m3" else 2.0 ** -15 if self.dtype == torch.bfloat16 else 2.0 ** -21
        terms = 6 if self.dtype == torch.float32 else 2
        for i, (n, ctx) in enumerate(self.lens):
            a, L = int(self.b.row0[i]), n + ctx
            k, v, seen = self.rows(0, i), self.rows(1, i), self.mask(i)
            mine = pos[a:a + n]
            keys = torch.cat([torch.arange(ctx), mine])
            if window:
                seen = seen & ((mine[:, None] - keys < window) | (keys < keep))
            for h in range(H):
                q = self.q[a:a + n, h * self.dim:(h + 1) * self.dim].double().cpu()
                f = scale * (1.0 if head_scale is None else float(head_scale[h]))
                s, Z = q @ k[:, h // (H // G)].T * f, q.abs() @ torch.nan_to_num(k[:, h // (H // G)]).abs().T * abs(f)
                if softcap:
                    s = softcap * torch.tanh(s / softcap)
                if dist is not None:
                    s = s - float(dist[0][h]) * torch.log1p(float(dist[1][h]) * (mine[:, None] - keys).clamp(min=0))
                vals = v[:, h // (H // G)]
                if logistic is not None:
                    w = torch.sigmoid(s + float(logistic[h])) * seen
                    den = torch.ones(n, 1, dtype=torch.float64)
                else:
                    s = s.masked_fill(~seen, -math.inf)
                    m = s.max(-1, keepdim=True).values.clamp(min=-1e300)
                    if sink is not None:
                        m = m.clamp(min=float(sink[h]))
                    w = torch.exp(s - m)
                    den = w.sum(-1, keepdim=True) + (0 if sink is None else math.exp(float(sink[h])) * torch.exp(-m))
                used = torch.where(seen[..., None], vals[None], 0.0)  # a value reaches only the rows that see it
                o = torch.einsum("nj,njd->nd", w, used)
                A = torch.einsum("nj,njd->nd", w, torch.nan_to_num(used).abs())
                den = torch.where(den == 0, 1.0, den)
                o, A = o / den, A / den
                delta = (2.0 ** -18 * (Z * seen).max(-1, keepdim=True).values + 2.0 ** -19)
                t = (2 * delta + weight_step + (L / 16 * terms + 8) * 2.0 ** -23) * A
                if gate is not None:
                    gt = gate[a:a + n].double().cpu()
                    gt = torch.sigmoid(gt[:, h:h + 1] if per_head else gt[:, h * vdim:(h + 1) * vdim])
                    o, t = o * gt, t * gt + 2.0 ** -21 * o.abs()
                out[a:a + n, h], tol[a:a + n, h] = o * out_scale, t * out_scale
        tol = tol + torch.finfo(self.dtype).eps / 2 * torch.nan_to_num(out).abs() + 1e-30
        return out, tol

    def check(self, scale=None, score=None, tree=True, **options):
        from paligemma_multimodal_system_b200 import seq_ops
        scale = self.dim ** -0.5 if scale is None else scale
        fn = seq_ops.attn_tree if tree else seq_ops.attn_ragged
        fn(self.q, *self.kv, options.get("gate"), self.out, self.b, self.H, self.G, self.dim, self.vdim, scale, options.get("softcap", 0.0), PAGE,
           gate_per_head=options.get("per_head", False), score=score)
        want, tol = self.want(scale, **options)
        got = self.out.double().cpu().view(want.shape)
        same(got, want, tol)
        return got


def same(got, want, tol):
    fine = torch.isfinite(want)
    assert torch.equal(torch.isfinite(got), fine), (got[~fine], torch.nonzero(torch.isfinite(got) != fine)[:4])
    over = ((got - want).abs() - tol)[fine]
    assert over.max() <= 0, (over.max(), tol[fine].max(), torch.nonzero(((got - want).abs() > tol) & fine)[:5])


def random_tree(n, seed):
    r = np.random.RandomState(seed)
    return [-1 if i == 0 or r.rand() < 0.15 else int(r.randint(max(0, i - 6), i)) for i in range(n)]


FORMS = [(torch.bfloat16, "e4m3"), (torch.float32, "e4m3"), (torch.bfloat16, "same"), (torch.float32, "same")]
HEADS = [(4, 2, 64, 64), (2, 2, 32, 32), (8, 1, 128, 128), (7, 1, 96, 64), (16, 2, 64, 128), (6, 2, 16, 16), (24, 1, 128, 32)]


@pytest.mark.parametrize("dtype,cache", FORMS)
@pytest.mark.parametrize("H,G,dim,vdim", HEADS)
def test_trees_of_every_kind(dtype, cache, H, G, dim, vdim):
    lens = [(1, 0), (2, 0), (5, 31), (3, 63), (9, 64), (33, 30), (17, 200)]
    Case(dtype, cache, lens, H, G, dim, vdim, [random_tree(n, i) for i, (n, _) in enumerate(lens)], seed=dim).check()


@pytest.mark.parametrize("dtype,cache", FORMS)
@pytest.mark.parametrize("lens", [[(1, 1500)], [(1, 2000), (1, 0), (1, 31), (1, 32), (1, 64), (1, 1111)], [(64, 900)], [(40, 3), (65, 70)]])
def test_lengths_and_chains(dtype, cache, lens):
    Case(dtype, cache, lens, 8, 2, 64, 64, seed=len(lens)).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,dim,vdim", HEADS)
def test_decoded_tokens(dtype, H, G, dim, vdim):
    Case(dtype, "e4m3", [(1, c) for c in (0, 1, 30, 31, 32, 63, 64, 65, 500, 1023, 1500)], H, G, dim, vdim, seed=3).check(tree=False)


def test_a_long_context():
    Case(torch.bfloat16, "e4m3", [(1, 20011)], 4, 1, 64, 64, seed=4).check(tree=False)
    Case(torch.bfloat16, "same", [(6, 9001)], 4, 1, 128, 128, [random_tree(6, 1)], seed=5).check()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("H,G,dim,vdim", [(4, 2, 64, 64), (8, 2, 128, 128), (3, 3, 48, 32)])
def test_mixed_steps_over_8_bit_pages(dtype, H, G, dim, vdim):
    """Prompt portions (rows read back, the attention of prompts) beside decoded tokens; tolerance of the prompt kernels: as the formula above."""
    Case(dtype, "e4m3", [(1, 77), (40, 30), (1, 0), (130, 0), (2, 600), (1, 300)], H, G, dim, vdim, seed=6).check(tree=False)


@pytest.mark.parametrize("dtype,cache", FORMS)
def test_score_options(dtype, cache):
    from paligemma_multimodal_system_b200 import seq_ops
    H, G = 6, 3
    g = torch.Generator(device="cuda").manual_seed(8)
    lens = [(9, 150), (1, 40), (20, 5), (4, 700)]
    parents = [random_tree(n, i + 50) for i, (n, _) in enumerate(lens)]

    def vec(lo, hi):
        return torch.rand(H, generator=g, device="cuda") * (hi - lo) + lo

    sink, da, db, hs, bias = vec(-1, 2), vec(0, 1), vec(0, 1), vec(0.5, 2), vec(-3, 0)
    for options, kw in [
        (dict(window=40), dict(window=40)),
        (dict(window=33, keep_first=5), dict(window=33, keep=5)),
        (dict(window=1, keep_first=70), dict(window=1, keep=70)),
        (dict(sink=sink), dict(sink=sink)),
        (dict(head_scale=hs), dict(head_scale=hs)),
        (dict(dist_a=da, dist_b=db), dict(dist=(da, db))),
        (dict(window=100, keep_first=4, sink=sink, dist_a=da, dist_b=db, head_scale=hs), dict(window=100, keep=4, sink=sink, dist=(da, db), head_scale=hs)),
        (dict(logistic=True, head_bias=bias), dict(logistic=bias)),
        (dict(logistic=True, head_bias=bias, out_scale=0.125), dict(logistic=bias, out_scale=0.125)),
    ]:
        c = Case(dtype, cache, lens, H, G, 64, 64, parents, seed=9)
        c.check(score=seq_ops.ScoreOptions(H, **options), **kw)
    for per_head in (False, True):
        c = Case(dtype, cache, lens, H, G, 64, 64, parents, seed=10)
        gate = torch.randn(c.b.T, (H if per_head else H * 64) + 5, generator=g, device="cuda").to(dtype)[:, 2:2 + (H if per_head else H * 64)]
        c.check(gate=gate, per_head=per_head, softcap=30.0)
    c = Case(dtype, cache, lens, H, G, 64, 64, parents, seed=11, spread=20.0)
    c.check(softcap=5.0)


@pytest.mark.parametrize("window", [0, 600])
def test_decoded_tokens_with_options(window):
    from paligemma_multimodal_system_b200 import seq_ops
    H = 8
    sink = torch.linspace(-1, 1, H, device="cuda")
    c = Case(torch.bfloat16, "e4m3", [(1, 2100), (1, 10), (1, 640)], H, 2, 64, 64, seed=12)
    gate = torch.randn(3, H * 64, device="cuda").to(torch.bfloat16)
    c.check(tree=False, score=seq_ops.ScoreOptions(H, window or None, 4, sink=sink), gate=gate, softcap=50.0, window=window, keep=4 if window else 0, sink=sink)


@pytest.mark.parametrize("dtype,cache", FORMS)
def test_rows_that_see_nothing_get_zeros(dtype, cache):
    c = Case(dtype, cache, [(5, 0), (3, 20), (40, 0)], 4, 2, 64, 64, [random_tree(5, 1), random_tree(3, 2), random_tree(40, 3)], seed=13)
    c.b.tree[1] = 0
    c.b.tree[6] = 0   # (sees the stored keys)
    c.b.tree[20] = 0
    got = c.check()
    assert not got[1].any() and not got[20].any() and got[6].any()


@pytest.mark.parametrize("dtype,cache", FORMS)
@pytest.mark.parametrize("what", [math.nan, math.inf, -math.inf])
def test_what_is_no_number_reaches_only_rows_that_see_it(dtype, cache, what):
    """A drafted key or value that overflowed: its own branch has it, the sibling branch does not."""
    n, ctx, G = 6, 35, 2
    parents = [-1, 0, 0, 1, 2, 4]  # 0 -> {1 -> 3, 2 -> 4 -> 5}
    for which in (0, 1):
        c = Case(dtype, cache, [(n, ctx), (2, 3)], 4, G, 64, 64, [parents, [-1, 0]], seed=14)
        clean = c.check().clone()
        j = ctx + 2
        p, slot = c.entries[0]["pages"][j // PAGE], j % PAGE
        if cache == "e4m3":
            c.kv[which].codes[p, slot, 70] = 0x7f
        else:
            c.kv[which][p, slot, 70] = what
        from paligemma_multimodal_system_b200 import seq_ops
        seq_ops.attn_tree(c.q, *c.kv, None, c.out, c.b, 4, G, 64, 64, 0.125, 0.0, PAGE)
        got = c.out.double().cpu().view(clean.shape)
        for t in (0, 1, 3, 6, 7):
            assert torch.equal(got[t], clean[t]), t
        assert torch.equal(got[:, :2], clean[:, :2])  # the other k/v head's
        for t in (2, 4, 5):
            if which == 1:
                assert not torch.isfinite(got[t, 2:, 6]).any() and torch.isfinite(got[t, 2:, :6]).all()
            elif what != what or cache == "e4m3":
                assert got[t, 2:].isnan().all()


def test_masks_wider_than_the_tree_and_bits_behind_it():
    c = Case(torch.bfloat16, "same", [(5, 10), (2, 30)], 4, 2, 64, 64, [random_tree(5, 1), [-1, 0]], seed=15)
    first = c.check()
    wide = torch.full((c.b.T, 4), -1, dtype=torch.int32, device="cuda")
    wide[:, :1] = c.b.tree
    wide[:5, 0] |= ~0x1f  # bits from n on are nobody's
    wide[5:, 0] |= ~0x3
    c.b.tree = wide
    c.out.fill_(3.0)
    assert torch.equal(c.check(), first)


def test_rows_outside_the_entries_are_left_alone():
    c = Case(torch.bfloat16, "e4m3", [(3, 40), (1, 90), (2, 5)], 4, 2, 64, 64, seed=16)
    c.b.n[1] = 0  # an entry that a padded step leaves out
    from paligemma_multimodal_system_b200 import seq_ops
    seq_ops.attn_tree(c.q, *c.kv, None, c.out, c.b, 4, 2, 64, 64, 0.125, 0.0, PAGE)
    want, tol = c.want(0.125)
    got = c.out.double().cpu().view(want.shape)
    rows = [0, 1, 2, 4, 5]
    same(got[rows], want[rows], tol[rows])
    assert (got[3] == 7.0).all()


def test_captured_and_replayed_beside_another_graph():
    """Two captured decode steps share no scratch; replays in turn give what the eager calls give."""
    from paligemma_multimodal_system_b200 import seq_ops
    cases = [Case(torch.bfloat16, "e4m3", [(1, 1700 + 100 * i), (1, 900)], 8, 2, 64, 64, seed=17 + i) for i in range(2)]

    def go(c):
        seq_ops.attn_ragged(c.q, *c.kv, None, c.out, c.b, 8, 2, 64, 64, 0.125, 0.0, PAGE)

    eager = []
    for c in cases:
        go(c)
        eager.append(c.out.clone())
    graphs = []
    side = torch.cuda.Stream()
    for c in cases:
        with torch.cuda.stream(side):
            g = torch.cuda.CUDAGraph()
            with torch.cuda.graph(g, stream=side):
                go(c)
        graphs.append(g)
    torch.cuda.synchronize()
    for c in cases:
        c.out.zero_()
    for _ in range(3):
        for g in graphs:
            g.replay()
    torch.cuda.synchronize()
    for c, e in zip(cases, eager):
        assert torch.equal(c.out, e)


def test_the_same_call_gives_the_same_bits():
    from paligemma_multimodal_system_b200 import seq_ops
    c = Case(torch.bfloat16, "same", [(12, 1500), (30, 400)], 8, 2, 64, 64, [random_tree(12, 1), random_tree(30, 2)], seed=20)
    seen = []
    for _ in range(4):
        seq_ops.attn_tree(c.q, *c.kv, None, c.out, c.b, 8, 2, 64, 64, 0.125, 0.0, PAGE)
        seen.append(c.out.clone())
    assert all(torch.equal(x, seen[0]) for x in seen)


@pytest.mark.parametrize("dtype,cache", [(torch.float32, "same"), (torch.float32, "e4m3")])
@pytest.mark.parametrize("nodes", [1, 13])
def test_long_sums_are_rounded_and_not_cut(dtype, cache, nodes):
    """Values of one sign under nearly equal weights, walks that nobody shares (24 entries x 8 heads): about 90 tiles are added to a growing sum.  Rounded to nearest they are off by
    half a step of 2^-24 each with random signs, sqrt(90) 2^-24 = 2^-20.8 together and a sixth of 2^-18; cut off, by half a step with one sign an instruction, six of them a tile:
    90 * 6 * 2^-25 = 2^-16.  Weights: three bf16 terms (2^-24) or two halves (2^-22 at random); what a score or the exponential is off has the same sign for all keys of a row and cancels."""
    c = Case(dtype, cache, [(nodes, 3000 - 9 * i) for i in range(24)], 16, 8, 64, 64, None if nodes == 1 else [random_tree(nodes, i) for i in range(24)], seed=30, spread=1e-3)
    v = c.kv[1]
    if cache == "e4m3":
        v.codes.bitwise_and_(0x7f)
        v.codes.copy_(torch.where(v.codes == 0x7f, v.codes, 0x38 + v.codes % 8))  # 1 .. 1.875
        v.powers.fill_(120)
        c.kv[0].powers.fill_(110)  # (small scores)
    else:
        v.abs_().add_(0.5)
    got = c.check()
    want, _ = c.want(c.dim ** -0.5)
    assert float(((got - want) / want).abs().max()) < 2.0 ** -18
