"""Verified drafts against 64 bits.  The outputs are whole numbers: weights are right to 1e-13, so a draw differs only where u lies within some 1e-12 of a token's border."""
import pytest
import torch

from paligemma_multimodal_system_b200 import seq_ops
from verify_reference import distribution, judge, pick

pytestmark = pytest.mark.gpu


def ints(x):
    return torch.tensor(x, dtype=torch.int32, device="cuda")


def tree(n, width, g):
    up, kids = [-1], [0] * n
    for i in range(1, n):
        free = [j for j in range(i) if kids[j] < width]
        j = free[int(torch.randint(0, len(free), (), generator=g))] if width > 1 else free[-1]
        kids[j] += 1
        up.append(j)
    return up


def batch(ns, parents, tokens):
    T, row0 = sum(ns), [sum(ns[:e]) for e in range(len(ns))]
    z = torch.zeros(T, dtype=torch.int32, device="cuda")
    return seq_ops.RequestBatch(T=T, E=len(ns), max_n=max(ns), tokens=ints(tokens), pos=z, row_entry=z, row0=ints(row0), n=ints(ns), ctx=z[:len(ns)], slot=z[:len(ns)],
                                page_table=z[:len(ns)].view(-1, 1), max_pages=1, parents=ints(parents))


def make(ns, V, width, seed, spread=4.0, temperature=1.0, top_p=1.0, agree=0.5):
    g = torch.Generator().manual_seed(seed)
    T = sum(ns)
    logits = torch.randn(T, V, generator=g) * spread
    draft = logits + agree * spread * torch.randn(T, V, generator=g)
    parents, tokens, r = [], [int(t) for t in torch.randint(0, V, (T,), generator=g)], 0
    for n in ns:
        up = tree(n, width, g)
        for i in range(1, n):
            tokens[r + i] = pick(distribution(draft[r + up[i]], temperature, top_p), float(torch.rand((), generator=g)))
        parents += up
        r += n
    return logits, draft, parents, tokens, torch.rand(T, 2, generator=g)


def check(got, ns, logits, parents, tokens, uniforms, draft, temperature, top_p, draft_temperature=None, draft_top_p=None):
    path, kept, nxt = (t.cpu() for t in got)
    assert path.dtype == kept.dtype == nxt.dtype == torch.int32 and path.shape == (len(ns), max(ns))
    r = 0
    for e, n in enumerate(ns):
        walk, last = judge(logits, tokens, parents, r, n, uniforms, draft, temperature, top_p, draft_temperature or temperature, top_p if draft_top_p is None else draft_top_p)
        assert path[e].tolist() == walk + [-1] * (max(ns) - len(walk)) and int(kept[e]) == len(walk) and int(nxt[e]) == last, f"entry {e}"
        r += n


@pytest.mark.parametrize("V", [1, 2, 3, 31, 257, 4099, 32000, 70001])
@pytest.mark.parametrize("drafts", ["greedy", "guessed", "model"])
@pytest.mark.parametrize("temperature,top_p", [(1.0, 1.0), (0.7, 0.9), (2.0, 0.4)])
def test_walks(V, drafts, temperature, top_p):
    ns = [5, 1, 9, 2]
    logits, draft, parents, tokens, u = make(ns, V, 3, V + len(drafts), temperature=temperature, top_p=top_p)
    if drafts != "model":  # the most likely tokens, so that some stay
        r = 0
        for n in ns:
            for i in range(1, n):
                tokens[r + i] = int(logits[r + parents[r + i]].argmax()) if i % 2 else tokens[r + i]
            r += n
    u = None if drafts == "greedy" else u
    draft = draft if drafts == "model" else None
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), None if u is None else u.cuda(), None if draft is None else draft.cuda(), temperature, top_p)
    check(got, ns, logits, parents, tokens, u, draft, temperature, top_p)


@pytest.mark.parametrize("V,spread", [(257216, 3.0), (257216, 0.01), (300001, 2.0), (700003, 2.0)])
def test_wide_rows(V, spread):
    ns = [4, 3]
    logits, draft, parents, tokens, u = make(ns, V, 2, 3, spread=spread, temperature=0.8, top_p=0.9, agree=0.3)
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda(), 0.8, 0.9)
    check(got, ns, logits, parents, tokens, u, draft, 0.8, 0.9)


def test_many_rows_and_chains():
    ns = [1 + i % 13 for i in range(70)]
    logits, draft, parents, tokens, u = make(ns, 2003, 1, 8, agree=0.1)
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda())
    check(got, ns, logits, parents, tokens, u, draft, 1.0, 1.0)


def test_the_draft_has_settings_of_its_own():
    ns = [6, 6, 6]
    logits, draft, parents, tokens, u = make(ns, 900, 3, 21, temperature=1.3, top_p=0.8)
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda(), 0.9, 0.95, 1.3, 0.8)
    check(got, ns, logits, parents, tokens, u, draft, 0.9, 0.95, 1.3, 0.8)


@pytest.mark.parametrize("pitch", [1003, 1008, 2048])
def test_rows_at_any_pitch(pitch):
    ns, V = [4, 5], 1001
    logits, draft, parents, tokens, u = make(ns, V, 2, pitch)
    held = torch.full((2, 9, pitch), float("nan"), device="cuda")
    held[0, :, 1:1 + V], held[1, :, 2:2 + V] = logits.cuda(), draft.cuda()
    got = seq_ops.verify_drafts(held[0, :, 1:1 + V], batch(ns, parents, tokens), u.cuda(), held[1, :, 2:2 + V])
    check(got, ns, logits, parents, tokens, u, draft, 1.0, 1.0)


def test_equal_logits_stay_together_and_masked_entries_are_never_drawn():
    ns, V = [3, 3, 3], 4000
    g = torch.Generator().manual_seed(2)
    logits = torch.randint(0, 3, (9, V), generator=g).float() * 2
    logits[3:6] = 0.25  # one number everywhere
    logits[6:, 7:] = float("-inf")
    logits[6:, :3] = torch.finfo(torch.float32).min
    draft = logits.clone()
    parents, tokens = [-1, 0, 1] * 3, [0, 5, 6, 0, 17, 30, 0, 4, 5]
    for top_p in (1.0, 0.5, 0.0):
        for k in range(3):
            u = torch.rand(9, 2, generator=g)
            got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), None if k == 0 else draft.cuda(), 1.0, top_p)
            check(got, ns, logits, parents, tokens, u, None if k == 0 else draft, 1.0, top_p)


def test_the_first_of_equal_entries_wins():
    ns = [2]
    logits = torch.zeros(2, 50000)
    logits[0, [49000, 123, 30000]] = 5.0
    logits[1, 7] = -0.0
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, [-1, 0], [0, 123]))
    assert [t.tolist() for t in got] == [[[0, 1]], [2], [0]]


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_rows_that_are_no_distribution_end_the_walk(bad):
    ns, V = [3, 3, 3], 5000
    logits, draft, parents, tokens, u = make(ns, V, 1, 6, agree=0.0)
    u[:, 0] = 0  # what is drafted stays
    logits[4] = bad if bad < 0 else logits[4]
    logits[4, 17] = bad
    draft[6] = bad if bad < 0 else draft[6]
    draft[6, 4999] = bad
    draft[2, 5] = float("nan")  # (a row without children: nothing is read of it)
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda())
    check(got, ns, logits, parents, tokens, u, draft, 1.0, 1.0)
    assert got[1].tolist() == [3, 2, 1] and got[2].tolist()[1:] == [-1, -1]


def test_random_numbers_at_their_borders_and_outside():
    ns, V = [1] * 6, 100
    logits, draft, parents, tokens, u = make(ns, V, 1, 9)
    logits[:, 0] = float("-inf")
    logits[:, 99] = float("-inf")
    u[:, 1] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 1.0, 2.0, -3.0, float("nan")])
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda())
    first, last = 1, pick(distribution(logits[1], 1.0, 1.0), 1.0 - 2.0 ** -24)
    assert got[2].tolist()[:2] == [first, last]
    assert got[2].tolist()[3:] == [pick(distribution(logits[3], 1.0, 1.0), 1.0 - 2.0 ** -24), first, first]


def test_rows_that_nothing_leads_to_and_tokens_outside_the_vocabulary():
    ns, V = [5, 3], 300
    logits, draft, _, tokens, u = make(ns, V, 1, 4, agree=0.0)
    u[:, 0] = 0
    parents = [-1, -1, 0, 1, 2] + [-1, 0, 9]  # row 1 of the first entry starts a tree of its own; a parent behind its child
    tokens[6] = V + 5
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda())
    assert got[0].tolist()[0] == [0, 2, 4, -1, -1] and got[1].tolist() == [3, 1]
    tokens[6] = -1
    again = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda())
    assert again[2].tolist() == got[2].tolist()


def test_the_same_child_twice():
    """Drawn with replacement, a draft's children may be equal: the second is tried against what the first one left."""
    V, ns = 40, [3] * 200
    g = torch.Generator().manual_seed(12)
    logits, draft = torch.randn(600, V, generator=g), torch.randn(600, V, generator=g)
    tokens, parents = [7] * 600, [-1, 0, 0] * 200
    draft[:, 7] += 3
    u = torch.rand(600, 2, generator=g)
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda())
    check(got, ns, logits, parents, tokens, u, draft, 1.0, 1.0)


def test_captured_and_replayed_and_on_another_stream():
    ns = [5, 4, 7]
    sets = [make(ns, 33000, 2, s, temperature=0.8, top_p=0.9) for s in (1, 2)]
    logits, draft, u = (torch.empty_like(t, device="cuda") for t in (sets[0][0], sets[0][1], sets[0][4]))
    b = batch(ns, sets[0][2], sets[0][3])

    def fill(s):
        for to, of in zip((logits, draft, u), (s[0], s[1], s[4])):
            to.copy_(of)
        b.tokens.copy_(ints(s[3])), b.parents.copy_(ints(s[2]))

    fill(sets[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        seq_ops.verify_drafts(logits, b, u, draft, 0.8, 0.9)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = seq_ops.verify_drafts(logits, b, u, draft, 0.8, 0.9)
    torch.cuda.current_stream().wait_stream(side)
    for s in (sets[1], sets[0]):
        fill(s)
        g.replay()
        check(out, ns, s[0], s[2], s[3], s[4], s[1], 0.8, 0.9)


@pytest.mark.parametrize("spread,top_p", [(0.05, 0.9), (1.0, 0.99), (1.0, 0.999999), (6.0, 0.9)])
@pytest.mark.parametrize("V", [9000, 150000])
def test_flat_and_steep_rows(V, spread, top_p):
    """More entries that may belong to the nucleus than are kept in shared memory, a border far down, and one among the first entries."""
    ns = [3, 4]
    logits, draft, parents, tokens, u = make(ns, V, 2, 31, spread=spread, top_p=top_p, agree=0.5)
    for d in (draft, None):
        got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), None if d is None else d.cuda(), 1.0, top_p)
        check(got, ns, logits, parents, tokens, u, d, 1.0, top_p)


@pytest.mark.parametrize("temperature", [1e-29, 1e-6, 0.01, 30.0, 1e6, 1e300])
@pytest.mark.parametrize("offset", [0.0, -500.0, 3e4, 1e30])
def test_temperatures_and_sizes_of_logits(temperature, offset):
    ns = [3]
    logits, draft, parents, tokens, u = make(ns, 5000, 1, 77, agree=0.0)
    logits, draft = logits + offset, draft + offset
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda(), temperature, 0.9)
    check(got, ns, logits, parents, tokens, u, draft, temperature, 0.9)


def test_two_streams_at_once():
    ns = [7, 3, 9, 1]
    logits, draft, parents, tokens, u = make(ns, 60000, 2, 5, temperature=0.8, top_p=0.9)
    dev = (logits.cuda(), batch(ns, parents, tokens), u.cuda(), draft.cuda(), 0.8, 0.9)
    torch.cuda.synchronize()
    streams, outs = [torch.cuda.Stream() for _ in range(3)], []
    for s in streams * 4:
        with torch.cuda.stream(s):
            outs.append(seq_ops.verify_drafts(*dev))
    torch.cuda.synchronize()
    for o in outs:
        check(o, ns, logits, parents, tokens, u, draft, 0.8, 0.9)


def test_a_long_chain():
    """More rows in front of one than a warp has lanes."""
    n, V = 90, 400
    g = torch.Generator().manual_seed(3)
    logits = torch.randn(n, V, generator=g)
    tokens = [0] + logits.argmax(-1).tolist()[:-1]
    parents = list(range(-1, n - 1))
    for wrong in (None, 40, 85):
        t = list(tokens)
        if wrong is not None:
            t[wrong] = (t[wrong] + 1) % V
        for copies in (1, 40):
            got = seq_ops.verify_drafts(logits.repeat(copies, 1).cuda(), batch([n] * copies, parents * copies, t * copies))
            stop = n if wrong is None else wrong
            assert got[1].tolist() == [stop] * copies and got[0][-1].tolist() == list(range(stop)) + [-1] * (n - stop)
            assert got[2].tolist() == [int(logits[stop - 1].argmax())] * copies


@pytest.mark.parametrize("step", ["bfloat16", 0.125, 0.002])
@pytest.mark.parametrize("V,spread,top_p", [(257216, 3.0, 0.9), (32000, 2.0, 0.7), (32000, 0.3, 0.5), (5000, 4.0, 0.95)])
def test_logits_of_few_values(step, V, spread, top_p):
    """Many entries equal the border's, in shares of several CTAs; runs of bit patterns that are divided until they are one."""
    ns = [3, 4, 2]
    logits, draft, parents, tokens, u = make(ns, V, 2, 13, spread=spread, temperature=0.8, top_p=top_p)
    coarse = (lambda t: t.bfloat16().float()) if step == "bfloat16" else (lambda t: (t / step).round() * step)
    logits, draft = coarse(logits), coarse(draft)
    for d in (None, draft):
        got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), u.cuda(), None if d is None else d.cuda(), 0.8, top_p)
        check(got, ns, logits, parents, tokens, u, d, 0.8, top_p)


@pytest.mark.parametrize("greedy,entries,n", [(True, 230, 9), (True, 300, 10), (False, 1900, 9)])
def test_more_rows_than_the_walk_keeps_in_shared_memory(greedy, entries, n):
    V, ns = 24, [n] * entries
    logits, draft, parents, tokens, u = make(ns, V, 2, 17, agree=0.2)
    u = None if greedy else u
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens), None if greedy else u.cuda(), None if greedy else draft.cuda())
    check(got, ns, logits, parents, tokens, u, None if greedy else draft, 1.0, 1.0)


def test_one_row_behind_another_that_is_not_drafted():
    """A step in which some entries bring prompts: their rows are a chain, their tokens are judged like guesses."""
    V, ns, g = 700, [1, 70, 5, 1], torch.Generator().manual_seed(23)
    logits = torch.randn(sum(ns), V, generator=g) * 3
    parents = [i - 1 for n in ns for i in range(n)]
    tokens = [int(t) for t in torch.randint(0, V, (sum(ns),), generator=g)]
    got = seq_ops.verify_drafts(logits.cuda(), batch(ns, parents, tokens))
    check(got, ns, logits, parents, tokens, None, None, 1.0, 1.0)
