"""Operators of what a request has of its own in the ragged-step engine, as cases that can be timed and checked: which of its drafted tokens stay, the
cache pages that it forks from another request and the rows that it keeps of a drafted tree, and its low-rank adapter.

A case is a dict of plain values; `kind` says which operator it takes:

  verify  drafted trees against the target's distributions, from given random numbers (`seq_ops.verify_drafts`)
  fork    the first rows of pages into other pages, all layers at once (`seq_ops.copy_pages`)
  keep    the rows of an accepted path move together behind the stored ones, all layers at once (`seq_ops.keep_rows`)
  adapt   low-rank adapters of the step's requests, added to a shared projection (`seq_ops.adapter_add`)

The rules of `verify`.  Row v of an entry holds the logits behind drafted token v; row 0 belongs to the request's pending token, which stays.  A row's
distribution is softmax(x / temperature) cut to its nucleus: a token belongs to it if the mass of the strictly more probable ones is at most top_p.
Without drafted distributions a token is drawn from the row (`greedy`: its first largest entry) and the walk goes on at the child that carries it.  With
them (row v of the draft's logits, from which v's children were drawn) children are tried in order against what the rejected ones left:
with c = 0 and S = 1, child x stays if u q(x) S < max(p(x) - c q(x), 0), and else c <- c + S, S <- sum max(p - c q, 0).  The token behind the walk is
drawn from max(p - c q, 0) of its last row, from p where that is nothing.  Drawn means the first id whose running sum is above u times the whole.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # one request checks four tokens that were guessed from its own text, PaliGemma's vocabulary (latency)
        dict(name="verify-one", kind="verify", entries=1, nodes=5, vocab=257216, drafts="guessed", width=1, temperature=0.8, top_p=0.9),
        # greedy decoding of a batch with guessed trees
        dict(name="verify-greedy", kind="verify", entries=16, nodes=8, vocab=257216, drafts="greedy", width=2, temperature=1.0, top_p=1.0),
        # a full batch with a drafting model, chains of seven behind the pending token
        dict(name="verify-batch", kind="verify", entries=32, nodes=8, vocab=257216, drafts="model", width=1, temperature=0.8, top_p=0.9),
        # a smaller vocabulary, trees with several children a node, whole distributions
        dict(name="verify-trees", kind="verify", entries=48, nodes=13, vocab=32000, drafts="model", width=3, temperature=1.0, top_p=1.0),
        # one request forks at a page that is filled to a third (latency)
        dict(name="fork-one", kind="fork", dtype="bfloat16", moves=1, rows=21, layers=12, width=512),
        # 32 requests with eight samples each
        dict(name="fork-samples", kind="fork", dtype="bfloat16", moves=256, rows=64, layers=12, width=512),
        # one request keeps five of its drafted tokens (latency)
        dict(name="keep-one", kind="keep", dtype="bfloat16", entries=1, nodes=8, context=1100, layers=12, width=512),
        # a batch with trees of up to 31 tokens, cache rows in full precision
        dict(name="keep-batch", kind="keep", dtype="float32", entries=48, nodes=31, context=150, layers=8, width=1024),
        # one decoding request, joint query, key and value projection (latency)
        dict(name="adapt-one", kind="adapt", dtype="bfloat16", out="bfloat16", prompts=0, longest=0, singles=1, adapters=1, rank=16, depth=2048, parts="2048,256,256"),
        # a full decode batch with 20 adapters, output projection into the residual stream
        dict(name="adapt-batch", kind="adapt", dtype="bfloat16", out="float32", prompts=0, longest=0, singles=64, adapters=20, rank=32, depth=2048, parts="2048"),
        # prompts of up to 1024 tokens beside decoding requests
        dict(name="adapt-prompts", kind="adapt", dtype="bfloat16", out="bfloat16", prompts=8, longest=1024, singles=32, adapters=7, rank=64, depth=2048, parts="2048,256,256"),
        # full precision
        dict(name="adapt-fp32", kind="adapt", dtype="float32", out="float32", prompts=3, longest=333, singles=5, adapters=4, rank=8, depth=1024, parts="1024,256"),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["verify", "verify", "fork", "keep", "adapt", "adapt", "adapt"])
    if kind == "verify":
        drafts = rng.choice(["guessed", "greedy", "model", "model"])
        vocab = rng.choice([32000, 257216, 257152, _spread(rng, 1000, 130001)])
        nodes = _spread(rng, 1, 24)
        entries = _spread(rng, 1, max(1, min(64, 40_000_000 // (vocab * nodes))))
        return dict(kind=kind, entries=entries, nodes=nodes, vocab=vocab, drafts=drafts, width=rng.choice([1, 1, 2, 4]), temperature=rng.choice([1.0, 0.8, 0.6]),
                    top_p=rng.choice([1.0, 0.9, 0.95, 0.5]))
    dtype = rng.choice(["bfloat16", "bfloat16", "float32"])
    if kind == "fork":
        return dict(kind=kind, dtype=dtype, moves=_spread(rng, 1, 128), rows=rng.randint(1, 64), layers=_spread(rng, 1, 12), width=rng.choice([64, 72, 256, 512, _spread(rng, 33, 500)]))
    if kind == "keep":
        return dict(kind=kind, dtype=dtype, entries=_spread(rng, 1, 48), nodes=_spread(rng, 1, 40), context=_spread(rng, 1, 300), layers=_spread(rng, 1, 8),
                    width=rng.choice([64, 72, 256, 512, 1024, _spread(rng, 33, 500)]))
    prompts = rng.choice([0, rng.randint(1, 6)])
    longest = _spread(rng, 2, 700) if prompts else 0
    parts = ",".join(str(8 * _spread(rng, 8, 256)) for _ in range(rng.randint(1, 3)))
    return dict(kind=kind, dtype=dtype, out=rng.choice([dtype, "float32"]), prompts=prompts, longest=longest, singles=_spread(rng, 1, 64), adapters=rng.randint(1, 24),
                rank=rng.choice([4, 8, 16, 16, 32, 64, 24]), depth=8 * _spread(rng, 8, 320), parts=parts)


# ------------------------------------------------------------------------------------------------------------------------ inputs
def _parents(n, width, r):
    """A drafted tree: node 0 is the pending token; up to `width` children a node, later nodes mostly below the newest ones."""
    up, kids = [-1], [0] * n
    for i in range(1, n):
        free = [j for j in range(i) if kids[j] < width]
        j = free[-1] if width == 1 or r.rand() < 0.5 else free[r.randint(0, len(free))]
        kids[j] += 1
        up.append(j)
    return up


def _nodes(c):
    """Rows of every entry."""
    return [max(1, c["nodes"] - (e * 3) % max(1, c["nodes"] // 2)) for e in range(c["entries"])]


def _entries(c):
    """Rows of every entry of an `adapt` case: prompts first, then decoded tokens."""
    return [max(2, c["longest"] - (i * 61) % max(1, c["longest"] // 2)) for i in range(c["prompts"])] + [1] * c["singles"]


def _adapter_of(c, r):
    """Adapters of the entries, -1 for one in eight that has none."""
    return [-1 if r.rand() < 0.125 and c["singles"] + c["prompts"] > 1 else int(r.randint(0, c["adapters"])) for _ in _entries(c)]


def _logits(g, rows, vocab):
    """A model's logits: most of the mass on some dozens of tokens."""
    x = torch.randn(rows, vocab, generator=g, device="cuda").mul_(2.5)
    liked = torch.randint(0, vocab, (rows, 24), generator=g, device="cuda")
    return x.scatter_add_(1, liked, torch.rand(rows, 24, generator=g, device="cuda") * 14)


def _pool(g, c, pages):
    return [torch.randn(pages, PAGE, c["width"], generator=g, device="cuda").to(DTYPES[c["dtype"]]) for _ in range(2 * c["layers"])]


def prepare(case, seed):
    c, kind = case, case["kind"]
    torch.cuda.set_device(0)
    g = torch.Generator(device="cuda").manual_seed((seed * 1000003 + 29) & 0x7FFFFFFF)
    r = np.random.RandomState((seed * 11 + 5) & 0x7FFFFFFF)
    s = dict(c)

    def ints(x):
        return torch.from_numpy(np.ascontiguousarray(np.asarray(x, np.int32))).cuda()

    if kind == "verify":
        ns, V = _nodes(c), c["vocab"]
        T = sum(ns)
        up = [_parents(n, c["width"], r) for n in ns]
        row0 = np.cumsum([0] + ns[:-1])
        s["parents"] = up
        logits = _logits(g, T, V)
        draft = logits + 0.6 * torch.randn(T, V, generator=g, device="cuda")  # what a smaller model thinks of the same text
        tokens = torch.randint(0, V, (T,), generator=g, device="cuda")
        for e, n in enumerate(ns):
            kids = {}
            for i in range(1, n):
                kids.setdefault(up[e][i], []).append(i)
            for v, cs in kids.items():
                at = torch.tensor([row0[e] + i for i in cs], device="cuda")
                if c["drafts"] == "model":  # drawn from the draft's own nucleus
                    w = torch.softmax(draft[row0[e] + v].double() / c["temperature"], 0)
                    top, ids = torch.sort(w, descending=True)
                    top = torch.where(torch.cumsum(top, 0) - top <= c["top_p"], top, 0.0)
                    u = torch.rand(len(cs), generator=g, device="cuda", dtype=torch.float64) * top.sum()
                    tokens[at] = ids[torch.searchsorted(torch.cumsum(top, 0), u, right=True).clamp(max=V - 1)]
                else:  # the most likely ones
                    tokens[at] = torch.topk(draft[row0[e] + v], len(cs)).indices
        s["logits"], s["draft"] = logits, draft if c["drafts"] == "model" else None
        s["uniforms"] = None if c["drafts"] == "greedy" else torch.rand(T, 2, generator=g, device="cuda")  # acceptance of token v, draw at row v
        n = np.array(ns, np.int32)
        entry = np.repeat(np.arange(len(ns)), ns)
        s["plan"] = dict(T=T, E=len(ns), max_n=max(ns), min_n=min(ns), tokens=tokens.int(), pos=ints(np.arange(T) - row0[entry]), row_entry=ints(entry), row0=ints(row0), n=ints(n),
                         ctx=ints(0 * n), slot=ints(0 * n), page_table=ints(np.zeros((len(ns), 1))), max_pages=1, parents=ints(np.concatenate(up)))
        return s
    if kind == "fork":  # pages in any order; a few that nothing touches
        pages = 2 * c["moves"] + 3
        order = r.permutation(pages)
        rows = [max(1, c["rows"] - (i * 7) % max(1, c["rows"])) for i in range(c["moves"])]
        s["moves"] = np.stack([order[:c["moves"]], order[c["moves"]:2 * c["moves"]], rows], 1).astype(np.int32)
        if c["moves"] > 8:  # samples of one request come from one page
            s["moves"][:, 0] = s["moves"][np.arange(c["moves"]) // 8 * 8, 0]
        s["pool"] = _pool(g, c, pages)
    elif kind == "keep":
        ns, E = _nodes(c), c["entries"]
        ctx = [max(0, c["context"] - (e * 53) % max(1, c["context"])) for e in range(E)]
        held = [-(-(x + n) // PAGE) for x, n in zip(ctx, ns)]
        order, table, at = r.permutation(sum(held) + 2), np.zeros((E, max(held)), np.int32), 0
        path, kept = np.full((E, max(ns)), -1, np.int32), np.zeros(E, np.int32)
        for e, n in enumerate(ns):
            table[e, :held[e]] = order[at:at + held[e]]
            at += held[e]
            # a main chain of half of the rows, then another continuation of it: the first `a` rows stay where they are, `d` of the others follow
            a = int(r.randint(0, n // 2 + 1))
            d = int(r.randint(0, max(1, min(n - n // 2, n // 2 - a) + 1))) if n > 1 else 0
            first = n // 2 + (int(r.randint(0, n - n // 2 - d + 1)) if d else 0)
            path[e, :a], path[e, a:a + d], kept[e] = np.arange(a), first + np.arange(d), a + d
        n = np.array(ns, np.int32)
        row0 = np.cumsum([0] + ns[:-1])
        entry = np.repeat(np.arange(E), ns)
        s["plan"] = dict(T=sum(ns), E=E, max_n=max(ns), min_n=min(ns), tokens=ints(entry), pos=ints(np.arange(sum(ns)) - row0[entry] + np.array(ctx)[entry]), row_entry=ints(entry),
                         row0=ints(row0), n=ints(n), ctx=ints(ctx), slot=ints(0 * n), page_table=ints(table), max_pages=max(held))
        s["path"], s["kept"] = ints(path), ints(kept)
        s["pool"] = _pool(g, c, len(order))
    if kind in ("fork", "keep"):
        if own:  # the handle that a program makes once for its cache
            from paligemma_multimodal_system_b200 import seq_ops
            s["cache"] = seq_ops.CachePages(s["pool"], PAGE)
        return s
    ns, who, parts = _entries(c), _adapter_of(c, r), [int(x) for x in c["parts"].split(",")]
    T, F, K, dtype = sum(ns), sum(parts), c["depth"], DTYPES[c["dtype"]]
    s.update(rows=ns, who=who, widths=parts)
    s["x"] = torch.randn(T, K, generator=g, device="cuda").to(dtype)
    s["y"] = torch.randn(T, F, generator=g, device="cuda").to(DTYPES[c["out"]])
    s["a"] = (torch.randn(c["adapters"], len(parts) * c["rank"], K, generator=g, device="cuda") * K ** -0.5).to(dtype)
    s["b"] = (torch.randn(c["adapters"], F, c["rank"], generator=g, device="cuda") * c["rank"] ** -0.5).to(dtype)
    s["scale"] = 0.25 + torch.rand(c["adapters"], generator=g, device="cuda")
    if own:  # the bank that a program keeps, and the step's plan
        from paligemma_multimodal_system_b200 import seq_ops
        s["bank"] = seq_ops.AdapterBank(s["a"], s["b"], s["scale"], parts)
        s["rows_of"] = seq_ops.AdapterPlan(ns, who)
    return s


# -------------------------------------------------------------------------------------------------------------------- plain forms
def _weights(x, c):
    """Probabilities of rows in 64 bits, cut to their nuclei: the walk's whole numbers hang on them."""
    z = x.double() / c["temperature"]
    w = torch.exp(z - z.amax(-1, keepdim=True))
    if c["top_p"] < 1:
        order = torch.sort(w, -1, descending=True).values
        before = torch.cumsum(order, -1) - order
        least = torch.where(before <= c["top_p"] * w.sum(-1, keepdim=True), order, math.inf).amin(-1, keepdim=True)
        w = torch.where(w >= least, w, 0.0)
    return w / w.sum(-1, keepdim=True)


def _drawn(p, u):
    """First id of every row whose running sum is above u times the whole."""
    run = torch.cumsum(p, -1)
    return torch.searchsorted(run, u.double()[:, None] * run[:, -1:], right=True)[:, 0].clamp(max=p.shape[1] - 1)


def _verify(s):
    p, c = s["plan"], s
    E, most, dev = p["E"], p["max_n"], p["tokens"].device
    up = torch.full((E, most), -2, dtype=torch.int64)
    for e, tree in enumerate(s["parents"]):
        up[e, :len(tree)] = torch.tensor(tree)
    deepest = widest = 0
    for tree in s["parents"]:
        depth = [0] * len(tree)
        for i in range(1, len(tree)):
            depth[i] = depth[tree[i]] + 1
        deepest, widest = max(deepest, max(depth)), max([widest] + [tree.count(i) for i in range(len(tree))])
    up, row0, place = up.to(dev), p["row0"].long(), torch.arange(most, device=dev)
    ids = torch.arange(E, device=dev)
    toks = p["tokens"].long()[(row0[:, None] + place).clamp(max=p["T"] - 1)]
    node, alive = torch.zeros(E, dtype=torch.int64, device=dev), torch.ones(E, dtype=torch.bool, device=dev)
    path = torch.full((E, most), -1, dtype=torch.int64, device=dev)
    path[:, 0] = 0
    kept, last = torch.ones(E, dtype=torch.int64, device=dev), torch.zeros(E, dtype=torch.int64, device=dev)
    for _ in range(deepest + 1):  # one node of every entry at a time
        row = row0 + node
        child = up == node[:, None]
        if c["drafts"] == "model":
            t, q = _weights(s["logits"][row], c), _weights(s["draft"][row], c)
            left, lost, mass = t, torch.zeros(E, 1, dtype=torch.float64, device=dev), torch.ones(E, 1, dtype=torch.float64, device=dev)
            onward, tried = torch.full_like(node, -1), child.clone()
            for _ in range(widest):
                i = tried.int().argmax(-1)
                some = tried.any(-1) & (onward < 0)
                x = toks[ids, i]
                u = s["uniforms"][row0 + i, 0].double()
                stays = some & (u * q[ids, x] * mass[:, 0] < left[ids, x])
                onward = torch.where(stays, i, onward)
                tried[ids, i] = False
                gone = (some & ~stays)[:, None]
                lost = torch.where(gone, lost + mass, lost)
                left = torch.where(gone, (t - lost * q).clamp(min=0), left)
                mass = torch.where(gone, left.sum(-1, keepdim=True), mass)
            token = _drawn(torch.where(mass > 0, left, t), s["uniforms"][row, 1])
        else:
            token = s["logits"][row].argmax(-1) if c["drafts"] == "greedy" else _drawn(_weights(s["logits"][row], c), s["uniforms"][row, 1])
            match = child & (toks == token[:, None])
            onward = torch.where(match.any(-1), match.int().argmax(-1), -1)
        last = torch.where(alive, token, last)
        alive = alive & (onward >= 0)
        path[ids, kept.clamp(max=most - 1)] = torch.where(alive, onward, path[ids, kept.clamp(max=most - 1)])
        kept = kept + alive
        node = torch.where(alive, onward, node)
    return [path.int(), kept.int(), last.int()]


def _fork(s):
    src, dst, rows = (torch.from_numpy(x).long().cuda() for x in s["moves"].T.copy())
    valid = torch.arange(PAGE, device="cuda") < rows[:, None]
    for x in s["pool"]:
        x[dst] = torch.where(valid[..., None], x[src], x[dst])
    return s["pool"]


def _keep(s):
    p = s["plan"]
    place = torch.arange(p["max_n"], device="cuda")
    e, i = torch.nonzero(place < s["kept"][:, None], as_tuple=True)
    table, ctx = p["page_table"].long(), p["ctx"].long()[e]
    to, at = ctx + i, ctx + s["path"].long()[e, i]
    for x in s["pool"]:
        x[table[e, to // PAGE], to % PAGE] = x[table[e, at // PAGE], at % PAGE]
    return s["pool"]


def _adapt(s):
    rows = torch.tensor(s["who"]).repeat_interleave(torch.tensor(s["rows"])).cuda()
    out, r = s["y"].clone(), s["rank"]
    for a in sorted(set(s["who"]) - {-1}):
        at = torch.nonzero(rows == a)[:, 0]
        v = s["x"][at].float() @ s["a"][a].float().T
        b = s["b"][a].float().split(s["widths"])
        add = torch.cat([v[:, i * r:(i + 1) * r] @ w.T for i, w in enumerate(b)], 1)
        out[at] = (s["y"][at].float() + s["scale"][a] * add).to(out.dtype)
    return out


# ---------------------------------------------------------------------------------------------------------------------------- run
def run(state):
    s, kind = state, state["kind"]
    if not own:
        return {"verify": _verify, "fork": _fork, "keep": _keep, "adapt": _adapt}[kind](s)
    from paligemma_multimodal_system_b200 import seq_ops
    if kind == "verify":
        return list(seq_ops.verify_drafts(s["logits"], seq_ops.RequestBatch(**s["plan"]), s["uniforms"], draft_logits=s["draft"], temperature=s["temperature"], top_p=s["top_p"]))
    if kind == "fork":
        seq_ops.copy_pages(s["cache"], s["moves"])
        return s["pool"]
    if kind == "keep":
        seq_ops.keep_rows(s["cache"], seq_ops.StepBatch(**s["plan"]), s["path"], s["kept"])
        return s["pool"]
    return seq_ops.adapter_add(s["x"], s["y"], s["bank"], s["rows_of"], out=torch.empty_like(s["y"]))


def work(case):
    c, kind = case, case["kind"]
    if kind == "verify":  # every row once; the draft's rows of nodes that have children
        rows = sum(_nodes(c))
        read = rows + (rows - c["entries"] if c["drafts"] == "model" and c["width"] == 1 else rows // 2 if c["drafts"] == "model" else 0)
        return {"bytes": 4.0 * read * c["vocab"], "flops": 3.0 * read * c["vocab"]}
    if kind in ("fork", "keep"):
        size = c["width"] * (2 if c["dtype"] == "bfloat16" else 4)
        if kind == "fork":
            rows = sum(max(1, c["rows"] - (i * 7) % max(1, c["rows"])) for i in range(c["moves"]))
        else:  # rows that move, about a quarter of the drafted ones
            rows = max(1, sum(_nodes(c)) // 8)
        return {"bytes": 2.0 * rows * 2 * c["layers"] * size, "flops": 0.0}
    ns, parts = _entries(c), [int(x) for x in c["parts"].split(",")]
    T, F, K, r, size, wide = sum(ns), sum(parts), c["depth"], c["rank"], 2 if c["dtype"] == "bfloat16" else 4, 2 if c["out"] == "bfloat16" else 4
    used = min(c["adapters"], len(ns))
    return {"bytes": float(T * K * size + 2 * T * F * wide + used * r * (len(parts) * K + F) * size), "flops": 2.0 * T * r * (len(parts) * K + F)}


# -------------------------------------------------------------------------------------------------------------------- 64 bits
def _exact_row(x, c):
    """Probabilities of one row, {id order}, from the definition."""
    z = x.double() / c["temperature"]
    p = torch.softmax(z, 0)
    if c["top_p"] >= 1:
        return p
    values, inverse = torch.unique(x, return_inverse=True)  # (ascending)
    mass = torch.zeros(len(values), dtype=torch.float64, device=x.device).index_add_(0, inverse, p)
    above = torch.flip(torch.cumsum(torch.flip(mass, [0]), 0), [0]) - mass
    p = p * (above <= c["top_p"])[inverse]
    return p / p.sum()


def _exact_pick(p, u):
    run = torch.cumsum(p, 0)
    return int((run <= u * run[-1]).sum().clamp(max=len(p) - 1))


def exact(case, seed):
    c, s = case, prepare(case, seed)
    kind = c["kind"]
    if kind == "verify":
        p = s["plan"]
        tokens, row0 = p["tokens"].tolist(), p["row0"].tolist()
        us = None if s["uniforms"] is None else s["uniforms"].double().tolist()
        path, kept, last = np.full((p["E"], p["max_n"]), -1, np.int32), [], []
        for e, tree in enumerate(s["parents"]):
            walk, go = [0], True
            while go:
                v, go = walk[-1], False
                row = row0[e] + v
                children = [i for i in range(v + 1, len(tree)) if tree[i] == v]
                if c["drafts"] == "model":
                    rest = whole = _exact_row(s["logits"][row], c)
                    q = _exact_row(s["draft"][row], c) if children else None
                    for i in children:  # the rest is normalised after every rejection
                        x = tokens[row0[e] + i]
                        if us[row0[e] + i][0] * float(q[x]) < float(rest[x]):
                            walk.append(i)
                            go = True
                            break
                        less = (rest - q).clamp(min=0)
                        if float(less.sum()) <= 0:
                            rest = whole
                            break
                        rest = less / less.sum()
                    if not go:
                        pick = _exact_pick(rest, us[row][1])
                else:
                    pick = int(torch.nonzero(s["logits"][row] == s["logits"][row].max())[0]) if us is None else _exact_pick(_exact_row(s["logits"][row], c), us[row][1])
                    same = [i for i in children if tokens[row0[e] + i] == pick]
                    if same:
                        walk.append(same[0])
                        go = True
            path[e, :len(walk)] = walk
            kept.append(len(walk))
            last.append(pick)
        return [torch.from_numpy(path), torch.tensor(kept, dtype=torch.int32), torch.tensor(last, dtype=torch.int32)]
    if kind == "fork":
        old = [x.clone() for x in s["pool"]]
        for a, b, n in s["moves"].tolist():
            for x, y in zip(s["pool"], old):
                x[b, :n] = y[a, :n]
        return [x.double() for x in s["pool"]]
    if kind == "keep":
        p = s["plan"]
        table, ctx, path = p["page_table"].tolist(), p["ctx"].tolist(), s["path"].tolist()
        for x in s["pool"]:
            for e, n in enumerate(s["kept"].tolist()):
                rows = [x[table[e][(ctx[e] + j) // PAGE], (ctx[e] + j) % PAGE].clone() if j != i else None for i, j in enumerate(path[e][:n])]
                for i, row in enumerate(rows):
                    if row is not None:
                        x[table[e][(ctx[e] + i) // PAGE], (ctx[e] + i) % PAGE] = row
        return [x.double() for x in s["pool"]]
    out, t = s["y"].double(), 0
    for n, a in zip(s["rows"], s["who"]):
        if a >= 0:
            col = 0
            for i, w in enumerate(s["widths"]):
                down = s["a"][a, i * s["rank"]:(i + 1) * s["rank"]].double()
                out[t:t + n, col:col + w] += s["scale"][a].double() * torch.einsum("tk,rk,fr->tf", s["x"][t:t + n].double(), down, s["b"][a, col:col + w].double())
                col += w
        t += n
    return out
