"""Operators of the ragged-step engine's 8-bit cache, of drafted tokens and of scored answers, as cases that can be timed and checked.

A case is a dict of plain values; `kind` says which operator it takes:

  store   a step's projected rows: norm, rotation, keys and values into the 8-bit paged cache as they are written, and the read-back of the
          rows that prompt attention goes over (`seq_ops.attn_prepare` with `QuantizedPages`, `seq_ops.kv_read`)
  decode  attention of decoded tokens over the 8-bit cache (`seq_ops.attn_ragged` with `QuantizedPages`)
  tree    attention of drafted trees over a cache of any type (`seq_ops.attn_tree`)
  score   log probability, rank and entropy of given tokens beside the top alternatives (`seq_ops.token_logprobs`)

The 8-bit format: an e4m3 code per element and a power of two per row and head, 2^(byte - 127), the least one that takes the largest of the
head's finite elements to 448 or below.
"""
import math

import numpy as np
import torch

own = False

PAGE = 64
DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def listed():
    return [
        # a short follow-up of one chat: 23 new tokens behind 105 (latency)
        dict(name="store-follow-up", kind="store", dtype="bfloat16", entries=1, new=23, spread=1, behind=105, heads=32, kv_heads=8, dim=64, turn=True),
        # the prompts of one step, 897 .. 1024 tokens each
        dict(name="store-prompts", kind="store", dtype="bfloat16", entries=8, new=1024, spread=128, behind=0, heads=32, kv_heads=8, dim=64, turn=True),
        # portions of two long prompts in full precision, no norm and no rotation, 128-wide heads
        dict(name="store-portions-fp32", kind="store", dtype="float32", entries=2, new=700, spread=40, behind=1400, heads=16, kv_heads=4, dim=128, turn=False),
        # one interactive request at a context of 3000 (latency)
        dict(name="decode-one", kind="decode", dtype="bfloat16", entries=1, context=3000, heads=32, kv_heads=8, dim=64, window=0, keep=0, softcap=0.0, gate=False),
        # a full decode batch with contexts of 1125 .. 2250, soft cap and output gate
        dict(name="decode-batch", kind="decode", dtype="bfloat16", entries=64, context=2250, heads=32, kv_heads=8, dim=64, window=0, keep=0, softcap=50.0, gate=True),
        # a few long documents, 128-wide heads, contexts of 16000 .. 32000
        dict(name="decode-long", kind="decode", dtype="bfloat16", entries=6, context=32000, heads=16, kv_heads=4, dim=128, window=0, keep=0, softcap=0.0, gate=False),
        # one request verifies eight drafted tokens (latency)
        dict(name="tree-one", kind="tree", dtype="bfloat16", cache="same", entries=1, nodes=8, context=1100, heads=32, kv_heads=8, dim=64, window=0, keep=0, softcap=0.0, gate=False),
        # a decode batch verifies trees of up to 31 tokens over the 8-bit cache
        dict(name="tree-batch-8bit", kind="tree", dtype="bfloat16", cache="e4m3", entries=24, nodes=31, context=1500, heads=32, kv_heads=8, dim=64, window=0, keep=0, softcap=0.0, gate=True),
        # a few requests served in full precision
        dict(name="tree-fp32", kind="tree", dtype="float32", cache="same", entries=4, nodes=13, context=800, heads=16, kv_heads=4, dim=64, window=512, keep=4, softcap=0.0, gate=False),
        # the answer of one request, PaliGemma's vocabulary, five alternatives (latency)
        dict(name="score-one", kind="score", rows=1, vocab=257216, top=5, temperature=1.0),
        # the decode step of a full batch at a sampling temperature
        dict(name="score-batch", kind="score", rows=64, vocab=257216, top=20, temperature=0.8),
        # every token of a prompt's portion
        dict(name="score-prompt", kind="score", rows=1500, vocab=32000, top=1, temperature=1.0),
    ]


def _spread(rng, lo, hi):
    """A whole number between lo and hi, even over the logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["store", "decode", "decode", "tree", "tree", "score"])
    if kind == "score":
        vocab = rng.choice([32000, 257216, 257152, _spread(rng, 1000, 130001)])
        return dict(kind=kind, rows=_spread(rng, 1, min(1500, 16_000_000 // vocab)), vocab=vocab, top=rng.choice([0, 1, 5, 20, 32]), temperature=rng.choice([1.0, 1.0, 0.8, 0.6]))
    dtype = rng.choice(["bfloat16", "bfloat16", "bfloat16", "float32"])
    dim = rng.choice([64, 64, 128, 96, 32])
    kv_heads = rng.choice([1, 2, 4, 8])
    heads = kv_heads * rng.choice([1, 2, 4, 4, 7, 8])
    c = dict(kind=kind, dtype=dtype, heads=heads, kv_heads=kv_heads, dim=dim)
    if kind == "store":
        entries = rng.randint(1, 8)
        new = _spread(rng, 2, 8192 // entries if dtype == "bfloat16" else 2048 // entries)
        new = min(new, 2048, 4_000_000 // (entries * heads * dim) + 2)
        return dict(c, entries=entries, new=new, spread=rng.randint(1, max(1, new // 2)), behind=rng.choice([0, 0, rng.randint(1, 1500)]), turn=dtype == "bfloat16" and rng.random() < 0.7)
    c.update(window=rng.choice([0, 0, 512, 1024]), keep=rng.choice([0, 4, 16]), softcap=rng.choice([0.0, 0.0, 50.0]), gate=rng.random() < 0.5)
    cells = 32_000_000 // (kv_heads * dim)  # keys of all entries: what the plain form holds in 32 bits stays within a GB
    if kind == "decode":
        entries = _spread(rng, 1, 64)
        return dict(c, entries=entries, context=_spread(rng, 1, min(32000, cells // entries)))
    entries, nodes = _spread(rng, 1, 24), _spread(rng, 2, 64)
    context = _spread(rng, 1, min(8000, cells // entries, 100_000_000 // (entries * nodes * heads)))
    return dict(c, cache=rng.choice(["same", "e4m3"]), entries=entries, nodes=nodes, context=context)


# ------------------------------------------------------------------------------------------------------------------------ inputs
def _lengths(c):
    """[(new tokens, tokens already stored)] of every entry."""
    n = c["entries"]
    if c["kind"] == "store":
        return [(max(1, c["new"] - (i * 37) % c["spread"]), c["behind"]) for i in range(n)]
    ctx = [max(0, c["context"] - (i * 53) % max(1, c["context"] // 2)) for i in range(n)]
    return [(1 if c["kind"] == "decode" else max(1, c["nodes"] - (i * 5) % max(1, c["nodes"] // 2)), x) for i, x in enumerate(ctx)]


def _parents(n, r):
    """A drafted tree: node 0 follows the last stored token, every later node one of those before it (mostly one of the last four)."""
    return [-1 if i == 0 else int(r.randint(max(0, i - 4) if r.rand() < 0.8 else 0, i)) for i in range(n)]


def _plan(c, seed):
    """The step's descriptors as a serving program keeps them: int32 on the GPU, in the layout of `seq_ops.StepBatch`."""
    r = np.random.RandomState((seed * 7 + 3) & 0x7FFFFFFF)
    rows = _lengths(c)
    E, T, most = len(rows), sum(n for n, _ in rows), max(n for n, _ in rows)
    pages = [(n + x + PAGE - 1) // PAGE for n, x in rows]
    width, words = max(pages), (most + 31) // 32
    order = r.permutation(sum(pages))  # pages come in any order
    table, dense, dense0 = np.zeros((E, width), np.int32), np.zeros((E, width), np.int32), np.zeros(E, np.int32)
    pos, at, entry, row0 = np.zeros(T, np.int32), np.zeros(T, np.int32), np.zeros(T, np.int32), np.zeros(E, np.int32)
    tree = np.zeros((T, words), np.uint32)
    t = p = d = 0
    for e, (n, x) in enumerate(rows):
        table[e, :pages[e]] = order[p:p + pages[e]]
        p += pages[e]
        if n > 1:
            dense[e, :pages[e]] = np.arange(d, d + pages[e])
            dense0[e] = d * PAGE
            d += pages[e]
        row0[e], entry[t:t + n], at[t:t + n], pos[t:t + n] = t, e, np.arange(x, x + n), np.arange(x, x + n)
        if c["kind"] == "tree":
            for i, up in enumerate(_parents(n, r)):
                if up >= 0:
                    tree[t + i] = tree[t + up]
                tree[t + i, i // 32] |= np.uint32(1 << (i % 32))
                pos[t + i] = pos[t + up] + 1 if up >= 0 else x
        t += n
    n, x = np.array([a for a, _ in rows], np.int32), np.array([a for _, a in rows], np.int32)
    dev = {k: torch.from_numpy(v).cuda() for k, v in dict(pos=pos, at=at, row_entry=entry, row0=row0, n=n, ctx=x, page_table=table, dense_row0=dense0, dense_pages=dense,
                                                         tree=tree.view(np.int32)).items()}
    dev.update(T=T, E=E, max_n=most, min_n=int(n.min()), tokens=dev["row_entry"], slot=dev["row0"], max_pages=width, singles=int((n == 1).sum()),
               max_single_ctx=max([b for a, b in rows if a == 1], default=0), dense_max_pages=width, dense_rows=d * PAGE,
               dense_max_len=max([a + b for a, b in rows if a > 1], default=0))
    if c["kind"] != "tree":
        dev.pop("tree"), dev.pop("at")
    return dev, sum(pages)


def _normal(g, *shape):
    return torch.randn(*shape, generator=g, device="cuda")


def _quantize(x, heads):
    """Rows [n, heads * dim] -> (codes uint8 [n, heads * dim], exponent bytes uint8 [n, heads])."""
    y = x.float().view(x.shape[0], heads, -1)
    top = y.abs().amax(-1)
    m, e = torch.frexp(top / 448)  # top / 448 = m 2^e, m in [1/2, 1): the least power not below it is 2^e, or 2^(e - 1) for m = 1/2
    e = torch.where(m == 0.5, e - 1, e)
    e = torch.where(torch.ldexp(torch.full_like(top, 448), e) < top, e + 1, e)  # (the quotient was rounded)
    e = torch.where(top == 0, -127, e).clamp(-127, 127)
    codes = torch.ldexp(y.double(), -e[..., None]).float().to(torch.float8_e4m3fn)
    return codes.view(torch.uint8).reshape(x.shape), (e + 127).to(torch.uint8)


def _values(codes, exps):
    """Codes [..., heads * dim] and exponent bytes [..., heads] -> fp32."""
    y = codes.view(torch.float8_e4m3fn).float().reshape(*exps.shape, -1)
    return (y * torch.ldexp(torch.ones_like(y[..., 0]), exps.int() - 127)[..., None]).reshape(codes.shape)


def _cache(rows, heads, g, shape):
    """A cached operand as the framework keeps it: pages of the rows' type, or 8-bit pages [pages, page, heads * dim] + exponents [pages, heads, page]."""
    pages, width = shape
    x = torch.empty(pages, PAGE, width, device="cuda", dtype=rows if rows != "e4m3" else torch.bfloat16)
    for a in range(0, pages, 256):  # (values of different tokens differ in size)
        part = _normal(g, min(256, pages - a), PAGE, width)
        x[a:a + 256] = part * torch.exp2(torch.randint(-2, 3, part.shape[:2] + (1,), generator=g, device="cuda").float())
    if rows != "e4m3":
        return x
    codes, exps = _quantize(x.view(-1, width), heads)
    return codes.view(pages, PAGE, width), exps.view(pages, PAGE, heads).transpose(1, 2).contiguous()


def prepare(case, seed):
    c, kind = case, case["kind"]
    torch.cuda.set_device(0)
    g = torch.Generator(device="cuda").manual_seed((seed * 1000003 + 17) & 0x7FFFFFFF)
    if kind == "score":
        R, V = c["rows"], c["vocab"]
        x = torch.randn(R, V, generator=g, device="cuda").mul_(2.5)  # a model's logits: most of the mass on some dozens of tokens
        liked = torch.randint(0, V, (R, 24), generator=g, device="cuda")
        x.scatter_add_(1, liked, torch.rand(R, 24, generator=g, device="cuda") * 14)
        given = torch.where(torch.rand(R, generator=g, device="cuda") < 0.7, liked[:, 0], torch.randint(0, V, (R,), generator=g, device="cuda"))
        return dict(c, logits=x, tokens=given.int())
    dtype, H, G, dim = DTYPES[c["dtype"]], c["heads"], c["kv_heads"], c["dim"]
    plan, pages = _plan(c, seed)
    s = dict(c, plan=plan, type=dtype, scale=dim ** -0.5)
    if kind == "store":
        s["proj"] = _normal(g, plan["T"], (H + 2 * G) * dim).to(dtype)
        s["freq"] = 1e6 ** (-2.0 * torch.arange(dim // 2, dtype=torch.float64, device="cuda") / dim)
        s["q_norm"], s["k_norm"] = 1 + 0.1 * _normal(g, dim), 1 + 0.1 * _normal(g, dim)
    else:
        s["q"] = _normal(g, plan["T"], H * dim).to(dtype)
        s["gates"] = _normal(g, plan["T"], H * dim).to(dtype) if c["gate"] else None
    form = "e4m3" if kind != "tree" or c["cache"] == "e4m3" else dtype
    s["k"], s["v"] = (_cache(form, G, g, (pages, G * dim)) for _ in "kv")
    return s


# -------------------------------------------------------------------------------------------------------------------- plain forms
def _turn(x, pos, freq):
    """Interleaved pairs (2 i, 2 i + 1) turned by pos * freq[i]; the angles in 64 bits."""
    a = pos.double()[:, None] * freq
    c, s = a.cos().float()[:, None], a.sin().float()[:, None]
    u, v = x[..., ::2], x[..., 1::2]
    return torch.stack((u * c - v * s, v * c + u * s), -1).flatten(-2)


def _store(s):
    p, H, G, dim, T = s["plan"], s["heads"], s["kv_heads"], s["dim"], s["plan"]["T"]
    x = s["proj"].float()
    q, k, v = x[:, :H * dim].view(T, H, dim), x[:, H * dim:(H + G) * dim].view(T, G, dim), x[:, (H + G) * dim:]
    if s["turn"]:
        q, k = (_turn(y / (y.square().mean(-1, keepdim=True) + 1e-6).sqrt() * w, p["pos"], s["freq"]) for y, w in ((q, s["q_norm"]), (k, s["k_norm"])))
    at = p["page_table"][p["row_entry"].long(), p["pos"].long() // PAGE].long()
    out = [q.reshape(T, H * dim).to(s["type"])]
    row = torch.arange(p["dense_rows"], device="cuda")  # the read-back: whole pages of every entry of several tokens, zeros behind its last row
    e = torch.searchsorted(p["dense_row0"], row, right=True, out_int32=True).long() - 1
    j = row - p["dense_row0"][e]
    held = j < (p["ctx"] + p["n"])[e]
    for rows, (codes, exps) in ((k.reshape(T, G * dim), s["k"]), (v, s["v"])):
        a, b = _quantize(rows, G)
        codes[at, p["pos"].long() % PAGE], exps[at, :, p["pos"].long() % PAGE] = a, b
        page = p["page_table"][e, j // PAGE].long()
        out.append((_values(codes[page, j % PAGE], exps[page, :, j % PAGE]) * held[:, None]).to(s["type"]))
    return out


def _plain_cache(x, table):
    """[entries, keys, width] in fp32 of an entry's pages one after another."""
    if isinstance(x, tuple):
        return _values(x[0][table].flatten(1, 2), x[1][table].transpose(2, 3).flatten(1, 2))
    return x[table].flatten(1, 2).float()


def _visible(s, keys, tree=None):
    """[entries, rows, keys] truth values (rows of an entry padded to the longest one's)."""
    p = s["plan"]
    i, j = torch.arange(p["max_n"], device="cuda")[:, None], torch.arange(keys, device="cuda")
    n, ctx = p["n"].long()[:, None, None], p["ctx"].long()[:, None, None]
    t = (p["row0"].long()[:, None, None] + i).clamp(max=p["T"] - 1)
    node = (j - ctx).clamp(min=0)  # the drafted token that key j is
    if "tree" in p:
        seen = p["tree"][t, (node // 32).clamp(max=p["tree"].shape[1] - 1)] >> (node % 32) & 1 == 1
    else:
        seen = node <= i
    vis = ((j < ctx) | ((node < n) & (j >= ctx) & seen)) & (i < n)
    if s["window"]:
        where = torch.where(j < ctx, j, p["pos"].long()[(p["row0"].long()[:, None, None] + node).clamp(max=p["T"] - 1)])
        vis &= (p["pos"].long()[t] - where < s["window"]) | (where < s["keep"])
    return vis


def _attend(s):
    p, H, G, dim = s["plan"], s["heads"], s["kv_heads"], s["dim"]
    k, v = (_plain_cache(s[x], p["page_table"].long()).unflatten(-1, (G, dim)) for x in "kv")
    row = (p["row0"].long()[:, None] + torch.arange(p["max_n"], device="cuda")).clamp(max=p["T"] - 1)
    q = s["q"].float()[row].view(p["E"], p["max_n"], G, H // G, dim)
    score = torch.einsum("engrd,ejgd->egnrj", q, k) * s["scale"]
    if s["softcap"]:
        score = s["softcap"] * torch.tanh(score / s["softcap"])
    vis = _visible(s, k.shape[1])[:, None, :, None]
    score = torch.where(vis, score, -math.inf)
    top = score.amax(-1, keepdim=True).clamp(min=torch.finfo(torch.float32).min)
    w = torch.exp(score - top)
    y = torch.einsum("egnrj,ejgd->engrd", w / w.sum(-1, keepdim=True), torch.where(vis.any(2).any(2)[..., None].transpose(1, 2), v, 0.0))
    y = y.flatten(2)[p["row_entry"].long(), torch.arange(p["T"], device="cuda") - p["row0"].long()[p["row_entry"].long()]]
    if s["gates"] is not None:
        y = y / (1 + torch.exp(-s["gates"].float()))
    return y.to(s["type"])


def _score(s):
    x, given = s["logits"], s["tokens"].long()[:, None]
    z = x / s["temperature"]
    z = z - z.amax(-1, keepdim=True)
    w = torch.exp(z)
    total = w.sum(-1, keepdim=True)
    logs = z - total.log()
    mine = x.gather(1, given)
    place = torch.arange(x.shape[1], device="cuda")
    rank = ((x > mine) | ((x == mine) & (place < given))).sum(-1)
    bits = x.view(torch.int32)
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits).long() << 32 | (0x7FFFFFFF - place)  # the larger value, then the lower index
    ids = torch.topk(order, s["top"], dim=-1, sorted=True).indices
    return [logs.gather(1, given)[:, 0], -(w / total * logs).sum(-1), rank.int(), ids.int(), logs.gather(1, ids)]


# ---------------------------------------------------------------------------------------------------------------------------- run
def run(state):
    s, kind = state, state["kind"]
    if not own:
        return _store(s) if kind == "store" else _score(s) if kind == "score" else _attend(s)
    from paligemma_multimodal_system_b200 import seq_ops
    if kind == "score":
        return list(seq_ops.token_logprobs(s["logits"], s["tokens"], top=s["top"], temperature=s["temperature"]))
    b, H, G, dim = seq_ops.StepBatch(**s["plan"]), s["heads"], s["kv_heads"], s["dim"]
    k, v = (seq_ops.QuantizedPages(*s[x]) if isinstance(s[x], tuple) else s[x] for x in "kv")
    if kind == "store":
        q = torch.empty(b.T, H * dim, device="cuda", dtype=s["type"])
        turn = s["turn"]
        seq_ops.attn_prepare(s["proj"], b, s["freq"], s["q_norm"] if turn else None, s["k_norm"] if turn else None, q, k, v, H, G, dim, dim, dim if turn else 0, 1e-6, PAGE,
                             norm_qk=turn, norm_v=False)
        return [q, *seq_ops.kv_read(k, v, b, s["type"])]
    out = torch.empty(b.T, H * dim, device="cuda", dtype=s["type"])
    score = seq_ops.ScoreOptions(H, s["window"], s["keep"]) if s["window"] else None
    attend = seq_ops.attn_tree if kind == "tree" else seq_ops.attn_ragged
    attend(s["q"], k, v, s["gates"], out, b, H, G, dim, dim, s["scale"], s["softcap"], PAGE, score=score)
    return out


def _seen(c):
    """(keys that are read, (row, key) pairs) of all entries."""
    keys = pairs = 0
    for n, x in _lengths(c):
        most = x + n if not c.get("window") else min(x + n, c["window"] + c["keep"] + n - 1)
        keys += most
        pairs += n * min(most, x + (n + 1) // 2)
    return keys, pairs


def work(case):
    c = case
    if c["kind"] == "score":
        return {"bytes": c["rows"] * (4.0 * c["vocab"] + 16 + 8 * c["top"]), "flops": 4.0 * c["rows"] * c["vocab"]}
    rows, size, H, G, dim = sum(n for n, _ in _lengths(c)), 2 if c["dtype"] == "bfloat16" else 4, c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "store":  # rows in; queries and 8-bit rows out; earlier rows in; every row out in the activations' type
        back = sum(n + x for n, x in _lengths(c) if n > 1)
        stored = 2 * G * (dim + 1)
        return {"bytes": float(rows * ((2 * H + 2 * G) * dim * size + stored) + (back - rows) * stored + back * 2 * G * dim * size), "flops": 6.0 * rows * (H + 2 * G) * dim}
    keys, pairs = _seen(c)
    row = 2 * G * (dim + 1) if c["kind"] == "decode" or c["cache"] == "e4m3" else 2 * G * dim * size
    return {"bytes": float(keys * row + rows * H * dim * size * (3 if c["gate"] else 2)), "flops": 4.0 * pairs * H * dim}


# -------------------------------------------------------------------------------------------------------------- in 64 bits, apart
def _exact_codes(x):
    """The value that a head's element has in the cache: [..., dim] in 64 bits, rounded to four bits in front of 2^(e - 9)."""
    top = x.abs().amax(-1, keepdim=True)
    e = torch.ceil(torch.log2(top / 448).clamp(min=-127, max=127))
    e = torch.where(448 * 2.0 ** (e - 1) >= top, e - 1, torch.where(448 * 2.0 ** e < top, e + 1, e)).clamp(-127, 127)  # (the logarithm is rounded)
    y = x / 2.0 ** e
    step = 2.0 ** (torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step * 2.0 ** e


def _exact_pages(x, e, pages):
    """One entry's pages in 64 bits: [keys, width]."""
    if not isinstance(x, tuple):
        return x[pages].flatten(0, 1).double()
    code, exp = x[0][pages].flatten(0, 1).int(), x[1][pages].transpose(1, 2).flatten(0, 1)
    low, mant = (code >> 3) & 15, code & 7
    y = torch.where(low == 0, mant / 8.0 * 2.0 ** -6, (1 + mant / 8.0) * 2.0 ** (low - 7).double()) * (1 - 2.0 * (code >> 7))
    return (y.double().unflatten(-1, (exp.shape[1], -1)) * 2.0 ** (exp.double() - 127)[..., None]).flatten(1)


def exact(case, seed):
    c, s = case, prepare(case, seed)
    if c["kind"] == "score":
        outs = [[], [], [], [], []]
        for row, t in zip(s["logits"].split(64), s["tokens"].split(64)):
            z = row.double() / c["temperature"]
            logs = z - torch.logsumexp(z, -1, keepdim=True)
            r = torch.arange(len(row), device="cuda")
            ids = torch.sort(row, descending=True, stable=True).indices
            lp, top = logs[r, t.long()], ids[:, :c["top"]]
            for o, v in zip(outs, (lp, -(logs.exp() * logs).sum(-1), (ids == t[:, None]).int().argmax(-1).int(), top.int(), torch.gather(logs, 1, top))):
                o.append(v)
        return [torch.cat(o) for o in outs]
    p, H, G, dim = s["plan"], c["heads"], c["kv_heads"], c["dim"]
    lens, table = _lengths(c), p["page_table"].long()
    row0 = p["row0"].tolist()
    if c["kind"] == "store":
        x = s["proj"].double().unflatten(1, (-1, dim))
        q, k, v = x[:, :H], x[:, H:H + G], x[:, H + G:]
        if c["turn"]:
            angle = p["pos"].double()[:, None, None] * s["freq"]
            wheel = torch.polar(torch.ones_like(angle), angle)

            def turned(y, w):
                y = y * w.double() / torch.sqrt((y * y).sum(-1, keepdim=True) / dim + 1e-6)
                return torch.view_as_real(torch.view_as_complex(y.unflatten(-1, (-1, 2)).contiguous()) * wheel).flatten(-2)

            q, k = turned(q, s["q_norm"]), turned(k, s["k_norm"])
        back = [torch.zeros(p["dense_rows"], G * dim, dtype=torch.float64, device="cuda") for _ in "kv"]
        for e, (n, behind) in enumerate(lens):
            if n > 1:
                at = int(p["dense_row0"][e])
                for o, old, new in zip(back, (s["k"], s["v"]), (k, v)):
                    o[at:at + behind] = _exact_pages(old, e, table[e])[:behind]
                    o[at + behind:at + behind + n] = _exact_codes(new[row0[e]:row0[e] + n]).flatten(1)
        return [q.flatten(1), *back]
    out = torch.zeros(p["T"], H * dim, dtype=torch.float64, device="cuda")
    for e, (n, ctx) in enumerate(lens):
        L, a = ctx + n, row0[e]
        k, v = (_exact_pages(s[x], e, table[e])[:L].unflatten(-1, (G, dim)) for x in "kv")
        vis = torch.ones(n, L, dtype=torch.bool, device="cuda")
        if c["kind"] == "tree":
            words = p["tree"][a:a + n].long() & 0xFFFFFFFF
            vis[:, ctx:] = ((words[:, :, None] >> torch.arange(32, device="cuda")) & 1).flatten(1)[:, :n].bool()
        if c["window"]:
            mine = p["pos"][a:a + n].long()
            keys = torch.cat([torch.arange(ctx, device="cuda"), mine])
            vis &= (mine[:, None] - keys < c["window"]) | (keys < c["keep"])
        for g in range(G):
            hs = range(g * (H // G), (g + 1) * (H // G))
            z = torch.stack([s["q"][a:a + n, h * dim:(h + 1) * dim].double() @ k[:, g].T for h in hs]) * s["scale"]
            if c["softcap"]:
                z = c["softcap"] * torch.tanh(z / c["softcap"])
            y = torch.softmax(z.masked_fill(~vis, -math.inf), -1) @ v[:, g]
            for i, h in enumerate(hs):
                out[a:a + n, h * dim:(h + 1) * dim] = y[i]
    return out * torch.sigmoid(s["gates"].double()) if c["gate"] else out
