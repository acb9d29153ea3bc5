"""Ragged-step engine for the token-sequence decoders: one step runs, as ONE batch, the next tokens of every request
that has some -- whole prompts, portions of prompts and single decoded tokens side by side.

  SequenceEngine.step(entries, end)   the step function: entries = [(request id, new token ids, wanted positions)];
                                      admits unknown ids, finds pages, runs the model's step over the shared page pool and
                                      state slots, returns the wanted logits; `end` releases requests afterwards
  SequenceEngine.generate(prompts)    continuous batching on top of it: serving.StepScheduler plans the steps, the
                                      framework's samplers (pg_argmax / pg_sample_top_p) pick the tokens

  SequenceEngine.score(prompts)       log probabilities of the prompts' own tokens (pg_token_logprobs)
  SequenceEngine.step_drafts(entries) drafted trees: logits of every drafted token in one step, nothing committed;
  SequenceEngine.accept(rid, path)    keeps the drafted tokens of one path and drops the others
  SequenceEngine.step_verify(entries) both at once: drafted tokens are judged against the model's own distributions and the accepted ones kept
  SequenceEngine.fork(rid, new)       new requests that go on where a live one stands (or stood), over shared pages
  adapters.AdapterSet                 low-rank adapters: every request may have one of its own

The model supplies `cache_layout()`, `step(batch, store, want_rows)`, `prec` and `vocab_size` (modeling_mapedra.py).
"""
import contextlib
import itertools
from typing import Callable, Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib, seq_ops
from .adapters import AdapterSet, StepAdapters
from .cache import SequenceStore
from .seq_ops import StaticDecodeBatch, make_step_batch
from .serving import StepScheduler, TokenRequest


@contextlib.contextmanager
def _weights_follow():
    """The products of a model's step take weights as their second operand: the kernels in front of them may let them come early."""
    L = _lib.lib()
    _lib.check(L.pg_weights_follow(1), "pg_weights_follow")
    try:
        yield
    finally:
        _lib.check(L.pg_weights_follow(0), "pg_weights_follow")


def _records(scores):
    """token_logprobs' tensors as a list of dicts."""
    lp, entropy, rank, ids, top = (t.tolist() for t in scores)
    return [dict(logprob=a, rank=r, entropy=h, top=list(zip(i, t))) for a, h, r, i, t in zip(lp, entropy, rank, ids, top)]


class LookupDrafter:
    """Drafts from a request's own text: what followed the last earlier place that reads as its newest `match` tokens (or fewer, down to one) does."""

    def __init__(self, most: int = 4, match: int = 3):
        if most < 1 or match < 1:
            raise ValueError("at least one drafted token, found by at least one")
        self.most, self.match = int(most), int(match)

    def __call__(self, history: List[int]):
        back = history[::-1]  # (newest first)
        for n in range(min(self.match, len(back) - 1), 0, -1):
            at = 0
            for _ in range(back.count(back[0]) - 1):
                at = back.index(back[0], at + 1)
                if back[at:at + n] == back[:n]:
                    tokens = back[max(0, at - self.most):at][::-1]
                    return tokens, list(range(-1, len(tokens) - 1))
        return [], []


class SequenceEngine:
    def __init__(self, model, max_tokens: int, num_slots: int = 4, use_cuda_graph: bool = True, kv_format: Optional[str] = None, adapters: Optional[AdapterSet] = None):
        """kv_format "e4m3": keys and values are cached in 8 bits (cache.py).  adapters: the model's low-rank adapters, which requests name when they are admitted."""
        _lib.require_device()
        self.model = model
        self.adapters = adapters
        self.store = SequenceStore(model.cache_layout(), max_tokens, num_slots, model.prec.dtype, kv_format=kv_format)
        self._drafted: Dict[object, List[int]] = {}  # request -> parents of the drafted tokens whose rows stand behind its own
        self._step_no = torch.zeros(1, device="cuda", dtype=torch.int32)
        # decode steps (every entry one token) replay a CUDA graph per (entries, page-table width, context bound); the second
        # step of a geometry captures it, the first ran eagerly (lazy kernel attributes are set by then)
        self.use_cuda_graph = use_cuda_graph
        self._decode_graphs = {}

    @torch.no_grad()
    def step(self, entries: Sequence[Tuple[object, Sequence[int], Sequence[int]]], end: Sequence[object] = (), trace=None, adapters: Optional[Dict[object, str]] = None):
        """Runs the new tokens of every entry; returns fp32 logits [sum(len(want)), vocab] in entry / want order (None when
        nothing is wanted).  A request id seen for the first time is admitted, with the adapter that `adapters` names for it, and keeps that one; ids in `end` are released
        after the step."""
        store = self.store
        batch, want, row = [], [], 0
        for rid, name in (adapters or {}).items():
            self._check_adapter(name, f"request {rid!r}")
            if rid in store.live and store.live[rid].adapter != name:
                raise ValueError(f"request {rid!r} is live: it keeps the adapter that it was admitted with")
        seen = set()
        for rid, toks, w in entries:
            if rid in seen:
                raise ValueError(f"request {rid!r} appears twice in one step")
            seen.add(rid)
            toks = self._checked(rid, toks)
            if rid not in store.live:
                store.admit(rid).adapter = (adapters or {}).get(rid)
            rec = store.reserve(rid, len(toks))
            batch.append(dict(tokens=toks, ctx=rec.length, slot=rec.slot, pages=rec.pages))
            for k in w:
                if not 0 <= int(k) < len(toks):
                    raise IndexError(f"request {rid!r}: wanted position {k} outside its {len(toks)} tokens")
                want.append(row + int(k))
            row += len(toks)
        for rid, _, _ in entries:
            self._drafted.pop(rid, None)  # (rows of drafts that were not accepted are written over)
        logits = None
        if batch and trace is None and self.use_cuda_graph and all(len(e["tokens"]) == 1 for e in batch):
            logits = self._decode_step(batch, want, self._slots_of([rid for rid, _, _ in entries]))
            for (rid, toks, _w) in entries:
                store.commit(rid, len(toks))
        elif batch:
            b = self._adapted(make_step_batch(batch), [rid for rid, _, _ in entries], [len(e["tokens"]) for e in batch])
            rows = torch.tensor(want, dtype=torch.int64).to("cuda", non_blocking=True) if want else None
            with _weights_follow():
                logits = self.model.step(b, store, rows, trace=trace)
            for (rid, toks, _w) in entries:
                store.commit(rid, len(toks))
        for rid in end:
            if rid in store.live:
                self.release(rid)
        return logits

    def _check_adapter(self, name, whose):
        if name is not None and (self.adapters is None or name not in self.adapters.names):
            raise KeyError(f"{whose}: no adapter {name!r} is loaded")

    def _checked(self, rid, toks):
        toks = [int(t) for t in toks]
        if not toks:
            raise ValueError(f"request {rid!r}: empty entry")
        if min(toks) < 0 or max(toks) >= self.model.vocab_size:
            raise IndexError(f"request {rid!r}: token id out of range")
        return toks

    # -- drafted trees -----------------------------------------------------------------------------------------------
    @torch.no_grad()
    def step_drafts(self, entries: Sequence[Tuple[object, Sequence[int], Sequence[int]]]):
        """entries: [(live request id, drafted tokens, parents)], parents[i] < i the drafted token that token i follows, -1 the request's last one.  Returns fp32
        logits of every drafted token, in entry / token order: row i belongs to the sequence that ends with token i's path.  The requests' lengths stay; the
        drafted rows stand behind them until `accept`, or until the request's next step writes over them.  Models whose layers keep nothing but keys
        and values."""
        store = self.store
        b, logits, batch = self._draft_step(entries)
        for rid, _, parents in batch:
            self._drafted[rid] = parents
        return logits

    def _slots_of(self, rids):
        """Adapters of requests by their places, None where no request has one."""
        names = [self.store.live[rid].adapter for rid in rids]
        return self.adapters.slots_of(names) if any(n is not None for n in names) else None

    def _adapted(self, b, rids, ns):
        slots = self._slots_of(rids)
        return b if slots is None else seq_ops.with_adapters(b, StepAdapters(self.adapters.banks, seq_ops.AdapterPlan(ns, slots)))

    def _draft_step(self, entries):
        """Runs drafted trees; the requests' lengths stay.  (step, logits of every row, [(request, tokens, parents)])."""
        store = self.store
        if any(spec is not None and spec[0] != "kv" for spec in store.layout):
            raise ValueError("drafted trees need a model whose layers keep nothing but keys and values: a state has no branches")
        if not entries:
            raise ValueError("a step of drafts needs at least one entry")
        if len({rid for rid, _, _ in entries}) != len(entries):
            raise ValueError("a request appears twice in one step")
        batch = []
        for rid, toks, parents in entries:
            if rid not in store.live:
                raise KeyError(f"request {rid!r} is not live")
            toks, parents = self._checked(rid, toks), [int(p) for p in parents]
            if len(parents) != len(toks) or any(not -1 <= p < i for i, p in enumerate(parents)):
                raise ValueError(f"request {rid!r}: parents are one for every token, an earlier drafted token or -1")
            batch.append((rid, toks, parents))
        rows = []
        for rid, toks, parents in batch:
            rec = store.reserve(rid, len(toks))
            rows.append(dict(tokens=toks, ctx=rec.length, slot=rec.slot, pages=rec.pages, parents=parents))
            self._drafted.pop(rid, None)  # (written over; nothing to accept should the step fail)
        b = self._adapted(make_step_batch(rows), [rid for rid, _, _ in batch], [len(toks) for _, toks, _ in batch])
        with _weights_follow():
            logits = self.model.step(b, store, torch.arange(b.T, device="cuda"))
        return b, logits, batch

    @torch.no_grad()
    def accept(self, rid, path: Sequence[int]):
        """Keeps the drafted tokens path[0], path[1], .. (indexes into the request's last step_drafts, each the parent of the next, the first a root): their cache rows
        move together behind the stored ones and count from here on.  An empty path drops all drafts."""
        parents = self._drafted.get(rid)
        if parents is None:
            raise KeyError(f"request {rid!r} has no drafted tokens")
        path = [int(p) for p in path]
        if any(not 0 <= p < len(parents) for p in path) or any(parents[p] != up for p, up in zip(path, [-1] + path)):
            raise ValueError("a path runs from a root of the drafted tree, every token the parent of the next")
        store, rec = self.store, self.store.live[rid]
        if any(i != p for i, p in enumerate(path)):
            n = len(parents)
            b = make_step_batch([dict(tokens=[0] * n, ctx=rec.length, slot=rec.slot, pages=rec.pages)])  # (says where the rows lie)
            where = torch.tensor([path + [len(path)]], dtype=torch.int32).to("cuda", non_blocking=True)
            seq_ops.keep_rows(store.operands()[0], b, where, where[:, -1])
        store.commit(rid, len(path))
        del self._drafted[rid]

    @torch.no_grad()
    def step_verify(self, entries: Sequence[Tuple[object, Sequence[int], Sequence[int]]], do_sample: bool = False, temperature: float = 0.8, top_p: float = 0.9,
                    uniforms: Optional[torch.Tensor] = None, draft_logits: Optional[torch.Tensor] = None, draft_temperature: Optional[float] = None,
                    draft_top_p: Optional[float] = None):
        """Runs drafted trees and keeps what the model itself would have said (seq_ops.verify_drafts): entries as step_drafts', the first token of each the request's pending
        one (chosen, not yet run), from which the others descend.  Returns per entry (path, next token): the rows that were kept, 0 in front, which the request has stored
        now, and the token behind them (-1: the logits there are no distribution).  Greedy, or with do_sample at `temperature` and `top_p`; uniforms: fp32 [rows, 2] (None: drawn here); draft_logits
        fp32 [rows, vocab]: what the children of every row were drawn from (None: guessed)."""
        out, _, _ = self._verified(entries, do_sample, temperature, top_p, uniforms, draft_logits, draft_temperature, draft_top_p)
        return out

    def _verified(self, entries, do_sample, temperature, top_p, uniforms=None, draft_logits=None, draft_temperature=None, draft_top_p=None):
        if not do_sample and (uniforms is not None or draft_logits is not None):
            raise ValueError("a greedy walk takes no random numbers and no drafted distributions")
        for rid, toks, parents in entries:
            if len(parents) == 0 or parents[0] != -1 or any(p < 0 for p in parents[1:]):
                raise ValueError(f"request {rid!r}: the first token is the pending one, the others descend from it")
        b, logits, batch = self._draft_step(entries)
        if do_sample and uniforms is None:
            uniforms = torch.rand(b.T, 2, device="cuda")
        how = dict(temperature=temperature, top_p=top_p) if do_sample else {}
        path, kept, last = seq_ops.verify_drafts(logits, b, uniforms, draft_logits, draft_temperature=draft_temperature, draft_top_p=draft_top_p, **how)
        seq_ops.keep_rows(self.store.operands()[0], b, path, kept)
        said = torch.cat([path, kept[:, None], last[:, None]], 1).tolist()
        out = []
        for (rid, _, _), (*row, n, token) in zip(batch, said):
            self.store.commit(rid, n)
            out.append((row[:n], token))
        return out, b, logits

    @torch.no_grad()
    def fork(self, rid, new: Sequence[object], length: Optional[int] = None):
        """New requests, admitted under the names `new`, that go on where the first `length` stored tokens (None: all) of `rid` end, with its adapter.  Full pages are
        shared; what each owns is a copy of the last, partly filled page and of the states.  Models with states fork behind the last token only."""
        self.store.fork(rid, new, length)

    def remove_adapter(self, name: str):
        users = [rid for rid, rec in self.store.live.items() if rec.adapter == name]
        if users:
            raise ValueError(f"adapter {name!r} is in use by {users[:4]}")
        self.adapters.remove(name)

    def _decode_step(self, batch, want, adapters=None):
        """A step of single-token entries through a captured graph (eagerly the first time a geometry is seen).  adapters: their places, or None."""
        E = len(batch)
        pages = max(len(e["pages"]) for e in batch)
        pages_cap = 4
        while pages_cap < pages:
            pages_cap *= 2
        ctx_cap = pages_cap * self.store.page  # every context of this page-table width; fixes the key split of the attention
        version = None if adapters is None else self.adapters.version
        key = (E, pages_cap) if adapters is None else (E, pages_cap, version)
        slot = self._decode_graphs.get(key)
        if slot is None:
            if adapters is not None:  # (steps that hold banks of before are not replayed again)
                self._decode_graphs = {k: v for k, v in self._decode_graphs.items() if len(k) == 2 or k[2] == version}
            slot = self._decode_graphs[key] = dict(static=StaticDecodeBatch(E, pages_cap, ctx_cap), graph=None, logits=None, seen=0)
            if adapters is not None:
                slot["plan"], slot["who"] = seq_ops.AdapterPlan([1] * E, adapters, tiles=E), list(adapters)
                slot["static"].batch = seq_ops.with_adapters(slot["static"].batch, StepAdapters(dict(self.adapters.banks), slot["plan"]))
        st = slot["static"]
        st.fill(batch)
        if adapters is not None and slot["who"] != adapters:
            slot["plan"].fill([1] * E, adapters)
            slot["who"] = list(adapters)
        slot["seen"] += 1
        if slot["graph"] is None and slot["seen"] >= 2:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                g = torch.cuda.CUDAGraph()
                with _lib.captured(g, side), _weights_follow():
                    slot["logits"] = self.model.step(st.batch, self.store, st.rows)
            torch.cuda.current_stream().wait_stream(side)
            slot["graph"] = g
        if slot["graph"] is not None:
            slot["graph"].replay()
            full = slot["logits"]
        else:
            with _weights_follow():
                full = self.model.step(st.batch, self.store, st.rows)
        if not want:
            return None
        return full.index_select(0, torch.tensor(want, dtype=torch.int64).to("cuda", non_blocking=True))

    def release(self, rid):
        self._drafted.pop(rid, None)
        self.store.release(rid)

    # -- generation ------------------------------------------------------------------------------------------------
    def _sample(self, logits, do_sample, temperature, top_p, seed):
        n, V = logits.shape
        out = torch.empty(n, device="cuda", dtype=torch.int32)
        L = _lib.lib()
        if do_sample:
            _lib.check(L.pg_sample_top_p(logits.data_ptr(), logits.stride(0), out.data_ptr(), 0, n, V, 1.0 / float(temperature), float(top_p),
                                         int(seed), self._step_no.data_ptr(), _lib.stream()), "pg_sample_top_p")
            self._step_no += 1
        else:
            _lib.check(L.pg_argmax(logits.data_ptr(), logits.stride(0), out.data_ptr(), n, V, _lib.stream()), "pg_argmax")
        return out

    @torch.no_grad()
    def generate(self, prompts: Sequence[Sequence[int]], max_new_tokens: int, do_sample: bool = False, temperature: float = 0.8,
                 top_p: float = 0.9, eos_token_id: Optional[int] = None, seed: int = 0, step_tokens: int = 512, logprobs: Optional[int] = None,
                 draft: Optional[Callable[[List[int]], Tuple[List[int], List[int]]]] = None, adapters: Optional[Sequence[Optional[str]]] = None):
        """Greedy (or temperature / top-p) continuation of every prompt; more prompts than slots queue up and take over slots
        and pages as earlier ones finish.  Returns the new tokens per prompt (EOS included when it was emitted): List[List[int]].
        logprobs = k (0 .. 32): (tokens, records), records per prompt and token a dict with its logprob, rank and entropy and the k most likely (id, logprob)
        pairs in `top`, under softmax(logits / temperature) where tokens are sampled and softmax(logits) else.
        draft: guesses how a request goes on -- its tokens so far -> (drafted tokens, parents), parents[i] the drafted token that token i follows or -1 the newest one
        (LookupDrafter) -- and steps of decoded tokens run the guesses along, `step_tokens` rows a step at most, and keep those that the model says as well: the tokens of a greedy
        run are the same where its logits are (a drafted step's kernels add in another order: near ties may fall otherwise, in bf16 above all), those of a sampled one have the same
        distribution.  adapters: one name or None for every prompt."""
        if draft is not None and any(spec is not None and spec[0] != "kv" for spec in self.store.layout):
            raise ValueError("drafted trees need a model whose layers keep nothing but keys and values: a state has no branches")
        if adapters is not None and len(adapters) != len(prompts):
            raise ValueError("one adapter (or None) for every prompt")
        for i, name in enumerate(adapters or ()):
            self._check_adapter(name, f"prompt {i}")
        rng = torch.Generator(device="cuda").manual_seed(int(seed)) if draft is not None and do_sample else None
        if logprobs is not None and not 0 <= logprobs <= min(32, self.model.vocab_size):
            raise ValueError(f"logprobs is 0 .. 32 and at most the vocabulary: got {logprobs}")
        if len(prompts) == 0:
            return [] if logprobs is None else ([], [])
        for left, what in ((self.store.free_slots, "sequence slots"), (self.store.pool.free, "cache pages")):
            if not left:
                raise MemoryError(f"live requests hold all {what}: release some before others are generated")
        # (names that no live request has: not the caller's, nor those of a generation whose `draft` asks for another)
        free = (("gen", i) for i in itertools.count())
        names = list(itertools.islice((rid for rid in free if rid not in self.store.live), len(prompts)))
        named = dict(zip(names, adapters or ()))
        records = {}
        # (what live requests hold stays theirs)
        sched = StepScheduler(len(self.store.free_slots), len(self.store.pool.free), self.store.page, step_tokens, eos_token_id)
        for rid, pr in zip(names, prompts):
            sched.submit(TokenRequest(rid, [int(t) for t in pr], int(max_new_tokens)))
        with self._released_on_errors(names):
            while not sched.idle():
                plan = sched.plan()
                if not plan:
                    raise RuntimeError("scheduler made no progress")
                if draft is not None and all(req.fed == len(req.prompt) for req, _, _ in plan):
                    guessed = self._guesses(plan, draft, sched.step_tokens)
                    if any(len(toks) > 1 for _, toks, _ in guessed):
                        self._drafted_turn(plan, guessed, sched, do_sample, temperature, top_p, rng, logprobs, records)
                        continue
                entries = [(req.rid, toks, [len(toks) - 1] if sample else []) for req, toks, sample in plan]
                logits = self.step(entries, adapters={rid: named.get(rid) for rid, _, _ in entries} if named else None)
                picked, said = [], None
                if logits is not None:
                    out = self._sample(logits, do_sample, temperature, top_p, seed)
                    if logprobs is not None:
                        said = _records(seq_ops.token_logprobs(logits, out, top=logprobs, temperature=temperature if do_sample else 1.0))
                    picked = out.tolist()
                it, told = iter(picked), iter(said or ())
                for req, toks, sample in plan:
                    if sample and said is not None:
                        records.setdefault(req.rid, []).append(next(told))
                    if sched.advance(req, len(toks), next(it) if sample else None):
                        self.release(req.rid)
        tokens = [sched.finished[rid] for rid in names]
        return tokens if logprobs is None else (tokens, [records.get(rid, []) for rid in names])

    @contextlib.contextmanager
    def _released_on_errors(self, rids):
        """What raises in between (a `draft` that the caller gave, rows that are no distribution) leaves none of these requests behind."""
        try:
            yield
        except BaseException:
            for rid in rids:
                if rid in self.store.live:
                    self.release(rid)
            raise

    def _guesses(self, plan, draft, step_tokens):
        """Entries of a drafted step: every decoding request's newest token and what is guessed behind it, `step_tokens` rows at most (each has its logits)."""
        entries, left = [], step_tokens - len(plan)
        for i, (req, toks, _) in enumerate(plan):
            tokens, parents = draft(req.prompt + req.tokens)
            # rows that the request's pages have room for beside the newest token's, and its share of the step's
            room = min(req.max_new_tokens - len(req.tokens) - 1, left // (len(plan) - i))
            tokens, parents = list(tokens)[:room], list(parents)[:room]
            left -= len(tokens)
            entries.append((req.rid, toks + tokens, [-1] + [int(p) + 1 for p in parents]))
        return entries

    def _drafted_turn(self, plan, entries, sched, do_sample, temperature, top_p, rng, logprobs, records):
        """One step of `generate` in which every request decodes, with its guesses."""
        T = sum(len(toks) for _, toks, _ in entries)
        uniforms = torch.rand(T, 2, device="cuda", generator=rng) if do_sample else None
        out, b, logits = self._verified(entries, do_sample, temperature, top_p, uniforms)
        if any(token < 0 for _, token in out):
            raise RuntimeError("a row of logits is no distribution")
        said, rows, row0 = [], [], 0
        for (_, toks, _), (path, token) in zip(entries, out):
            said.append([toks[i] for i in path[1:]] + [token])
            rows += [row0 + i for i in path]
            row0 += len(toks)
        if logprobs is not None:
            idx = torch.tensor(rows + [t for ts in said for t in ts], dtype=torch.int64).to("cuda", non_blocking=True)
            told = iter(_records(seq_ops.token_logprobs(logits.index_select(0, idx[:len(rows)]), idx[len(rows):].int(), top=logprobs, temperature=temperature if do_sample else 1.0)))
        for (req, _, _), tokens in zip(plan, said):
            told_here = [next(told) for _ in tokens] if logprobs is not None else []
            for i, t in enumerate(tokens):
                if logprobs is not None:
                    records.setdefault(req.rid, []).append(told_here[i])
                if sched.advance(req, 1, t):
                    self.release(req.rid)
                    break

    @torch.no_grad()
    def score(self, prompts: Sequence[Sequence[int]], top: int = 0, step_tokens: int = 512):
        """Records (as `generate`'s) of every prompt's tokens but its first, each under the tokens in front of it: prompts of one token have none.  Prompts run one
        after another in portions of up to `step_tokens` tokens, whose logits are held at once."""
        if step_tokens < 1:
            raise ValueError("a portion has at least one token")
        if not 0 <= top <= min(32, self.model.vocab_size):
            raise ValueError(f"top is 0 .. 32 and at most the vocabulary: got {top}")
        prompts = [self._checked(("score", i), pr) for i, pr in enumerate(prompts)]
        scored = []
        for pr in prompts:
            rid, got = object(), []  # (a name that no live request has)
            try:
                for lo in range(0, len(pr) - 1, step_tokens):
                    part = pr[lo:min(lo + step_tokens, len(pr) - 1)]  # (nothing follows the last token)
                    logits = self.step([(rid, part, range(len(part)))])
                    given = torch.tensor(pr[lo + 1:lo + 1 + len(part)], dtype=torch.int32).to("cuda", non_blocking=True)
                    got += _records(seq_ops.token_logprobs(logits, given, top=top))
            finally:
                if rid in self.store.live:
                    self.release(rid)
            scored.append(got)
        return scored
