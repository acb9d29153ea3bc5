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

The model supplies `cache_layout()`, `step(batch, store, want_rows)`, `prec` and `vocab_size` (modeling_mapedra.py).
"""
import contextlib
from typing import Dict, List, Optional, Sequence, Tuple

import torch

from . import _lib, seq_ops
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


class SequenceEngine:
    def __init__(self, model, max_tokens: int, num_slots: int = 4, use_cuda_graph: bool = True, kv_format: Optional[str] = None):
        """kv_format "e4m3": keys and values are cached in 8 bits (cache.py)."""
        _lib.require_device()
        self.model = model
        self.store = SequenceStore(model.cache_layout(), max_tokens, num_slots, model.prec.dtype, kv_format=kv_format)
        self._drafted: Dict[object, List[int]] = {}  # request -> parents of the drafted tokens whose rows stand behind its own
        self._step_no = torch.zeros(1, device="cuda", dtype=torch.int32)
        # decode steps (every entry one token) replay a CUDA graph per (entries, page-table width, context bound); the second
        # step of a geometry captures it, the first ran eagerly (lazy kernel attributes are set by then)
        self.use_cuda_graph = use_cuda_graph
        self._decode_graphs = {}

    @torch.no_grad()
    def step(self, entries: Sequence[Tuple[object, Sequence[int], Sequence[int]]], end: Sequence[object] = (), trace=None):
        """Runs the new tokens of every entry; returns fp32 logits [sum(len(want)), vocab] in entry / want order (None when
        nothing is wanted).  A request id seen for the first time is admitted; ids in `end` are released after the step."""
        store = self.store
        batch, want, row = [], [], 0
        seen = set()
        for rid, toks, w in entries:
            if rid in seen:
                raise ValueError(f"request {rid!r} appears twice in one step")
            seen.add(rid)
            toks = self._checked(rid, toks)
            if rid not in store.live:
                store.admit(rid)
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
            logits = self._decode_step(batch, want)
            for (rid, toks, _w) in entries:
                store.commit(rid, len(toks))
        elif batch:
            b = make_step_batch(batch)
            rows = torch.tensor(want, dtype=torch.int64).to("cuda", non_blocking=True) if want else None
            with _weights_follow():
                logits = self.model.step(b, store, rows, trace=trace)
            for (rid, toks, _w) in entries:
                store.commit(rid, len(toks))
        for rid in end:
            if rid in store.live:
                self.release(rid)
        return logits

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
        b = make_step_batch(rows)
        with _weights_follow():
            logits = self.model.step(b, store, torch.arange(b.T, device="cuda"))
        for rid, _, parents in batch:
            self._drafted[rid] = parents
        return logits

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
        moved = [(i, p) for i, p in enumerate(path) if i != p]
        if moved:
            page = store.page
            at = torch.tensor([[rec.length + x for x in m] for m in moved], dtype=torch.int64)
            pages = torch.tensor(rec.pages, dtype=torch.int64)
            idx = torch.cat([pages[at // page], at % page], 1).to("cuda", non_blocking=True)
            (dst, src), (dslot, sslot) = (idx[:, 0], idx[:, 1]), (idx[:, 2], idx[:, 3])
            for kind in (store.k_pages, store.v_pages):
                for p in kind:
                    if isinstance(p, seq_ops.QuantizedPages):
                        p.codes[dst, dslot] = p.codes[src, sslot]
                        p.powers[dst, :, dslot] = p.powers[src, :, sslot]
                    elif p is not None:
                        p[dst, dslot] = p[src, sslot]
        store.commit(rid, len(path))
        del self._drafted[rid]

    def _decode_step(self, batch, want):
        """A step of single-token entries through a captured graph (eagerly the first time a geometry is seen)."""
        E = len(batch)
        pages = max(len(e["pages"]) for e in batch)
        pages_cap = 4
        while pages_cap < pages:
            pages_cap *= 2
        ctx_cap = pages_cap * self.store.page  # every context of this page-table width; fixes the key split of the attention
        key = (E, pages_cap)
        slot = self._decode_graphs.get(key)
        if slot is None:
            slot = self._decode_graphs[key] = dict(static=StaticDecodeBatch(E, pages_cap, ctx_cap), graph=None, logits=None, seen=0)
        st = slot["static"]
        st.fill(batch)
        slot["seen"] += 1
        if slot["graph"] is None and slot["seen"] >= 2:
            side = torch.cuda.Stream()
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                g = torch.cuda.CUDAGraph()
                with torch.cuda.graph(g, stream=side), _weights_follow():
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
                 top_p: float = 0.9, eos_token_id: Optional[int] = None, seed: int = 0, step_tokens: int = 512, logprobs: Optional[int] = None):
        """Greedy (or temperature / top-p) continuation of every prompt; more prompts than slots queue up and take over slots
        and pages as earlier ones finish.  Returns the new tokens per prompt (EOS included when it was emitted): List[List[int]].
        logprobs = k (0 .. 32): (tokens, records), records per prompt and token a dict with its logprob, rank and entropy and the k most likely (id, logprob)
        pairs in `top`, under softmax(logits / temperature) where tokens are sampled and softmax(logits) else."""
        if logprobs is not None and not 0 <= logprobs <= min(32, self.model.vocab_size):
            raise ValueError(f"logprobs is 0 .. 32 and at most the vocabulary: got {logprobs}")
        records = {}
        sched = StepScheduler(self.store.num_slots, self.store.pool.num_pages, self.store.page, step_tokens, eos_token_id)
        for i, pr in enumerate(prompts):
            sched.submit(TokenRequest(("gen", i), [int(t) for t in pr], int(max_new_tokens)))
        while not sched.idle():
            plan = sched.plan()
            if not plan:
                raise RuntimeError("scheduler made no progress")
            entries = [(req.rid, toks, [len(toks) - 1] if sample else []) for req, toks, sample in plan]
            logits = self.step(entries)
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
        tokens = [sched.finished[("gen", i)] for i in range(len(prompts))]
        return tokens if logprobs is None else (tokens, [records.get(("gen", i), []) for i in range(len(prompts))])

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
