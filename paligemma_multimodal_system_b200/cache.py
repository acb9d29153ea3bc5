"""Sequence storage for the ragged-step engine: a shared pool of 64-token KV pages and a pool of recurrent-state slots.

The `KVCache` of modeling_gemma.py gives every batch row a fixed run of pages; here pages belong to whoever asks first.
A model describes what each of its layers keeps per sequence (`cache_layout()`):

    ("kv", key_width, value_width)      one key row and one value row per token  -> pages [num_pages, 64, width]
    ("latent", width)                   ONE row per token from which keys and values of every head are derived (latent
                                        attention: compressed kv vector + shared rotated key part) -> k_pages only
    ("state", shape)                    one fp32 tensor per sequence             -> [num_slots, *shape]
    None                                nothing

A "kv" layer that says how many heads its rows hold (`KvSpec`) can keep them in 8 bits (`kv_format="e4m3"`: seq_ops.QuantizedPages, an e4m3 code per element
and a power of two per row and head, a little over half of bfloat16's bytes); latent rows and states keep their types.

`SequenceStore` owns the device tensors and the host-side bookkeeping (free lists, per-request page lists and lengths).
Requests that fork (`fork`) share their full pages, which have as many owners, and have copies of the last, partly filled one and of the states.
Pages and slots go back to the free lists when a request is released and are handed out again, lowest id first, so a
second request really does land on memory a finished one used.  Nothing is cleared on reuse: a sequence's first step
starts from length zero (attention reads no stale key; recurrent layers start from a zero state when their context is empty).
"""
from typing import Dict, List, Optional, Sequence

import torch

from .modeling_gemma import PAGE
from .seq_ops import CachePages, QuantizedPages, copy_pages

KV_FORMATS = (None, "e4m3")


class KvSpec(tuple):
    """("kv", key_width, value_width) that also knows the number of key / value heads in a row."""

    def __new__(cls, key_width: int, value_width: int, heads: int):
        self = super().__new__(cls, ("kv", int(key_width), int(value_width)))
        self.heads = int(heads)
        return self

    def __getnewargs__(self):  # (copies and pickles make it anew)
        return self[1], self[2], self.heads


class PagePool:
    """Host-side free list of page ids (no tensors; CPU-testable)."""

    def __init__(self, num_pages: int):
        if num_pages <= 0:
            raise ValueError("a page pool needs at least one page")
        self.num_pages = int(num_pages)
        self.free: List[int] = list(range(self.num_pages))
        self.shared: Dict[int, int] = {}  # page -> owners, of pages with more than one

    def take(self, n: int) -> List[int]:
        if n > len(self.free):
            raise MemoryError(f"KV page pool exhausted: {n} pages wanted, {len(self.free)} of {self.num_pages} free")
        self.free.sort()
        got, self.free = self.free[:n], self.free[n:]
        return got

    def share(self, pages: Sequence[int]):
        """One more owner for each page: it is free again when all have given it back."""
        for p in pages:
            self.shared[p] = self.shared.get(p, 1) + 1

    def give(self, pages: Sequence[int]):
        dup = set(pages) & set(self.free)
        if dup:
            raise RuntimeError(f"pages freed twice: {sorted(dup)[:4]}")
        for p in pages:
            owners = self.shared.get(p, 1)
            if owners == 1:
                self.free.append(p)
            elif owners == 2:
                del self.shared[p]
            else:
                self.shared[p] = owners - 1


class SequenceRecord:
    __slots__ = ("rid", "slot", "pages", "length", "adapter")

    def __init__(self, rid, slot):
        self.rid, self.slot, self.pages, self.length, self.adapter = rid, slot, [], 0, None  # (adapter: its name, None for the shared weights alone)


class SequenceStore:
    """Pages + state slots of the live requests of one engine."""

    def __init__(self, layout, max_tokens: int, num_slots: int, dtype: torch.dtype, device="cuda", allocate: bool = True,
                 kv_format: Optional[str] = None):
        if kv_format not in KV_FORMATS:
            raise ValueError(f"unknown cache format {kv_format!r} (known: {KV_FORMATS})")
        self.page = PAGE
        self.kv_format = kv_format
        self.num_slots = int(num_slots)
        num_pages = (int(max_tokens) + PAGE - 1) // PAGE
        self.pool = PagePool(num_pages)
        self.free_slots: List[int] = list(range(self.num_slots))
        self.live: Dict[object, SequenceRecord] = {}
        self.layout = list(layout)
        self.k_pages: List[Optional[torch.Tensor]] = []
        self.v_pages: List[Optional[torch.Tensor]] = []
        self.state: List[Optional[torch.Tensor]] = []
        for spec in self.layout:
            k = v = s = None
            if kv_format is not None and spec is not None and spec[0] == "kv":
                heads = getattr(spec, "heads", None)
                if heads is None:
                    raise ValueError("a layer that does not say how many heads its rows hold cannot be kept in 8 bits")
                sizes = (spec[1] // heads, spec[2] // heads)
                if any(n % 16 or n > 128 for n in sizes):
                    raise ValueError(f"the 8-bit cache serves heads of a multiple of 16 elements up to 128: got {sizes[0]} and {sizes[1]}")
                if allocate:
                    k, v = (QuantizedPages.empty(num_pages, PAGE, heads, n, device) for n in sizes)
            elif allocate and spec is not None and spec[0] == "kv":
                k = torch.zeros(num_pages, PAGE, spec[1], device=device, dtype=dtype)
                v = torch.zeros(num_pages, PAGE, spec[2], device=device, dtype=dtype)
            elif allocate and spec is not None and spec[0] == "latent":
                k = torch.zeros(num_pages, PAGE, spec[1], device=device, dtype=dtype)
            elif allocate and spec is not None and spec[0] == "state":
                s = torch.zeros(self.num_slots, *spec[1], device=device, dtype=torch.float32)
            elif spec is not None and spec[0] not in ("kv", "latent", "state"):
                raise ValueError(f"unknown cache kind {spec[0]!r}")
            self.k_pages.append(k)
            self.v_pages.append(v)
            self.state.append(s)
        self._operands = None

    def operands(self):
        """(CachePages of the layers' pages, CachePages of the states as pages of one row): what moves with a request; None where there is none."""
        if self._operands is None:
            pages = [p for p in self.k_pages + self.v_pages if p is not None]
            states = [s.view(self.num_slots, 1, -1) for s in self.state if s is not None]
            self._operands = (CachePages(pages, self.page) if pages else None, CachePages(states, 1) if states else None)
        return self._operands

    # -- bookkeeping ---------------------------------------------------------------------------------------------------
    def admit(self, rid) -> SequenceRecord:
        if rid in self.live:
            raise KeyError(f"request {rid!r} is already live")
        if not self.free_slots:
            raise MemoryError(f"all {self.num_slots} sequence slots are taken")
        self.free_slots.sort()
        rec = SequenceRecord(rid, self.free_slots.pop(0))
        self.live[rid] = rec
        return rec

    def reserve(self, rid, new_tokens: int) -> SequenceRecord:
        """Makes sure the request owns pages for `new_tokens` more tokens (its length is advanced by `commit`)."""
        rec = self.live[rid]
        need = (rec.length + new_tokens + PAGE - 1) // PAGE - len(rec.pages)
        if need > 0:
            rec.pages.extend(self.pool.take(need))
        return rec

    def commit(self, rid, new_tokens: int):
        self.live[rid].length += int(new_tokens)

    def fork(self, rid, new: Sequence, length: Optional[int] = None) -> List[SequenceRecord]:
        """New requests that go on where the first `length` (None: all) stored tokens of `rid` end.  They share its full pages, which nobody writes again, and have copies of the
        rest of the last one and of its states: one launch for all of them."""
        if rid not in self.live:
            raise KeyError(f"request {rid!r} is not live")
        rec, new = self.live[rid], list(new)
        length = rec.length if length is None else int(length)
        if not 0 < length <= rec.length:
            raise ValueError(f"request {rid!r} has {rec.length} stored tokens: no fork behind {length}")
        if length != rec.length and any(spec is not None and spec[0] == "state" for spec in self.layout):
            raise ValueError("a model that keeps states forks behind its last token: there is no state of an earlier one")
        if len(set(new)) != len(new) or any(n in self.live for n in new):
            raise KeyError("a fork needs names that no live request has, each once")
        full, rest = divmod(length, self.page)
        if len(new) > len(self.free_slots):
            raise MemoryError(f"{len(new)} forks wanted, {len(self.free_slots)} of {self.num_slots} sequence slots free")
        mine = self.pool.take(len(new)) if rest else []
        made = [self.admit(n) for n in new]
        for i, r in enumerate(made):
            r.pages, r.length, r.adapter = rec.pages[:full] + mine[i:i + 1], length, rec.adapter
            self.pool.share(rec.pages[:full])
        pages, states = self.operands()
        try:
            if pages is not None and mine:
                copy_pages(pages, [(rec.pages[full], p, rest) for p in mine])
            if states is not None and made:
                copy_pages(states, [(rec.slot, r.slot, 1) for r in made])
        except BaseException:
            for n in new:
                self.release(n)
            raise
        return made

    def release(self, rid):
        rec = self.live.pop(rid)
        self.pool.give(rec.pages)
        self.free_slots.append(rec.slot)

    def max_pages(self, rids) -> int:
        return max(1, max(len(self.live[r].pages) for r in rids))
