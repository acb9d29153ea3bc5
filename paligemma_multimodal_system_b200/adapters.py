"""Low-rank adapters of a text decoder: every request of an engine may have one of its own, beside the weights that all of them share.

    adapters = AdapterSet(model, slots=16, rank=32)
    adapters.load("french", tensors, scale=0.5)             # y += 0.5 * B (A x) beside every projection that `tensors` names
    engine = SequenceEngine(model, max_tokens, num_slots, adapters=adapters)
    engine.step([("a", prompt, [])], adapters={"a": "french"})

`tensors` holds A [r, K] and B [columns, r] as "<weight>.A" and "<weight>.B" beside the names that the checkpoint gives the weights: "l3.mix.q.A" stands beside "l3.mix.q".
Which weights can be adapted is the sub-layers' to say (`adapter_sites`): the attention layers' query, key, value, gate and output projections (latent attention:
the output), the linear attention's, the down projections of dense feed-forwards and the polynomial-of-norms one's up projection.  Adapters of a lower rank than the set's are padded with zeros.
"""
from typing import Dict, List, Optional, Sequence

import torch

from . import seq_ops


class StepAdapters:
    """What the sub-layers see of a step's adapters: they add to a projection by its name (`add`)."""

    def __init__(self, banks: Dict[str, seq_ops.AdapterBank], plan: seq_ops.AdapterPlan):
        self.banks, self.plan = banks, plan

    def add(self, site: str, x: torch.Tensor, y: torch.Tensor, gain: float = 1.0):
        bank = self.banks.get(site)
        if bank is not None:
            seq_ops.adapter_add(x[:, :bank.K], y[:, :bank.F], bank, self.plan, gain=gain)  # (products pad their columns)


class AdapterSet:
    """Up to `slots` named adapters of a rank up to `rank` for one model."""

    def __init__(self, model, slots: int, rank: int):
        if slots < 1 or not 1 <= rank <= seq_ops.ADAPTER_MOST_RANK:
            raise ValueError(f"at least one adapter, of a rank of 1 .. {seq_ops.ADAPTER_MOST_RANK}: got {slots} and {rank}")
        self.slots, self.rank, self.dtype = int(slots), int(rank), model.prec.dtype
        self.sites: Dict[str, tuple] = {}    # projection -> (depth, [(weight, columns)])
        for blk in model.blocks:
            for sub in (blk.mixer, blk.ff):
                if hasattr(sub, "adapter_sites"):
                    self.sites.update(sub.adapter_sites())
        self.places = {w: (site, i) for site, (_, parts) in self.sites.items() for i, (w, _) in enumerate(parts)}
        self.banks: Dict[str, seq_ops.AdapterBank] = {}  # of the projections that some adapter stands beside
        self.names: Dict[str, int] = {}
        self.version = 0                     # counts changes of `banks`: a captured step holds the banks that it was captured with

    def load(self, name: str, tensors: Dict[str, torch.Tensor], scale: float = 1.0):
        """Takes a free place for `name`.  Every tensor must have a place in the model, with its partner."""
        if name in self.names:
            raise KeyError(f"adapter {name!r} is loaded already")
        free = sorted(set(range(self.slots)) - set(self.names.values()))
        if not free:
            raise MemoryError(f"all {self.slots} places for adapters are taken")
        weights = sorted({k[:-2] for k in tensors})
        found = []
        for w in weights:
            if w not in self.places or f"{w}.A" not in tensors or f"{w}.B" not in tensors:
                raise KeyError(f"adapter {name!r}: {w} is no weight that can be adapted, or one of {w}.A and {w}.B is missing")
            site, part = self.places[w]
            depth, parts = self.sites[site]
            a, b = tensors[f"{w}.A"], tensors[f"{w}.B"]
            if a.dim() != 2 or tuple(b.shape) != (parts[part][1], a.shape[0]) or a.shape[1] != depth or not 1 <= a.shape[0] <= self.rank:
                raise ValueError(f"adapter {name!r}: {w}.A {tuple(a.shape)} and {w}.B {tuple(b.shape)} for {parts[part][1]} columns of a depth of {depth} and ranks up to {self.rank}")
            found.append((site, part, a, b))
        if len(tensors) != 2 * len(weights) or not found:
            raise KeyError(f"adapter {name!r}: tensors are pairs <weight>.A and <weight>.B")
        slot = free[0]
        for site, _, _, _ in found:
            if site not in self.banks:
                depth, parts = self.sites[site]
                self.banks[site] = seq_ops.AdapterBank.empty(self.slots, self.rank, depth, [n for _, n in parts], self.dtype)
                self.version += 1
        for bank in self.banks.values():  # (what the place held before)
            bank.clear(slot)
        for site, part, a, b in found:
            self.banks[site].put(slot, part, a, b)
            self.banks[site].scale[slot] = float(scale)
        self.names[name] = slot
        return slot

    def remove(self, name: str):
        """The caller's engines have no live request with it (SequenceEngine.remove_adapter looks)."""
        del self.names[name]

    def slots_of(self, names: Sequence[Optional[str]]) -> List[int]:
        return [-1 if n is None else self.names[n] for n in names]
