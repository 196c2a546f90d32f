"""The cache on the device: page pools for keys and values, and fixed-size state per slot.

Each schedule entry of the model states what its parts need (a ``KVSpec``, a
``StateSpec``, a list of them with at most one ``KVSpec`` and states of different names, or nothing). Entries with equal ``KVSpec`` share one group: one tensor
``[entries, pages, kv_heads, 64, head_dim]`` for keys and one for values, in the compute
type, and one page pool. Entries with equal ``StateSpec`` share one tensor
``[entries, slots, *shape]``. An entry that reads another entry's cache has no storage.
The dense Llama decoder has one group (all keys, every layer) and no state.

The reference's device cache is ``cache_k/cache_v`` as ``[kv_head][position][head_dim]``
per layer (src/cuda_resident.rs:5424-5428, :1568-1583), sized from the configuration and
refused before allocation when it does not fit (src/inference/kv_cache.rs:285-299).
"""
from __future__ import annotations

from typing import Optional

import torch

from ..errors import CacheError
from .book import PAGE, CacheBook, KVSpec, StateSpec, flatten_specs

_STATE_DTYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "int32": torch.int32}


class SequenceCache:
    def __init__(self, entry_specs: list, entry_sources: list, *, max_tokens: int, max_position: int,
                 dtype: torch.dtype, device, max_slots: Optional[int] = None, track_weights: bool = False, weights_scratch: int = 0):
        n_pages = max(1, (int(max_tokens) + PAGE - 1) // PAGE)
        n_slots = int(max_slots) if max_slots else n_pages
        self.dtype = dtype
        self.device = torch.device(device)
        self.entry_specs = list(entry_specs)
        self.entry_sources = list(entry_sources)
        kv_specs: list = []
        state_specs: list = []
        self.entry_kv: list = [None] * len(entry_specs)        # (group, index in group)
        self.entry_state: list = [None] * len(entry_specs)
        counts_kv: list = []
        counts_state: list = []
        for i, (spec, src) in enumerate(zip(entry_specs, entry_sources)):
            if src is not None:
                continue
            for one in flatten_specs(spec):
                if isinstance(one, KVSpec):
                    if self.entry_kv[i] is not None:
                        raise CacheError(f"schedule entry {i} asks for two sets of keys and values")
                    if one not in kv_specs:
                        kv_specs.append(one)
                        counts_kv.append(0)
                    g = kv_specs.index(one)
                    self.entry_kv[i] = (g, counts_kv[g])
                    counts_kv[g] += 1
                elif isinstance(one, StateSpec):
                    if self.entry_state[i] is None:
                        self.entry_state[i] = {}
                    if one.name in self.entry_state[i]:
                        raise CacheError(f"schedule entry {i} keeps two states named {one.name!r}")
                    if one not in state_specs:
                        state_specs.append(one)
                        counts_state.append(0)
                    g = state_specs.index(one)
                    self.entry_state[i][one.name] = (g, counts_state[g])
                    counts_state[g] += 1
                else:
                    raise CacheError(f"schedule entry {i}: unknown cache need {one!r}")
        for i, src in enumerate(entry_sources):
            if src is not None:
                if self.entry_kv[src] is None:
                    raise CacheError(f"schedule entry {i} reads the keys of entry {src}, which keeps none")
                self.entry_kv[i] = self.entry_kv[src]
        if track_weights and (state_specs or not kv_specs or any(s.forgets for s in kv_specs)):
            raise CacheError("attention weights are kept only by caches that keep all keys and no per-sequence state of fixed size")
        self.book = CacheBook(kv_specs, n_pages, n_slots, max_position)
        need = self.bytes_needed(kv_specs, counts_kv, state_specs, counts_state, n_pages, n_slots, dtype)
        if track_weights:
            need += sum(self.score_bytes(s, c, n_pages) for s, c in zip(kv_specs, counts_kv)) + 4 * int(weights_scratch)
        if self.device.type == "cuda":
            free, _total = torch.cuda.mem_get_info(self.device)
            if need > free:
                raise CacheError(f"the cache needs {need} bytes ({n_pages} pages of {PAGE} tokens) but only {free} are free on {self.device}")
        # zero-filled once; kernels never count rows beyond a sequence's length
        self.k = [torch.zeros((counts_kv[g], n_pages, s.n_kv_heads, PAGE, s.head_dim), dtype=dtype, device=self.device)
                  for g, s in enumerate(kv_specs)]
        # (a group whose values are channels of its key rows keeps no value pages: its keys are handed out for both)
        self.v = [self.k[g] if s.values_in_keys else
                  torch.zeros((counts_kv[g], n_pages, s.n_kv_heads, PAGE, s.value_dim), dtype=dtype, device=self.device)
                  for g, s in enumerate(kv_specs)]
        self.state = [torch.zeros((counts_state[g], n_slots) + tuple(s.shape), dtype=_STATE_DTYPES[s.dtype],
                                  device=self.device) for g, s in enumerate(state_specs)]
        # with ``track_weights``: what every position was weighed by the queries since, float32 [entries, pages, kv_heads, 64] a
        # group (attention sets a position's score when it writes its key, so pages need no clearing); else None
        self.scores = None
        if track_weights:
            self.scores = [torch.zeros(t.shape[:-1], dtype=torch.float32, device=self.device) for t in self.k]
        # ``weights_scratch`` float32 numbers for the attention that keeps weights: one piece for all layers, steps and captured
        # graphs of this cache, which never run at the same time
        self.weights_scratch = torch.empty(int(weights_scratch), dtype=torch.float32, device=self.device) if track_weights else None
        self.bytes = need

    @staticmethod
    def score_bytes(spec: KVSpec, entries: int, n_pages: int) -> int:
        return 4 * entries * n_pages * spec.n_kv_heads * PAGE

    @staticmethod
    def bytes_needed(kv_specs, counts_kv, state_specs, counts_state, n_pages, n_slots, dtype) -> int:
        size = torch.empty((), dtype=dtype).element_size()
        total = 0
        for s, c in zip(kv_specs, counts_kv):
            total += c * n_pages * s.n_kv_heads * PAGE * (s.head_dim + s.stored_value_dim) * size
        for s, c in zip(state_specs, counts_state):
            n = 1
            for d in s.shape:
                n *= d
            total += c * n_slots * n * torch.empty((), dtype=_STATE_DTYPES[s.dtype]).element_size()
        return total

    # ---- slots ----
    def alloc_slot(self) -> int:
        slot = self.book.alloc_slot()
        for t in self.state:
            t[:, slot].zero_()
        return slot

    def free_slot(self, slot: int) -> None:
        self.book.free_slot(slot)

    def length(self, slot: int) -> int:
        self.book._check_slot(slot)
        return self.book.length[slot]

    def truncate(self, slot: int, length: int) -> None:
        """Forget the positions of ``slot`` at and beyond ``length`` (the reference's
        ``rollback_to_position``, src/inference/kv_cache.rs:246-269). State of fixed size has no
        positions to go back to: a cache that keeps any refuses."""
        if self.state and length < self.length(slot):
            raise CacheError(f"slot {slot}: this model keeps per-sequence state of fixed size, which cannot be rolled back")
        self.book.truncate(slot, length)

    # ---- storage of one schedule entry ----
    def kv_pages(self, entry: int):
        """(group, keys [pages, kv_heads, 64, head_dim], values) of a schedule entry."""
        where = self.entry_kv[entry]
        if where is None:
            raise CacheError(f"schedule entry {entry} keeps no keys and values")
        g, i = where
        return g, self.k[g][i], self.v[g][i]

    def scores_of(self, entry: int):
        """The kept attention weights [pages, kv_heads, 64] of a schedule entry (None if the cache keeps none)."""
        where = self.entry_kv[entry]
        return None if self.scores is None or where is None else self.scores[where[0]][where[1]]

    def state_of(self, entry: int, name: str | None = None) -> torch.Tensor:
        """[slots, *shape] state of a schedule entry; ``name`` picks one where the entry keeps several."""
        where = self.entry_state[entry]
        if where is None:
            raise CacheError(f"schedule entry {entry} keeps no per-sequence state")
        if name is None:
            if len(where) != 1:
                raise CacheError(f"schedule entry {entry} keeps the states {sorted(where)}: name one")
            name = next(iter(where))
        if name not in where:
            raise CacheError(f"schedule entry {entry} keeps no state named {name!r} (it keeps {sorted(where)})")
        g, i = where[name]
        return self.state[g][i]
