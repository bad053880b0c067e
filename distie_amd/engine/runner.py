"""The step function: a batch of (request, its next tokens) in, logits at the wanted
places out.

It runs only the tokens it is given, as one flattened batch, from the cache that earlier
steps left: portions of prompts beside single decoded tokens, cut anywhere. It samples
nothing (the reference's step also samples: worker/src/inference/model_runner.py:51-62).
Pages for the new tokens are reserved here unless the caller (the scheduler) has done so,
and the cache's counts advance when the step is done.
"""

from __future__ import annotations

from dataclasses import dataclass
from typing import Dict, Hashable, List, Mapping, Optional, Sequence

import numpy as np
import torch

from ..cache.manager import CacheManager, RequestCache
from ..parts import PAGE
from .batch import BatchBuilder, StepEntry
from .model import Model


@dataclass
class _Draft:
    """What a step of drafted tokens left of one request: its place in the cache then, and the parents of its tokens."""

    state: RequestCache
    resets: int
    cached: int
    parents: List[int]

    def lies_in(self, state: Optional[RequestCache]) -> bool:
        """Whether the drafted entries are still there: in the request's own pages (not in those of one that came behind it under the same
        name), none of which were given back since, behind the same cached ones."""
        return state is self.state and state.resets == self.resets and state.num_cached == self.cached


class ModelRunner:
    def __init__(self, model: Model, cache: CacheManager, ops, act_dtype: torch.dtype,
                 max_model_len: Optional[int] = None) -> None:
        self.model = model
        self.cache = cache
        self.ops = ops
        self.act_dtype = act_dtype
        self.max_model_len = int(max_model_len or model.spec.max_positions)
        self.builder = BatchBuilder(cache, self.max_model_len, ops.device, model.spec.vocab_size, ops)
        self._drafts: Dict[Hashable, _Draft] = {}          # between `step` and `keep`
        self.graphs = None          # set by the engine when captured decode steps are on
        model.prepare(ops)
        cache.clear_rows_with(ops)

    def step(self, entries: Sequence[StepEntry], reserve: bool = True,
             feed: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
        """-> float32 [wanted, vocab] in the order of the entries and of their `want`
        (None if nothing is wanted). A request not yet known to the cache is added.

        `feed` (int32 [F], on the device, F <= len(entries)): each of the first F entries brings one
        token, and the token of entry i is feed[i], which need not have reached the host (those
        entries' own tokens are placeholders)."""
        if feed is not None and (feed.shape[0] > len(entries) or
                                 any(len(e.tokens) != 1 for e in entries[:feed.shape[0]])):
            raise ValueError("a fed step takes one token for each of its first entries")
        if not entries:
            raise ValueError("empty step")
        drafted = any(entry.parents is not None for entry in entries)
        if drafted and not self.model.takes_trees:
            raise ValueError("this model does not take trees of drafted tokens: every mixer has to be attention over pages with plain scores")
        for entry in entries:
            if entry.request_id not in self.cache:
                self.cache.add(entry.request_id)
        if reserve:
            # if a reservation fails nothing was written yet; pages taken for this step stay with
            # their requests and are returned when those end
            for entry in entries:
                self.cache.reserve(entry.request_id, len(entry.tokens))
        logits, ran = None, False
        if self.graphs is not None and not drafted:
            logits = self.graphs.try_run(entries, feed)   # a view of the bucket's buffer: use it before the next step
            ran = logits is not None
            if ran and logits.shape[0] == 0:
                logits = None
        if not ran:
            ids, meta, want_rows = self.builder.build(entries)       # (what it refuses has written nothing: drafts stay)
        for entry in entries:
            self._drafts.pop(entry.request_id, None)
        if not ran:
            if feed is not None and feed.shape[0]:
                ids[:feed.shape[0]].copy_(feed)           # one-token entries lead the step: entry i is token i
            logits = self.model.forward(self.ops, ids, meta, self.cache, self.act_dtype, want_rows)
        for entry in entries:
            if drafted:
                state = self.cache.request(entry.request_id)
                parents = range(-1, len(entry.tokens) - 1) if entry.parents is None else entry.parents
                self._drafts[entry.request_id] = _Draft(state, state.resets, state.num_cached, [int(p) for p in parents])
            else:
                self.cache.commit(entry.request_id, len(entry.tokens))
        return logits

    def keep(self, paths: Mapping[Hashable, Sequence[int]]) -> None:
        """Behind a step of drafted tokens: `paths[request]` names the accepted ones by their places in the request's entry, from one
        that follows what is cached on, each the parent of the next (empty: none). What they left in the cache moves to the places of
        their positions and counts as cached from now on; all else of the drafted tokens is forgotten. A request of that step that `paths`
        does not name may still be kept later, until its next step."""
        for request_id, path in paths.items():
            draft = self._drafts.get(request_id)
            if draft is None or not draft.lies_in(self.cache.request(request_id) if request_id in self.cache else None):
                raise ValueError(f"request {request_id!r} has no drafted tokens")
            before, parents = -1, draft.parents
            for place in path:
                if not 0 <= int(place) < len(parents) or parents[int(place)] != before:
                    raise ValueError(f"request {request_id!r}: token {place} does not follow token {before} in its tree")
                before = int(place)
        moved = [(request_id, [int(p) for p in path]) for request_id, path in paths.items() if list(path) != list(range(len(path)))]
        if moved:
            length = max(len(path) for _, path in moved)
            states = [self.cache.request(request_id) for request_id, _ in moved]
            packed = np.full((len(moved), 2 + length), -1, dtype=np.int32)
            for row, (_, path), state in zip(packed, moved, states):
                row[:2] = state.slot, state.num_cached
                row[2:2 + len(path)] = path
            rows, past, path = (self.ops.upload(np.ascontiguousarray(a)) for a in (packed[:, 0], packed[:, 1], packed[:, 2:]))
            for group in self.cache.groups:
                for decl in group.requirement.tensors:
                    self.ops.keep_drafted(group.tensors[decl.name], 2 + decl.shape.index(PAGE), group.table, rows, past, path)
        for request_id, path in paths.items():
            del self._drafts[request_id]
            if len(path):
                self.cache.commit(request_id, len(path))

    def finish(self, request_id) -> None:
        self._drafts.pop(request_id, None)
        if request_id in self.cache:
            self.cache.release(request_id)
