"""Steps whose requests hold the same leading pages: when their attention reads those pages once for all of them.

The cache manager lets requests share the pages of a common prefix; attention as a rule reads them once per request.  A runner made with
``shared_prefix=True`` gives steps of few tokens a request (decode steps, drafted tokens) a plan of the shared pages
(``kernels.shared_prefix_plan``) where that saves more time than it costs: a plan takes the host some hundred microseconds, and a decode
step that takes one runs its launches one by one instead of replaying a capture (a plan changes with every step's contexts).  Results
then differ from the other kernels' in the order of float32 additions, as between batch sizes.
"""
from __future__ import annotations

import weakref

import numpy as np
import torch

from .. import kernels
from ..prefix_plan import MEMBER_TOKENS

BYTES_PER_US = 6.4e6               # what attention streams keys and values at
# A plan, for each request of it, and a layer's launches one by one beside a replay of them (measured: 64 requests of the 0.5B shape over
# 4,096 shared keys take 1.55 ms a step as a replay and 4.3 with a plan; over 32,768, 4.3 and 4.5)
PLAN_US, PLAN_REQUEST_US, EAGER_LAYER_US = 600.0, 10.0, 130.0


def shared_keys(table: np.ndarray, whole: np.ndarray, page_tokens: int) -> int:
    """Key reads that reading common leading pages once saves, at least: over the requests with the same first page, the pages that all of
    them hold; ``whole``: a request's pages that its tokens all see in full."""
    saved = 0
    for first in np.unique(table[:, 0]):
        group = np.flatnonzero((table[:, 0] == first) & (whole > 0))
        if len(group) > 1:
            rows = table[group, :int(whole[group].min())]
            same = (rows == rows[0]).all(axis=0)
            saved += (len(group) - 1) * (int(same.argmin()) if not same.all() else rows.shape[1]) * page_tokens
    return saved


class SharedPrefixSteps:
    """Decides for a runner's steps; ``always`` takes a plan whenever pages are shared (tests)."""

    def __init__(self, runner):
        self.runner = runner
        self.always = False
        self.steps = 0                     # steps that took a plan
        self.tables: dict = {}             # the last such step's block tables as arrays, by group
        manager, runtime = runner.manager, runner.runtime
        self.group = next((g for g in runner._groups_in_use if manager.groups[g].kind == "full"), None)
        self._tables = weakref.WeakKeyDictionary()          # request's cache -> its block table as an array (a full group's only grows)
        # how many layer calls have attention of which sizes
        self.sizes: dict = {}
        if runtime.dtype == torch.bfloat16 and self.group is not None:
            for call in runner.model.spec.order:
                sizes = getattr(runner.model.blocks[call.layer].mixer, "shared_prefix_sizes", lambda: None)()
                if sizes is not None and runner.storage.slot_group[call.cache] == self.group:
                    self.sizes[sizes] = self.sizes.get(sizes, 0) + 1

    def _table(self, seq) -> np.ndarray:
        pages, held = seq.tables[self.group], self._tables.get(seq)
        known = 0 if held is None else len(held)
        if known > len(pages):
            known = 0                      # given back meanwhile
        if held is None or known != len(pages):
            new = np.array(pages[known:], dtype=np.int32)
            held = self._tables[seq] = np.concatenate([held[:known], new]) if known else new
        return held

    def plans(self, entries, replayed: bool):
        """{sizes: plan} for a step, or None; ``replayed``: the step would be a capture's replay otherwise."""
        if not self.sizes or len(entries) < 2 or max(len(e.tokens) for e in entries) > MEMBER_TOKENS:
            return None
        counts = np.array([len(e.tokens) for e in entries])
        contexts = np.array([e.seq.length for e in entries]) + counts
        per_key = sum(n * kv_heads * head_dim * 4 for (_, kv_heads, head_dim), n in self.sizes.items())
        cost = PLAN_US + PLAN_REQUEST_US * len(entries) + (EAGER_LAYER_US * sum(self.sizes.values()) if replayed else 0.0)
        page_tokens = self.runner.page_tokens
        if not self.always and int(contexts.sum()) * per_key / BYTES_PER_US < cost:
            return None                    # not if every key were shared
        rows = [self._table(e.seq) for e in entries]
        table = np.full((len(entries), max(map(len, rows))), -1, dtype=np.int32)
        for at, row in zip(table, rows):
            at[:len(row)] = row
        saved = shared_keys(table, (contexts - counts + 1) // page_tokens, page_tokens)
        if not saved or (not self.always and saved * per_key / BYTES_PER_US < cost):
            return None
        q_start = np.concatenate([[0], np.cumsum(counts)])
        self.steps += 1
        self.tables = {self.group: table}
        return {sizes: kernels.shared_prefix_plan(table, q_start, contexts, page_tokens, *sizes, torch.bfloat16, self.runner.runtime.device)
                for sizes in self.sizes}
