"""Steps whose requests hold the same leading pages: when their attention reads those pages once for all of them.

The cache manager lets requests share the pages of a common prefix; attention as a rule reads them once per request.  A runner made with
``shared_prefix=True`` gives steps of few tokens a request (decode steps, drafted tokens) a plan of the shared pages
(``kernels.shared_prefix_plan``) where that saves more time than it costs.

Decode steps replay captures, and a plan is part of what is captured.  So once the same requests have decoded for a while, a plan for their
next ``STRETCH`` steps is made and a step captured over it; it is replayed until those are over (then the next is made) or another
request joins or leaves.  Other steps take a plan of their own and run their launches one by one.  Results differ from the other
kernels' in the order of float32 additions, as between batch sizes.
"""
from __future__ import annotations

import weakref

import numpy as np
import torch

from .. import kernels
from ..prefix_plan import MEMBER_TOKENS

BYTES_PER_US = 6.4e6               # what attention streams keys and values at
# A plan, for each request of it, and a layer's launches one by one beside a replay of them (measured: 64 requests of the 0.5B shape over
# 4,096 shared keys take 1.55 ms a step as a replay and 4.6 with a plan of its own; over 32,768, 4.4 and 4.5)
PLAN_US, PLAN_REQUEST_US, EAGER_LAYER_US = 600.0, 10.0, 130.0
# What of the reads' time is saved (the shared keys still meet every request's queries), and what a layer's attention takes longer otherwise.
# Replayed steps of 64 requests without and with a plan: the 0.5B shape, 24 layers, over 1,024, 4,096 and 32,768 shared keys 1.14 and 1.11 ms,
# 1.55 and 1.23, 4.36 and 1.65; of 8 over 4,096 and 16,384 0.74 and 0.77, 0.91 and 0.84; the 7B shape, 4 layers, 64 over 1,024 and 8,192
# 0.84 and 0.79, 1.25 and 0.84.
SAVED, REPLAY_LAYER_US = 0.7, 3.0
CAPTURE_US, CAPTURE_LAYER_US = 1500.0, 300.0         # a capture beside its plan (the first step of the above: 10 to 30 ms)
STRETCH = 128                      # steps that a captured one's plan serves behind its first


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


class Plans(dict):
    """{(query heads, key/value heads, head size): plan} for the layers whose pages are those of page group ``group``."""

    def __init__(self, group: int, plans):
        super().__init__(plans)
        self.group = group


class SharedPrefixSteps:
    """Decides for a runner's steps; ``always`` takes a plan whenever pages are shared (tests)."""

    _width = float("inf")                  # of the captured step's block tables, in pages

    def __init__(self, runner):
        self.runner = runner
        self.always = False
        self.steps = 0                     # steps that took a plan
        self.tables: dict = {}             # the last such step's block tables as arrays, by group
        self.after = 8                     # decode steps of the same requests before a capture over their pages is thought of (a power of two)
        self._seqs: list = []              # the last decode step's requests, for how many steps they have been those,
        self._same = 0
        self._graph = None                 # the step captured over their shared pages, and their lengths at its plan's first step
        self._base: list = []
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

    def _arrays(self, entries):
        """The requests' block tables as an array, their contexts and numbers of tokens in the step."""
        counts = np.array([len(e.tokens) for e in entries])
        rows = [self._table(e.seq) for e in entries]
        table = np.full((len(entries), max(map(len, rows))), -1, dtype=np.int32)
        for at, row in zip(table, rows):
            at[:len(row)] = row
        return table, np.array([e.seq.length for e in entries]) + counts, counts

    def _key_bytes(self) -> int:
        """What a key and its value take in all layers that read them over a plan."""
        return sum(n * kv_heads * head_dim * 4 for (_, kv_heads, head_dim), n in self.sizes.items())

    def _plans(self, table, q_start, contexts, stretch: int = 0):
        return Plans(self.group, {sizes: kernels.shared_prefix_plan(table, q_start, contexts, self.runner.page_tokens, *sizes, torch.bfloat16, self.runner.runtime.device, stretch)
                                  for sizes in self.sizes})

    # ------------------------------------------------------------------ captured decode steps
    def _are(self, entries) -> bool:
        return len(entries) == len(self._seqs) and all(e.seq is s for e, s in zip(entries, self._seqs))

    def captured(self, entries, shift: int = 0):
        """The step captured over these requests' shared pages if it serves them ``shift`` tokens on, else None: their lengths are within its
        plan's, and their block tables (a caller may have reserved far ahead meanwhile) within its width."""
        if self._graph is not None and self._are(entries) and all(0 <= e.seq.length + shift - n <= STRETCH for e, n in zip(entries, self._base)) \
                and all(len(t) <= self._width for e in entries for t in e.seq.tables):
            return self._graph
        return None

    def due(self, entries, behind: int = 0) -> bool:
        """Whether the decode step of these requests (``behind`` the last one) is one to think of a capture at: the one they have is used up,
        or they have been the same for 8, 16, 32 .. steps."""
        if not self.sizes or len(entries) < 2 or not self._are(entries):
            return False
        same = self._same + behind
        return self._graph is not None or (same >= self.after and same & (same - 1) == 0)

    def decode_graph(self, entries, capture: bool):
        """The captured step for this decode step, or None; one is made (to run as it is captured) where it is due and pays."""
        if not self._are(entries):
            self._seqs, self._same, self._graph = [e.seq for e in entries], 0, None
        self._same += 1
        if not capture:
            return None
        graph = self.captured(entries)
        return self._capture(entries) if graph is None and self.due(entries) else graph

    def _capture(self, entries):
        from .graphs import DecodeGraph
        self._graph = None                 # before the next capture begins
        runner, page_tokens, layers = self.runner, self.runner.page_tokens, sum(self.sizes.values())
        table, contexts, counts = self._arrays(entries)
        saved = shared_keys(table, (contexts - counts) // page_tokens, page_tokens)
        # as many steps more as they have been the same
        gain = (SAVED * saved * self._key_bytes() / BYTES_PER_US - REPLAY_LAYER_US * layers) * min(self._same, STRETCH)
        if not saved or (not self.always and gain < PLAN_US + PLAN_REQUEST_US * len(entries) + CAPTURE_US + CAPTURE_LAYER_US * layers):
            return None
        longest = int(contexts.max()) + STRETCH
        multiple = runner.graphs.page_multiple
        width = -(-max(-(-longest // page_tokens), *(len(t) for e in entries for t in e.seq.tables)) // multiple) * multiple
        plans = self._plans(table, np.arange(len(entries) + 1), contexts, STRETCH)
        self._base, self._width = [e.seq.length for e in entries], width
        self._graph = DecodeGraph(runner, len(entries), width, min(width * page_tokens, -(-longest // 128) * 128), plans)
        return self._graph

    # ------------------------------------------------------------------ steps with a plan of their own
    def plans(self, entries, replayed: bool):
        """{sizes: plan} for a step, or None; ``replayed``: the step would be a capture's replay otherwise."""
        if not self.sizes or len(entries) < 2 or max(len(e.tokens) for e in entries) > MEMBER_TOKENS:
            return None
        per_key = self._key_bytes()
        cost = PLAN_US + PLAN_REQUEST_US * len(entries) + (EAGER_LAYER_US * sum(self.sizes.values()) if replayed else 0.0)
        if not self.always and sum(e.seq.length + len(e.tokens) for e in entries) * per_key / BYTES_PER_US < cost:
            return None                    # not if every key were shared
        table, contexts, counts = self._arrays(entries)
        saved = shared_keys(table, (contexts - counts) // self.runner.page_tokens, self.runner.page_tokens)
        if not saved or (not self.always and SAVED * saved * per_key / BYTES_PER_US < cost):
            return None
        self.steps += 1
        self.tables = {self.group: table}
        return self._plans(table, np.concatenate([[0], np.cumsum(counts)]), contexts)
