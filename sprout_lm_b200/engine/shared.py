"""Steps whose requests hold the same leading pages: when their attention reads those pages once for all of them.

The cache manager lets requests share the pages of a common prefix; attention as a rule reads them once per request.  A runner made with
``shared_prefix=True`` gives steps of few tokens a request (decode steps, drafted tokens) a plan of the shared pages
(``kernels.shared_prefix_plan``) where that saves more time than it costs: a plan takes the host some hundred microseconds, and a decode
step that takes one runs its launches one by one instead of replaying a capture (a plan changes with every step's contexts).  Results
then differ from the other kernels' in the order of float32 additions, as between batch sizes.
"""
from __future__ import annotations

import numpy as np
import torch

from .. import kernels
from ..prefix_plan import MEMBER_TOKENS

BYTES_PER_US = 6.4e6               # what attention streams keys and values at
PLAN_US, PLAN_REQUEST_US = 400.0, 10.0         # a plan, and for each request of it
EAGER_LAYER_US = 90.0              # a layer's launches one by one beside a replay of them


def shared_keys(tables, page_tokens: int) -> int:
    """Key reads that reading common leading pages once saves, at least: over the requests with the same first page, what all of them hold.
    The lists between the least and the greatest in order share what those two do."""
    groups: dict = {}
    for table in tables:
        if table:
            groups.setdefault(table[0], []).append(table)
    saved = 0
    for group in groups.values():
        if len(group) > 1:
            low, high = min(group), max(group)
            common = 0
            for a, b in zip(low, high):
                if a != b:
                    break
                common += 1
            saved += (len(group) - 1) * common * page_tokens
    return saved


class SharedPrefixSteps:
    """Decides for a runner's steps; ``always`` takes a plan whenever pages are shared (tests)."""

    def __init__(self, runner):
        self.runner = runner
        self.always = False
        self.steps = 0                     # steps that took a plan
        manager, runtime = runner.manager, runner.runtime
        self.group = next((g for g in runner._groups_in_use if manager.groups[g].kind == "full"), None)
        # how many layer calls have attention of which sizes
        self.sizes: dict = {}
        if runtime.dtype == torch.bfloat16 and self.group is not None:
            for call in runner.model.spec.order:
                sizes = getattr(runner.model.blocks[call.layer].mixer, "shared_prefix_sizes", lambda: None)()
                if sizes is not None and runner.storage.slot_group[call.cache] == self.group:
                    self.sizes[sizes] = self.sizes.get(sizes, 0) + 1

    def plans(self, entries, replayed: bool):
        """{sizes: plan} for a step, or None; ``replayed``: the step would be a capture's replay otherwise."""
        if not self.sizes or len(entries) < 2 or max(len(e.tokens) for e in entries) > MEMBER_TOKENS:
            return None
        tables = [e.seq.tables[self.group] for e in entries]
        saved = shared_keys(tables, self.runner.page_tokens)
        if not saved:
            return None
        if not self.always:
            layers = sum(self.sizes.values())
            won = saved * sum(n * kv_heads * head_dim * 4 for (_, kv_heads, head_dim), n in self.sizes.items()) / BYTES_PER_US
            if won < PLAN_US + PLAN_REQUEST_US * len(entries) + (EAGER_LAYER_US * layers if replayed else 0.0):
                return None
        counts = [len(e.tokens) for e in entries]
        table = np.full((len(entries), max(map(len, tables))), -1, dtype=np.int32)
        for row, pages in zip(table, tables):
            row[:len(pages)] = pages
        q_start = np.concatenate([[0], np.cumsum(counts)])
        contexts = np.array([e.seq.length + n for e, n in zip(entries, counts)])
        self.steps += 1
        return {sizes: kernels.shared_prefix_plan(table, q_start, contexts, self.runner.page_tokens, *sizes, torch.bfloat16, self.runner.runtime.device)
                for sizes in self.sizes}
