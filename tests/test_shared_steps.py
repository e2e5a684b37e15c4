"""When a step takes a plan of shared pages, and the numbers that check drafted tokens (host only)."""
import random

import numpy as np
import pytest

from sprout_lm_b200.engine import shared
from sprout_lm_b200.engine.shared import shared_keys
from sprout_lm_b200.sampling import uniform_for, verify_uniforms


def table_of(tables):
    table = np.full((len(tables), max(map(len, tables))), -1, dtype=np.int32)
    for row, pages in zip(table, tables):
        row[:len(pages)] = pages
    return table, np.array([len(t) for t in tables])


def test_shared_keys_counts_what_all_of_a_group_hold():
    assert shared_keys(*table_of([[1, 2, 3, 4], [1, 2, 3, 9], [1, 2, 7]]), 16) == 2 * 2 * 16
    assert shared_keys(*table_of([[1, 2], [3, 2], [4]]), 16) == 0
    assert shared_keys(*table_of([[1, 2], [1, 2], [5, 6, 7], [5, 6]]), 8) == 2 * 8 + 2 * 8
    # pages that a request's tokens do not all see in full are not shared
    table, whole = table_of([[1, 2, 3], [1, 2, 3]])
    assert shared_keys(table, whole - 1, 8) == 2 * 8 and shared_keys(table, whole * 0, 8) == 0


@pytest.mark.parametrize("seed", range(5))
def test_shared_keys_against_every_pair(seed):
    rng = random.Random(seed)
    tables = [[rng.randint(0, 1) for _ in range(rng.randint(1, 6))] for _ in range(8)]
    groups = {first: [t for t in tables if t[0] == first] for first in (0, 1)}
    want = 0
    for group in groups.values():
        common = 0
        while group and all(len(t) > common for t in group) and len({t[common] for t in group}) == 1:
            common += 1
        want += max(0, len(group) - 1) * common * 4
    assert shared_keys(*table_of(tables), 4) == want


def test_numbers_follow_the_output_index_alone():
    accept, draw = verify_uniforms(5, "a", 10, 4)
    assert (accept[2:], draw[2:]) == verify_uniforms(5, "a", 12, 2)
    assert draw == [uniform_for(5, "a", 10 + i) for i in range(4)] and accept != draw
    assert all(0.0 <= u < 1.0 for u in accept + draw)


class Request:
    length, tables = 100, [[1, 2, 3]]


class Entry:
    def __init__(self, seq):
        self.seq, self.tokens, self.want = seq, [5], [0]


def test_when_a_capture_is_thought_of(monkeypatch):
    """At 8, 16, 32 .. decode steps of the same requests; behind one's last step at once; a step launched ahead makes way for it."""
    steps = shared.SharedPrefixSteps.__new__(shared.SharedPrefixSteps)
    steps.sizes, steps.after, steps._seqs, steps._same, steps._graph, steps._base = {(4, 1, 64): 1}, 8, [], 0, None, []
    asked = []
    monkeypatch.setattr(steps, "_capture", lambda entries: asked.append(steps._same), raising=False)
    entries = [Entry(Request()), Entry(Request())]
    for _ in range(40):
        ahead = steps.due(entries, behind=1)
        assert steps.decode_graph(entries, True) is None
        assert ahead == (asked[-1:] == [steps._same])
    assert asked == [8, 16, 32]
    assert steps.decode_graph(entries[::-1], True) is None and steps._same == 1          # their order is the plan's
    steps._graph, steps._base = "captured", [100, 100]
    assert steps.decode_graph(entries[::-1], True) == "captured" and steps.captured(entries, 0) is None
    assert steps.captured(entries[::-1], shared.STRETCH) == "captured" and steps.captured(entries[::-1], shared.STRETCH + 1) is None
    entries[0].seq.length = 99
    assert steps.decode_graph(entries[::-1], False) is None and asked == [8, 16, 32]     # launched ahead: nothing is made
    assert steps.decode_graph(entries[::-1], True) is None and asked == [8, 16, 32, steps._same]
    assert steps.decode_graph(entries[:1], True) is None and steps._graph is None and not steps.due(entries[:1], behind=7)


def test_engine_option_is_a_boolean():
    from sprout_lm_b200 import EngineOptions
    EngineOptions(shared_prefix=True).validate()
    with pytest.raises(ValueError, match="shared_prefix must be a boolean"):
        EngineOptions(shared_prefix=1).validate()


def test_a_capture_serves_tables_within_its_width(monkeypatch):
    """A caller may reserve pages far ahead (a device-side loop does): the captured step, whose tables have a fixed width, is not taken then, now
    or ahead, and the next is thought of at once."""
    steps = shared.SharedPrefixSteps.__new__(shared.SharedPrefixSteps)
    steps.sizes, steps.after, steps._seqs, steps._same, steps._base, steps._width = {(4, 1, 64): 1}, 8, [], 0, [100, 100], 4
    monkeypatch.setattr(steps, "_capture", lambda entries: "another", raising=False)
    entries = [Entry(Request()), Entry(Request())]
    steps._seqs, steps._graph = [e.seq for e in entries], "captured"
    assert steps.captured(entries) == steps.captured(entries, 1) == "captured"
    entries[1].seq.tables = [[1, 2, 3, 4]]
    assert steps.captured(entries) == "captured"
    entries[1].seq.tables = [[1, 2, 3, 4, 5]]
    assert steps.captured(entries) is None and steps.captured(entries, 1) is None
    assert steps.due(entries, behind=1) and steps.decode_graph(entries, True) == "another"


def context_of(groups, group, plans):
    import torch
    from sprout_lm_b200.engine.batch import StepContext
    tables = [torch.full((2, 3), g, dtype=torch.int32) for g in range(groups)]
    none = torch.zeros(0, dtype=torch.int32)
    ctx = StepContext(num_tokens=2, num_seqs=2, max_q_len=1, max_context=9, token_ids=none, positions=none, seq_of_token=none, q_start=none,
                      context_lens=none, state_slots=none, logits_rows=none, block_tables=tables, page_tokens=16)
    ctx.shared = plans and shared.Plans(group, plans)
    return ctx


def test_a_plan_is_its_page_groups_alone(monkeypatch):
    """Layers of another page group have pages of their own, whatever their sizes: they take no plan of the first's, and keep the kernels that
    they have without one."""
    from types import SimpleNamespace
    from sprout_lm_b200.parts import attention
    monkeypatch.setattr(attention.kernels, "decode_fusable", lambda *sizes: True)
    mixer = attention.PagedGQAttention.__new__(attention.PagedGQAttention)
    mixer.heads, mixer.kv_heads, mixer.head_dim = 4, 2, 16
    view = lambda table: SimpleNamespace(block_table=table, page_tokens=16, write=True)
    for group in (0, 1):
        ctx = context_of(2, group, {(4, 2, 16): "plan"})
        mine, other = ctx.block_tables[group], ctx.block_tables[1 - group]
        assert ctx.shared_plan((4, 2, 16), mine) == "plan" and ctx.shared_plan((4, 2, 32), mine) is None and ctx.shared_plan((4, 2, 16), other) is None
        assert not mixer._decodes_fused(2, ctx, view(mine)) and mixer._decodes_fused(2, ctx, view(other))
    ctx = context_of(1, 0, None)
    assert ctx.shared_plan((4, 2, 16), ctx.block_tables[0]) is None and mixer._decodes_fused(2, ctx, view(ctx.block_tables[0]))


def test_drafts_have_numbers_of_their_own():
    from sprout_lm_b200.sampling import draft_uniforms
    drafts = draft_uniforms(5, "a", 10, 4)
    assert drafts[2:] == draft_uniforms(5, "a", 12, 2) and all(0.0 <= u < 1.0 for u in drafts)
    accept, draw = verify_uniforms(5, "a", 10, 4)
    assert not set(drafts) & {*accept, *draw}


def test_emitted_tokens_follow_the_target_with_the_drafts_own_numbers():
    """Drafts drawn with ``draft_uniforms`` and checked with ``verify_uniforms``, the definition in 64 bits, 40,000 requests under one seed: the
    first token's frequencies are the target's within five standard deviations (the binomial's).  With the draws' own numbers for the
    drafts they are not."""
    from sprout_lm_b200.sampling import draft_uniforms
    rng = np.random.default_rng(0)
    p, q = (np.exp(1.2 * rng.standard_normal(8)) for _ in range(2))
    p, q = p / p.sum(), q / q.sum()
    left = np.maximum(p - q, 0.0)
    pick = lambda weights, u: int(np.searchsorted(np.cumsum(weights), u * weights.sum(), side="right"))
    count = 40000
    seen = {"own": np.zeros(8), "draws": np.zeros(8)}
    for r in range(count):
        (u, _), (w, _) = verify_uniforms(3, f"r{r}", 0, 2)
        for name, number in (("own", draft_uniforms(3, f"r{r}", 0, 1)[0]), ("draws", w)):
            draft = pick(q, number)
            seen[name][draft if u * q[draft] < p[draft] else pick(left, w)] += 1 / count
    off = {name: np.abs(f - p) / np.sqrt(p * (1 - p) / count) for name, f in seen.items()}
    assert (off["own"] <= 5).all() and off["draws"].max() > 5
