"""The plan of attention over shared prefixes, on the host: every (token, key) pair exactly once, through a page that the token's request
holds there, whatever the tables share."""
import random

import numpy as np
import pytest

from sprout_lm_b200.prefix_plan import MEMBER_TOKENS, MIN_SAVED_KEYS, HostPlan, PlanError


def batch(rng, requests, page, stems, counts, own):
    """Tables, starts and contexts of requests whose leading pages come from common stems."""
    fresh = iter(range(1000, 10 ** 9))
    stems = [[next(fresh) for _ in range(n)] for n in stems]
    stems.append(stems[0][:max(1, len(stems[0]) // 2)] + [next(fresh) for _ in range(9)])       # branches off the first
    tables, contexts, tokens = [], [], []
    for _ in range(requests):
        stem = rng.choice(stems)
        held = stem[:rng.randint(0, len(stem))] if rng.random() < 0.4 else stem
        n = rng.choice(counts)
        contexts.append(len(held) * page + rng.randint(0, own) + n)
        tables.append(held + [next(fresh) for _ in range(-(-contexts[-1] // page) - len(held))])
        tokens.append(n)
    table = np.full((requests, max(map(len, tables))), -1, dtype=np.int32)
    for row, pages in zip(table, tables):
        row[:len(pages)] = pages
    return table, np.concatenate([[0], np.cumsum(tokens)]), np.asarray(contexts)


def covered(plan, tables, group):
    """Per (place, head of the group): the (key, page) pairs of the plan's items."""
    pairs = {}
    for table, key_begin, key_end, token_begin, row_begin, rows, part, _ in plan.items.tolist():
        for i in range(rows):
            place, head = token_begin + (row_begin + i) // group, (row_begin + i) % group
            assert 0 <= part < plan.part_start[place + 1] - plan.part_start[place]
            pairs.setdefault((place, head), []).append((part, key_begin, key_end, table))
    return pairs


@pytest.mark.parametrize("seed", range(40))
def test_every_key_once(seed):
    rng = random.Random(seed)
    page, group, kv_heads = rng.choice([1, 4, 8, 32]), rng.choice([1, 3, 7]), rng.choice([1, 2])
    tables, q_start, contexts = batch(rng, rng.randint(1, 12), page, [rng.randint(1, 30) for _ in range(3)], rng.choice([[1], [1, 2, 5], [1, 16, 17, 40]]), 60)
    for tensor_cores in (True, False):
        plan = HostPlan(tables, q_start, contexts, page, group * kv_heads, kv_heads, tensor_cores, rng.choice([1, 8, 60, 600]), rng.choice([0, 1, 148]))
        assert sorted(plan.order.tolist()) == list(range(plan.tokens))
        assert plan.simple_items + plan.matrix_items + plan.narrow_items + plan.wide_items == len(plan.items) and (plan.simple_items > 0) != tensor_cores
        pairs = covered(plan, tables, group)
        for place, token in enumerate(plan.order.tolist()):
            request = int(plan.table_of[place])
            assert q_start[request] <= token < q_start[request + 1]
            position = contexts[request] - (q_start[request + 1] - token)
            assert plan.seen[place] + plan.extra[place] == position + 1 and 0 <= plan.extra[place] < MEMBER_TOKENS
            for head in range(group):
                held = sorted(pairs[place, head])
                assert [part for part, *_ in held] == list(range(plan.part_start[place + 1] - plan.part_start[place]))     # a result each
                keys = sorted((k, int(tables[table, k // page])) for _, begin, end, table in held for k in range(begin, end))
                assert keys == [(k, int(tables[request, k // page])) for k in range(plan.seen[place])]


@pytest.mark.parametrize("seed", range(20))
def test_every_key_once_in_later_steps(seed):
    """A plan for steps whose requests are each up to ``stretch`` positions further: open items end with their member's first token."""
    rng = random.Random(100 + seed)
    page, group, kv_heads, stretch = rng.choice([1, 4, 8, 32]), rng.choice([1, 3, 7]), rng.choice([1, 2]), rng.choice([1, 17, 128, 1024])
    tables, q_start, contexts = batch(rng, rng.randint(1, 12), page, [rng.randint(1, 30) for _ in range(3)], rng.choice([[1], [1, 2, 5], [1, 16, 17, 40]]), 60)
    room = np.full((len(tables), -(-stretch // page)), -1, dtype=np.int32)
    ahead = np.array([rng.choice([0, stretch, rng.randint(0, stretch)]) for _ in contexts])
    for tensor_cores in (True, False):
        plan = HostPlan(tables, q_start, contexts, page, group * kv_heads, kv_heads, tensor_cores, rng.choice([1, 8, 60, 600]), rng.choice([0, 1, 148]), stretch=stretch)
        own = HostPlan(tables, q_start, contexts, page, group * kv_heads, kv_heads, tensor_cores, 60, 0)
        assert plan.pages * page >= contexts.max() + stretch and plan.pages <= tables.shape[1] + room.shape[1]
        assert (plan.order == own.order).all() and (plan.seen == own.seen).all() and (plan.extra == own.extra).all()
        assert not plan.items[:plan.matrix_items, 7].any()
        keys = np.zeros((plan.tokens, group), dtype=np.int64)
        for table, key_begin, key_end, token_begin, row_begin, rows, _, is_open in plan.items.tolist():
            if is_open:                # as csrc/attention_prefix.cuh has it: to the member's first token
                first = plan.seen[token_begin] + ahead[plan.table_of[token_begin]]
                assert key_begin < plan.seen[token_begin] <= first <= key_end
                key_end = first
            keys[token_begin:].reshape(-1)[row_begin:row_begin + rows] += key_end - key_begin
        assert (keys == (plan.seen + ahead[plan.table_of])[:, None]).all()


@pytest.mark.parametrize("stretch", [-1, 1025, 2.0, True, None])
def test_stretch_is_checked(stretch):
    with pytest.raises(PlanError, match="stretch"):
        HostPlan([[0, 1]], [0, 1], [5], 8, 4, 1, True, 60, stretch=stretch)


def test_a_shared_prefix_is_read_once():
    requests, page, prefix = 50, 16, 1600
    tables = np.arange(requests * 110, dtype=np.int32).reshape(requests, 110)
    tables[:, :100] = tables[0, :100]
    plan = HostPlan(tables, np.arange(requests + 1), np.full(requests, prefix + 40), page, 14, 2, True, 592)
    assert plan.read_keys == prefix + 40 * requests and plan.context_keys == requests * (prefix + 40)
    assert len(plan.segments) == requests + 1 and plan.segments[0].token_end == requests


def test_branching_prefixes():
    """Two documents behind one system prompt, four requests each."""
    page = 8
    tables = np.arange(8 * 60, dtype=np.int32).reshape(8, 60)
    tables[:, :20] = tables[0, :20]
    tables[:4, 20:50], tables[4:, 20:50] = tables[0, 20:50], tables[7, 20:50]
    plan = HostPlan(tables, np.arange(9), np.full(8, 60 * page), page, 4, 1, True, 592)
    assert plan.read_keys == (20 + 2 * 30 + 8 * 10) * page
    assert sorted(s.token_end - s.token_begin for s in plan.segments) == [1] * 8 + [4, 4, 8]


def test_short_runs_stay_the_requests_own():
    page = 8
    tables = np.arange(2 * 20, dtype=np.int32).reshape(2, 20)
    for shared in (MIN_SAVED_KEYS // page - 1, MIN_SAVED_KEYS // page):
        tables[1, :shared] = tables[0, :shared]
        plan = HostPlan(tables, [0, 1, 2], [100, 120], page, 4, 1, True, 592)
        assert len(plan.segments) == (2 if shared * page < MIN_SAVED_KEYS else 3)


@pytest.mark.parametrize("matrix_slots", [0, 148])
def test_no_range_is_much_longer_than_an_even_share(matrix_slots):
    """A long prefix for many requests is divided so far that its items fill a few rounds of the device evenly."""
    requests, page = 200, 16
    tables = np.arange(requests * 1030, dtype=np.int32).reshape(requests, 1030)
    tables[:, :1000] = tables[0, :1000]
    plan = HostPlan(tables, np.arange(requests + 1), np.full(requests, 16000 + 200), page, 28, 4, True, 444, matrix_slots)
    prefix = plan.items[plan.items[:, 5] > 16]
    assert (plan.matrix_items > 0) == (matrix_slots > 0) and len(prefix) == (plan.matrix_items or plan.wide_items)
    lengths = -(-(prefix[:, 2] - prefix[:, 1]) // 128)
    assert int(lengths.max()) * (matrix_slots or 444) <= 1.3 * int(lengths.sum()) * 4


@pytest.mark.parametrize("tokens, context", [(20000, 20000), (5000, 30000)])
def test_a_long_prompt_among_the_requests(tokens, context):
    """A request's pages of the step itself are read by its members, each with one result: no chain of a segment a page."""
    page, cached = 16, context - tokens
    tables = np.arange(3 * (context // page), dtype=np.int32).reshape(3, -1)
    tables[:, :cached // page] = tables[0, :cached // page]
    plan = HostPlan(tables, [0, tokens, tokens + 1, tokens + 2], [context, cached + 1, cached + 1], page, 28, 4, True, 592, 148, 296, 128)
    assert plan.tokens == tokens + 2 and len(plan.segments) <= -(-tokens // MEMBER_TOKENS) + 3
    assert plan.parts <= 12 * plan.tokens        # a segment of the cached pages in ranges, and the member's own


@pytest.mark.parametrize("group", [1, 7])
def test_many_requests_that_leave_a_document_page_by_page(group):
    """Request i holds i pages of a document: as many branches one inside the other."""
    page, requests = 16, 1300
    tables = np.full((requests, requests + 1), -1, dtype=np.int32)
    for i in range(requests):
        tables[i, :i] = np.arange(i)
        tables[i, i] = 10000 + i
    contexts = np.arange(requests) * page + 3
    plan = HostPlan(tables, np.arange(requests + 1), contexts, page, group, 1, True, 592, 148, 296, 128)
    keys = np.zeros(plan.tokens * group, dtype=np.int64)
    for table, begin, end, token_begin, row_begin, rows, _, _ in plan.items.tolist():
        keys[token_begin * group + row_begin:][:rows] += end - begin
        assert (tables[table, begin // page:-(-end // page)] >= 0).all()
    assert (keys.reshape(-1, group) == contexts[plan.table_of][:, None]).all()


def test_one_token_of_context():
    plan = HostPlan([[3]], [0, 1], [1], 16, 4, 2, True, 592)
    assert plan.items[:, :7].tolist() == [[0, 0, 1, 0, 0, 2, 0]] and plan.parts == 1


@pytest.mark.parametrize("change", [dict(q_start=[0, 1]), dict(q_start=[1, 2, 3]), dict(q_start=[0, 0, 2]), dict(contexts=[0, 5]), dict(contexts=[5, 33]),
                                    dict(tables=[1, 2]), dict(tables=[[1, 2]]), dict(contexts=[5.0, 6.0]), dict(page_tokens=0), dict(heads=3), dict(contexts=[], q_start=[0])])
def test_refusals(change):
    given = dict(tables=[[1, 2], [1, 3]], q_start=[0, 1, 3], contexts=[5, 9], page_tokens=16, heads=4, kv_heads=2, tensor_cores=True, slots=10)
    HostPlan(**given)
    with pytest.raises(PlanError):
        HostPlan(**{**given, **change})


def test_kernel_binding_refuses_what_it_cannot_run():
    import torch
    from sprout_lm_b200 import kernels
    for head_dim in (0, 7, 258):
        with pytest.raises(kernels.KernelError, match="head_dim"):
            kernels.shared_prefix_plan([[1]], [0, 1], [1], 16, 4, 2, head_dim, torch.bfloat16, "cpu")
    with pytest.raises(kernels.KernelError, match="unsupported element type"):
        kernels.shared_prefix_plan([[1]], [0, 1], [1], 16, 4, 2, 64, torch.float16, "cpu")
    with pytest.raises(kernels.KernelError, match="context"):
        kernels.shared_prefix_plan([[1]], [0, 1], [17], 16, 4, 2, 64, torch.bfloat16, "cpu")
    # tensors that are not on a GPU are refused, whichever they are, before anything else is looked at
    plan = kernels.shared_prefix_plan([[1]], [0, 1], [1], 16, 4, 2, 64, torch.bfloat16, "cpu")
    q, cache = torch.zeros(1, 256, dtype=torch.bfloat16), torch.zeros(2, 2, 16, 64, dtype=torch.bfloat16)
    word = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(kernels.KernelError, match="q must be a CUDA tensor"):
        kernels.attention_shared_prefix(q, cache, cache.clone(), torch.ones(1, 1, dtype=torch.int32), word, plan, torch.zeros_like(q), word)
    with pytest.raises(kernels.KernelError, match="logits must be a CUDA tensor"):
        kernels.verify_drafts(torch.zeros(2, 5), torch.zeros(2, dtype=torch.int32), torch.tensor([0, 2], dtype=torch.int32), word)


class OnDevice:
    """What the device check sees of a tensor."""

    def __init__(self, index):
        self.index, self.device = index, f"device {index}"

    def get_device(self):
        return self.index


def test_device_check(monkeypatch):
    """One tensor off the GPU, or on another GPU than the current one, is found at any place among the others."""
    import torch
    from sprout_lm_b200 import kernels
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 1)
    kernels._one_device("name", [("a", OnDevice(1)), ("b", None), ("c", OnDevice(1))])
    for at in range(3):
        for index, text in ((-1, "CUDA tensor"), (0, "the current device is cuda:1")):
            tensors = [(f"t{i}", OnDevice(index if i == at else 1)) for i in range(3)]
            with pytest.raises(kernels.KernelError, match=f"t{at} .*{text}"):
                kernels._one_device("name", tensors)
    with pytest.raises(kernels.KernelError, match="t0 is on"):
        kernels._one_device("name", [("t0", OnDevice(0)), ("t1", OnDevice(0))])


def test_overlap_check():
    import torch
    from sprout_lm_b200 import kernels
    whole = torch.zeros(40)
    for a0 in range(0, 40, 3):
        for a1 in range(a0 + 1, 41, 4):
            for b0 in range(0, 40, 5):
                for b1 in range(b0 + 1, 41, 3):
                    assert kernels._overlap(whole[a0:a1], whole[b0:b1]) == (a0 < b1 and b0 < a1)
    rows = torch.zeros(4, 10)
    assert kernels._overlap(rows[:, :3], rows[:, 5:]) and not kernels._overlap(rows[:2, 5:], rows[2:, :3])      # from the first to the last element
    assert not kernels._overlap(whole[3:3], whole)


def test_ragged_tables_are_refused():
    with pytest.raises(PlanError, match="arrays on the host"):
        HostPlan([[1, 2], [3]], [0, 1, 2], [5, 5], 8, 4, 1, True, 60)


@pytest.mark.timeout(60)
@pytest.mark.parametrize("seed", range(12))
def test_pages_outside_the_pool(seed):
    """Negative pages inside contexts, beside requests of every length: the plan ends, and has every key once (the kernels skip and flag such
    pages).  They are nobody's in common: runs end before them."""
    rng = random.Random(seed)
    page, group, kv_heads = rng.choice([1, 4, 16]), rng.choice([1, 4]), rng.choice([1, 2])
    tables, q_start, contexts = batch(rng, rng.randint(2, 14), page, [rng.randint(1, 30) for _ in range(3)], rng.choice([[1], [1, 2, 5], [1, 17]]), 60)
    for row, context in zip(tables, contexts):
        for at in range(-(-int(context) // page)):
            if rng.random() < (0.5 if at == 0 else 0.1):
                row[at] = -rng.randint(1, 2 * len(tables))
    if seed % 3 == 0:
        tables[:, 1:2] = -1                               # all of them, in the same place
    for tensor_cores in (True, False):
        plan = HostPlan(tables, q_start, contexts, page, group * kv_heads, kv_heads, tensor_cores, 60, 148)
        pairs = covered(plan, tables, group)
        for place in range(plan.tokens):
            request = int(plan.table_of[place])
            for head in range(group):
                keys = sorted((k, int(tables[table, k // page])) for _, begin, end, table in pairs[place, head] for k in range(begin, end))
                assert keys == [(k, int(tables[request, k // page])) for k in range(plan.seen[place])]
        for s in plan.segments:
            assert s.own or (tables[s.table, s.key_begin // page:s.key_end // page] >= 0).all()


@pytest.mark.timeout(60)
def test_a_short_request_beside_a_negative_page():
    plan = HostPlan([[5, 6, 7, 8], [-1, 9, 10, 11], [3, 4, 5, 6]], [0, 1, 2, 3], [3, 40, 40], 16, 8, 2, True, 60)
    assert len(plan.segments) == 3 and plan.read_keys == 83


def test_columns_of_one_buffer_do_not_share_memory():
    """Against the elements themselves."""
    from sprout_lm_b200 import kernels
    for stride in (4, 9, 13):
        for width in range(1, 5):
            for gap in range(-30, 31):
                places = lambda start: {start + r * stride + c for r in range(3) for c in range(width)}
                apart = not places(0) & places(gap)
                said = kernels._columns_apart(gap, width, 3, stride, stride)
                assert not said or apart                  # never side by side when they meet
                if apart and gap % stride:                # and found wherever both keep to columns of their own
                    assert said == (width <= gap % stride <= stride - width)
    assert not kernels._columns_apart(5, 4, 3, 9, 10) and not kernels._columns_apart(0, 4, 1, 9, 9)
