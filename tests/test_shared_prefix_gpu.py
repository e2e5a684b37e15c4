"""Attention over shared prefixes against a plain implementation in 64 bits.

Tolerances, with A = sum_k w_k |v_k| and o the exact output (w the softmax weights).  bfloat16: the weights are rounded to bfloat16 where
they multiply the values (2^-8 of each: 2^-8 A), and so is the output (2^-8 |o|); the rest is float32: a score is off by (d + 4) 2^-24
of the sum of its products' sizes, its weight by as much, relative, and the sums by 2^-24 for every key, twice that with the
denominator's.  float32: those last terms alone, and 2^-24 |o|."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

DEV = "cuda:0"


@pytest.fixture()
def status():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


class Step:
    """A step's tensors: requests of `groups` prefixes (pages each), own keys and new tokens per request."""

    def __init__(self, heads, kv_heads, dim, dtype, page, group, prefix_pages, own, tokens, seed=0, spare=5, sharp=1.0, table_pad=0, pool=None):
        g = torch.Generator().manual_seed(seed)
        self.heads, self.kv_heads, self.dim, self.dtype, self.page = heads, kv_heads, dim, dtype, page
        self.contexts = [prefix_pages[group[r]] * page + own[r] + tokens[r] for r in range(len(own))]
        own_pages = [-(-(o + t) // page) for o, t in zip(own, tokens)]
        total = sum(prefix_pages) + sum(own_pages) + spare
        free = torch.randperm(total, generator=g).tolist()
        if pool is not None:                              # the same pages at the end of a pool that large
            free = [pool - total + f for f in free]
        shared = [[free.pop() for _ in range(n)] for n in prefix_pages]
        self.pages = [shared[group[r]] + [free.pop() for _ in range(own_pages[r])] for r in range(len(own))]
        width = max(map(len, self.pages)) + table_pad
        self.tables = np.full((len(own), width), -1, dtype=np.int32)
        for row, pages in zip(self.tables, self.pages):
            row[:len(pages)] = pages
        self.q_start = np.concatenate([[0], np.cumsum(tokens)]).astype(np.int32)
        self.positions = torch.cat([torch.arange(c - t, c, dtype=torch.int32) for c, t in zip(self.contexts, tokens)]).to(DEV)
        shape = (pool or total, kv_heads, page, dim)
        # unused pages and rows behind a context hold NaN
        if pool is None:
            self.k, self.v = (torch.full(shape, float("nan"), dtype=dtype, device=DEV) for _ in range(2))
        else:
            self.k, self.v = (torch.empty(shape, dtype=dtype, device=DEV) for _ in range(2))
            self.k[-total:] = float("nan")
            self.v[-total:] = float("nan")
        filled = set()
        for pages, context in zip(self.pages, self.contexts):
            for i, p in enumerate(pages):
                rows = min(page, context - i * page)
                if rows > 0 and p not in filled:
                    filled.add(p)
                    for cache in (self.k, self.v):
                        cache[p, :, :rows] = torch.randn(kv_heads, rows, dim, generator=g).to(dtype).to(DEV)
        self.q = (torch.randn(int(self.q_start[-1]), heads * dim, generator=g) * sharp).to(dtype).to(DEV)
        self.block_table = torch.from_numpy(self.tables).to(DEV)

    def plan(self):
        from sprout_lm_b200 import kernels
        return kernels.shared_prefix_plan(self.tables, self.q_start, self.contexts, self.page, self.heads, self.kv_heads, self.dim, self.dtype, DEV)

    def run(self, status, out=None, plan=None):
        from sprout_lm_b200 import kernels
        out = torch.full_like(self.q, float("nan")) if out is None else out
        kernels.attention_shared_prefix(self.q, self.k, self.v, self.block_table, self.positions, plan or self.plan(), out, status)
        return out

    def exact(self):
        """(outputs, tolerances) in 64 bits."""
        group = self.heads // self.kv_heads
        outs, tols = [], []
        for r, context in enumerate(self.contexts):
            place = torch.arange(context, device=DEV)
            pages = torch.tensor(self.pages[r], device=DEV)[place // self.page]
            k, v = (c[pages, :, place % self.page].double().permute(1, 0, 2) for c in (self.k, self.v))        # [kv_heads, context, dim]
            for t in range(int(self.q_start[r]), int(self.q_start[r + 1])):
                seen = int(self.positions[t]) + 1
                q = self.q[t].double().view(self.kv_heads, group, self.dim)
                scores = q @ k[:, :seen].transpose(1, 2) / math.sqrt(self.dim)
                sizes = (q.abs() @ k[:, :seen].abs().transpose(1, 2)).amax() / math.sqrt(self.dim)
                w = torch.softmax(scores, -1)
                o, a = (w @ v[:, :seen]).reshape(-1), (w @ v[:, :seen].abs()).reshape(-1)
                fp32 = 2.0 ** -24 * a * (4 * (self.dim + 4) * sizes + 4 * seen + 64)
                half = 2.0 ** -8 if self.dtype == torch.bfloat16 else 2.0 ** -24
                tols.append(fp32 + half * o.abs() + (half * a if self.dtype == torch.bfloat16 else 0))
                outs.append(o)
        return torch.stack(outs), torch.stack(tols)

    def check(self, status, out=None):
        out = self.run(status, out)
        want, tol = self.exact()
        assert int(status.item()) == 0
        error = (out.double() - want).abs()
        assert bool((error <= tol).all()), f"off by {float((error / tol).max()):.2f} of what it may be"
        return out


BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("heads,kv_heads,dim,dtype", [(14, 2, 64, BF16), (28, 4, 128, BF16), (40, 8, 128, BF16), (5, 1, 48, BF16), (3, 3, 80, BF16), (16, 1, 16, BF16),
                                                     (20, 1, 96, BF16), (4, 2, 112, BF16), (2, 1, 32, BF16), (4, 2, 256, BF16), (6, 3, 40, BF16), (3, 1, 144, BF16),
                                                     (14, 2, 64, F32), (4, 2, 128, F32), (3, 1, 6, F32), (2, 2, 130, F32), (4, 1, 256, F32)])
@pytest.mark.parametrize("page", [16, 5])
def test_head_layouts(heads, kv_heads, dim, dtype, page, status):
    Step(heads, kv_heads, dim, dtype, page, [0, 0, 0, 0, 0], [20], [0, 3, 41, 130, 17], [1, 2, 1, 6, 1], seed=dim).check(status)


@pytest.mark.parametrize("requests,prefix,own,tokens", [(1, 0, 1, 1), (1, 0, 0, 1), (2, 9, 0, 1), (3, 40, 300, 1), (17, 70, 33, 1), (33, 130, 20, 2), (64, 33, 5, 1),
                                                        (4, 25, 10, 16), (3, 20, 50, 17), (2, 12, 8, 45), (9, 300, 400, 4), (150, 20, 30, 1)])
@pytest.mark.parametrize("shape", [(14, 2, 64), (28, 4, 128)])
def test_batches(requests, prefix, own, tokens, shape, status):
    rng = np.random.default_rng(requests)
    owns = [int(n) for n in rng.integers(0, own + 1, requests)]
    Step(*shape, BF16, 16, [0] * requests, [prefix], owns, [int(n) for n in rng.integers(1, tokens + 1, requests)], seed=1, sharp=2.0).check(status)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_groups(dtype, status):
    rng = np.random.default_rng(5)
    group = [int(g) for g in rng.integers(0, 4, 23)]
    Step(14, 2, 64, dtype, 8, group, [30, 3, 77, 150], [int(n) for n in rng.integers(0, 90, 23)], [int(n) for n in rng.integers(1, 4, 23)], seed=2, table_pad=7).check(status)


@pytest.mark.parametrize("page", [1, 8, 32, 64, 128, 100])
def test_page_sizes(page, status):
    Step(28, 4, 128, BF16, page, [0] * 12, [-(-700 // page)], [int(n) for n in range(0, 240, 20)], [1] * 12, seed=3).check(status)


def test_branching_prefixes(status):
    step = Step(14, 2, 64, BF16, 16, [0, 0, 0, 1, 1, 1], [64, 64], [10, 20, 30, 40, 50, 60], [1] * 6, seed=4)
    step.tables[3:, :30] = step.tables[0, :30]            # the second group's prefix begins with the first one's
    for pages in step.pages[3:]:
        pages[:30] = step.pages[0][:30]
    step.block_table.copy_(torch.from_numpy(step.tables))
    assert len(step.plan().host.segments) == 6 + 3
    step.check(status)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F32, 64), (F32, 34), (BF16, 40)])
def test_strided_rows(dtype, dim, status):
    step = Step(14, 2, dim, dtype, 16, [0] * 5, [20], [5, 9, 0, 30, 100], [2, 1, 1, 3, 1], seed=6)
    wide = torch.full((step.q.shape[0], step.q.shape[1] + (256 if dim == 64 and dtype == BF16 else 3)), float("nan"), dtype=dtype, device=DEV)
    wide[:, :step.q.shape[1]] = step.q
    step.q = wide[:, :step.q.shape[1]]
    out = torch.full((step.q.shape[0], step.q.shape[1] + 3), 7.0, dtype=dtype, device=DEV)
    step.check(status, out[:, :step.q.shape[1]])
    assert bool((out[:, step.q.shape[1]:] == 7.0).all())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("q_first", [True, False])
def test_queries_and_outputs_in_columns_of_one_buffer(dtype, q_first, status):
    from sprout_lm_b200 import kernels
    step = Step(14, 2, 64, dtype, 16, [0] * 5, [20], [5, 9, 0, 30, 100], [2, 1, 1, 3, 1], seed=6)
    width = step.q.shape[1]
    both = torch.full((step.q.shape[0], 2 * width + 64), 7.0, dtype=dtype, device=DEV)
    mine, out = (both[:, :width], both[:, width:2 * width]) if q_first else (both[:, width:2 * width], both[:, :width])
    mine.copy_(step.q)
    step.q = mine
    step.check(status, out)
    assert bool((both[:, 2 * width:] == 7.0).all())
    with pytest.raises(kernels.KernelError, match="q and out share memory"):
        step.run(status, both[:, 64:64 + width])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_later_tokens_do_not_reach_earlier_ones(dtype, status):
    """Non-finite keys and values of a request's later tokens leave its earlier tokens, and all other requests, as they were."""
    step = Step(14, 2, 64, dtype, 16, [0] * 4, [20], [5, 9, 0, 30], [6, 1, 20, 3], seed=7)
    before = step.run(status)
    for r, first in ((0, 3), (2, 17)):                    # from this token of the request on
        for i in range(first, int(step.q_start[r + 1] - step.q_start[r])):
            position = step.contexts[r] - int(step.q_start[r + 1] - step.q_start[r]) + i
            page, row = step.pages[r][position // 16], position % 16
            step.v[page, :, row] = float("inf") if i % 2 else float("nan")
            step.k[page, :, row] = float("nan")
    after = step.run(status)
    touched = torch.zeros(step.q.shape[0], dtype=torch.bool, device=DEV)
    touched[3:6] = True
    touched[int(step.q_start[2]) + 17:int(step.q_start[3])] = True
    assert torch.equal(after[~touched], before[~touched]) and bool(after[touched].isnan().any())


def test_nan_in_a_seen_key_is_not_lost(status):
    """A NaN in a key or value that a row sees makes the row NaN, wherever in a tile it lies: a shared key every row, an own key its request's."""
    step = Step(28, 4, 128, BF16, 16, [0] * 24, [600], [30] * 24, [1] * 24, seed=15)
    assert step.plan().host.matrix_items > 0
    for key in range(0, 64):
        saved = step.k[step.pages[0][key // 16], 1, key % 16, 5].clone()
        step.k[step.pages[0][key // 16], 1, key % 16, 5] = float("nan")
        out = step.run(status).view(24, 28, 128)
        step.k[step.pages[0][key // 16], 1, key % 16, 5] = saved
        assert bool(out[:, 7:14].isnan().all()) and not bool(out[:, :7].isnan().any()) and not bool(out[:, 14:].isnan().any())
    step.v[step.pages[3][601], 0, 3, 9] = float("nan")
    out = step.run(status).view(24, 28, 128)
    assert bool(out[3, :7, 9].isnan().all()) and int(out.isnan().sum()) == 7


@pytest.mark.parametrize("page", [8, 16, 32])
@pytest.mark.parametrize("dtype,ways", [(BF16, (0, 1)), (BF16, (2, 2)), (BF16, (1, 1)), (F32, (1, 1))])
def test_an_infinite_value_stays_one(page, dtype, ways, monkeypatch, status):
    """An infinity among the values that a row sees makes the column infinite, as the definition has it, where a range ends inside a tile and
    where a page lies outside the pool: what an earlier tile left in shared memory there does not come into it."""
    import sprout_lm_b200.prefix_plan as prefix_plan
    monkeypatch.setattr(prefix_plan, "choose_kinds", lambda rows, steps, whole, *rest: np.where(rows <= 16, 1, np.where(whole, *ways)))
    monkeypatch.setattr(prefix_plan, "divide", lambda tiles, steps, *rest: (np.ones_like(steps), 0.0))       # one range: ten tiles of 64 keys
    step = Step(28, 4, 128, dtype, page, [0] * 24, [(9 * 64 + page) // page], [30] * 24, [1] * 24, seed=19)
    if dtype == BF16:
        assert (step.plan().host.matrix_items > 0) == (ways[0] == 0)
    for tile in range(9):
        for g, sign in ((1, 1.0), (2, -1.0)):
            key = tile * 64 + 63                          # a row that no copy fills in the last tile
            step.v[step.pages[0][key // page], g, key % page, 40 + g] = sign * float("inf")
    out, (want, tol) = step.run(status).double(), step.exact()
    infinite = want.isinf()
    assert int(infinite.sum()) == 24 * 7 * 2 and bool((out[infinite] == want[infinite]).all())
    assert bool(((out - want).abs()[~infinite] <= tol[~infinite]).all()) and int(status.item()) == 0
    step.tables[:, (6 * 64 + 63) // page] = step.k.shape[0]
    step.block_table.copy_(torch.from_numpy(step.tables))
    out = step.run(status).double()
    assert bool((out[infinite] == want[infinite]).all()) and bool(out[~infinite].isfinite().all()) and int(status.item()) == 1


def test_large_scores(status):
    """Scores of hundreds either way: the running maximum carries them."""
    step = Step(14, 2, 64, BF16, 16, [0] * 6, [40], [5, 9, 0, 30, 200, 77], [1] * 6, seed=8, sharp=60.0)
    step.check(status)


def test_same_results_every_time(status):
    step = Step(28, 4, 128, BF16, 16, [0] * 40, [80], [30] * 40, [2] * 40, seed=9)
    plan = step.plan()
    first = step.run(status, plan=plan)
    for _ in range(5):
        assert torch.equal(step.run(status, plan=plan), first)


def test_offsets_beyond_32_bits(status):
    """Pages at the end of a pool of more than 2^31 elements."""
    pool = (1 << 31) // (4 * 16 * 128) + 4096
    step = Step(28, 4, 128, BF16, 16, [0] * 6, [40], [5, 9, 0, 30, 200, 77], [1, 1, 2, 1, 1, 1], seed=10, pool=pool)
    assert int(step.tables.max()) * 4 * 16 * 128 > 1 << 31
    step.check(status)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bad_pages_are_flagged(dtype, status):
    """Pages outside the pool are left out and set a status bit: a shared one, a request's own, and all of a request's."""
    step = Step(14, 2, 64, dtype, 16, [0] * 4, [30], [50, 90, 0, 30], [1, 2, 1, 1], seed=11)
    step.tables[:, 3] = step.k.shape[0]
    step.tables[1, 31] = -5
    step.block_table.copy_(torch.from_numpy(step.tables))
    out = step.run(status)
    assert int(status.item()) == 1 and bool(out.isfinite().all())
    status.zero_()
    step.tables[:] = 1 << 30
    step.block_table.copy_(torch.from_numpy(step.tables))
    assert bool((step.run(status) == 0).all()) and int(status.item()) == 1


def test_another_steps_plan_is_flagged(status):
    step = Step(14, 2, 64, BF16, 16, [0] * 4, [30], [50, 90, 0, 30], [1, 2, 1, 1], seed=12)
    plan = step.plan()
    step.positions += 1
    step.run(status, plan=plan)
    assert int(status.item()) == 16


def test_captured_and_on_another_stream(status):
    """A captured call replayed with other contents, two captures side by side, a call on a stream of its own: what eager calls give."""
    steps = [Step(28, 4, 128, BF16, 16, [0] * 9, [50], list(range(0, 90, 10)), [3] * 9, seed=s) for s in (21, 22)]
    eager = [s.run(status) for s in steps]
    held, plan = steps[0], steps[0].plan()
    graphs = []
    torch.cuda.synchronize()
    for _ in range(2):
        graph, out = torch.cuda.CUDAGraph(), torch.empty_like(held.q)
        with torch.cuda.graph(graph):
            held.run(status, out=out, plan=plan)
        graphs.append((graph, out))
    for step, want in zip(steps, eager):
        for name in ("q", "k", "v", "block_table", "positions"):
            getattr(held, name).copy_(getattr(step, name))
        for graph, _ in graphs:
            graph.replay()
        assert all(torch.equal(out, want) for _, out in graphs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = held.run(status, plan=plan)
    side.synchronize()
    assert torch.equal(again, eager[-1]) and int(status.item()) == 0


def test_launches_one_behind_the_other(status):
    """Without programmatic dependent launch the items' launches follow one another; the results are the same bits."""
    from sprout_lm_b200 import kernels
    step = Step(28, 4, 128, BF16, 16, [0] * 30, [600], list(range(0, 600, 20)), [1, 2, 3] * 10, seed=14)
    plan = step.plan()
    assert plan.host.matrix_items > 0 and plan.host.narrow_items > 0
    want = step.run(status, plan=plan)
    try:
        kernels.set_pdl(False)
        assert torch.equal(step.run(status, plan=plan), want)
    finally:
        kernels.set_pdl(True)
    step.check(status)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_a_chain_of_calls_each_reading_the_one_before(dtype, status):
    """Each call's queries are the outputs of the call before, in scratch that all of them share, whatever was in it: the same bits as launches
    that follow one another.  The gate between a call's launches is shut behind each."""
    from sprout_lm_b200 import kernels
    step = Step(14, 2, 64, dtype, 16, [0] * 30, [200], list(range(0, 600, 20)), [1, 2, 3] * 10, seed=20)
    plan = step.plan()
    assert dtype == F32 or plan.host.matrix_items > 0 and plan.host.narrow_items > 0
    scratch = torch.full((plan.scratch_floats,), float("nan"), device=DEV)

    def chain():
        outs, q = [torch.empty_like(step.q) for _ in range(25)], step.q
        for out in outs:
            kernels.attention_shared_prefix(q, step.k, step.v, step.block_table, step.positions, plan, out, status, scratch)
            q = out
        return outs

    try:
        kernels.set_pdl(False)
        want = chain()
    finally:
        kernels.set_pdl(True)
    for _ in range(4):
        assert all(torch.equal(a, b) for a, b in zip(chain(), want))
        assert scratch[-2:].tolist() == [0.0, 0.0]
    assert int(status.item()) == 0


def test_two_calls_at_once(status):
    """Calls of one plan on two streams, each with scratch of its own, while a third runs on the current one."""
    step = Step(28, 4, 128, BF16, 16, [0] * 20, [300], list(range(0, 400, 20)), [1] * 20, seed=16)
    plan = step.plan()
    want = step.run(status, plan=plan)
    torch.cuda.synchronize()
    outs = []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(4):
        for stream in streams:
            with torch.cuda.stream(stream):
                outs.append(step.run(status, plan=plan))
        outs.append(step.run(status, plan=plan))
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs) and int(status.item()) == 0


def test_a_plan_let_go_while_another_stream_reads_it(status):
    """The plan's memory is not given to others before a call on another stream than its own is done, whoever held it last."""
    step = Step(28, 4, 128, BF16, 16, [0] * 20, [300], list(range(0, 400, 20)), [1] * 20, seed=16)
    want = step.run(status)
    side, scratch = torch.cuda.Stream(), torch.empty(step.plan().scratch_floats, device=DEV)
    from sprout_lm_b200 import kernels
    for _ in range(3):
        plan, out = step.plan(), torch.full_like(step.q, float("nan"))
        size, at = plan.buffer.numel(), plan.buffer.data_ptr()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            torch.cuda._sleep(100_000_000)               # fifty milliseconds or so
            kernels.attention_shared_prefix(step.q, step.k, step.v, step.block_table, step.positions, plan, out, status, scratch)
        del plan
        held = [torch.zeros(size, dtype=torch.int32, device=DEV) for _ in range(20)]      # what the allocator has to give of that size
        assert side.query() or at not in [t.data_ptr() for t in held]
        side.synchronize()
        assert torch.equal(out, want) and int(status.item()) == 0
        del held


@pytest.mark.parametrize("shape", [(128, 1, 64), (64, 1, 128), (17, 1, 16)])
def test_many_query_heads_a_key_value_head(shape, status):
    """More query rows a token than an item of few rows holds."""
    Step(*shape, BF16, 16, [0] * 5, [30], [5, 70, 0, 33, 200], [1, 3, 1, 2, 1], seed=17).check(status)


def test_every_kind_of_item(status):
    """Each kind alone and all of them in one call, whatever the plan's model would pick."""
    import sprout_lm_b200.prefix_plan as prefix_plan
    step = Step(14, 2, 64, BF16, 16, [0] * 20, [100], [7 * i for i in range(20)], [1 + i % 6 for i in range(20)], seed=18)
    want, tol = step.exact()
    pick, seen = prefix_plan.choose_kinds, set()
    try:
        for ways in ((1, 1), (2, 2), (0, 1), (0, 2)):
            prefix_plan.choose_kinds = lambda rows, steps, whole, *rest, ways=ways: np.where(rows <= 16, 1, np.where(whole, *ways))
            plan = step.plan()
            seen.add((plan.host.matrix_items > 0, plan.host.narrow_items > 0, plan.host.wide_items > 0))
            assert bool(((step.run(status, plan=plan).double() - want).abs() <= tol).all())
    finally:
        prefix_plan.choose_kinds = pick
    assert seen == {(False, True, False), (False, True, True), (True, True, False), (True, True, True)}


def test_refusals(status):
    from sprout_lm_b200 import kernels
    step = Step(14, 2, 64, BF16, 16, [0] * 3, [10], [5, 9, 0], [1, 2, 1], seed=13)
    plan, out = step.plan(), torch.empty_like(step.q)

    def refused(match, **changes):
        given = dict(q=step.q, k_cache=step.k, v_cache=step.v, block_table=step.block_table, positions=step.positions, plan=plan, out=out, status=status)
        given.update(changes)
        with pytest.raises(kernels.KernelError, match=match):
            kernels.attention_shared_prefix(**given)

    refused("CUDA tensor", q=step.q.cpu())
    refused("the plan's tokens", q=step.q[:2])
    refused("the plan's tokens", out=out[:, :64])
    refused("the plan's type", q=step.q.float())
    refused("the plan's type", k_cache=step.k.float(), v_cache=step.v.float())
    refused("the plan's sizes", k_cache=step.k[:, :, :8].contiguous(), v_cache=step.v[:, :, :8].contiguous())
    refused("caches must be contiguous", v_cache=step.v[:3])
    refused("caches must be contiguous", k_cache=step.k.transpose(2, 3).contiguous().transpose(2, 3), v_cache=step.v)
    refused("block_table must hold", block_table=step.block_table[:2])
    refused("block_table must hold", block_table=step.block_table[:, :5])
    refused("must be torch.int32", block_table=step.block_table.long())
    refused("positions must be", positions=step.positions.long())
    refused("positions must be", positions=step.positions[:2])
    refused("share memory", out=step.q)
    refused("scratch must be", scratch=torch.empty(10, device=DEV))
    refused("unit inner stride", q=step.q.t())
    refused("16-byte", q=torch.empty(step.q.numel() + 1, dtype=BF16, device=DEV)[1:].view_as(step.q))
    assert int(status.item()) == 0


def test_memory_that_meets_itself_is_refused(status):
    """Rows of the output that share memory, and a given scratch inside another argument: nothing is launched."""
    from sprout_lm_b200 import kernels
    step = Step(14, 2, 64, F32, 16, [0] * 3, [10], [5, 9, 0], [1, 2, 1], seed=13)
    plan, width = step.plan(), 14 * 64
    whole = torch.full((plan.scratch_floats + 8 * width,), 7.0, device=DEV)
    call = lambda q, out, scratch=None: kernels.attention_shared_prefix(q, step.k, step.v, step.block_table, step.positions, plan, out, status, scratch)
    for apart in (0, 64, width - 1):
        with pytest.raises(kernels.KernelError, match="rows share memory"):
            call(step.q, whole.as_strided((4, width), (apart, 1)))
    scratch = whole[:plan.scratch_floats]
    for at in (plan.scratch_floats - 1, 0, plan.scratch_floats // 2):
        with pytest.raises(kernels.KernelError, match="scratch shares memory"):
            call(step.q, whole[at:at + 4 * width].view(4, width), scratch)
        with pytest.raises(kernels.KernelError, match="scratch shares memory"):
            call(whole[at:at + 4 * width].view(4, width), torch.empty_like(step.q), scratch)
    with pytest.raises(kernels.KernelError, match="scratch shares memory"):
        call(step.q, torch.empty_like(step.q), step.k.view(-1)[:plan.scratch_floats])
    assert bool((whole == 7.0).all()) and int(status.item()) == 0
    out = whole[plan.scratch_floats:][:4 * width].view(4, width)
    call(step.q, out, scratch)
    want, tol = step.exact()
    assert bool(((out.double() - want).abs() <= tol).all())


# ---------------------------------------------------------------------------------- plans for later steps

LATER = [(14, 2, 64, BF16, 16), (28, 4, 128, BF16, 16), (14, 2, 64, BF16, 5), (5, 1, 48, BF16, 16), (28, 4, 128, BF16, 128), (6, 3, 40, BF16, 8), (14, 2, 64, F32, 16), (3, 1, 144, BF16, 16)]


def earlier_plan(step, ahead, stretch):
    """The plan that the step's requests would have had `ahead` tokens before, good for `stretch` more."""
    from sprout_lm_b200 import kernels
    contexts = [c - a for c, a in zip(step.contexts, ahead)]
    tables = step.tables.copy()
    for row, c in zip(tables, contexts):
        row[-(-c // step.page):] = -1                     # pages that the requests did not have yet
    tables = tables[:, :-(-max(contexts) // step.page)]
    return kernels.shared_prefix_plan(tables, step.q_start, contexts, step.page, step.heads, step.kv_heads, step.dim, step.dtype, DEV, stretch=stretch)


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,page", LATER)
@pytest.mark.parametrize("tokens", [1, 5, 20])
def test_a_plan_for_later_steps(heads, kv_heads, dim, dtype, page, tokens, status):
    rng = np.random.default_rng(tokens)
    own = [130, 20, 300, 64, 200, 128, 1, 160]
    ahead = [0, 5, 128, 64, 17, 128, 0, 1]
    counts = [int(n) for n in rng.integers(1, tokens + 1, len(own))]
    step = Step(heads, kv_heads, dim, dtype, page, [0] * len(own), [40], own, counts, seed=tokens, table_pad=-(-128 // page))
    plan = earlier_plan(step, ahead, 128)
    out = step.run(status, plan=plan)
    want, tol = step.exact()
    assert int(status.item()) == 0
    assert bool(((out.double() - want).abs() <= tol).all())


@pytest.mark.parametrize("requests,prefix", [(20, 130), (48, 400)])
def test_a_captured_step_replayed_for_later_ones(requests, prefix, status):
    """One capture for decode steps 0 to 70 positions behind its plan: items of few rows and, over the prefix, matrix items."""
    from sprout_lm_b200 import kernels
    rng = np.random.default_rng(requests)
    own = [70 + int(n) for n in rng.integers(0, 200, requests)]
    last = Step(28, 4, 128, BF16, 16, [0] * requests, [prefix], own, [1] * requests, seed=7, table_pad=5)
    plan, out, scratch = earlier_plan(last, [70] * requests, 70), torch.empty_like(last.q), None
    assert plan.host.matrix_items > 0 and plan.host.narrow_items > 0
    scratch = torch.empty(plan.scratch_floats, device=DEV)
    positions = last.positions.clone()
    last.positions -= 70
    call = lambda: kernels.attention_shared_prefix(last.q, last.k, last.v, last.block_table, last.positions, plan, out, status, scratch)
    call()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call()
    for behind in (70, 69, 41, 0, 13):
        last.positions.copy_(positions - behind)
        out.fill_(float("nan"))
        graph.replay()
        want, tol = last.exact()
        assert bool(((out.double() - want).abs() <= tol).all()), behind
    assert int(status.item()) == 0


@pytest.mark.parametrize("heads,kv_heads,dim,dtype,page", LATER[:4])
@pytest.mark.parametrize("off", [-1, 129])
def test_a_step_that_the_plan_does_not_serve(heads, kv_heads, dim, dtype, page, off, status):
    """Further back than the plan's own, or beyond its stretch: a status bit, and the other requests' rows are as they should be."""
    own = [300, 310, 320]
    step = Step(heads, kv_heads, dim, dtype, page, [0, 0, 0], [40], own, [1, 1, 1], seed=3, table_pad=-(-200 // page))
    plan = earlier_plan(step, [100, 129 if off > 0 else 0, 128], 128)
    if off < 0:
        step.positions[1] -= 1
    out = step.run(status, plan=plan)
    assert int(status.item()) == 16
    want, tol = step.exact()
    keep = torch.tensor([0, 2], device=DEV)
    assert bool(((out.double() - want).abs() <= tol)[keep].all()) and bool(torch.isfinite(out).all())
