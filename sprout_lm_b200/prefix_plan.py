"""How attention divides the keys of a step whose requests hold the same leading pages (host only; csrc/attention_prefix.cuh says what
the kernels make of it).

The step's tokens are taken in *members*: up to ``MEMBER_TOKENS`` tokens of one request.  Members' block tables are a trie over pages:
a run of pages that several members hold is a *segment* read once for all of them; what lies behind its last shared run is a member's own
segment.  Runs may branch: all requests share a system prompt, some of them a document behind it.  Only keys that all of a member's tokens
see are divided this way; what its later tokens see of one another is added where the parts are put together.

A segment's rows (its tokens times the query heads of a key/value head) are cut into tiles and its keys into ranges, so that the tiles'
ranges, the *items*, fill the device once.  Everything is arrays: a plan is made once a step and serves all layers.
"""
from __future__ import annotations

import numpy as np

MEMBER_TOKENS = 16          # attention_prefix.cuh: MEMBER_TOKENS
KEY_STEP = 128              # keys that a CTA takes at a time: ranges are whole steps
NARROW_ROWS, WIDE_ROWS, SIMPLE_ROWS, MATRIX_ROWS = 16, 64, 16, 256      # rows of an item of each kind
MATRIX_FROM = 48            # rows of a segment
MATRIX_US, MATRIX_STEP_US, NARROW_STEP_US = 8.0, 2.0, 2.0      # of items beside one another: a matrix item's start and step, a step of few rows
# Microseconds on a B200 by kind (0: matrix, 2: 64 rows), at head sizes up to 64 and above: an item's start and its step of 128 keys, what a
# launch takes beside; the step of a walk over items of few rows; a row's partial result, written and put together, and the chain of
# reads that a part of a row adds.  Fitted to launches of 60 batches in ten forms each (kinds, ranges of 1 to 12 steps); over 35 others the
# form that they choose takes 1 to 2 % more than the best of the ten.
KIND_US = {0: ((0.6, 2.2), (2.5, 2.6)), 2: ((0.0, 5.0), (0.0, 7.5))}
BESIDE_US = {0: (2.0, 0.5), 2: (1.0, 1.0)}
WALK_US = 2.2
PART_US, DEPTH_US = 2.6e-4, 0.05
ITEM_STEPS = 0.5            # what an item of few rows costs beside its steps
MAX_RANGES = 64             # of a segment
MAX_STRETCH = 1024          # positions that a plan's steps may be behind its own: its items are sized for its own
# A shared run is a segment of its own if reading it once saves this many key reads (a member fewer than hold it, times its keys): below,
# the members read it themselves.
MIN_SAVED_KEYS = 64
PART_KEYS = 2               # and more than its rows' partial results cost: float32 written and read, the bytes of two bfloat16 keys and values a row


class PlanError(ValueError):
    pass


class Segment:
    """Keys ``key_begin`` to ``key_end`` of the pages in block table row ``table``, seen by the places ``token_begin`` to ``token_end`` of the
    plan's order; ``part``: the first of its partial results at each of these places (``ranges`` of them); ``own``: one member's, what it
    sees behind its last shared run."""
    __slots__ = ("table", "key_begin", "key_end", "token_begin", "token_end", "part", "ranges", "own")

    def __init__(self, table, key_begin, key_end, token_begin=0, token_end=0, own=False):
        self.table, self.key_begin, self.key_end, self.token_begin, self.token_end = table, key_begin, key_end, token_begin, token_end
        self.part, self.ranges, self.own = 0, 1, own


def find_segments(tables: np.ndarray, q_start: np.ndarray, contexts: np.ndarray, page_tokens: int, group: int = 1):
    """(segments, order, seen, extra, table_of): the trie's segments, parents before their children; per place of the plan's order the
    step's token there, the keys that its member's tokens all see, the further ones that it sees itself, and its request.  The
    parent of a segment is in ``parents`` of the result (-1: none).  ``group``: query heads of a key/value head."""
    counts = np.diff(q_start)
    # members: request, first token, tokens, keys that all of them see
    blocks = -(-counts // MEMBER_TOKENS)
    request = np.repeat(np.arange(len(counts)), blocks)
    offset = (np.arange(len(request)) - np.repeat(np.cumsum(blocks) - blocks, blocks)) * MEMBER_TOKENS
    tokens = np.minimum(MEMBER_TOKENS, counts[request] - offset)
    first = q_start[request] + offset
    sees = contexts[request] - counts[request] + offset + 1
    whole = np.minimum(sees, contexts[request] - counts[request]) // page_tokens       # full pages of earlier steps: what may be shared
    segments, parents, leaves = [], [], []               # leaves: members in the plan's order
    placed = 0
    # Work that is left, the next last: members that hold the same pages up to ``depth``, of which those from ``start`` on are in no
    # segment yet; or a segment whose members are all placed.
    left = []

    def branch(members, start, depth, parent):
        groups = {}
        for member in members:
            page = int(tables[request[member], depth]) if whole[member] > depth else -1
            # by itself, under a key that is no page: it has no full page here, or one outside the pool (which the kernels skip and flag)
            groups.setdefault(page if page >= 0 else -1 - int(member), []).append(member)
        left.extend((group, start, depth, parent) for group in reversed(groups.values()))

    branch(np.arange(len(request)), 0, 0, -1)
    while left:
        members, start, depth, parent = left.pop()
        if members is None:
            segments[parent].token_end = placed
        elif len(members) == 1:
            member = members[0]
            # never empty: what is shared ends before the step's own tokens
            segments.append(Segment(int(request[member]), int(start) * page_tokens, int(sees[member]), placed, placed + int(tokens[member]), own=True))
            parents.append(parent)
            leaves.append(member)
            placed += int(tokens[member])
        else:
            members = np.asarray(members)
            rows = tables[request[members], depth:int(whole[members].min())]
            same = (rows == rows[0]).all(axis=0) & (rows[0] >= 0)
            end = depth + (int(same.argmin()) if not same.all() else rows.shape[1])
            if (len(members) - 1) * (end - start) * page_tokens >= max(MIN_SAVED_KEYS, PART_KEYS * group * int(tokens[members].sum())):
                segments.append(Segment(int(request[members[0]]), start * page_tokens, end * page_tokens, placed))
                parents.append(parent)
                parent, start = len(segments) - 1, end
                left.append((None, 0, 0, parent))
            branch(members, start, end, parent)
    leaves = np.asarray(leaves)
    lengths = tokens[leaves]
    within = np.arange(placed) - np.repeat(np.cumsum(lengths) - lengths, lengths)
    return segments, parents, np.repeat(first[leaves], lengths) + within, np.repeat(sees[leaves], lengths), within, np.repeat(request[leaves], lengths)


def choose_kinds(rows, steps, whole, kv_heads: int, head_dim: int, slots: int, matrix_slots: int, narrow_slots: int) -> np.ndarray:
    """The kind of every segment: 0 where ``whole`` allows it (tiles of 256 rows on tcgen05), 1 (tiles of 16 rows) or 2 (of 64).  Segments of
    up to 16 rows are 1; of the four ways for the rest (0 or not where it may be, and 1 or 2 for all others) the one that a rough model of
    the launches finds shortest.  Measured, head size 128 as 0, 2, 1: 24 requests of up to 6 tokens over 2,000 keys (28 heads over 4) 21.7, 28.5,
    36.5 us; 14 of 2 over two prompts of 5,000 (40 over 8) 18.8, 18.5, 20.9; 42 over six of 6,800 50, 61, 54; head size 64 (14 over 2): 64
    over 4,096 15.3, 18.5, 19.7; 90 of 2 over six of 5,000 20.1, 24.0, 30.7; 10 of 5 over 230 12.9, 9.6, 8.4."""
    few = rows <= NARROW_ROWS
    if few.all():
        return np.ones(len(rows), dtype=np.int64)
    wide_head = head_dim > 64
    best = None
    for matrix in ((True, False) if whole.any() else (False,)):
        for others in (1, 2):
            kind = np.where(few, 1, others)
            if matrix:
                kind[whole] = 0
            cost, walk = 0.0, walk_us(rows, steps, kind, kv_heads, narrow_slots)
            for which, tile, places in ((0, MATRIX_ROWS, matrix_slots), (2, WIDE_ROWS, slots)):
                of = kind == which
                if of.any():
                    time = divide(-(-rows[of] // tile), steps[of], rows[of], kv_heads, places, *KIND_US[which][wide_head], walk if which == 0 else None)[1]
                    if which == 0:
                        walk = None                          # beside or behind the matrix items, and counted with them
                    elif walk is not None:                   # among the others
                        time += max(0.0, walk[0] - 0.5 * time)
                        walk = None
                    cost += BESIDE_US[which][wide_head] + time
            if walk is not None:
                cost += walk[0]
            if best is None or cost < best[0]:
                best = cost, kind
    return best[1]


def walk_us(rows, steps, kind, kv_heads: int, narrow_slots: int):
    """What the items of few rows take with the device to themselves, and a function of the share of it that they have; None without any."""
    of = kind == 1
    if not of.any():
        return None
    share = float((-(-rows[of] // NARROW_ROWS) * kv_heads * steps[of]).sum()) / narrow_slots
    parts = float((rows[of] * -(-steps[of] // np.ceil(max(1.0, share)))).sum()) * kv_heads * PART_US
    time = lambda free: WALK_US * np.maximum(1.5, share / free + 1.25) + parts       # some CTA has more than its share
    return time(1.0), time


def divide(tiles: np.ndarray, steps: np.ndarray, rows: np.ndarray, kv_heads: int, slots: int, start: float, step: float, walk=None):
    """Into how many ranges each segment's keys go (``steps`` key steps, ``tiles`` tiles of ``rows`` rows), on a device that runs ``slots`` items
    at once, an item of n steps taking ``start + n * step``, and the time that takes: the rounds of items, what their partial results cost,
    and what ``walk`` (``walk_us``) takes behind them, or beside them where they leave room."""
    if not len(tiles):
        return steps, 0.0
    most = int(steps.max())
    lengths = np.unique(-(-most // np.arange(1, min(most, MAX_RANGES) + 1)))[:, None]
    ranges = np.minimum(-(-steps // lengths), MAX_RANGES)
    items = (tiles * ranges).sum(1) * kv_heads
    time = -(-items // slots) * (start + step * (-(-steps // ranges)).max(1))
    total = time + (rows * ranges).sum(1) * kv_heads * PART_US + np.minimum(ranges.max(1), 24) * DEPTH_US
    if walk is not None:
        free = np.maximum(1e-9, 1.0 - items / slots)
        total += np.minimum(walk[0], np.maximum(0.0, walk[1](free) - time))
    best = int(total.argmin())
    return ranges[best], float(total[best])


def spread(tiles: np.ndarray, steps: np.ndarray, kv_heads: int, slots: int) -> np.ndarray:
    """The same for items that ``slots`` CTAs walk, each taking one of every ``slots`` of them, longest first, forwards and backwards in
    turn: ranges of the length with which the CTA that has most to do has least (an item costs ``ITEM_STEPS`` steps beside its own), and
    how much that is."""
    if not len(tiles):
        return steps, 0.0

    def busiest(length):
        ranges = np.minimum(-(-steps // length), MAX_RANGES)
        each = -(-steps // ranges)
        items = np.repeat(np.concatenate([each, steps - each * (ranges - 1)]), np.concatenate([tiles * (ranges - 1), tiles]) * kv_heads)
        rounds = -(-len(items) // slots)
        loads = np.zeros(rounds * slots)
        loads[:len(items)] = np.sort(items)[::-1] + ITEM_STEPS
        loads = loads.reshape(rounds, slots)
        loads[1::2] = loads[1::2, ::-1]
        return loads.sum(0).max()

    share = int((tiles * steps).sum()) * kv_heads / slots
    count = lambda n: int((tiles * np.minimum(-(-steps // n), MAX_RANGES)).sum()) * kv_heads
    lengths = {int(steps.max())} | {max(1, -(-int(share * 16) // k)) for k in (8, 12, 16, 24, 32, 48, 64)}
    low, high = 1, int(steps.max())                      # and the shortest ranges that are one round
    if count(high) <= slots:
        while low < high:
            middle = (low + high) // 2
            low, high = (low, middle) if count(middle) <= slots else (middle + 1, high)
        lengths.add(low)
    most, best = min((busiest(n), -n) for n in lengths)
    return np.minimum(-(-steps // -best), MAX_RANGES), float(most)


class HostPlan:
    """The plan's arrays on the host, for a step and for those of the same requests and numbers of tokens up to ``stretch`` positions behind
    it: ``items`` [n, 8] (simple ones, or matrix, narrow and wide ones), ``order``, ``part_start``, ``seen``,
    ``extra``, ``table_of``."""

    def __init__(self, tables, q_start, contexts, page_tokens: int, heads: int, kv_heads: int, tensor_cores: bool, slots: int, matrix_slots: int = 0, narrow_slots: int | None = None, head_dim: int = 64,
                 stretch: int = 0):
        try:
            tables, q_start, contexts = (np.asarray(a) for a in (tables, q_start, contexts))
        except (TypeError, ValueError) as error:             # ragged rows, or tensors of a device
            raise PlanError(f"tables, starts and contexts are arrays on the host ({error})") from None
        if tables.ndim != 2 or q_start.ndim != 1 or contexts.ndim != 1 or len(contexts) == 0 or len(q_start) != len(contexts) + 1 or len(tables) < len(contexts):
            raise PlanError("a block table row and a context per request, and where each request's tokens start")
        if any(a.dtype.kind not in "iu" for a in (tables, q_start, contexts)):
            raise PlanError("tables, starts and contexts are whole numbers")
        q_start, contexts = q_start.astype(np.int64), contexts.astype(np.int64)
        counts = np.diff(q_start)
        if q_start[0] != 0 or (counts < 1).any() or (contexts < counts).any():
            raise PlanError("every request brings a token or more, and its context holds them")
        if page_tokens < 1 or int(contexts.max()) > tables.shape[1] * page_tokens or int(contexts.max()) > 0x7fffffff - MAX_STRETCH:
            raise PlanError("a context reaches beyond its block table")
        if type(stretch) is not int or not 0 <= stretch <= MAX_STRETCH:
            raise PlanError(f"stretch must be a whole number up to {MAX_STRETCH} (got {stretch!r})")
        if kv_heads < 1 or heads < 1 or heads % kv_heads:
            raise PlanError(f"heads ({heads}) must be a multiple of the key/value heads ({kv_heads})")
        self.narrow_ctas = 0                             # that walk the narrow items
        self.tokens, self.requests = int(q_start[-1]), len(contexts)
        self.stretch, self.pages = stretch, int(-(-(contexts.max() + stretch) // page_tokens))       # pages: of a call's block tables
        group = heads // kv_heads
        segments, parents, order, seen, extra, table_of = find_segments(tables, q_start, contexts, page_tokens, group)
        begin = np.array([s.key_begin for s in segments])
        end = np.array([s.key_end for s in segments])
        token_begin, own = np.array([s.token_begin for s in segments]), np.array([s.own for s in segments])
        rows = (np.array([s.token_end for s in segments]) - token_begin) * group
        # the kinds: 0 a matrix product's worth of rows over whole pages, 1 few rows, 2 more; all of 1 on the CUDA cores
        if tensor_cores:
            whole = (rows >= MATRIX_FROM) & ~(own & (stretch > 0)) & (end % page_tokens == 0) & (begin % page_tokens == 0) if matrix_slots else np.zeros(len(segments), dtype=bool)
            kind = choose_kinds(rows, -(-(end - begin) // KEY_STEP), whole, kv_heads, head_dim, slots, matrix_slots, narrow_slots or slots)
            tile_rows = np.array([MATRIX_ROWS, NARROW_ROWS, WIDE_ROWS])[kind]
        else:
            kind, tile_rows = np.ones(len(segments), dtype=np.int64), np.full(len(segments), SIMPLE_ROWS)
        tiles, steps = -(-rows // tile_rows), -(-(end - begin) // KEY_STEP)
        ranges = np.empty(len(segments), dtype=np.int64)
        matrix = kind == 0
        if tensor_cores:
            ranges[matrix] = divide(tiles[matrix], steps[matrix], rows[matrix], kv_heads, max(1, matrix_slots), *KIND_US[0][head_dim > 64],
                                    walk_us(rows, steps, kind, kv_heads, narrow_slots or slots))[0]
            wide, narrow = kind == 2, kind == 1
            ranges[wide] = divide(tiles[wide], steps[wide], rows[wide], kv_heads, slots, *KIND_US[2][head_dim > 64])[0]
            self.narrow_ctas = narrow_slots or slots
            ranges[narrow], most = spread(tiles[narrow], steps[narrow], kv_heads, self.narrow_ctas)
            ctas = int((tiles[matrix] * ranges[matrix]).sum()) * kv_heads
            if narrow.any() and 0 < ctas < matrix_slots:
                # beside matrix items that leave some SMs: all there, if that is done before both one behind the other would be
                beside = (matrix_slots - ctas) * self.narrow_ctas // matrix_slots
                alone_us = -(-steps[matrix] // ranges[matrix]).max() * MATRIX_STEP_US + MATRIX_US
                apart, there = spread(tiles[narrow], steps[narrow], kv_heads, beside)
                if max(alone_us, there * NARROW_STEP_US) < alone_us + most * NARROW_STEP_US:
                    ranges[narrow], self.narrow_ctas = apart, beside
        else:
            ranges[:] = divide(tiles, steps, rows, kv_heads, slots, 4.0, 1.5)[0]
        per_range = -(-steps // ranges)                  # steps of a range
        ranges = -(-steps // per_range)
        parts = np.zeros(self.tokens, dtype=np.int64)    # of each place
        for i, s in enumerate(segments):
            s.ranges = int(ranges[i])
            s.part = 0 if parents[i] < 0 else segments[parents[i]].part + segments[parents[i]].ranges
            parts[s.token_begin:s.token_end] = s.part + s.ranges
        part = np.array([s.part for s in segments])
        # the items: segment by segment, tile by tile, range by range
        count = tiles * ranges
        of = np.repeat(np.arange(len(segments)), count)
        index = np.arange(len(of)) - np.repeat(np.cumsum(count) - count, count)
        tile, rng = index // ranges[of], index % ranges[of]
        items = np.zeros((len(of), 8), dtype=np.int32)
        items[:, 0] = np.array([s.table for s in segments])[of]
        items[:, 1] = begin[of] + rng * per_range[of] * KEY_STEP
        items[:, 2] = np.minimum(end[of], items[:, 1] + per_range[of] * KEY_STEP)
        items[:, 3] = token_begin[of]
        items[:, 4] = tile * tile_rows[of]
        items[:, 5] = np.minimum(rows[of] - items[:, 4], tile_rows[of])
        items[:, 6] = part[of] + rng
        if stretch:
            items[:, 7] = own[of] & (rng == ranges[of] - 1)                 # a member's last own range grows with the steps
            items[:, 2] += items[:, 7] * stretch
        of_kind = kind[of]
        items = items[np.lexsort((items[:, 1] - items[:, 2], of_kind))]     # longest first within a kind
        counts = np.bincount(of_kind, minlength=3).tolist()
        self.matrix_items, self.wide_items = counts[0], counts[2]
        self.simple_items, self.narrow_items = (0, counts[1]) if tensor_cores else (counts[1], 0)
        self.items, self.segments, self.parents = items, segments, parents
        self.order, self.seen, self.extra, self.table_of = (a.astype(np.int32) for a in (order, seen, extra, table_of))
        self.part_start = np.concatenate([[0], np.cumsum(parts)]).astype(np.int32)
        self.parts = int(self.part_start[-1])
        # keys that the items read, and those that the requests' contexts hold
        self.read_keys, self.context_keys = int((end - begin).sum()), int(contexts.sum())

    def pack(self) -> np.ndarray:
        """All arrays in one of int32, each starting on a multiple of four."""
        arrays = (self.items.reshape(-1), self.order, self.part_start, self.seen, self.extra, self.table_of)
        self.offsets, at = [], 0
        for a in arrays:
            self.offsets.append((at, len(a)))
            at += -(-len(a) // 4) * 4
        packed = np.zeros(at, dtype=np.int32)
        for (where, n), a in zip(self.offsets, arrays):
            packed[where:where + n] = a
        return packed
