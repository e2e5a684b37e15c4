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
            groups.setdefault(int(tables[request[member], depth]) if whole[member] > depth else -1 - int(member), []).append(member)
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
            same = (rows == rows[0]).all(axis=0)
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
    the launches finds shortest.  Its constants are microseconds on a B200 at head size 64 and 128: a CTA's time for a step of 128 keys,
    what it takes beside, and the partial results' way through memory.  Measured, head size 128: 20 requests over 16,384 keys
    (28 heads over 4) as 0, 1, 2: 23.1, 48.4, 40.3 us; 24 of 4 tokens over 2,000: 26.4, 40.3, 33.4; 6 over 30,000 (40 over 8): -, 42.8,
    56.0; head size 64 (14 over 2): 64 over 1,024: 12.0, 9.7, 11.3; 90 pairs of tokens over 1,000: 20.4, 17.6, 16.8."""
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
            cost = 0.0
            for which, tile, places, beside, step in ((0, MATRIX_ROWS, matrix_slots, 6.5 if wide_head else 7.5, 2.0 if wide_head else 1.4), (2, WIDE_ROWS, slots, 3.5, 7.5 if wide_head else 3.5),
                                                      (1, NARROW_ROWS, narrow_slots, 2.0, 2.7 if wide_head else 2.2)):
                of = kind == which
                if not of.any():
                    continue
                tiles = -(-rows[of] // tile) * kv_heads
                share = float((tiles * steps[of]).sum()) / places
                length = max(1.0, share)
                time = beside + step * (length + 0.75 if which == 1 else np.ceil(length))      # items of few rows are walked: some CTA has more
                if which == 0:
                    ctas = float((tiles * -(-steps[of] // np.ceil(length))).sum())
                    alone, free = time, max(0.0, 1.0 - ctas / places)
                elif matrix and free > 0:                # on the SMs that the matrix items leave, or behind them
                    time = min(time, max(0.0, beside + step * (max(1.0, share / free) + 0.75) - alone))
                cost += 1.0 + time
                cost += float((rows[of] * -(-steps[of] // np.ceil(length))).sum()) * kv_heads * head_dim * 8 / 6e6
            if best is None or cost < best[0]:
                best = cost, kind
    return best[1]


def divide(tiles: np.ndarray, steps: np.ndarray, kv_heads: int, slots: int, start: float, step: float) -> np.ndarray:
    """Into how many ranges each segment's keys go (``steps`` key steps, ``tiles`` tiles of rows), on a device that runs ``slots`` items at
    once, an item of n steps taking ``start + n * step``: ranges of the length that makes the fewest full rounds of items the shortest."""
    if not len(tiles):
        return steps
    items = lambda n: int((tiles * np.minimum(-(-steps // n), MAX_RANGES)).sum()) * kv_heads
    best = None
    for rounds in range(1, 9):
        low, high = 1, int(steps.max())                  # the shortest ranges whose items fit that many rounds
        if items(high) > rounds * slots:
            continue
        while low < high:
            middle = (low + high) // 2
            if items(middle) <= rounds * slots:
                high = middle
            else:
                low = middle + 1
        cost = -(-items(low) // slots) * (start + low * step)
        if best is None or cost < best[0]:
            best = cost, low
        if low == 1:
            break
    # more segments than eight rounds hold: an even share of the steps
    length = best[1] if best is not None else max(1, -(-int((tiles * steps).sum()) * kv_heads // (8 * slots)))
    return np.minimum(-(-steps // length), MAX_RANGES)


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
        ranges[matrix] = divide(tiles[matrix], steps[matrix], kv_heads, max(1, matrix_slots), 7.0, 2.4)
        if tensor_cores:
            wide, narrow = kind == 2, kind == 1
            ranges[wide] = divide(tiles[wide], steps[wide], kv_heads, slots, 4.0, 1.5)
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
            ranges[:] = divide(tiles, steps, kv_heads, slots, 4.0, 1.5)
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
