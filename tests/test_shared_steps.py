"""When a step takes a plan of shared pages, and the numbers that check drafted tokens (host only)."""
import random

import numpy as np
import pytest

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


def test_engine_option_is_a_boolean():
    from sprout_lm_b200 import EngineOptions
    EngineOptions(shared_prefix=True).validate()
    with pytest.raises(ValueError, match="shared_prefix must be a boolean"):
        EngineOptions(shared_prefix=1).validate()
