"""The grouping of sequences by the pages that they name first."""

import random
import time

import pytest

import microserve_amd as M
from microserve_amd.shared_prefix import MAX_GROUPS


def _saved(tables, groups):
    def common(g):
        a, b = min(tables[i] for i in g), max(tables[i] for i in g)
        return next((j for j, (x, y) in enumerate(zip(a, b)) if x != y), min(len(a), len(b)))
    return sum((len(g) - 1) * common(g) for g in groups)


def _groups(tables, block=16):
    order, cu, prefixes = M.group_by_prefix(tables, block)
    assert sorted(order) == list(range(len(tables)))
    assert cu[0] == 0 and cu[-1] == len(tables) and len(prefixes) == len(cu) - 1
    groups = [order[a:b] for a, b in zip(cu, cu[1:])]
    for g, p in zip(groups, prefixes):
        assert len(g) > 0 and p % block == 0
        for i in g:  # what the group is said to share it shares
            assert tables[i][:p // block] == tables[g[0]][:p // block]
            assert len(tables[i]) >= p // block
    return groups, [p // block for p in prefixes]


def test_an_outsider_does_not_shorten_the_prefix():
    tables = [list(range(32)) + [100 + i] for i in range(8)] + [[0, 77, 78]]
    groups, pages = _groups(tables)
    assert groups == [list(range(8)), [8]] and pages == [32, 0]
    # two such share their one page with one another
    groups, pages = _groups([[0, 90]] + tables)
    assert sorted(map(len, groups)) == [2, 8] and sorted(pages) == [1, 32]
    # and many of them are worth a group of all
    groups, pages = _groups([[0, 1, 50 + i] for i in range(9)] + [[0, 1, 2, 3], [0, 1, 2, 4]])
    assert [len(g) for g in groups] == [11] and pages == [2]


def _partitions(items):
    if not items:
        yield []
        return
    first, rest = items[0], items[1:]
    for part in _partitions(rest):
        yield [[first]] + part
        for i in range(len(part)):
            yield part[:i] + [[first] + part[i]] + part[i + 1:]


@pytest.mark.parametrize("seed", range(60))
def test_no_partition_saves_more(seed):
    rng = random.Random(seed)
    tables = []
    for _ in range(rng.randint(1, 7)):
        if tables and rng.random() < 0.8:
            base = rng.choice(tables)
            tables.append(base[:rng.randint(0, len(base))]
                          + [rng.randint(0, 3) for _ in range(rng.randint(0, 6))])
        else:
            tables.append([rng.randint(0, 2) for _ in range(rng.randint(0, 12))])
    groups, _ = _groups(tables)
    best = max(_saved(tables, p) for p in _partitions(list(range(len(tables)))))
    assert _saved(tables, groups) == best


def test_more_groups_than_a_call_takes():
    lone = [[i] for i in range(1100)]
    groups, pages = _groups(lone)
    assert len(groups) <= MAX_GROUPS and not any(pages)
    # the pairs that share most stay, whatever lies beside them
    pairs = [[5000 + i // 2, *range(i // 2 % 7)] for i in range(2400)]
    groups, pages = _groups(pairs + lone)
    assert len(groups) == MAX_GROUPS and pages[-1] == 0
    assert all(len(g) == 2 and p > 0 for g, p in zip(groups[:-1], pages))
    dropped = {1 + i // 2 % 7 for i in groups[-1] if i < 2400}
    assert max(dropped) <= min(pages[:-1])


def test_nested_prefixes_and_time():
    """A chain of sequences, each longer than the one before, and a large batch."""
    begin = time.time()
    groups, _ = _groups([list(range(n)) for n in range(1500)])
    assert sum(map(len, groups)) == 1500
    prompts = [[1000 * a + j for j in range(32)] for a in range(8)]
    groups, pages = _groups([prompts[i % 8][:8 + i % 25] + [10 ** 6 + i] for i in range(1000)])
    assert len(groups) >= 8 and max(pages) <= 32
    assert time.time() - begin < 20
