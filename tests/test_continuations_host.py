"""The host side of steps whose sequences share pages, without a GPU."""
import random

import pytest

pytest.importorskip("torch")

from llm_accelerator_b200 import paged  # noqa: E402


def users(held, n=64, more=()):
    count = [0] * n
    for pages in list(held) + list(more):
        for p in pages:
            count[p] += 1
    return count


@pytest.mark.parametrize("held,more,runs", [
    ([], (), []),
    ([[]], (), [(1, 0)]),
    ([[], []], (), [(1, 0), (1, 0)]),
    ([[1, 2], [3]], (), [(1, 0), (1, 0)]),
    ([[1, 2, 3], [1, 2, 4]], (), [(2, 2)]),
    ([[1, 2, 3], [1, 2, 4], [1, 5]], (), [(3, 1)]),
    ([[1, 5], [1, 2, 3], [1, 2, 4]], (), [(3, 1)]),
    ([[1, 2, 3], [9], [1, 2, 4]], (), [(1, 0), (1, 0), (1, 0)]),
    ([[1, 2], [1, 2], [7, 8, 9], [7, 8, 10]], (), [(2, 2), (2, 2)]),
    ([[1, 2, 3, 4], [1, 2]], ([1, 2, 3],), [(2, 2)]),      # a third page is shared with one that is not in the step
    ([[1, 2, 3]], ([1, 2],), [(1, 0)]),
    ([[1, 2], [], [1, 2]], (), [(1, 0), (1, 0), (1, 0)]),
])
def test_runs(held, more, runs):
    assert paged.shared_runs(held, users(held, more=more)) == runs


def test_runs_of_random_forks():
    rng = random.Random(0)
    for _ in range(300):
        trunk, free = [], iter(range(1000))
        held = []
        for _ in range(rng.randint(1, 4)):
            trunk = [next(free) for _ in range(rng.randint(0, 5))]
            for _ in range(rng.randint(1, 4)):
                held.append(trunk[:rng.randint(0, len(trunk))] + [next(free) for _ in range(rng.randint(0, 3))])
        got = paged.shared_runs(held, users(held, 1000))
        assert sum(n for n, _ in got) == len(held)
        at = 0
        for n, pages in got:
            group = held[at:at + n]
            assert all(g[:pages] == group[0][:pages] and len(g) >= pages for g in group)
            # no longer one is shared by all of them
            assert n == 1 or len({tuple(g[:pages + 1]) for g in group if len(g) > pages}) > 1 or \
                any(len(g) == pages for g in group)
            at += n
