"""The largest block counts a shared-prefix plan takes, and those it refuses, on the host."""

import pytest

from tests.test_shared_prefix_host import check_covers, lib, plan_of  # noqa: F401

MOST = 2 ** 27 - 1  # blocks of 16 keys, the keys counted in 31 bits


@pytest.mark.parametrize("n", [MOST + 1, 2 ** 31 - 8, 2 ** 31 - 1])
def test_counts_past_31_bits_of_keys_are_refused(lib, n):  # noqa: F811
    for groups, prefix, rows in (([[0, 1]], [n], [n, n, 4]), ([[0, 1]], [n - 5], [n, n, 4]),
                                 ([], [], [4, n, 4]), ([[0, 2]], [3], [4, n, 4])):
        with pytest.raises(ValueError, match="row_blocks past"):
            plan_of(groups, prefix, rows)
    with pytest.raises(ValueError, match="fewer blocks"):
        plan_of([[0, 1]], [n], [4, 4, 4])


@pytest.mark.parametrize("full", [False, True])
def test_the_largest_counts_are_divided(lib, full):  # noqa: F811
    groups, prefix, rows = [[0, 1], [2, 3]], [MOST, MOST - 9], [MOST] * 4 + [MOST, 0]
    check_covers(plan_of(groups, prefix, rows, full_grid=full), groups, prefix, rows)
