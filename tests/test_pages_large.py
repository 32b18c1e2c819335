"""Sharing and moving blocks at the sizes where the calls go round their loops: as many rows as are allowed, and pools of
10^6 blocks. Rules and checks are those of test_pages.py."""
import numpy as np
import pytest

from test_pages import check_compact, check_fork, make_pools, random_rows


@pytest.mark.gpu
@pytest.mark.parametrize("in_place", [True, False])
def test_fork_of_as_many_rows_as_are_allowed(in_place):
    rng, B, MB, bs = np.random.default_rng(1), 8192, 3, 4
    lens = rng.integers(0, MB * bs + 1, size=B)
    NB = int((-(-lens // bs)).sum()) + 5000
    table, left = random_rows(rng, B, MB, bs, NB, lens, share=0.5)
    parents = rng.integers(-1, B, size=B)
    parents[::3] = np.arange(B)[::3]
    parents[5::11] = 4000  # one row that hundreds continue
    free = np.full(NB, -1, np.int32)
    count = min(len(left), 3000)  # too few for all copies
    free[:count] = left[:count]
    pools = make_pools(NB, 1, bs, 16, "bhtd", 1)
    check_fork(parents, lens, table, free, count, bs, pools, "bhtd", in_place)


@pytest.mark.gpu
@pytest.mark.parametrize("fill", [0.02, 0.6])
def test_pools_of_a_million_blocks(fill):
    rng, B, bs, NB = np.random.default_rng(2), 40, 2, 1 << 20
    MB = NB // B
    lens = np.minimum((rng.random(B) * 2 * fill * MB * bs).astype(np.int64), MB * bs)
    table, left = random_rows(rng, B, MB, bs, NB, lens, share=0.1)
    free = np.full(NB, -1, np.int32)
    count = len(left) - 1000  # some belong to others
    free[:count] = left[:count]
    pools = make_pools(NB, 1, bs, 4, "bhtd", 2)
    parents = rng.integers(-1, B, size=B)
    table, lens, free, count, *_ = check_fork(parents, lens, table, free, count, bs, pools, "bhtd", True)
    check_compact(lens, table, free, count, bs, pools, "bhtd", True)
