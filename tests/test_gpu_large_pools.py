"""Pools of so many blocks that a workgroup goes through their counts in several rounds: more than 16,384 in a
fork, more than 262,144 in a compaction."""

import random

import pytest

from kvserve_amd import paged

from _shared_ref import compact, fork
from test_gpu_shared_blocks import Pool, i32, random_step, run_fork

pytestmark = pytest.mark.gpu


def take(pool, parents, new, tokens):
    pool.take(fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, pool.S, tokens))


@pytest.mark.parametrize("R,C,S,N,seed", [(300, 40, 4, 16385, 0), (30, 900, 2, 40000, 1), (150, 2000, 1, 300001, 2)])
@pytest.mark.parametrize("in_place", [False, True])
def test_forks_in_large_pools(cuda, R, C, S, N, seed, in_place):
    r = random.Random(seed)
    pool = Pool(r, R, C, S, N, (5, N - 1))
    workspace = paged.fork_workspace(N, R, C, cuda)
    served = 0
    for step in range(4):
        if step == 2:  # most of the rows end: their blocks are counted all over the pool
            parents, new = list(range(R)), [n if i % 5 == 0 else 0 for i, n in enumerate(pool.lengths)]
        else:
            parents, new = random_step(r, pool.lengths, C, S)
            if step == 0:
                new = [r.randint(C * S // 2, C * S) for _ in range(R)]
        tokens = sum(max(0, n - (pool.lengths[p] if p >= 0 else 0)) for n, p in zip(new, parents))
        want = fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, tokens)
        got, err = run_fork(cuda, pool, parents, new, tokens, in_place, workspace)
        assert err == {None: 0, "blocks": 64}[want[8]]
        for k in range(8):
            assert got[k] == want[k], (step, k)
        served += want[8] is None
        pool.take(want)
    assert served >= 3


# held blocks all over the pool: the pool's n-th id lies in one of the last ranges, in the middle, at the
# beginning, and there is none
@pytest.mark.parametrize("rows", [140, 60, 1, 0])
@pytest.mark.parametrize("in_place", [False, True])
def test_compactions_of_large_pools(cuda, rows, in_place):
    r, R, C, S, N = random.Random(rows), 140, 1950, 1, 300001
    pool = Pool(r, R, C, S, N, (7, N // 2, N - 2))
    if rows:
        take(pool, [-1] * R, [C if i < rows else 0 for i in range(R)], C * R)
        take(pool, [0 if i == 1 and rows > 1 else i for i in range(R)], pool.lengths, 0)  # a shared row
    held = len({b for row in pool.tables for b in row} - {-1})
    assert held == (C * (rows - (rows > 1)) if rows else 0)
    lengths, tables, shares, ring, state = pool.device(cuda)
    want = compact(pool.lengths, pool.tables, pool.shares, pool.ring, pool.state, S)
    out = None
    if in_place:
        out = (tables, shares, ring, state, i32([[-7] * 3] * (N // 2), cuda))
    err = i32([0], cuda)
    workspace = paged.compact_workspace(N, cuda)
    got = paged.compact_block_tables(lengths, tables, shares, ring, state, S, out=out, workspace=workspace, check=False,
                                     err=err)
    assert int(err) == 0
    for k, (a, b) in enumerate(zip(got, want)):
        assert a.tolist() == b, k
    assert int(workspace[:-(-N // 16) * 8].abs().sum()) == 0
