"""The crowded tiles of beam search's selection, step by step on the host: which elements the search for the
`count`-th largest counts, and which are collected behind it, with NaN among them."""

import numpy as np
import pytest

THREADS, ROOM, VECTORS = 256, 1024, 128
INF = np.float32(np.inf)


def order(x):
    """The kernel's words: unsigned, in the order of the values; NaN lies outside, by its sign."""
    u = (np.asarray(x, np.float32) + np.float32(0)).view(np.uint32).astype(np.int64)
    return np.where(u >> 31, u ^ 0xffffffff, u | 0x80000000)


def value(word):
    u = np.uint32(word & 0x7fffffff if word >> 31 else word ^ 0xffffffff)
    return np.array([u]).view(np.float32)[0]


def tile(x, nv, vec):
    """Elements of a tile as [vector of a thread, thread, element]."""
    return np.asarray(x, np.float32).reshape(nv, THREADS, vec)


def crowded(x, count):
    """(the search's word, vectors that reach the bound) of a tile."""
    with np.errstate(invalid="ignore"):
        words = np.sort(order(x.max(axis=(0, 2))))[::-1]  # (NaN wins over all, as in the kernel)
        bound = max(int(words[count - 1]), int(order(-INF)) + 1)
        hits = int((x.max(axis=2) >= value(bound)).sum())
        lo, hi = bound, 0xffffffff
        while hi - lo > 1:
            mid = lo + (hi - lo) // 2
            if int((x >= value(mid)).sum()) >= count:
                lo = mid
            else:
                hi = mid
    return lo, hits


def collected(x, count, lo, by_value):
    """Elements above the word, by the search's comparison or by their words, and those at it."""
    with np.errstate(invalid="ignore"):
        above = int((x >= value(lo + 1)).sum()) if by_value else int((order(x) > lo).sum())
    return above + max(0, min(count - above, int((order(x) == lo).sum())))


def plateau(nv, vec, nan_threads, level=0.0):
    x = np.full((nv, THREADS, vec), level, np.float32)
    x[:, :nan_threads] = np.nan
    return x


@pytest.mark.parametrize("nv,vec,count,nans", [(16, 8, 16, 15), (16, 8, 16, 12), (8, 4, 64, 40), (4, 8, 64, 63)])
@pytest.mark.parametrize("level", [0.0, -0.0, 3.5, float(np.finfo(np.float32).min)])
def test_a_plateau_with_nan_in_a_few_threads(nv, vec, count, nans, level):
    x = plateau(nv, vec, nans, level)
    lo, hits = crowded(x, count)
    assert hits > VECTORS and lo == int(order(np.float32(level)))
    assert collected(x, count, lo, True) == count
    assert collected(x, count, lo, False) > ROOM  # what the words would have put into the list


def test_random_tiles_collect_what_was_counted():
    r = np.random.default_rng(0)
    specials = np.array([np.nan, -np.nan, np.inf, -np.inf, 0.0, -0.0, 1e-45, -1e-45, 3e38, -3e38], np.float32)
    crowds = 0
    for i in range(300):
        nv, vec = int(r.choice([1, 2, 4])), int(r.choice([4, 8]))
        count = int(r.integers(1, 65))
        x = r.integers(-1, 2, (nv, THREADS, vec)).astype(np.float32)
        if i % 3 == 0:
            x *= np.float32(1e-45)
        some = r.random((1, THREADS, 1)) < r.choice([0.0, 0.05, 0.2])
        x = np.where(some & (r.random(x.shape) < 0.9), r.choice(specials, x.shape), x).astype(np.float32)
        lo, hits = crowded(x, count)
        if hits <= VECTORS:
            continue
        crowds += 1
        with np.errstate(invalid="ignore"):
            assert int((x >= value(lo + 1)).sum()) < count <= int((x >= value(lo)).sum())
        assert collected(x, count, lo, True) == count
    assert crowds > 100
