"""Every attention kernel on the batches that it is chosen for: each case asserts its kernel, its
waves, the rows of a workgroup and whether keys are split, and is held to the 64-bit definition."""

import ctypes
import math
import random

import pytest
import torch

from kvserve_amd import _lib, paged

from test_gpu_tree_attention import BF16, FP16, call, hold, make

pytestmark = pytest.mark.gpu


def kernels(d, max_length=None):
    """(kernel, waves, rows, parts) of the call."""
    args, _query = paged._attention_args(d["query"], d["cache"], d["tables"], d["lengths"], d["starts"], d["max_query"],
                                         max_length, d["mask"], None, torch.empty_like(d["query"]), None)
    shape = (ctypes.c_int32 * 4)()
    kind = _lib.load().kvmi_attention_kernels(args, shape)
    return kind, shape[0], shape[1], shape[2]


def longest(lens):
    return max(n for n, _ in lens)


# ------------------------------------------------------------------ tiles of 256 rows, 8 waves
def wide_batch(requests, t, seed, context=150, ragged=True):
    """Requests of up to t queries; with `ragged` some of one query, of none, without a cache, and
    shorter than their queries."""
    r = random.Random(seed)
    lens = [(r.randint(0, context) + t, t) for _ in range(requests)]
    if ragged:
        odd = [(0, 1), (90, 0), (t // 2, t), (77, 1), (64, 33), (1, 1)]
        lens[1:1 + len(odd)] = odd
    return lens


EIGHT = [
    # requests, queries, KV heads, query heads a KV head: rows of a request
    (24, 50, 32, 4),   # 200 of 256
    (40, 128, 16, 2),  # 256
    (12, 300, 16, 4),  # 1200: four tiles and 176 rows
    (24, 64, 32, 8),   # 512
    (70, 129, 8, 3),   # 387: one tile and 131 rows
]


@pytest.mark.parametrize("D", [104, 112, 120, 128])
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("requests,t,H,G", EIGHT)
def test_tiles_of_256_rows(cuda, D, dtype, tree, requests, t, H, G):
    lens = wide_batch(requests, t, D + t)
    d = make(cuda, lens, H, G, D, 16, dtype, "kv_adjacent" if t == 50 else "flash", tree, seed=D + t)
    assert kernels(d, longest(lens)) == (_lib.ATTENTION_TILES, 8, 256, 1)
    hold(d, *call(d, return_lse=True, max_length=longest(lens)))


@pytest.mark.parametrize("D,dtype,G", [(128, BF16, 4), (128, FP16, 2), (104, BF16, 3)])
def test_prompts_in_tiles_of_256_rows(cuda, D, dtype, G):
    """Whole prompts and long contexts: tiles that only some of the waves see, in many tiles of keys."""
    for lens in ([(2048, 2048)] * 4, [(1500, 1024), (1024, 1024), (3000, 1000), (2222, 700)]):
        d = make(cuda, lens, 32, G, D, 16, dtype, seed=D + G)
        assert kernels(d, longest(lens)) == (_lib.ATTENTION_TILES, 8, 256, 1)
        hold(d, *call(d, return_lse=True, max_length=longest(lens)))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("D", [120, 128])
def test_hidden_places_in_tiles_of_256_rows(cuda, value, tree, D):
    """A draft's key or value that is not finite reaches only the queries that see it."""
    t, H, G = 50, 32, 4
    lens = wide_batch(24, t, 3)
    d = make(cuda, lens, H, G, D, 16, BF16, tree=tree, seed=D)
    assert kernels(d, longest(lens))[1] == 8
    j = 7 if tree else t - 1  # of the first request
    if tree:
        d["mask"][:t, 0] &= ~(1 << j)
        d["mask"][j, 0] |= 1 << j
    clean = call(d, max_length=longest(lens))
    hold(d, clean)
    p = lens[0][0] - t + j
    block, others = int(d["tables"][0, p // 16]), [i for i in range(d["query"].shape[0]) if i != j]
    for part in (0, 1):
        held = d["cache"][part, block, p % 16].clone()
        d["cache"][part, block, p % 16] = value
        got = call(d, max_length=longest(lens))
        assert torch.equal(got[others], clean[others]), part
        if part == 1:
            assert (torch.isnan(got[j]) if math.isnan(value) else got[j] == value).all()
        d["cache"][part, block, p % 16] = held


def test_a_query_of_nan_in_tiles_of_256_rows(cuda):
    lens = wide_batch(24, 50, 4)
    d = make(cuda, lens, 32, 4, 128, 16, seed=4)
    assert kernels(d, longest(lens))[1] == 8
    clean, clean_lse = call(d, return_lse=True, max_length=longest(lens))
    for row, head in ((0, 0), (17, 63), (d["query"].shape[0] - 1, 127)):
        bad = dict(d, query=d["query"].clone())
        bad["query"][row, head, 3] = math.nan
        out, lse = call(bad, return_lse=True, max_length=longest(lens))
        assert torch.isnan(out[row, head]).all() and torch.isnan(lse[row, head])
        out[row, head], lse[row, head] = clean[row, head], clean_lse[row, head]
        assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


# ------------------------------------------------------------------ few rows, 4 waves
HEADS = [(40, 1), (64, 1), (80, 1), (128, 1), (136, 1), (160, 1), (192, 1), (200, 1), (224, 1), (256, 1), (24, 2),
         (64, 2), (96, 2), (128, 2)]


@pytest.mark.parametrize("D,groups", HEADS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("length,split", [(300, False), (1700, True)])
def test_decode_batches(cuda, D, groups, dtype, length, split):
    """Batches that fill the chip: 4 waves a workgroup, whole requests and parts of them; 1 to 16
    rows a KV head, and 17 to 32 where the kernel takes them."""
    r = random.Random(D + length)
    for t, G, tree in ((1, 16 * groups, False), (4, 3 + 4 * (groups - 1), True), (5 * groups, 3, False)):
        rows = t * G
        assert rows <= 16 if groups == 1 else 16 < rows <= 32
        lens = [(r.randint(length // 3, length) + t, t) for _ in range(32)]
        lens[3:6] = [(length + t, t), (0, 1), (t, t)]
        d = make(cuda, lens, 8, G, D, 16, dtype, tree=tree, seed=D + t)
        kind, waves, held, parts = kernels(d, longest(lens))
        assert (kind, waves, held) == (_lib.ATTENTION_ROWS, 4, 16 * groups) and (parts > 1) == split
        hold(d, *call(d, return_lse=True, max_length=longest(lens)))


@pytest.mark.parametrize("D,groups", [(64, 2), (128, 2), (192, 1), (256, 1)])
def test_hidden_places_in_decode_batches(cuda, D, groups):
    t, G = 4, 4 * groups
    lens = [(250 + 10 * i, t) for i in range(32)]
    d = make(cuda, lens, 8, G, D, 16, tree=True, seed=D)
    assert kernels(d, longest(lens))[:3] == (_lib.ATTENTION_ROWS, 4, 16 * groups)
    d["mask"][:t, 0] &= ~(1 << 2)
    d["mask"][2, 0] |= 1 << 2
    clean = call(d, max_length=longest(lens))
    hold(d, clean)
    p = lens[0][0] - t + 2
    block, others = int(d["tables"][0, p // 16]), [i for i in range(32 * t) if i != 2]
    for part in (0, 1):
        held = d["cache"][part, block, p % 16].clone()
        d["cache"][part, block, p % 16] = math.nan
        got = call(d, max_length=longest(lens))
        assert torch.equal(got[others], clean[others]) and torch.isnan(got[2]).all()
        d["cache"][part, block, p % 16] = held
