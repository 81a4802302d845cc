"""Attention of drafted tokens over the paged cache against its definition in 64 bits.  Every
output is held to its own bound (`_paged_ref.attention`), derived from the roundings taken."""

import math
import random

import pytest
import torch

from kvserve_amd import paged

from _paged_ref import attention, parts

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def make(cuda, lens, H, G, D, S, dtype=BF16, layout="flash", tree=False, seed=0, extra_columns=1):
    """Inputs for lens = [(cache length, queries)]; blocks of no request hold NaN, and so do the
    places of a request's last block behind its length."""
    gen = torch.Generator(device=cuda).manual_seed(seed)
    counts = [-(-n // S) for n, _ in lens]
    C, P = max(counts + [1]) + extra_columns, sum(counts) + 3
    shape = (2, P, S, H, D) if layout == "flash" else (P, 2, S, H, D)
    cache = torch.full(shape, math.nan, device=cuda, dtype=dtype)
    ids = torch.randperm(P, generator=gen, device=cuda)[:sum(counts)]
    tables = torch.full((len(lens), C), -1, dtype=torch.int32, device=cuda)
    at = 0
    for r, ((n, _), k) in enumerate(zip(lens, counts)):
        tables[r, :k] = ids[at:at + k].int()
        p = torch.arange(n, device=cuda)
        for part in parts(cache):
            part[tables[r].long()[p // S], p % S] = torch.randn((n, H, D), generator=gen, device=cuda).to(dtype)
        at += k
    total = sum(t for _, t in lens)
    query = (2 * torch.randn((total, H * G, D), generator=gen, device=cuda)).to(dtype)
    starts = [0]
    for _, t in lens:
        starts.append(starts[-1] + t)
    top = max([t for _, t in lens] + [1])
    mask = None
    if tree:
        r = random.Random(seed)
        words = (top + 63) // 64
        rows = [paged.tree_mask([r.randint(-1, i - 1) for i in range(t)], words, cuda) for _, t in lens]
        mask = torch.cat(rows)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device=cuda)
    return dict(query=query, cache=cache, tables=tables, lengths=i32([n for n, _ in lens]), starts=i32(starts),
                mask=mask, max_query=top)


def call(d, **kw):
    return paged.tree_attention(d["query"], d["cache"], d["tables"], d["lengths"], d["starts"],
                                max_query=kw.pop("max_query", d["max_query"]), tree_mask=d["mask"], **kw)


def hold(d, got, lse=None, scale=None):
    out, want_lse, bound = attention(d["query"], d["cache"], d["tables"], d["lengths"], d["starts"], d["mask"], scale)
    off = (got.double() - out).abs()
    assert torch.isfinite(got).all()
    worst = (off - bound).max()
    assert worst <= 0, (float(worst), float(off.max()))
    if lse is not None:
        assert torch.equal(torch.isinf(lse), torch.isinf(want_lse))
        fine = ~torch.isinf(want_lse)
        # the scores' and sums' errors of the bound, and the log's own in 32 bits
        assert float((lse.double() - want_lse)[fine].abs().max() if fine.any() else 0.0) <= 2e-4


HEAD_SIZES = [8, 16, 24, 40, 64, 72, 80, 96, 104, 112, 120, 128, 136, 160, 192, 200, 224, 248, 256]


@pytest.mark.parametrize("D", HEAD_SIZES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_head_sizes(cuda, D, dtype):
    """Every head size, from single tokens to rows enough for every kernel."""
    for G, lens in ((1, [(70, 1)]), (4, [(333, 1), (5, 5), (64, 2)]), (3, [(257, 40), (300, 90)])):
        d = make(cuda, lens, 2, G, D, 16, dtype, tree=G == 4, seed=D + G)
        hold(d, *call(d, return_lse=True))


@pytest.mark.parametrize("G", [1, 2, 3, 5, 7, 8, 16, 17, 32])
@pytest.mark.parametrize("t", [1, 2, 9, 33, 100])
def test_shared_heads_and_row_counts(cuda, G, t):
    for tree in (False, True):
        d = make(cuda, [(t + 130, t), (t, t), (1, 1)], 3, G, 64, 16, BF16, "kv_adjacent", tree, seed=G * t)
        hold(d, *call(d, return_lse=True))


@pytest.mark.parametrize("S", [1, 2, 12, 16, 17, 64, 128, 1000])
@pytest.mark.parametrize("layout", ["flash", "kv_adjacent"])
def test_block_sizes(cuda, S, layout):
    for t, tree in ((1, False), (20, True), (150, False)):
        d = make(cuda, [(n + t, t) for n in (0, 1, 63, 64, 65, 500)], 2, 4, 128, S, BF16, layout, tree, seed=S + t)
        hold(d, *call(d, return_lse=True))


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("n,t,G", [(9000, 1, 4), (9000, 1, 8), (20011, 3, 5), (12345, 64, 8), (6000, 129, 2),
                                   (2048, 2048, 4), (3001, 1500, 1)])
def test_long(cuda, dtype, n, t, G):
    """Lengths that are split over workgroups and joined, and whole prompts."""
    d = make(cuda, [(n, t), (n // 3 + t, t)], 2, G, 128, 16, dtype, tree=t <= 64, seed=n + t)
    hold(d, *call(d, return_lse=True))
    hold(d, call(d, max_length=n))
    hold(d, call(d, max_length=1))  # a poor launch, the same sums


def test_many_requests(cuda):
    r = random.Random(5)
    lens = [(r.randint(0, 700) + t, t) for t in (r.choice([0, 1, 1, 2, 30]) for _ in range(200))]
    d = make(cuda, lens, 2, 6, 64, 16, seed=11)
    hold(d, *call(d, return_lse=True))


def test_rows_that_see_nothing(cuda):
    """Empty requests, requests shorter than their queries, and mask rows of zero."""
    d = make(cuda, [(0, 1), (0, 7), (3, 9), (40, 0), (5, 5), (0, 0)], 2, 4, 64, 4, seed=1)
    out, lse = call(d, return_lse=True)
    hold(d, out, lse)
    assert not out[:8].any() and torch.isinf(lse[:8]).all()
    d = make(cuda, [(6, 6), (70, 70), (90, 20)], 2, 4, 64, 16, tree=True, seed=2)
    d["mask"][2] = 0
    d["mask"][10:50] = 0
    d["mask"][80] = 0
    out, lse = call(d, return_lse=True)
    hold(d, out, lse)
    assert not out[2].any() and not out[10:50].any() and out[80].any()


def test_masks_beyond_the_queries_and_dense(cuda):
    """Bits of drafts that a request has not got say nothing; any pattern is served, not only trees."""
    d = make(cuda, [(50, 20), (130, 100), (64, 64)], 2, 3, 64, 16, tree=True, seed=3)
    gen = torch.Generator(device=cuda).manual_seed(3)
    d["mask"] = torch.randint(-2**62, 2**62, d["mask"].shape, generator=gen, device=cuda) * 2 + 1
    hold(d, *call(d, return_lse=True))
    d["mask"] = torch.full_like(d["mask"], -1)
    hold(d, *call(d, return_lse=True))


@pytest.mark.parametrize("value", [math.nan, math.inf, -math.inf, 1e30])
@pytest.mark.parametrize("tree", [False, True])
@pytest.mark.parametrize("G,t,D", [(2, 5, 64), (4, 20, 128), (8, 70, 80), (1, 200, 256)])
def test_hidden_places_have_no_part(cuda, value, tree, G, t, D):
    """Non-finite keys or values of a draft reach only the queries that see it."""
    n = t + 90
    d = make(cuda, [(n, t), (t, t)], 2, G, D, 16, BF16, tree=tree, seed=t + D)
    if tree:  # nobody but the draft itself sees it
        d["mask"] = d["mask"] & ~(1 << 3) if d["mask"].shape[1] == 1 else d["mask"]
        d["mask"][:, 0] &= ~(1 << 3)
        d["mask"][3, 0] |= 1 << 3
    clean = call(d)
    hold(d, clean)
    j = 3 if tree else t - 1
    p = n - t + j
    block, place = int(d["tables"][0, p // 16]), p % 16
    for part in (0, 1):
        held = d["cache"][part, block, place].clone()
        d["cache"][part, block, place] = value
        got = call(d)
        others = [i for i in range(2 * t) if i != j]
        assert torch.equal(got[others], clean[others]), part
        if part == 1 and not math.isfinite(value):
            # the query that sees it gets what its sum is
            assert (torch.isnan(got[j]) if math.isnan(value) else got[j] == value).all()
        d["cache"][part, block, place] = held


def test_infinite_values_of_both_signs(cuda):
    d = make(cuda, [(30, 4)], 1, 2, 64, 16, seed=9)
    for p, v in ((27, math.inf), (28, -math.inf)):
        d["cache"][1, int(d["tables"][0, p // 16]), p % 16] = v
    got = call(d)
    assert torch.isfinite(got[0]).all() and (got[1] == math.inf).all() and torch.isnan(got[2:]).all()


def test_strided_and_misaligned_queries(cuda):
    d = make(cuda, [(100, 3), (40, 8)], 2, 4, 128, 16, seed=4)
    want = call(d)
    n = d["query"].shape[0]
    fused = torch.zeros((n, 12, 128), dtype=BF16, device=cuda)
    fused[:, 2:10] = d["query"]
    heads = d["query"].transpose(0, 1).contiguous().transpose(0, 1)
    odd = torch.zeros(d["query"].numel() + 1, dtype=BF16, device=cuda)[1:].view_as(d["query"])
    odd.copy_(d["query"])
    for q in (fused[:, 2:10], heads, odd):
        assert torch.equal(call(dict(d, query=q)), want)
    out = torch.zeros_like(want)
    assert call(d, out=out) is out and torch.equal(out, want)


def test_scales(cuda):
    d = make(cuda, [(200, 2), (77, 5)], 2, 4, 64, 16, seed=6)
    for scale in (1e-6, 0.05, 1.0):
        hold(d, *call(d, scale=scale, return_lse=True), scale=scale)


def test_scores_far_apart(cuda):
    """Maxima that rise late, by a little and by a lot, and one that leads from the first key."""
    d = make(cuda, [(1000, 2), (700, 1)], 1, 4, 64, 16, seed=7)
    for r, where in ((0, (3, 500, 501, 997)), (1, (0,))):
        for k, p in enumerate(where):
            q = d["query"][0 if r == 0 else 2, 0].float()
            d["cache"][0, int(d["tables"][r, p // 16]), p % 16, 0] = ((1.5 + k) * q / q.norm() * 8).to(BF16)
    hold(d, *call(d, return_lse=True))


def test_rows_of_no_request_are_left(cuda):
    d = make(cuda, [(20, 4), (30, 4)], 1, 2, 64, 16, seed=8)
    d["starts"] = torch.tensor([0, 4, 6], dtype=torch.int32, device=cuda)
    out = torch.full_like(d["query"], 7.0)
    got = call(d, out=out)
    assert (got[6:] == 7.0).all() and not (got[:6] == 7.0).all(-1).any()


def test_past_32_bit_offsets(cuda):
    """Blocks behind 2^32 elements of a part."""
    P, S, H, D, n = 270000, 16, 8, 128, 100
    cache = torch.empty((2, P, S, H, D), dtype=BF16, device=cuda)
    ids = torch.tensor([P - 1, 0, P - 2, 1, P - 70000, P - 3, 5], dtype=torch.int32, device=cuda)
    cache[:, ids.long()] = torch.randn((2, 7, S, H, D), device=cuda).to(BF16)
    for t in (1, 50):
        d = dict(query=torch.randn((t, 2 * H, D), device=cuda).to(BF16), cache=cache, tables=ids.view(1, 7),
                 lengths=torch.tensor([n], dtype=torch.int32, device=cuda), mask=None, max_query=t,
                 starts=torch.tensor([0, t], dtype=torch.int32, device=cuda))
        hold(d, call(d))


def test_bad_pages_and_lengths_are_flagged(cuda):
    """A bad id, length or range reads nothing outside the cache and is reported."""
    for t in (1, 40):
        d = make(cuda, [(100, t), (60, t)], 2, 4, 64, 16, seed=t)
        good = call(d)
        for name, index, value, exc, code in (("tables", (0, 2), -1, IndexError, 16),
                                              ("tables", (0, 0), 10**9, IndexError, 16),
                                              ("lengths", 0, 10**6, ValueError, 128), ("lengths", 0, -5, ValueError, 128),
                                              ("starts", 2, 10**6, ValueError, 128), ("starts", 0, -3, ValueError, 128)):
            bad = dict(d, **{name: d[name].clone()})
            bad[name][index] = value
            with pytest.raises(exc):
                call(bad, check=True)
            err = torch.zeros(1, dtype=torch.int32, device=cuda)
            got = call(bad, check=False, err=err)
            assert int(err) & code
            if name != "starts":
                assert torch.equal(got[t:], good[t:])
        with pytest.raises(ValueError):
            call(d, max_query=t - 1, check=True) if t > 1 else call(d, max_length=-1)


def test_graph_replays(cuda):
    """Captured once and replayed on rewritten inputs, with eager work in between."""
    d = make(cuda, [(900, 5), (300, 5), (0, 5)], 2, 4, 128, 16, seed=12)
    out = torch.empty_like(d["query"])
    call(d, out=out, check=False)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(d, out=out)
    for step in range(5):
        d["query"].mul_(0.9)
        d["lengths"].copy_(torch.tensor([900 - 100 * step, 300 - step, 0], dtype=torch.int32, device=cuda))
        out.fill_(3.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, call(d))
        hold(d, out)


def test_repeats_are_bitwise_alike(cuda):
    d = make(cuda, [(5000, 3), (100, 3)], 2, 4, 128, 16, seed=13)
    first = call(d)
    for _ in range(3):
        assert torch.equal(call(d), first)


def test_nothing_to_do(cuda):
    d = make(cuda, [(10, 0)], 1, 1, 64, 16)
    assert call(d).shape == (0, 1, 64)
    d = make(cuda, [(10, 2)], 1, 1, 64, 16)
    none = dict(d, tables=d["tables"][:0], lengths=d["lengths"][:0], starts=d["starts"][:1])
    out = torch.full_like(d["query"], 5.0)
    assert (call(none, out=out) == 5.0).all()
