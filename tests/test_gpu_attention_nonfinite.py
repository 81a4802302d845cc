"""Attention over the paged cache where scores are not finite: a row whose scores are NaN gives NaN,
and an infinity gives what its score gives, however the keys are split and whichever kernel runs."""

import math

import pytest
import torch

from test_gpu_tree_attention import BF16, FP16, call, hold, make

pytestmark = pytest.mark.gpu

# (requests' (length, queries), KV heads, query heads a KV head, channels): one part and many, few
# rows and tiles
SHAPES = [([(40, 1)], 2, 4, 128), ([(3000, 1)], 2, 4, 128), ([(3000, 4), (70, 2)], 2, 4, 64),
          ([(9000, 3)], 1, 9, 64), ([(5000, 1), (500, 1)], 2, 16, 256), ([(90, 60)], 2, 4, 128),
          ([(3000, 60)], 2, 4, 128), ([(2500, 50), (300, 50)], 1, 3, 80)]


@pytest.mark.parametrize("lens,H,G,D", SHAPES)
@pytest.mark.parametrize("dtype", [BF16, FP16])
def test_a_query_of_nan_gives_nan(cuda, lens, H, G, D, dtype):
    """One NaN channel of one query head: NaN in that row and its lse, all others as they were."""
    d = make(cuda, lens, H, G, D, 16, dtype, seed=D + G)
    top = max(n for n, _ in lens)
    for max_length in (top, 1, None):  # many parts, one part, the tables' length
        clean, clean_lse = call(d, return_lse=True, max_length=max_length)
        hold(d, clean, clean_lse)
        for row, head in ((0, 0), (d["query"].shape[0] - 1, H * G - 1)):
            bad = dict(d, query=d["query"].clone())
            bad["query"][row, head, D // 2] = math.nan
            out, lse = call(bad, return_lse=True, max_length=max_length)
            assert torch.isnan(out[row, head]).all() and torch.isnan(lse[row, head])
            out[row, head], lse[row, head] = clean[row, head], clean_lse[row, head]
            assert torch.equal(out, clean) and torch.equal(lse, clean_lse)


@pytest.mark.parametrize("t,G", [(1, 4), (2, 16), (40, 4)])
@pytest.mark.parametrize("first", [0, 64, 700])
def test_keys_of_nan_give_nan_to_all_who_see_them(cuda, t, G, first):
    """From one NaN key to whole parts of them, from and to each 64th key, among keys that are finite."""
    d = make(cuda, [(3000, t), (200, t)], 2, G, 128, 16, seed=t + first)
    held, clean = d["cache"].clone(), call(d, max_length=3000)
    for last in [first + 1, *range(first // 64 * 64 + 64, 2944, 64)]:
        p = torch.arange(first, last, device=cuda)
        d["cache"][0, d["tables"][0].long()[p // 16], p % 16, 0, 5] = math.nan
        for max_length in (3000, 1):
            out, lse = call(d, return_lse=True, max_length=max_length)
            assert torch.isnan(out[:t, :G]).all() and torch.isnan(lse[:t, :G]).all(), last
            assert torch.isfinite(out[:t, G:]).all() and torch.isfinite(lse).sum() == lse.numel() - t * G
        assert torch.equal(call(d, max_length=3000)[t:], clean[t:])
        d["cache"].copy_(held)


@pytest.mark.parametrize("D", [8, 24, 40, 56, 72, 80, 96, 104, 120, 128, 136, 160, 200, 224, 248, 256])
@pytest.mark.parametrize("t,G", [(1, 4), (5, 3), (40, 4)])
def test_a_score_of_minus_infinity_weighs_nothing(cuda, D, t, G):
    """A key with an infinity whose scores are all -inf: as if it were not there, at every head size."""
    for first in (0, D - 1):
        d = make(cuda, [(700, t), (90, t)], 2, G, D, 16, seed=D + t)
        d["query"][..., first] = -d["query"][..., first].abs() - 0.5
        cache, tables = d["cache"], d["tables"].long()
        for p in (0, 130, 699 - t):
            cache[0, tables[0, p // 16], p % 16, :, first] = math.inf
        out, lse = call(d, return_lse=True)
        assert torch.isfinite(out).all() and torch.isfinite(lse).all()
        # the definition drops the keys; a key far on the other side of every query comes near it
        cache[0, tables[0, 0], 0, :, first] = 1e30
        for p in (130, 699 - t):
            cache[0, tables[0, p // 16], p % 16, :, first] = 1e30
        assert torch.equal(call(d), out)
