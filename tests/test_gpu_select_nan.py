"""Beams with NaN among equal logits, in tiles that take several vectors a thread: the beam is dropped and
reported, and nothing of the other beams changes."""

import math

import pytest
import torch

from kvserve_amd import paged

pytestmark = pytest.mark.gpu


def expect(x, s, beams, count, bad):
    """What is chosen without the beams `bad`, which are clean here and out of use."""
    s = s.clone()
    s[bad] = -math.inf
    return paged.select_beams(x, s, beams, count, check=True)


# rows enough for 16, 8 and 4 vectors a thread; NaN in fewer threads of a tile than candidates are asked for
@pytest.mark.parametrize("dtype,rows,V,count,vec,nans", [
    (torch.bfloat16, 400, 131072, 16, 8, 15), (torch.float16, 400, 131072, 16, 8, 12),
    (torch.float32, 64, 70000, 64, 4, 40), (torch.bfloat16, 64, 70000, 64, 8, 63)])
@pytest.mark.parametrize("level", [0.0, "lowest"])
@pytest.mark.parametrize("sign", [1, -1])
def test_nan_on_a_plateau(cuda, dtype, rows, V, count, vec, nans, level, sign):
    beams = 4
    low = torch.finfo(dtype).min if level == "lowest" else level
    x = torch.full((rows, V), low, dtype=dtype, device=cuda)
    s = -torch.rand(rows, generator=torch.Generator(device=cuda).manual_seed(rows), device=cuda)
    x[:, 5] = 1.0  # (a log-sum that 64 bits hold beside the lowest value too)
    bad = torch.zeros(rows, dtype=torch.bool, device=cuda)
    bad[1::3] = True
    want = expect(x, s, beams, count, bad)
    column = torch.arange(V, device=cuda) // vec % 256 < nans
    nan = torch.full((), math.nan, dtype=dtype, device=cuda)
    nan = nan if sign > 0 else -nan
    y = torch.where(bad.unsqueeze(1) & column, nan, x)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = paged.select_beams(y, s, beams, count, check=False, err=err)
    assert int(err) == 256
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    parents = got.all_parents[got.all_parents >= 0].long()
    assert not bool(bad[parents].any()) and parents.numel() == rows // beams * count
    # a request all of whose beams are dropped has no candidates
    y[:beams] = torch.where(column, nan, x[:beams])
    got = paged.select_beams(y, s, beams, count, check=False, err=err)
    assert got.all_parents[0].tolist() == [-1] * count and got.parents[:beams].tolist() == [-1] * beams
    for a, b in zip(got[3:], want[3:]):
        assert torch.equal(a[1:], b[1:])


@pytest.mark.parametrize("count", [3, 17, 64])
def test_nan_anywhere_in_crowded_tiles(cuda, count):
    """Few values, so that most tiles are crowded, and NaN of either sign in random places and threads."""
    gen = torch.Generator(device=cuda).manual_seed(count)
    rows, V, beams = 96, 65000, 3
    x = torch.randint(-1, 2, (rows, V), generator=gen, device=cuda).to(torch.bfloat16)
    s = -torch.rand(rows, generator=gen, device=cuda)
    share = torch.rand((rows, 1), generator=gen, device=cuda) * 0.2
    few = torch.rand((rows, V), generator=gen, device=cuda) < share
    some = torch.rand((rows, 256), generator=gen, device=cuda) < 0.1
    thread = some[:, torch.arange(V, device=cuda) // 8 % 256]
    place = torch.where(torch.arange(rows, device=cuda).unsqueeze(1) % 2 == 0, few, thread)
    place &= torch.arange(rows, device=cuda).unsqueeze(1) % 4 != 3
    nan = torch.where(torch.rand((rows, V), generator=gen, device=cuda) < 0.5, math.nan, -math.nan).to(x.dtype)
    bad = place.any(1)
    assert 0 < int(bad.sum()) < rows
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    got = paged.select_beams(torch.where(place, nan, x), s, beams, count, check=False, err=err)
    assert int(err) == 256
    for a, b in zip(got, expect(x, s, beams, count, bad)):
        assert torch.equal(a, b)
