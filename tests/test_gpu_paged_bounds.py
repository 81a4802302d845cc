"""The paged operators on arguments that are wrong in the middle: nothing outside the arrays they
were given is read or written."""

import pytest
import torch

from kvserve_amd import paged

from test_gpu_paged import i32

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("S,C,base,path", [(4, 2, 6, [0, 1, 0, 1]), (1, 8, 3, [3, 0, 1, 2, 0, 1, -1]),
                                           (4, 20, 72, [0, 1, 2, 0] + [0, 1] * 30), (2, 40, 70, [0, 1] * 400)])
def test_paths_that_fall_back_stay_in_their_row(cuda, S, C, base, path):
    """A path that stops increasing has places behind its request's row: the row behind it, here of
    ids outside the cache, is not looked at."""
    cache = torch.randn((2, C, S, 2, 64), device=cuda).to(torch.bfloat16)
    before = cache.clone()
    whole = torch.full((40, C), 9999, dtype=torch.int32, device=cuda)
    whole[0] = torch.arange(C, device=cuda)
    err = i32([0], cuda)
    got = paged.keep_drafts([cache], whole[:1], i32([base], cuda), i32([path], cuda), check=False, err=err)
    assert got.tolist() == [base] and int(err) == 128 and torch.equal(cache, before)
