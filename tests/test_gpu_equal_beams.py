"""Beams with the same logits and score, in rows that begin anywhere within 16 bytes: their values are the same to
the last bit, so the lower beam comes first."""

import numpy as np
import pytest
import torch

from kvserve_amd import paged

pytestmark = pytest.mark.gpu


def expected(x, beams, count):
    """[requests, count] beams and tokens, from one row of logits a request: larger logits first (beams are
    alike, so that is the order of the values), then the lower beam, then the lower token."""
    parents, tokens = [], []
    for r, row in enumerate(x.float().cpu().numpy()):
        t = np.argsort(-row, kind="stable")[:count]
        all_t, beam = np.tile(t, beams), np.repeat(np.arange(beams), t.size)
        best = np.lexsort((all_t, beam, -row[all_t]))[:count]
        parents.append(r * beams + beam[best])
        tokens.append(all_t[best])
    return torch.tensor(np.array(parents)), torch.tensor(np.array(tokens))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("requests,beams,V,pad,offset", [
    (3000, 2, 1003, 0, 0), (3000, 3, 777, 2, 1), (2000, 4, 2047, 0, 3), (600, 2, 5001, 4, 0), (300, 5, 9006, 1, 0),
    (96, 4, 30001, 0, 1), (100, 4, 66001, 1, 0),
    (2000, 4, 1000, 0, 0)])
def test_equal_beams_stand_in_their_order(cuda, dtype, requests, beams, V, pad, offset):
    gen = torch.Generator(device=cuda).manual_seed(V)
    one = (torch.randn((requests, V), generator=gen, device=cuda) * 2.5).to(dtype)
    rows, stride, count = requests * beams, V + pad, 2 * beams + 1
    room = torch.zeros(rows * stride + offset, dtype=dtype, device=cuda)
    x = room[offset:].view(rows, stride)[:, :V]
    x.copy_(one.repeat_interleave(beams, 0))
    s = (-20.0 * torch.rand(requests, generator=gen, device=cuda)).repeat_interleave(beams)
    got = paged.select_beams(x, s, beams, count)
    parents, tokens = expected(one, beams, count)
    assert torch.equal(got.all_tokens.cpu().long(), tokens)
    assert torch.equal(got.all_parents.cpu().long(), parents)
