"""The paged operators on arguments that are wrong in the middle: nothing outside the arrays they
were given is read or written."""

import sys

import pytest
import torch

from kvserve_amd import paged

from test_gpu_paged import i32
from test_gpu_tree_attention import call, hold, make

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


@pytest.mark.parametrize("in_place", [False, True])
def test_a_ring_without_room_keeps_its_free_blocks(cuda, in_place):
    """Blocks given back past the ring's room are dropped and reported, in order, and those that
    are free stay so; a count of more blocks than the ring has is reported."""
    S = 4
    # (lengths, new lengths, tables, ring, state) -> (tables, ring, state)
    cases = [
        ([8, 4], [0, 4], [[0, 1], [2, -1]], [8, 9], [0, 2], [[-1, -1], [2, -1]], [8, 9], [0, 2]),
        ([8, 8], [4, 0], [[0, 1], [2, 3]], [-1, -1, 7], [2, 1], [[0, -1], [-1, -1]], [1, 2, 7], [2, 3]),
        ([8, 0, 4], [0, 5, 0], [[0, 1], [-1, -1], [2, -1]], [6, 7, 8, -1], [0, 3], [[-1, -1], [6, 7], [-1, -1]],
         [6, 7, 8, 0], [2, 2]),
        ([4], [8], [[0, -1]], [5, 6], [1, 3], [[0, 6]], [5, 6], [0, 1]),
    ]
    for now, new, tables, ring, state, want_tables, want_ring, want_state in cases:
        for check in (False, True):
            t = [i32(v, cuda) for v in (now, new, tables, ring, state)]
            kw = {}
            if in_place:
                slots, starts = torch.empty(9, dtype=torch.int64, device=cuda), i32([0] * (len(now) + 1), cuda)
                kw = dict(out=(t[2], t[0], t[4], slots, starts), ticket=i32([0], cuda))
            err = i32([0], cuda)
            args = (t[0], t[1], t[2], t[3], t[4], S, 9)
            if check:
                with pytest.raises(ValueError, match="ring of free blocks"):
                    paged.build_block_tables(*args, check=True, **kw)
                continue
            got = paged.build_block_tables(*args, check=False, err=err, **kw)
            assert int(err) == 128
            assert got.tables.tolist() == want_tables and got.lengths.tolist() == new
            assert t[3].tolist() == want_ring and got.state.tolist() == want_state


@pytest.mark.parametrize("check", [True, False])
def test_any_longest_length_is_taken(cuda, check):
    """`max_length` shapes the launch alone, whatever its size."""
    d = make(cuda, [(900, 2), (70, 1)], 2, 4, 64, 16, seed=1)
    want = call(d, max_length=2**31 - 1, check=check)
    hold(d, want)
    for n in (2**31, 2**32, 2**32 + 7, sys.maxsize):
        assert torch.equal(call(d, max_length=n, check=check), want)


def test_layers_in_one_memory_are_refused(cuda):
    """Rows that two layers' workgroups would both move."""
    one = torch.zeros((2, 6, 4, 1, 8), dtype=torch.bfloat16, device=cuda)
    both = torch.zeros((3, 2, 6, 4, 1, 8), dtype=torch.bfloat16, device=cuda)
    overlapping = both.flatten()[both[0].numel() // 2:][:both[0].numel()].view_as(both[0])
    for caches in ([one, one], [both[0], one, both[0]], [both[0], overlapping], [both[1], both[2], overlapping]):
        with pytest.raises(ValueError, match="share"):
            paged.LayerCaches(caches)
        with pytest.raises(ValueError, match="share"):
            paged.keep_drafts(caches, i32([[0, 1]], cuda), i32([0], cuda), i32([[0]], cuda))
    assert paged.LayerCaches([both[2], both[0], both[1]]).bases.tolist() == [c.data_ptr() for c in (both[2], both[0], both[1])]


def test_more_tokens_than_slots_move_the_tables_on(cuda):
    """A `max_tokens` that does not hold is an error, found after lengths and tables have changed."""
    own = paged.BlockTables(6, 4, 2, 3, cuda)
    slots = torch.full((7,), -9, dtype=torch.int64, device=cuda)
    with pytest.raises(ValueError):
        own.update(i32([6, 5], cuda), 7, slots=slots, check=True)
    assert own.lengths.tolist() == [6, 5] and own.state.tolist() == [4, 2]
    assert own.tables.tolist() == [[0, 1, -1], [2, 3, -1]] and slots.tolist() == [0, 1, 2, 3, 4, 5, 8]
