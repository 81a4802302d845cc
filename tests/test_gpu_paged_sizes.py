"""The paged operators at the sizes where their kernels change: rows of tables in pieces and one by
one, requests by the thousand, paths of 64 and 65 drafts, keys split up to 64 times, row tiles of
every remainder, and shared heads on every XCD."""

import math
import random

import pytest
import torch

from kvserve_amd import paged

from _paged_ref import build_tables, parts
from test_gpu_paged import i32, random_state
from test_gpu_tree_attention import call, hold, make

pytestmark = pytest.mark.gpu


def run_tables(cuda, now, new, tables, ring, state, S, tokens, offset=0, in_place=False):
    """The kernel's update, tables and their copies `offset` words behind a 256-byte border."""
    R, C = len(now), len(tables[0])
    room = lambda: torch.full((R * C + offset,), -9, dtype=torch.int32, device=cuda)[offset:].view(R, C)
    t_tab, t_now, t_ring, t_state = room().copy_(i32(tables, cuda)), i32(now, cuda), i32(ring, cuda), i32(state, cuda)
    slots = torch.full((tokens,), -9, dtype=torch.int64, device=cuda)
    out = (t_tab if in_place else room(), t_now if in_place else i32([0] * R, cuda),
           t_state if in_place else i32([0, 0], cuda), slots, i32([0] * (R + 1), cuda))
    err = i32([0], cuda)
    got = paged.build_block_tables(t_now, i32(new, cuda), t_tab, t_ring, t_state, S, tokens, out=out, check=False,
                                   ticket=i32([0], cuda) if in_place else None, err=err)
    return [got.tables.tolist(), got.lengths.tolist(), got.state.tolist(), got.slots.tolist(), got.starts.tolist(),
            t_ring.tolist()], int(err)


@pytest.mark.parametrize("R,C,S,spare", [(1, 4, 3, 5), (2, 8, 16, 9), (3, 12, 1, 3), (7, 1100, 2, 4000), (2, 2052, 16, 4200),
                                         (1030, 4, 16, 700), (2100, 8, 5, 3000), (5000, 3, 16, 4000)])
@pytest.mark.parametrize("offset", [0, 1, 2, 4])
@pytest.mark.parametrize("in_place", [False, True])
def test_table_rows_in_pieces(cuda, R, C, S, spare, offset, in_place):
    r = random.Random(R + C)
    now, tables, ring, state = random_state(r, R, C, S, spare)
    new = [r.choice([n, 0, C * S, min(n + 1, C * S), r.randint(0, C * S), max(0, n - 1)]) for n in now]
    tokens = sum(max(0, b - a) for a, b in zip(now, new)) + 2
    want = build_tables(now, new, tables, ring, state, S, tokens)
    got, err = run_tables(cuda, now, new, tables, ring, state, S, tokens, offset, in_place)
    assert got == list(want[:6]) and err == (64 if want[6] else 0)


@pytest.mark.parametrize("tokens", [1, 255, 256, 257, 1023, 1024, 1025, 4096, 5000, 70000])
@pytest.mark.parametrize("have", [0, 5])
def test_slots_of_one_long_request(cuda, tokens, have):
    S = 7
    C = -(-(tokens + have) // S)
    ids = random.Random(tokens).sample(range(C + 3), C + 3)
    held = -(-have // S)
    tables, ring, state = [ids[:held] + [-1] * (C - held)], ids[held:] + [-1] * held, [0, C + 3 - held]
    want = build_tables([have], [have + tokens], tables, ring, state, S, tokens + 1)
    got, err = run_tables(cuda, [have], [have + tokens], tables, ring, state, S, tokens + 1)
    assert got == list(want[:6]) and err == 0


@pytest.mark.parametrize("width,drafts", [(1, 1), (63, 70), (64, 64), (64, 200), (65, 65), (65, 300), (1024, 1100)])
@pytest.mark.parametrize("H,D", [(1, 8), (3, 7), (8, 128)])
def test_kept_paths_of_every_width(cuda, width, drafts, H, D):
    r, S, base = random.Random(width), 16, 13
    C = -(-(base + drafts) // S)
    ids = r.sample(range(C + 2), C)
    caches = [torch.randn((2, C + 2, S, H, D), device=cuda).to(torch.float16) for _ in range(2)]
    for n in {0, 1, width // 2, width}:
        path = sorted(r.sample(range(drafts), n))
        want = [c.clone() for c in caches]
        for cache in want:
            for part in parts(cache):
                for i, j in enumerate(path):
                    a, b = base + j, base + i
                    part[ids[b // S], b % S] = part[ids[a // S], a % S].clone()
        got = paged.keep_drafts(caches, i32([ids], cuda), i32([base], cuda), i32([path + [-1] * (width - n)], cuda),
                                check=True)
        assert got.tolist() == [base + n] and all(torch.equal(a, b) for a, b in zip(caches, want))


@pytest.mark.parametrize("H", [1, 2, 3, 5, 7, 8, 9, 16])
@pytest.mark.parametrize("R", [1, 3, 8])
def test_heads_and_requests_of_every_remainder(cuda, H, R):
    r = random.Random(H * R)
    for t, G in ((1, 2), (40, 3), (70, 4)):
        lens = [(r.randint(0, 300) + t, t) for _ in range(R)]
        d = make(cuda, lens, H, G, 64, 16, seed=H + R + t)
        hold(d, *call(d, return_lse=True))


@pytest.mark.parametrize("rows", [1, 15, 16, 17, 31, 32, 33, 63, 96, 97, 127, 128, 129, 160, 255, 256, 257])
@pytest.mark.parametrize("D", [64, 80, 128, 160, 256])
def test_every_count_of_rows(cuda, rows, D):
    """One query head a KV head, so that rows are queries; some requests have fewer."""
    lens = [(rows + 77, rows), (rows, rows), (200, max(1, rows // 3)), (0, 1)]
    for tree in (False, True):
        d = make(cuda, lens, 2, 1, D, 16, tree=tree, seed=rows + D)
        hold(d, *call(d, return_lse=True))


@pytest.mark.parametrize("n", [63, 64, 65, 127, 128, 255, 256, 257, 1023, 1024, 1025, 4095, 4097, 70000])
@pytest.mark.parametrize("t,G", [(1, 1), (1, 16), (2, 16), (9, 8)])
def test_every_count_of_parts(cuda, n, t, G):
    """Lengths around the parts that keys are split into, and past 64 of them."""
    d = make(cuda, [(n + t, t), (n // 2 + t, t), (t, t)], 1, G, 128, 16, seed=n)
    hold(d, *call(d, return_lse=True))
    hold(d, call(d, max_length=n + t))


@pytest.mark.parametrize("value", [math.nan, -math.inf])
@pytest.mark.parametrize("n,t,G", [(3000, 4, 4), (3000, 12, 2), (3000, 60, 4)])
def test_hidden_places_in_split_keys(cuda, value, n, t, G):
    """The last draft's place, seen by itself alone, in a request whose keys are split."""
    d = make(cuda, [(n, t)], 2, G, 128, 16, tree=True, seed=t)
    clean = call(d, max_length=n)
    hold(d, clean)
    d["mask"][:-1] &= ~(1 << (t - 1))
    clean = call(d, max_length=n)
    p = n - 1
    d["cache"][1, int(d["tables"][0, p // 16]), p % 16] = value
    got = call(d, max_length=n)
    assert torch.equal(got[:-1], clean[:-1])
    assert (torch.isnan(got[-1]) if math.isnan(value) else got[-1] == value).all()


def test_pages_that_end_inside_a_tile_hold_what_they_will(cuda):
    """Blocks of 100 tokens, lengths inside them; the places behind the length hold NaN."""
    for t, G in ((1, 4), (20, 8)):
        lens = [(n + t, t) for n in (0, 1, 62, 63, 64, 65, 99, 100, 101, 163, 164, 165, 499)]
        d = make(cuda, lens, 2, G, 128, 100, seed=t)
        hold(d, *call(d, return_lse=True))


def test_outputs_off_their_alignment(cuda):
    """Any contiguous output will do; rows of no request stay as they are."""
    d = make(cuda, [(90, 3), (20, 20)], 2, 4, 64, 16, seed=21)
    want = call(d)
    for check in (True, False):
        for skip in (1, 2, 4):
            out = torch.full((want.numel() + skip,), 7.0, dtype=want.dtype, device=cuda)[skip:].view_as(want)
            assert call(d, out=out, check=check) is out and torch.equal(out, want)
            short = dict(d, starts=torch.tensor([0, 3, 10], dtype=torch.int32, device=cuda))
            out.fill_(7.0)
            call(short, out=out, check=check)
            assert (out[10:] == 7.0).all() and not (out[:10] == 7.0).all(-1).any()
