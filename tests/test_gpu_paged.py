"""Block tables, slot writes and kept drafts on the GPU against plain host programs."""

import random

import pytest
import torch

from kvserve_amd import paged

from _paged_ref import build_tables, parts

pytestmark = pytest.mark.gpu


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


# ------------------------------------------------------------------ block tables
def random_state(r, R, C, S, spare):
    """Lengths, tables and a turned ring of free blocks that belong together."""
    now = [r.choice([0, 1, S, S + 1, r.randint(0, C * S), C * S]) for _ in range(R)]
    now = [min(n, C * S) for n in now]
    held = sum(-(-n // S) for n in now)
    N = max(1, held + spare)
    ids = list(range(N))
    r.shuffle(ids)
    tables, at = [], 0
    for n in now:
        k = -(-n // S)
        tables.append(ids[at:at + k] + [-1] * (C - k))
        at += k
    head = r.randrange(N)
    ring = [-1] * N
    for i, b in enumerate(ids[at:]):
        ring[(head + i) % N] = b
    return now, tables, ring, [head, N - held]


@pytest.mark.parametrize("R,C,S,spare,seed", [(1, 1, 1, 0, 0), (1, 7, 16, 9, 1), (3, 5, 12, 2, 2), (5, 40, 1, 60, 3),
                                              (64, 9, 16, 200, 4), (257, 33, 16, 3000, 5), (300, 20, 128, 400, 6),
                                              (1000, 12, 16, 100, 7)])
@pytest.mark.parametrize("in_place", [False, True])
def test_tables_match_a_host_program(cuda, R, C, S, spare, seed, in_place):
    r = random.Random(seed)
    now, tables, ring, state = random_state(r, R, C, S, spare)
    new = [r.choice([n, 0, min(n + 1, C * S), r.randint(0, C * S), max(0, n - 1)]) for n in now]
    tokens = sum(max(0, b - a) for a, b in zip(now, new)) + r.choice([0, 3])
    want = build_tables(now, new, tables, ring, state, S, tokens)
    t_now, t_tab, t_ring, t_state = i32(now, cuda), i32(tables, cuda), i32(ring, cuda), i32(state, cuda)
    err = torch.zeros(1, dtype=torch.int32, device=cuda)
    out, ticket = None, None
    if in_place:
        ticket = torch.zeros(1, dtype=torch.int32, device=cuda)
        out = (t_tab, t_now, t_state, torch.full((tokens,), -7, dtype=torch.int64, device=cuda),
               torch.full((R + 1,), -7, dtype=torch.int32, device=cuda))
    got = paged.build_block_tables(t_now, i32(new, cuda), t_tab, t_ring, t_state, S, tokens, out=out, ticket=ticket,
                                   check=False, err=err)
    assert got.tables.tolist() == want[0]
    assert got.lengths.tolist() == want[1]
    assert got.state.tolist() == want[2]
    assert got.slots.tolist() == want[3]
    assert got.starts.tolist() == want[4]
    assert t_ring.tolist() == want[5]
    assert int(err) == (64 if want[6] else 0)
    if in_place:
        assert int(ticket) == 0
    else:
        assert t_now.tolist() == now and t_tab.tolist() == tables and t_state.tolist() == state


def test_tables_refusals_and_bad_lengths(cuda):
    now, tables, ring, state = [4, 0, 8], [[0, -1, -1], [-1, -1, -1], [1, 2, -1]], [3, 4, -1, -1, -1], [0, 2]
    for new, code, exc in (([4, 12, 9], 64, RuntimeError), ([4, -1, 8], 128, ValueError),
                           ([13, 4, 8], 128, ValueError), ([5, 8, 9], 64, RuntimeError)):
        want = build_tables(now, new, tables, ring, state, 4, 30)
        for in_place in (False, True):
            t = [i32(v, cuda) for v in (now, new, tables, ring, state)]
            out = (t[2], t[0], t[4], torch.empty(30, dtype=torch.int64, device=cuda), i32([0] * 4, cuda))
            ticket = i32([0], cuda)
            kw = dict(out=out, ticket=ticket) if in_place else {}
            with pytest.raises(exc):
                paged.build_block_tables(t[0], t[1], t[2], t[3], t[4], 4, 30, check=True, **kw)
            t = [i32(v, cuda) for v in (now, new, tables, ring, state)]
            kw = dict(out=(t[2], t[0], t[4], out[3], out[4]), ticket=ticket) if in_place else {}
            err = i32([0], cuda)
            got = paged.build_block_tables(t[0], t[1], t[2], t[3], t[4], 4, 30, check=False, err=err, **kw)
            assert int(err) == code
            assert [got.tables.tolist(), got.lengths.tolist(), got.state.tolist(), got.slots.tolist(),
                    got.starts.tolist(), t[3].tolist()] == list(want[:6])
    # more tokens than slots: those that fit are right, the rest is not written
    err = i32([0], cuda)
    got = paged.build_block_tables(i32(now, cuda), i32([8, 0, 8], cuda), i32(tables, cuda), i32(ring, cuda),
                                   i32(state, cuda), 4, 2, check=False, err=err)
    assert int(err) == 128 and got.slots.tolist() == [12, 13] and got.starts.tolist() == [0, 4, 4, 4]


def test_tables_of_no_requests(cuda):
    got = paged.build_block_tables(i32([], cuda), i32([], cuda), torch.empty((0, 4), dtype=torch.int32, device=cuda),
                                   i32([1, 2], cuda), i32([1, 2], cuda), 16, 3)
    assert got.state.tolist() == [1, 2] and got.slots.tolist() == [-1] * 3 and got.starts.tolist() == [0]


def test_block_tables_over_many_steps_and_in_a_graph(cuda):
    """The class keeps lengths, tables and ring in step with the host program over growing,
    shrinking and ending requests, eager and replayed."""
    r, R, C, S, N = random.Random(3), 9, 11, 8, 60
    own = paged.BlockTables(N, S, R, C, cuda, free_blocks=range(1, N))
    assert own.tables.shape == (R, C) and own.lengths.tolist() == [0] * R
    now, tables, ring, state = [0] * R, [[-1] * C for _ in range(R)], list(range(1, N)) + [-1], [0, N - 1]
    new = i32([0] * R, cuda)
    slots, starts = torch.empty(400, dtype=torch.int64, device=cuda), i32([0] * (R + 1), cuda)
    err = i32([0], cuda)
    graph = None
    for step in range(12):
        target = [r.choice([n, 0, min(n + r.randint(1, 20), C * S), max(0, n - 5)]) for n in now]
        new.copy_(i32(target, cuda))
        if step == 6:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                own.update(new, 400, slots=slots, starts=starts, err=err)
        if graph is None:
            own.update(new, 400, slots=slots, starts=starts, check=False, err=err)
        else:
            graph.replay()
        tables, now, state, want_slots, want_starts, ring, _, _ = build_tables(now, target, tables, ring, state, S, 400)
        torch.cuda.synchronize()
        assert own.tables.tolist() == tables and own.lengths.tolist() == now and own.state.tolist() == state
        assert slots.tolist() == want_slots and starts.tolist() == want_starts and own.free.tolist() == ring
    held = [b for row in own.tables.tolist() for b in row if b >= 0]
    assert len(set(held)) == len(held) and 0 not in held


# ------------------------------------------------------------------ slot writes
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.int16])
@pytest.mark.parametrize("T,H,D,S,layout,view", [
    (1, 1, 8, 1, "flash", "plain"), (5, 3, 80, 12, "kv_adjacent", "fused"), (33, 8, 128, 16, "flash", "fused"),
    (64, 2, 64, 64, "kv_adjacent", "heads_first"), (17, 5, 7, 4, "flash", "plain"),
    (40, 4, 128, 16, "flash", "off_by_one"), (300, 1, 256, 16, "flash", "fused"), (9, 40, 128, 16, "flash", "plain")])
def test_write_kv(cuda, dtype, T, H, D, S, layout, view):
    gen = torch.Generator(device=cuda).manual_seed(T * H + D)
    rand = lambda *s: torch.randint(-30000, 30000, s, generator=gen, device=cuda).to(torch.int16).view(dtype)
    P = (T + S - 1) // S + 3
    cache = rand(2, P, S, H, D) if layout == "flash" else rand(P, 2, S, H, D)
    if view == "plain":
        key, value = rand(T, H, D), rand(T, H, D)
    elif view == "fused":
        both = rand(T, 4 * H, D)
        key, value = both[:, H:2 * H], both[:, 3 * H:]
    elif view == "heads_first":
        key, value = rand(H, T, D).transpose(0, 1), rand(H, T, D).transpose(0, 1)
    else:
        key, value = rand(T * H * D + 1)[1:].view(T, H, D), rand(T, H, D)
    slots = torch.randperm(P * S, generator=gen, device=cuda)[:T]
    slots[torch.rand(T, generator=gen, device=cuda) < 0.2] = -1
    want = cache.clone()
    for i, s in enumerate(slots.tolist()):
        if s >= 0:
            for part, rows in zip(parts(want), (key, value)):
                part[s // S, s % S] = rows[i]
    paged.write_kv(key, value, cache, slots)
    assert torch.equal(cache.view(torch.int16), want.view(torch.int16))


def test_write_kv_skips_and_flags_bad_slots(cuda):
    cache = torch.zeros((2, 3, 4, 2, 8), dtype=torch.bfloat16, device=cuda)
    rows = torch.ones((4, 2, 8), dtype=torch.bfloat16, device=cuda)
    slots = torch.tensor([12, -2, 1 << 40, 5], device=cuda)
    with pytest.raises(IndexError):
        paged.write_kv(rows, rows, cache, slots, check=True)
    assert float(cache.sum()) == 2 * 2 * 8 and float(cache[:, 1, 1].sum()) == 2 * 2 * 8
    err = i32([0], cuda)
    paged.write_kv(rows, rows, cache, slots, check=False, err=err)
    assert int(err) == 16
    paged.write_kv(rows[:0], rows[:0], cache, slots[:0])


def test_write_kv_past_32_bit_offsets(cuda):
    """A part of 2^32 elements and more: rows behind it land where they should."""
    P, S, H, D = 270000, 16, 8, 128
    cache = torch.empty((2, P, S, H, D), dtype=torch.bfloat16, device=cuda)
    rows = torch.randn((2, 3, H, D), device=cuda).to(torch.bfloat16)
    slots = torch.tensor([0, P * S - 1, P * S - 40000], device=cuda)
    paged.write_kv(rows[0], rows[1], cache, slots)
    for i, s in enumerate(slots.tolist()):
        for part in (0, 1):
            assert torch.equal(cache[part, s // S, s % S], rows[part, i])


# ------------------------------------------------------------------ kept drafts
@pytest.mark.parametrize("R,H,D,S,layers,drafts,width,layout,seed", [
    (1, 1, 8, 1, 1, 1, 1, "flash", 0), (3, 4, 128, 16, 28, 26, 5, "flash", 1), (7, 2, 80, 12, 3, 64, 20, "kv_adjacent", 2),
    (5, 3, 7, 4, 2, 30, 30, "flash", 3), (2, 8, 128, 16, 2, 300, 150, "flash", 4)])
def test_keep_drafts(cuda, R, H, D, S, layers, drafts, width, layout, seed):
    r = random.Random(seed)
    base = [r.choice([0, 1, S - 1, r.randint(0, 60)]) for _ in range(R)]
    C = max(-(-(n + drafts) // S) for n in base)
    P = R * C + 2
    ids = r.sample(range(P), R * C)
    tables = i32([ids[i * C:(i + 1) * C] for i in range(R)], cuda)
    paths = []
    for _ in range(R):
        n = r.randint(0, min(width, drafts))
        paths.append(sorted(r.sample(range(drafts), n)) + [-1] * (width - n))
    paths[0] = sorted(r.sample(range(drafts), min(width, drafts))) + [-1] * (width - min(width, drafts))
    shape = (2, P, S, H, D) if layout == "flash" else (P, 2, S, H, D)
    caches = [torch.randn(shape, device=cuda).to(torch.bfloat16) for _ in range(layers)]
    want = [c.clone() for c in caches]
    for cache in want:
        for part in parts(cache):
            for n, path, row in zip(base, paths, tables.tolist()):
                for i, j in enumerate(p for p in path if p >= 0):
                    a, b = n + j, n + i
                    part[row[b // S], b % S] = part[row[a // S], a % S].clone()
    got = paged.keep_drafts(paged.LayerCaches(caches), tables, i32(base, cuda), i32(paths, cuda))
    assert got.tolist() == [n + sum(j >= 0 for j in p) for n, p in zip(base, paths)]
    for c, w in zip(caches, want):
        assert torch.equal(c, w)


def test_keep_drafts_leaves_bad_paths_alone(cuda):
    cache = torch.randn((2, 6, 4, 1, 8), device=cuda).to(torch.bfloat16)
    before = cache.clone()
    lengths = i32([3, 2, 1, 0], cuda)
    tables = i32([[0, 1], [2, 9], [3, 4], [-1, 5]], cuda)
    for path, code, kept in (([2, 2, -1], 128, 3), ([1, 0, -1], 128, 3), ([0, 5, -1], 128, 3)):
        err = i32([0], cuda)
        got = paged.keep_drafts([cache], tables[:1], lengths[:1], i32([path], cuda), check=False, err=err)
        assert int(err) == code and got.tolist() == [kept] and torch.equal(cache, before)
        with pytest.raises(ValueError):
            paged.keep_drafts([cache], tables[:1], lengths[:1], i32([path], cuda), check=True)
    for r, path in ((1, [1, 2]), (3, [0, 4])):
        with pytest.raises(IndexError):
            paged.keep_drafts([cache], tables[r:r + 1], lengths[r:r + 1], i32([path], cuda), check=True)
        assert torch.equal(cache, before)
    # a bad request does not keep a good one from being served
    err = i32([0], cuda)
    got = paged.keep_drafts([cache], tables[1:3].contiguous(), lengths[1:3].contiguous(), i32([[1, 2], [1, 3]], cuda),
                            check=False, err=err)
    assert int(err) == 16 and got.tolist() == [2, 3]
    assert torch.equal(cache[:, 3, 1], before[:, 3, 2]) and torch.equal(cache[:, 3, 2], before[:, 4, 0])


def test_paged_operators_on_another_stream(cuda):
    """Work is enqueued on the stream that is current at the call."""
    side = torch.cuda.Stream()
    cache = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16, device=cuda)
    rows = torch.randn((5, 2, 64), device=cuda).to(torch.bfloat16)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own = paged.BlockTables(4, 16, 1, 4, cuda)
        slots, starts = own.update(i32([5], cuda), 5, check=False)
        paged.write_kv(rows, rows, cache, slots, check=False)
        out = paged.tree_attention(rows, cache, own.tables, own.lengths, starts, max_query=5, check=False)
        kept = paged.keep_drafts([cache], own.tables, i32([0], cuda), i32([[1, 3]], cuda), check=False)
    side.synchronize()
    assert own.lengths.tolist() == [5] and kept.tolist() == [2]
    assert torch.equal(cache[0, 0, 0], rows[1]) and torch.equal(cache[1, 0, 1], rows[3])
    assert torch.equal(out[0], rows[0])  # the first query sees itself alone
