"""Rows that share blocks on the GPU against plain host programs: forked tables, copied blocks, a
compacted pool."""

import random

import pytest
import torch

from kvserve_amd import paged

from _paged_ref import parts
from _shared_ref import blocks, compact, consistent, fork

pytestmark = pytest.mark.gpu


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def random_step(r, lengths, C, S):
    """Parents and new lengths of all sorts."""
    R, top = len(lengths), C * S
    parents, new = [], []
    for i in range(R):
        u = r.random()
        if u < 0.1:
            p, n = -1, 0
        elif u < 0.25:
            p, n = -1, r.randint(0, top)
        elif u < 0.4:
            p, n = i, lengths[i]
        elif u < 0.6:
            p = r.randrange(R)
            n = r.randint(0, lengths[p])
        else:
            p = r.randrange(max(0, i - 3), min(R, i + 4))
            n = lengths[p] + r.choice([0, 1, 1, 5, S])
        parents.append(p)
        new.append(min(n, top))
    return parents, new


class Pool:
    """A host program's rows and ring, kept over steps."""

    def __init__(self, r, R, C, S, N, away=()):
        ids = [b for b in range(N) if b not in away]
        r.shuffle(ids)
        head = r.randrange(N)
        self.S, self.away = S, away
        self.tables, self.lengths, self.shares = [[-1] * C for _ in range(R)], [0] * R, [0] * N
        self.ring = [-1] * N
        for i, b in enumerate(ids):
            self.ring[(head + i) % N] = b
        self.state = [head, len(ids)]

    def device(self, dev):
        return [i32(v, dev) for v in (self.lengths, self.tables, self.shares, self.ring, self.state)]

    def take(self, want):
        self.tables, self.lengths, self.shares, self.state, _, _, _, self.ring, _ = want
        consistent(self.tables, self.lengths, self.shares, self.ring, self.state, self.S, self.away)


def run_fork(dev, pool, parents, new, tokens, in_place, workspace):
    lengths, tables, shares, ring, state = pool.device(dev)
    R = len(pool.lengths)
    err, out = i32([0], dev), None
    if in_place:
        out = (tables, lengths, shares, state, torch.full((tokens,), -7, dtype=torch.int64, device=dev),
               torch.full((R + 1,), -7, dtype=torch.int32, device=dev),
               torch.full((R, 3), -7, dtype=torch.int32, device=dev))
    got = paged.fork_block_tables(lengths, None if parents is None else i32(parents, dev),
                                  new if isinstance(new, int) else i32(new, dev), tables, shares, ring, state, pool.S,
                                  tokens, out=out, workspace=workspace, check=False, err=err)
    if not in_place:
        assert [t.tolist() for t in (lengths, tables, shares, state)] == [pool.lengths, pool.tables, pool.shares,
                                                                          pool.state]
    return [t.tolist() for t in got] + [ring.tolist()], int(err)


@pytest.mark.parametrize("R,C,S,N,seed", [(1, 1, 1, 3, 0), (2, 3, 4, 9, 1), (4, 7, 16, 40, 2), (9, 12, 12, 90, 3),
                                          (33, 40, 1, 900, 4), (70, 9, 16, 1023, 5), (257, 16, 16, 2500, 6),
                                          (600, 33, 128, 9000, 7)])
@pytest.mark.parametrize("in_place", [False, True])
def test_forks_match_a_host_program(cuda, R, C, S, N, seed, in_place):
    r = random.Random(seed)
    away = (0, N // 2) if N > 5 else ()
    pool = Pool(r, R, C, S, N, away)
    workspace = paged.fork_workspace(N, R, C, cuda)
    refused = 0
    for step in range(8):
        parents, new = random_step(r, pool.lengths, C, S)
        if step == 3:
            parents = None
            new = [r.randint(0, n) if r.random() < 0.7 else n for n in pool.lengths]
        if step == 5:
            new = 1
        tokens = 0
        if not isinstance(new, int):
            tokens = sum(max(0, n - (pool.lengths[p] if p >= 0 else 0))
                         for n, p in zip(new, parents or range(R))) + r.choice([0, 3])
        else:
            tokens = R
        want = fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, tokens)
        got, err = run_fork(cuda, pool, parents, new, tokens, in_place, workspace)
        assert err == {None: 0, "blocks": 64, "length": 128}[want[8]]
        for k in range(8):
            assert got[k] == want[k], (step, k)
        refused += want[8] is not None
        pool.take(want)
        assert int(workspace[:N].abs().sum()) == 0  # a block's holders are counted anew in every call
    assert refused < 8


def test_fork_of_one_prompt_into_many_and_a_long_list_of_children(cuda):
    """4096 rows of one parent, cut at every length: the longest list of children there is."""
    r, R, C, S = random.Random(1), 4096, 40, 4
    N = R * 3
    pool = Pool(r, R, C, S, N)
    first = [150] + [0] * (R - 1)
    pool.take(fork(pool.lengths, None, first, pool.tables, pool.shares, pool.ring, pool.state, S, 150))
    for parents, new in (([0] * R, [r.randint(0, 152) for _ in range(R)]),
                         ([r.randrange(R) for _ in range(R)], 0), ([r.choice([-1, -1, i]) for i in range(R)], 0)):
        want = fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, 3 * R)
        got, err = run_fork(cuda, pool, parents, new, 3 * R, True, None)
        assert err == {None: 0, "blocks": 64}[want[8]] and got == list(want[:8])
        pool.take(want)


def test_unaligned_rows_and_long_rows(cuda):
    """Rows whose entries are not 16-byte aligned, and rows of many parts."""
    for C, offset in ((5, 0), (3000, 0), (8, 1), (2048, 3)):
        r = random.Random(C)
        R, S, N = 3, 2, 3 * C + 5
        pool = Pool(r, R, C, S, N)
        for step in range(4):
            parents, new = random_step(r, pool.lengths, C, S)
            tokens = sum(max(0, n - (pool.lengths[p] if p >= 0 else 0)) for n, p in zip(new, parents))
            want = fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, tokens)
            lengths, tables, shares, ring, state = pool.device(cuda)
            room = torch.zeros(R * C + offset, dtype=torch.int32, device=cuda)
            room[offset:] = tables.flatten()
            err = i32([0], cuda)
            got = paged.fork_block_tables(lengths, i32(parents, cuda), i32(new, cuda), room[offset:].view(R, C), shares,
                                          ring, state, S, tokens, check=False, err=err)
            assert [t.tolist() for t in got] == list(want[:7]) and ring.tolist() == want[7]
            assert int(err) == {None: 0, "blocks": 64}[want[8]]
            pool.take(want)


def test_refused_forks_change_nothing(cuda):
    r, R, C, S, N = random.Random(2), 4, 3, 4, 10
    pool = Pool(r, R, C, S, N)
    pool.take(fork(pool.lengths, None, [12, 9, 0, 4], pool.tables, pool.shares, pool.ring, pool.state, S, 25))
    keep = [0, 1, 2, 3]
    for parents, new, tokens, code, exc in (
            (keep, [12, 9, 12, 12], 40, 64, RuntimeError),     # five blocks, three are free
            (keep, [12, 9, 1, 4], 0, 128, ValueError),         # a token more than slots
            (keep, [12, 9, 13, 4], 40, 128, ValueError),       # past the row's end
            (keep, [12, -1, 0, 4], 40, 128, ValueError),
            ([0, 4, 2, 3], [12, 9, 0, 4], 40, 128, ValueError),
            ([0, -2, 2, 3], [12, 9, 0, 4], 40, 128, ValueError),
            ([0, 0, 0, 0], 1, 40, 128, ValueError)):           # 12 + 1 past the row's end
        want = fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, tokens)
        assert want[8] == {64: "blocks", 128: "length"}[code]
        for in_place in (False, True):
            got, err = run_fork(cuda, pool, parents, new, tokens, in_place, None)
            assert err == code and got == list(want[:8])
        lengths, tables, shares, ring, state = pool.device(cuda)
        with pytest.raises(exc):
            paged.fork_block_tables(lengths, i32(parents, cuda), new if isinstance(new, int) else i32(new, cuda), tables,
                                    shares, ring, state, S, tokens, check=True)
    # a ring's count and a length that cannot be
    for at, value in ((4, [0, N + 1]), (4, [0, -1]), (0, [12, 13, 0, 4]), (0, [12, -9, 0, 4])):
        held = pool.device(cuda)
        held[at] = i32(value, cuda)
        lengths, tables, shares, ring, state = held
        err = i32([0], cuda)
        got = paged.fork_block_tables(lengths, None, 0, tables, shares, ring, state, S, 4, check=False, err=err)
        assert int(err) == 128 and torch.equal(got.tables, tables) and torch.equal(got.state, state)
        assert torch.equal(got.lengths, lengths) and got.slots.tolist() == [-1] * 4


def test_ids_outside_the_pool_are_flagged(cuda):
    tables, lengths = i32([[0, 99], [-5, 1]], cuda), i32([8, 8], cuda)
    shares, ring, state = i32([0] * 4, cuda), i32([2, 3, -1, -1], cuda), i32([0, 2], cuda)
    err = i32([0], cuda)
    got = paged.fork_block_tables(lengths, i32([-1, -1], cuda), 0, tables, shares, ring, state, 4, 0, check=False,
                                  err=err)
    assert int(err) == 16 and ring.tolist() == [2, 3, 0, 1] and got.state.tolist() == [0, 4]
    with pytest.raises(IndexError):
        paged.fork_block_tables(lengths, i32([0, 0], cuda), 0, tables, shares, ring.clone(), state, 4, 0, check=True)


def test_no_rows(cuda):
    e = i32([], cuda)
    got = paged.fork_block_tables(e, e, e, torch.empty((0, 4), dtype=torch.int32, device=cuda), i32([0] * 3, cuda),
                                  i32([1, 2, 0], cuda), i32([1, 2], cuda), 16, 3)
    assert got.state.tolist() == [1, 2] and got.slots.tolist() == [-1] * 3 and got.starts.tolist() == [0]
    assert got.shares.tolist() == [0] * 3
    got = paged.compact_block_tables(e, torch.empty((0, 4), dtype=torch.int32, device=cuda), i32([0] * 3, cuda),
                                     i32([1, 2, 0], cuda), i32([2, 2], cuda), 16)
    assert got.free.tolist() == [0, 1, -1] and got.state.tolist() == [0, 2]


def test_shared_tables_over_many_steps_and_in_a_graph(cuda):
    r, R, C, S, N = random.Random(4), 12, 9, 8, 80
    own = paged.SharedBlockTables(N, S, R, C, cuda, free_blocks=range(1, N))
    pool = Pool(random.Random(0), R, C, S, N, (0,))
    pool.ring, pool.state = list(range(1, N)) + [-1], [0, N - 1]
    parents_t, new_t, err = i32([0] * R, cuda), i32([0] * R, cuda), i32([0], cuda)
    slots, starts = torch.empty(900, dtype=torch.int64, device=cuda), i32([0] * (R + 1), cuda)
    graph, done = None, 0
    for step in range(16):
        parents, new = random_step(r, pool.lengths, C, S)
        parents_t.copy_(i32(parents, cuda))
        new_t.copy_(i32(new, cuda))
        if step == 6:
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                own.fork(parents_t, new_t, 900, slots=slots, starts=starts, err=err)
        err.zero_()
        if graph is None:
            own.fork(parents_t, new_t, 900, slots=slots, starts=starts, check=False, err=err)
        else:
            graph.replay()
        torch.cuda.synchronize()
        want = fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, 900)
        got = (own.tables, own.lengths, own.shares, own.state, slots, starts, own.copies, own.free)
        assert [t.tolist() for t in got] == list(want[:8]) and int(err) == {None: 0, "blocks": 64}[want[8]]
        done += want[8] is None
        pool.take(want)
        if step in (4, 9, 13):
            moves = own.compact()
            torch.cuda.synchronize()
            want = compact(pool.lengths, pool.tables, pool.shares, pool.ring, pool.state, S)
            assert [t.tolist() for t in (own.tables, own.shares, own.free, own.state, moves)] == list(want)
            pool.tables, pool.shares, pool.ring, pool.state = want[:4]
    assert done > 8
    # shrinking into shared blocks keeps the others' tokens
    own.fork(i32([-1] * R, cuda), i32([20] + [0] * (R - 1), cuda), 20)
    own.fork(i32([0] * R, cuda), i32([20] * R, cuda), 0)
    own.update(i32([13] + [20] * (R - 1), cuda), 0)
    torch.cuda.synchronize()
    assert own.copies[0, 2] == 5 and own.tables[0, 1] != own.tables[1, 1] and own.tables[0, 0] == own.tables[1, 0]


# ------------------------------------------------------------------ copied blocks
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("H,D,S,layers,n,layout,offset", [
    (1, 8, 1, 1, 1, "flash", 0), (4, 128, 16, 28, 7, "flash", 0), (5, 80, 12, 3, 50, "kv_adjacent", 0),
    (3, 7, 4, 2, 30, "flash", 0), (2, 64, 16, 2, 20, "flash", 1), (8, 256, 64, 1, 5, "kv_adjacent", 0),
    (1, 2, 3, 1, 9000, "flash", 0), (1, 8, 2, 1, 20000, "kv_adjacent", 0)])
def test_copy_blocks(cuda, dtype, H, D, S, layers, n, layout, offset):
    r = random.Random(n)
    P = 2 * n + 1
    shape = (2, P, S, H, D) if layout == "flash" else (P, 2, S, H, D)
    size = 2 * P * S * H * D
    caches = [torch.randint(-30000, 30000, (size + offset,), device=cuda).to(torch.int16).view(dtype)[offset:].view(shape)
              for _ in range(layers)]
    ids = list(range(P))
    r.shuffle(ids)
    rows = []
    for i in range(n):
        t = r.choice([0, 1, S, r.randint(0, S)])
        rows.append([ids[2 * i], ids[2 * i + 1], t] if r.random() < 0.8 or n == 1 else [-1, -1, -1])
    want = [c.clone() for c in caches]
    moves = i32(rows, cuda).long()
    moves = moves[moves[:, 0] >= 0]
    place = torch.arange(S, device=cuda)
    used = place.unsqueeze(0) < moves[:, 2:]
    for cache in want:
        for part in parts(cache):
            mixed = torch.where(used[:, :, None, None], part[moves[:, 0]].view(torch.int16),
                                part[moves[:, 1]].view(torch.int16))
            part.view(torch.int16)[moves[:, 1]] = mixed
    paged.copy_blocks(paged.LayerCaches(caches), i32(rows, cuda))
    for c, w in zip(caches, want):
        assert torch.equal(c.view(torch.int16), w.view(torch.int16))


def test_copy_blocks_refuses_bad_rows_one_by_one(cuda):
    cache = torch.randn((2, 6, 4, 1, 8), device=cuda).to(torch.bfloat16)
    before = cache.clone()
    for row, code, exc in (([0, 6, 4], 16, IndexError), ([6, 0, 4], 16, IndexError), ([0, -1, 4], 16, IndexError),
                           ([0, 1, 5], 128, ValueError), ([0, 1, -1], 128, ValueError)):
        err = i32([0], cuda)
        paged.copy_blocks([cache], i32([row], cuda), check=False, err=err)
        assert int(err) == code and torch.equal(cache, before)
        with pytest.raises(exc):
            paged.copy_blocks([cache], i32([row], cuda), check=True)
        err.zero_()
        paged.copy_blocks([cache], i32([row, [2, 3, 3], [-1, -1, -1]], cuda), check=False, err=err)
        assert int(err) == code and torch.equal(cache[:, 3, :3], before[:, 2, :3])
        assert torch.equal(cache[:, 3, 3:], before[:, 3, 3:])
        cache.copy_(before)
    paged.copy_blocks([cache], i32([[1, 1, 4]], cuda))
    paged.copy_blocks([cache], i32([], cuda).view(0, 3))
    assert torch.equal(cache, before)


def test_copy_blocks_past_32_bit_offsets(cuda):
    P, S, H, D = 270000, 16, 8, 128
    cache = torch.empty((2, P, S, H, D), dtype=torch.bfloat16, device=cuda)
    cache[:, P - 1] = torch.randn((2, S, H, D), device=cuda).to(torch.bfloat16)
    cache[:, 1] = 0
    cache[:, P - 7] = 0
    paged.copy_blocks([cache], i32([[P - 1, 1, S], [-1, 0, 0]], cuda))
    paged.copy_blocks([cache], i32([[1, P - 7, 9]], cuda))
    assert torch.equal(cache[:, 1], cache[:, P - 1]) and torch.equal(cache[:, P - 7, :9], cache[:, P - 1, :9])
    assert float(cache[:, P - 7, 9:].abs().sum()) == 0


# ------------------------------------------------------------------ a compacted pool
@pytest.mark.parametrize("R,C,S,N,seed", [(1, 1, 1, 1, 0), (1, 3, 4, 2, 1), (3, 5, 16, 17, 2), (20, 9, 12, 200, 3),
                                          (40, 60, 1, 1023, 4), (40, 60, 2, 1024, 5), (40, 60, 1, 1025, 6),
                                          (300, 30, 16, 5000, 7), (90, 1500, 1, 70000, 8)])
@pytest.mark.parametrize("in_place", [False, True])
def test_compactions_match_a_host_program(cuda, R, C, S, N, seed, in_place):
    r = random.Random(seed)
    away = r.sample(range(N), min(3, N // 4))
    pool = Pool(r, R, C, S, N, away)
    workspace = paged.compact_workspace(N, cuda)
    for step in range(5):
        lengths, tables, shares, ring, state = pool.device(cuda)
        want = compact(pool.lengths, pool.tables, pool.shares, pool.ring, pool.state, S)
        out = None
        if in_place:
            out = (tables, shares, ring, state, torch.full((N // 2, 3), -7, dtype=torch.int32, device=cuda))
        err = i32([0], cuda)
        got = paged.compact_block_tables(lengths, tables, shares, ring, state, S, out=out, workspace=workspace,
                                         check=False, err=err)
        assert int(err) == 0 and [t.tolist() for t in got] == list(want)
        if not in_place:
            assert [t.tolist() for t in (tables, shares, ring, state)] == [pool.tables, pool.shares, pool.ring, pool.state]
        assert int(workspace[:-(-N // 16) * 8].abs().sum()) == 0
        for _ in range(3):
            parents, new = random_step(r, pool.lengths, C, S)
            if step == 3:
                new = [0] * R  # nothing held
            pool.take(fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, R * C * S))


def test_a_full_pool_and_bad_ids(cuda):
    i = lambda v: i32(v, cuda)
    got = paged.compact_block_tables(i([8, 8]), i([[3, 0], [1, 2]]), i([0] * 4), i([-1] * 4), i([2, 0]), 4)
    assert got.tables.tolist() == [[3, 0], [1, 2]] and got.state.tolist() == [0, 0]
    assert got.copies.tolist() == [[-1] * 3] * 2 and got.free.tolist() == [-1] * 4
    err = i([0])
    # an id outside the pool keeps its name; one that is held and free is held
    got = paged.compact_block_tables(i([8, 4]), i([[3, 9], [5, -1]]), i([0] * 6), i([1, 0, 3, -1, -1, 9]), i([5, 4]), 4,
                                     check=False, err=err)
    assert int(err) == 16
    assert got.tables.tolist() == [[0, 9], [1, -1]] and got.free.tolist()[:2] == [3, 5]
    assert got.copies.tolist() == [[3, 0, 4], [5, 1, 4], [-1] * 3]
    for lengths, state in (([9, 4], [0, 0]), ([-1, 4], [0, 0]), ([4, 4], [0, 7]), ([4, 4], [0, -1])):
        with pytest.raises(ValueError):
            paged.compact_block_tables(i(lengths), i([[3, 4], [5, -1]]), i([0] * 6), i([0, 1, 2, 0, 1, 2]), i(state), 4,
                                       check=True)


def test_rows_behind_a_sequence_do_not_matter(cuda):
    """Entries behind a row's tokens may hold anything."""
    i = lambda v: i32(v, cuda)
    got = paged.compact_block_tables(i([4]), i([[2, 1 << 30, -9]]), i([0] * 3), i([0, 1, -1]), i([0, 2]), 4)
    assert got.tables.tolist() == [[0, -1, -1]]
    got = paged.fork_block_tables(i([4]), None, 1, i([[2, 1 << 30, -9]]), i([0] * 3), i([0, 1, -1]), i([0, 2]), 4, 1)
    assert got.tables.tolist() == [[2, 0, -1]] and got.slots.tolist() == [0]


def test_on_another_stream_with_work_before_it(cuda):
    """Every call goes to the stream that is current, behind what is there."""
    side = torch.cuda.Stream()
    big = torch.randn((3000, 3000), device=cuda)
    cache = torch.zeros((2, 8, 4, 1, 8), dtype=torch.bfloat16, device=cuda)
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        own = paged.SharedBlockTables(8, 4, 3, 2, cuda)
        for _ in range(20):
            big = big @ big * 1e-3
        first = i32([6, 0, 0], cuda)
        logits = torch.zeros((3, 50), device=cuda) + big.sum() * 0
        logits[0, 7], logits[0, 9] = 3.0, 2.0
        scores = torch.tensor([0.0, float("-inf"), float("-inf")], device=cuda)
        slots, _ = own.update(first, 6, check=False)
        rows = torch.arange(48, device=cuda).view(6, 1, 8).to(torch.bfloat16)
        paged.write_kv(rows, rows, cache, slots, check=False)
        best = paged.select_beams(logits, scores, 3, check=False)
        slots, starts = own.fork(best.parents, 1, 3, check=False)
        paged.copy_blocks([cache], own.copies, check=False)
        paged.copy_blocks([cache], own.compact(check=False), check=False)
    side.synchronize()
    assert best.tokens.tolist() == [7, 9, 0] and own.lengths.tolist() == [7, 7, 7] and own.shares.tolist()[0] == 2
    for row in own.tables.tolist():
        assert torch.equal(torch.cat([cache[0, row[0]], cache[0, row[1], :2]]), rows)


def test_two_tables_side_by_side(cuda):
    """Tables have workspaces of their own: their calls may overlap."""
    r, streams = random.Random(9), [torch.cuda.Stream() for _ in range(2)]
    R, C, S, N = 40, 12, 4, 600
    own = [paged.SharedBlockTables(N, S, R, C, cuda) for _ in streams]
    pools = [Pool(random.Random(0), R, C, S, N) for _ in streams]
    for pool in pools:
        pool.ring, pool.state = list(range(N)), [0, N]
    for _ in range(6):
        steps = []
        for pool in pools:
            parents, new = random_step(r, pool.lengths, C, S)
            steps.append((i32(parents, cuda), i32(new, cuda)))
            pool.take(fork(pool.lengths, parents, new, pool.tables, pool.shares, pool.ring, pool.state, S, 4000))
        torch.cuda.synchronize()
        for stream, tables, (parents, new) in zip(streams, own, steps):
            with torch.cuda.stream(stream):
                tables.fork(parents, new, 4000, check=False)
        torch.cuda.synchronize()
        for tables, pool in zip(own, pools):
            got = (tables.tables, tables.lengths, tables.shares, tables.state, tables.free)
            assert [t.tolist() for t in got] == [pool.tables, pool.lengths, pool.shares, pool.state, pool.ring]
