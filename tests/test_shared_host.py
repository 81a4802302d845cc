"""Refusals and host logic of the operators of rows that share blocks that need no GPU (nothing is
launched), and their host programs held to what they describe."""

import ctypes
import random

import pytest
import torch

from kvserve_amd import _lib, paged

from _shared_ref import compact, consistent, fork, select

P = 4096  # an address that is never read: the calls are refused first


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(_lib.ForkArgs) == 17 * 8 + 6 * 4
    assert ctypes.sizeof(_lib.CompactArgs) == 13 * 8 + 4 * 4
    assert ctypes.sizeof(_lib.SelectArgs) == 12 * 8 + 6 * 4


def fork_args(**kw):
    a = {n: P * (i + 1) for i, (n, t) in enumerate(_lib.ForkArgs._fields_) if t is ctypes.c_void_p}
    a.update(workspace_bytes=1 << 40, rows=4, columns=8, blocks=64, block_size=16, max_tokens=9, grow=0)
    a.update(kw)
    return _lib.ForkArgs(**a)


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(rows=4097), dict(columns=0), dict(blocks=0), dict(block_size=0), dict(max_tokens=-1),
    dict(grow=-1), dict(columns=1 << 27), dict(blocks=1 << 27), dict(blocks=(1 << 24) + 1, block_size=1), dict(rows=4096, columns=1 << 20, block_size=1),
    dict(workspace_bytes=0), dict(workspace=None), dict(workspace=P + 4), dict(lengths=None), dict(tables=None),
    dict(shares=None), dict(free_blocks=None), dict(state=None), dict(out_tables=None), dict(out_lengths=None),
    dict(out_shares=None), dict(out_state=None), dict(slots=None), dict(starts=None), dict(copies=None)])
def test_fork_refuses_bad_arguments(kw):
    assert _lib.load().kvmi_fork_tables(fork_args(**kw), None) == _lib.EINVAL


def test_fork_refuses_outputs_over_some_inputs():
    lib, good = _lib.load(), fork_args()
    pairs = [("out_tables", "tables"), ("out_lengths", "lengths"), ("out_shares", "shares"), ("out_state", "state")]
    for i in range(1, 15):  # every mixture
        kw = {o: getattr(good, n) for k, (o, n) in enumerate(pairs) if i >> k & 1}
        assert lib.kvmi_fork_tables(fork_args(**kw), None) == _lib.EINVAL
    for name in ("parents", "new_lengths"):
        assert lib.kvmi_fork_tables(fork_args(out_lengths=getattr(good, name)), None) == _lib.EINVAL
    assert lib.kvmi_fork_tables(None, None) == _lib.EINVAL
    assert lib.kvmi_fork_tables(fork_args(rows=0), None) == 0


@pytest.mark.parametrize("kw", [
    dict(rows=-1), dict(columns=0), dict(blocks=0), dict(block_size=0), dict(columns=1 << 27), dict(blocks=1 << 27),
    dict(blocks=(1 << 24) + 1, block_size=1), dict(rows=1 << 20, columns=1 << 20, block_size=1), dict(workspace=None), dict(workspace=P + 4),
    dict(workspace_bytes=8), dict(lengths=None), dict(tables=None), dict(shares=None), dict(free_blocks=None),
    dict(state=None), dict(out_tables=None), dict(out_shares=None), dict(out_free=None), dict(out_state=None),
    dict(copies=None), dict(out_tables=2 * P), dict(out_shares=3 * P), dict(out_free=4 * P), dict(out_state=5 * P)])
def test_compact_refuses_bad_arguments(kw):
    a = {n: P * (i + 1) for i, (n, t) in enumerate(_lib.CompactArgs._fields_) if t is ctypes.c_void_p}
    a.update(workspace_bytes=1 << 40, rows=4, columns=8, blocks=64, block_size=16)
    a.update(kw)
    assert _lib.load().kvmi_compact_tables(_lib.CompactArgs(**a), None) == _lib.EINVAL


def select_args(**kw):
    a = {n: P * (i + 1) for i, (n, t) in enumerate(_lib.SelectArgs._fields_) if t is ctypes.c_void_p}
    a.update(workspace_bytes=1 << 40, row_stride=1000, dtype=0, requests=2, beams=4, vocab=1000, count=8, end_token=-1)
    a.update(kw)
    return _lib.SelectArgs(**a)


@pytest.mark.parametrize("kw", [
    dict(requests=-1), dict(requests=20000), dict(beams=0), dict(beams=65, count=64), dict(count=3), dict(count=65),
    dict(vocab=0), dict(vocab=0x7fffffff), dict(end_token=-2), dict(row_stride=-1), dict(dtype=3), dict(dtype=-1)])
def test_select_refuses_bad_sizes(kw):
    lib = _lib.load()
    assert lib.kvmi_select_beams(select_args(**kw), None) == _lib.EINVAL
    assert lib.kvmi_select_workspace_bytes(select_args(**kw)) == _lib.EINVAL


@pytest.mark.parametrize("kw", [dict(workspace=None), dict(workspace=P + 8), dict(workspace_bytes=16),
                                dict(logits=P + 1), dict(logits=P + 2, dtype=2)] + [
    {n: None} for n in ("logits", "scores", "parents", "tokens", "next_scores", "all_parents", "all_tokens",
                        "all_scores")])
def test_select_refuses_bad_addresses(kw):
    assert _lib.load().kvmi_select_beams(select_args(**kw), None) == _lib.EINVAL
    assert _lib.load().kvmi_select_beams(select_args(requests=0), None) == 0


@pytest.mark.parametrize("cache", [dict(num_blocks=0), dict(block_size=0), dict(num_heads=0), dict(head_dim=0),
                                   dict(part_stride=-1), dict(block_stride=8)])
def test_copy_refuses_bad_caches_and_sizes(cache):
    c = dict(base=0, part_stride=4 * 16 * 128, block_stride=16 * 128, num_blocks=4, block_size=16, num_heads=2, head_dim=64)
    lib = _lib.load()
    good = _lib.Cache(*c.values())
    assert lib.kvmi_copy_blocks(good, P, 1, P, 0, None, None) == 0
    for bases, layers, copies, n in ((P, 0, P, 1), (P, 32768, P, 1), (P, 1, P, -1), (None, 1, P, 1), (P, 1, None, 1)):
        assert lib.kvmi_copy_blocks(good, bases, layers, copies, n, None, None) == _lib.EINVAL
    c.update(cache)
    assert lib.kvmi_copy_blocks(_lib.Cache(*c.values()), P, 1, P, 1, None, None) == _lib.EINVAL


def test_workspaces_take_positive_sizes():
    lib = _lib.load()
    assert lib.kvmi_fork_workspace_bytes(0, 1, 1) == _lib.EINVAL and lib.kvmi_fork_workspace_bytes(1, -1, 1) == _lib.EINVAL
    assert lib.kvmi_compact_workspace_bytes(0) == _lib.EINVAL
    assert lib.kvmi_compact_workspace_bytes((1 << 24) + 1) == lib.kvmi_fork_workspace_bytes((1 << 24) + 1, 1, 1) == _lib.EINVAL
    assert paged.fork_workspace(100, 4, 8, "cpu").sum() == 0 and paged.compact_workspace(100, "cpu").numel() > 50
    for bad in ((0, 1, 1), (1, 0, 1), (1, 1, 1 << 31), (1.0, 1, 1), (True, 1, 1)):
        with pytest.raises(ValueError):
            paged.fork_workspace(*bad, "cpu")
    with pytest.raises(ValueError):
        paged.compact_workspace(-3, "cpu")


def test_wrappers_refuse_host_tensors_and_bad_sizes():
    i = lambda *s: torch.zeros(s, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        paged.fork_block_tables(i(1), None, 1, i(1, 2), i(4), i(4), i(2), 16, 5)
    for size, tokens in ((0, 5), (16, -1), (1.0, 5), (16, 1 << 31)):
        with pytest.raises(ValueError):
            paged.fork_block_tables(i(1), None, 1, i(1, 2), i(4), i(4), i(2), size, tokens)
    with pytest.raises(TypeError):
        paged.fork_block_tables(i(1).long(), None, 1, i(1, 2), i(4), i(4), i(2), 16, 5)
    with pytest.raises(ValueError, match="CUDA"):
        paged.compact_block_tables(i(1), i(1, 2), i(4), i(4), i(2), 16)
    with pytest.raises(ValueError):
        paged.compact_block_tables(i(1), i(1, 2), i(4), i(4), i(2), 0)
    with pytest.raises(TypeError):
        paged.select_beams(torch.zeros(4, 9), torch.zeros(4), 2)
    with pytest.raises(ValueError, match="4096"):
        paged.SharedBlockTables(8, 16, 4097, 4, "cpu")


def test_tables_begin_empty():
    own = paged.SharedBlockTables(9, 16, 3, 4, "cpu", free_blocks=[5, 2])
    assert own.shares.tolist() == [0] * 9 and own.copies.tolist() == [[-1] * 3] * 3 and own.state.tolist() == [0, 2]


def test_the_host_programs_keep_a_pool_whole():
    """Random forks of all sorts: every block stays held or free, counted as often as it is held."""
    r = random.Random(0)
    for R, C, S, N in ((3, 5, 4, 12), (20, 8, 16, 90), (9, 30, 1, 120)):
        tables, lengths, shares, ring, state = [[-1] * C for _ in range(R)], [0] * R, [0] * N, list(range(N)), [0, N]
        served = 0
        for step in range(40):
            parents = [r.choice([-1, i, r.randrange(R)]) for i in range(R)]
            new = [r.randint(0, C * S // 2) for _ in range(R)]
            got = fork(lengths, parents, new, tables, shares, ring, state, S, R * C * S)
            tables, lengths, shares, state, slots, starts, copies, ring, error = got
            served += error is None
            consistent(tables, lengths, shares, ring, state, S)
            assert len(set(s for s in slots if s >= 0)) == starts[-1]
            fresh = {b for row in tables for b in row}
            assert all(b in fresh and a != b for a, b, t in copies if t > 0)
            if step % 7 == 0:
                tables, shares, ring, state, moves = compact(lengths, tables, shares, ring, state, S)
                consistent(tables, lengths, shares, ring, state, S)
                assert max([b for row in tables for b in row], default=-1) < N - state[1]
        assert served > 5


def test_the_selection_in_64_bits_is_the_sorted_list():
    gen = torch.Generator().manual_seed(1)
    for beams, V, count in ((1, 5, 3), (3, 40, 7), (4, 9, 40)):
        x, s = torch.randint(-3, 4, (2 * beams, V), generator=gen).float(), torch.randint(-2, 0, (2 * beams,), generator=gen).float()
        got = select(x, s, beams, count, end=2)
        v = torch.log_softmax(x.double(), 1) + s.double()[:, None]
        for q in range(2):
            part = v[q * beams:(q + 1) * beams].flatten()
            want = sorted(part.tolist(), reverse=True)[:count]
            have = got[5][q][:len(want)]
            assert torch.allclose(have, torch.tensor(want, dtype=torch.float64), atol=1e-12)
            at = (got[3][q].long() - q * beams) * V + got[4][q].long()
            assert torch.allclose(part[at[:len(want)]], have, atol=1e-12) and len(set(at[:len(want)].tolist())) == len(want)
