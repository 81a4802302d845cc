"""Refusals and host logic of the paged operators that need no GPU (nothing is launched)."""

import ctypes

import pytest
import torch

from kvserve_amd import _lib, paged

from _paged_ref import build_tables

SOME = ctypes.c_void_p(4096)  # never dereferenced: the calls are refused first


def cache_struct(**kw):
    c = dict(base=4096, part_stride=4 * 16 * 2 * 64, block_stride=16 * 2 * 64, num_blocks=4, block_size=16, num_heads=2,
             head_dim=64)
    c.update(kw)
    return _lib.Cache(*c.values())


def test_struct_sizes_match_the_header():
    assert ctypes.sizeof(_lib.Cache) == 40
    assert ctypes.sizeof(_lib.TablesArgs) == 12 * 8 + 6 * 4
    assert ctypes.sizeof(_lib.AttentionArgs) == 40 + 8 * 8 + 8 + 8 + 16 + 10 * 4


BAD_CACHES = [dict(base=None), dict(num_blocks=0), dict(block_size=0), dict(num_heads=0), dict(head_dim=0),
              dict(part_stride=-1), dict(block_stride=16 * 2 * 64 - 8), dict(num_blocks=1 << 30)]


def attention_args(cache=None, **kw):
    a = dict(query=4096, out=4096, lse=None, tables=4096, lengths=4096, starts=4096, mask=None, workspace=4096,
             workspace_bytes=1 << 40, err=None, query_token_stride=8 * 64, query_head_stride=64, scale=0.1, dtype=0,
             requests=1, columns=4, total_queries=3, query_heads=8, max_query=3, max_length=64, mask_words=0, reserved=0)
    a.update(kw)
    return _lib.AttentionArgs(cache or cache_struct(), *a.values())


@pytest.mark.parametrize("kw", BAD_CACHES + [dict(head_dim=60), dict(head_dim=264, block_stride=1 << 20),
                                             dict(part_stride=4), dict(block_stride=16 * 2 * 64 + 4), dict(base=4098)])
def test_attention_refuses_bad_caches(kw):
    args = attention_args(cache_struct(**kw))
    lib = _lib.load()
    assert lib.kvmi_tree_attention(args, None) == _lib.EINVAL
    assert lib.kvmi_attention_workspace_bytes(args) == _lib.EINVAL


@pytest.mark.parametrize("kw", [
    dict(requests=-1), dict(requests=70000), dict(columns=0), dict(columns=1 << 28), dict(total_queries=-1),
    dict(max_query=-1), dict(max_length=-1), dict(query_heads=0), dict(query_heads=5), dict(dtype=2), dict(scale=0.0),
    dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")), dict(mask=4096, mask_words=0)])
def test_attention_refuses_bad_sizes(kw):
    lib = _lib.load()
    assert lib.kvmi_tree_attention(attention_args(**kw), None) == _lib.EINVAL
    assert lib.kvmi_attention_workspace_bytes(attention_args(**kw)) == _lib.EINVAL


@pytest.mark.parametrize("kw", [dict(query=None), dict(out=None), dict(tables=None), dict(lengths=None),
                                dict(starts=None), dict(query=4104), dict(query_token_stride=4),
                                dict(query_head_stride=12)])
def test_attention_refuses_bad_pointers(kw):
    assert _lib.load().kvmi_tree_attention(attention_args(**kw), None) == _lib.EINVAL
    assert _lib.load().kvmi_tree_attention(None, None) == _lib.EINVAL


def test_attention_with_nothing_to_do_is_fine():
    lib = _lib.load()
    for kw in (dict(requests=0), dict(total_queries=0), dict(max_query=0)):
        assert lib.kvmi_tree_attention(attention_args(**kw), None) == _lib.OK


def test_write_and_keep_refuse_bad_arguments():
    lib = _lib.load()
    c = cache_struct()
    write = lambda c, key=SOME, value=SOME, slots=SOME, n=3: lib.kvmi_write_kv(
        c, key, value, 128, 64, 128, 64, slots, n, None, None)
    for kw in BAD_CACHES:
        assert write(cache_struct(**kw)) == _lib.EINVAL
    assert write(c, n=-1) == write(c, key=None) == write(c, value=None) == write(c, slots=None) == _lib.EINVAL
    assert write(c, n=0) == _lib.OK
    keep = lambda c, layers=2, columns=4, R=1, width=3, lengths=SOME, out=ctypes.c_void_p(8192), bases=SOME, acc=SOME: \
        lib.kvmi_keep_drafts(c, bases, layers, SOME, columns, lengths, acc, R, width, out, None, None)
    for kw in BAD_CACHES[1:]:
        assert keep(cache_struct(**kw)) == _lib.EINVAL
    for kw in (dict(layers=0), dict(layers=65536), dict(columns=0), dict(columns=1 << 28), dict(R=-1), dict(width=-1),
               dict(width=1025), dict(lengths=None), dict(out=None), dict(bases=None), dict(acc=None), dict(out=SOME)):
        assert keep(c, **kw) == _lib.EINVAL, kw
    assert keep(c, R=0) == _lib.OK


def test_tables_refuse_bad_arguments():
    lib = _lib.load()
    names = [f for f, _ in _lib.TablesArgs._fields_]

    def call(**kw):
        a = {n: 4096 * (i + 1) for i, n in enumerate(names[:12])}
        a.update(err=None, requests=2, columns=4, ring=8, block_size=16, max_tokens=10, reserved=0)
        a.update(kw)
        return lib.kvmi_build_tables(_lib.TablesArgs(*(a[n] for n in names)), None)

    for n in ("lengths", "new_lengths", "tables", "free_blocks", "state", "out_tables", "out_lengths", "out_state",
              "slots", "starts"):
        assert call(**{n: None}) == _lib.EINVAL, n
    for kw in (dict(requests=-1), dict(columns=0), dict(ring=0), dict(block_size=0), dict(max_tokens=-1),
               dict(columns=1 << 28), dict(ring=1 << 28), dict(out_lengths=4096), dict(out_state=5 * 4096),
               dict(out_lengths=4096, out_state=5 * 4096, ticket=None), dict(out_lengths=2 * 4096)):
        assert call(**kw) == _lib.EINVAL, kw
    assert lib.kvmi_build_tables(None, None) == _lib.EINVAL
    assert call(requests=0) == _lib.OK


def test_wrappers_refuse_host_tensors_and_wrong_types():
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    cache = torch.zeros((2, 3, 4, 2, 8), dtype=torch.bfloat16)
    rows = torch.zeros((3, 2, 8), dtype=torch.bfloat16)
    with pytest.raises(ValueError):
        paged.write_kv(rows, rows, cache, torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        paged.write_kv(rows, rows, cache.float(), torch.zeros(3, dtype=torch.int64))
    with pytest.raises(ValueError):
        paged.write_kv(rows, rows, cache[0], torch.zeros(3, dtype=torch.int64))
    with pytest.raises(TypeError):
        paged.tree_attention(rows, cache, i32(1, 2), i32(1), i32(2), max_query=3)
    with pytest.raises(ValueError):
        paged.keep_drafts([cache], i32(1, 2), i32(1), i32(1, 2))
    with pytest.raises(ValueError):
        paged.keep_drafts([], i32(1, 2), i32(1), i32(1, 2))
    with pytest.raises(TypeError):
        paged.build_block_tables(i32(1).long(), i32(1), i32(1, 2), i32(4), i32(2), 16, 5)
    with pytest.raises(ValueError):
        paged.build_block_tables(i32(1), i32(1), i32(1, 2), i32(4), i32(2), 16, 5)
    for kw in (dict(block_size=0), dict(max_tokens=-1), dict(max_tokens=1.5)):
        kw = dict(dict(block_size=16, max_tokens=5), **kw)
        with pytest.raises(ValueError):
            paged.build_block_tables(i32(1), i32(1), i32(1, 2), i32(4), i32(2), **kw)
    for kw in (dict(num_blocks=0), dict(block_size=0), dict(requests=0), dict(columns=0), dict(free_blocks=[1, 1]),
               dict(free_blocks=[4]), dict(free_blocks=[-1])):
        with pytest.raises(ValueError):
            paged.BlockTables(**dict(dict(num_blocks=4, block_size=16, requests=2, columns=3, device="cpu"), **kw))


def test_block_tables_begin_empty():
    own = paged.BlockTables(5, 16, 2, 3, device="cpu", free_blocks=[4, 1])
    assert own.free.tolist() == [4, 1, -1, -1, -1] and own.state.tolist() == [0, 2]
    assert own.tables.tolist() == [[-1] * 3] * 2 and own.lengths.tolist() == [0, 0]


def test_tree_mask_words():
    mask = paged.tree_mask([-1, 0, 0, 1, -1], device="cpu")
    assert mask.tolist() == [[0b1], [0b11], [0b101], [0b1011], [0b10000]]
    chain = paged.tree_mask(list(range(-1, 69)), device="cpu")
    assert chain.shape == (70, 2)
    for i in range(70):
        whole = (int(chain[i, 1]) % 2**64) << 64 | int(chain[i, 0]) % 2**64
        assert whole == (1 << (i + 1)) - 1
    assert paged.tree_mask([], device="cpu").shape == (0, 1) and paged.tree_mask([-1], 3, "cpu").shape == (1, 3)
    for bad in ([0], [-2], [-1, 2]):
        with pytest.raises(ValueError):
            paged.tree_mask(bad, device="cpu")
    with pytest.raises(ValueError):
        paged.tree_mask([-1] * 65, 1, "cpu")


def test_host_program_of_the_tables():
    """The restatement that the GPU tests compare with, on a case worked by hand."""
    got = build_tables([4, 0, 8], [5, 8, 0], [[0, -1, -1], [-1, -1, -1], [1, 2, -1]], [4, 5, -1, -1, -1, 3], [5, 3], 4, 10)
    tables, after, state, slots, starts, ring, refused, bad = got
    assert tables == [[0, 3, -1], [4, 5, -1], [-1, -1, -1]] and after == [5, 8, 0]
    assert state == [2, 2] and ring == [4, 5, 1, 2, -1, 3]
    assert slots == [12, 16, 17, 18, 19, 20, 21, 22, 23, -1] and starts == [0, 1, 9, 9] and not refused and not bad
