"""What the library decides on the host, where nothing is launched: sizes at the end of 31 bits and
past it are refused, and an attention call names its kernels."""

import ctypes

import pytest
import torch

from kvserve_amd import _lib, paged

from test_paged_host import SOME, attention_args, cache_struct

MOST = 2**31 - 2**20 - 1  # tokens of a table's row, rows of a request's queries


def one_token_blocks():
    return cache_struct(block_size=1, block_stride=2 * 64, part_stride=4 * 2 * 64)


def test_attention_refuses_places_that_its_counters_would_pass():
    lib = _lib.load()
    size = lambda **kw: lib.kvmi_attention_workspace_bytes(attention_args(one_token_blocks(), **kw))
    assert size(columns=MOST) >= 0
    assert size(columns=MOST + 1) == size(columns=2**31 - 1) == _lib.EINVAL
    assert lib.kvmi_tree_attention(attention_args(one_token_blocks(), columns=2**31 - 1), None) == _lib.EINVAL
    rows = lambda n: size(max_query=n, query_heads=2, total_queries=n)
    assert rows(MOST // 2) >= 0
    assert rows(MOST // 2 + 1) == rows(2**30 - 1) == _lib.EINVAL


def test_any_longest_length_is_taken():
    lib = _lib.load()
    for n in (0, 1, 64, 10**6, 2**31 - 1):
        assert lib.kvmi_attention_workspace_bytes(attention_args(max_length=n)) >= 0


@pytest.mark.parametrize("columns,fine", [(MOST, True), (MOST + 1, False), (2**31 - 1, False)])
def test_tables_and_kept_drafts_refuse_longer_rows(columns, fine):
    lib = _lib.load()
    want = _lib.OK if fine else _lib.EINVAL
    names = [f for f, _ in _lib.TablesArgs._fields_]
    a = {n: 4096 * (i + 1) for i, n in enumerate(names[:12])}
    a.update(err=None, requests=0, columns=columns, ring=8, block_size=1, max_tokens=10, reserved=0)
    assert lib.kvmi_build_tables(_lib.TablesArgs(*(a[n] for n in names)), None) == want
    c = one_token_blocks()
    assert lib.kvmi_keep_drafts(c, SOME, 1, SOME, columns, SOME, SOME, 0, 3, SOME, None, None) == want


def test_sizes_past_31_bits_are_not_cut():
    """Python's integers are refused where the structs' words would keep their low bits only."""
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    build = lambda S, n: paged.build_block_tables(i32(1), i32(1), i32(1, 2), i32(4), i32(2), S, n)
    for S, n in ((2**32 + 16, 5), (2**31, 5), (16, 2**32 + 5), (16, 2**31)):
        with pytest.raises(ValueError, match="block_size .* max_tokens"):
            build(S, n)
    with pytest.raises(ValueError, match="block_size"):
        paged.BlockTables(4, 2**32 + 16, 2, 3, device="cpu")
    cache = torch.empty((2, 1, 2**31, 1, 1), dtype=torch.bfloat16, device="meta")
    with pytest.raises(ValueError, match="31 bits"):
        paged._cache_struct(cache)


def test_attention_names_its_kernels():
    """Few rows or tiles, waves, rows of a workgroup, parts and keys of a part, for batches that
    are not the GPU's to decide."""
    lib, shape = _lib.load(), (ctypes.c_int32 * 4)()

    def kernels(D=128, H=8, **kw):
        c = cache_struct(head_dim=D, num_heads=H, block_stride=16 * H * D, part_stride=4 * 16 * H * D)
        return lib.kvmi_attention_kernels(attention_args(c, columns=4096, **kw), shape), *shape

    few, tiles = _lib.ATTENTION_ROWS, _lib.ATTENTION_TILES
    one = dict(requests=1, total_queries=1, query_heads=32, max_query=1)
    assert kernels(**one, max_length=512) == (few, 2, 16, 8, 64)
    batch = dict(requests=64, total_queries=64, query_heads=32, max_query=1)
    assert kernels(**batch, max_length=12289) == (few, 4, 16, 18, 704)
    prompt = dict(requests=1, total_queries=8192, query_heads=32, max_query=8192)
    assert kernels(**prompt, max_length=8192) == (tiles, 8, 256, 1, 8192)
    assert kernels(D=64, **prompt, max_length=8192) == (tiles, 4, 128, 1, 8192)
    # 16 rows, 32, and 33; above 128 channels 16 and 17
    for D, rows, want in ((128, 16, (few, 16)), (128, 17, (few, 32)), (128, 32, (few, 32)), (128, 33, (tiles, 128)),
                          (136, 16, (few, 16)), (136, 17, (tiles, 128))):
        got = kernels(D=D, requests=1, total_queries=rows, query_heads=8, max_query=rows, max_length=100)
        assert (got[0], got[2]) == want
    assert lib.kvmi_attention_kernels(attention_args(), None) == few
    for kw in (dict(requests=0), dict(total_queries=0), dict(max_query=0), dict(scale=0.0)):
        assert lib.kvmi_attention_kernels(attention_args(**kw), shape) == _lib.EINVAL
    assert lib.kvmi_attention_kernels(None, shape) == _lib.EINVAL
