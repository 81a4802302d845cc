"""The module behind the paged operators' unchecked calls: what it takes gives the same as the
checked way, and what it does not take is left to the wrappers' checks."""

import ctypes

import pytest
import torch

from kvserve_amd import _lib, paged

BF16 = torch.bfloat16


def i32(values, dev):
    return torch.tensor(values, dtype=torch.int32, device=dev)


def arguments(dev):
    """Right arguments of each function of the module (right on a GPU)."""
    cache = torch.zeros((2, 4, 16, 2, 64), dtype=BF16, device=dev)
    rows = torch.ones((5, 2, 64), dtype=BF16, device=dev)
    tables, lengths = i32([[0, 1], [2, 3]], dev), i32([20, 17], dev)
    layers = paged._lib.Cache(cache.data_ptr(), 4 * 16 * 128, 16 * 128, 4, 16, 2, 64)
    out = paged.TablesUpdate(i32([[0] * 2] * 2, dev), i32([0, 0], dev), i32([0, 0], dev),
                             torch.zeros(6, dtype=torch.int64, device=dev), i32([0] * 3, dev))
    return {
        "write_kv": [rows, rows, cache, torch.arange(5, device=dev), None],
        "build_block_tables": [lengths, i32([22, 17], dev), tables, i32([-1] * 4, dev), i32([0, 0], dev), 16, 6, out,
                               None, None],
        "tree_attention": [torch.ones((5, 4, 64), dtype=BF16, device=dev), cache, tables, lengths, i32([0, 3, 5], dev),
                           3, 20, None, None, torch.empty((5, 4, 64), dtype=BF16, device=dev), None],
        "keep_drafts": [ctypes.addressof(layers), torch.tensor([cache.data_ptr()], device=dev), tables, lengths,
                        i32([[0, 2], [1, -1]], dev), i32([0, 0], dev), None],
    }, layers


def test_host_tensors_and_junk_are_not_taken():
    args, _keep = arguments("cpu")
    for name, good in args.items():
        call = getattr(paged._calls, name)
        assert call(*good) is False
        assert call() is False and call(*good, None) is False
        for i in range(len(good)):
            for junk in (None, 3, -1, 1 << 70, "x", 1.5, (), torch.zeros(2)):
                if name == "keep_drafts" and i == 0 and isinstance(junk, int):
                    continue  # an address is the caller's word
                assert call(*good[:i], junk, *good[i + 1:]) is False, (name, i, junk)


def test_a_missing_module_is_named():
    with pytest.raises(_lib.KvmiError, match="kvserve_amd.build"):
        _lib._NoCalls(ImportError("no such file")).write_kv


# what is wrong with one argument: (function, its number, change)
WRONG = [
    ("write_kv", 0, lambda t: t.half()), ("write_kv", 0, lambda t: t[:4]), ("write_kv", 1, lambda t: t[:, :1]),
    ("write_kv", 1, lambda t: t.transpose(0, 2)), ("write_kv", 2, lambda t: t.float()), ("write_kv", 2, lambda t: t[0]),
    ("write_kv", 3, lambda t: t.int()), ("write_kv", 3, lambda t: t[:4]), ("write_kv", 3, lambda t: t.repeat(2)[::2]),
    ("write_kv", 4, lambda t: torch.zeros(1, dtype=torch.int64, device="cuda")),
    ("build_block_tables", 0, lambda t: t.long()), ("build_block_tables", 1, lambda t: t[:1]),
    ("build_block_tables", 2, lambda t: t[:1]), ("build_block_tables", 2, lambda t: t.t()),
    ("build_block_tables", 4, lambda t: t[:1]), ("build_block_tables", 5, lambda t: 0),
    ("build_block_tables", 6, lambda t: 7), ("build_block_tables", 6, lambda t: True),
    ("build_block_tables", 7, lambda t: t[:4]), ("build_block_tables", 7, lambda t: list(t)),
    ("build_block_tables", 8, lambda t: torch.zeros(2, dtype=torch.int32, device="cuda")),
    ("tree_attention", 0, lambda t: t.half()), ("tree_attention", 0, lambda t: t[:, :3]),
    ("tree_attention", 0, lambda t: t[..., :32]), ("tree_attention", 1, lambda t: t.view(torch.int16)),
    ("tree_attention", 2, lambda t: t[:1]), ("tree_attention", 3, lambda t: t.cpu()),
    ("tree_attention", 4, lambda t: t[:2]), ("tree_attention", 5, lambda t: -1), ("tree_attention", 6, lambda t: 1.0),
    ("tree_attention", 7, lambda t: torch.zeros((4, 1), dtype=torch.int64, device="cuda")),
    ("tree_attention", 8, lambda t: 0.0), ("tree_attention", 8, lambda t: float("nan")),
    ("tree_attention", 9, lambda t: t[:4]), ("tree_attention", 9, lambda t: t.transpose(0, 1)),
    ("keep_drafts", 1, lambda t: t.int()), ("keep_drafts", 2, lambda t: t[:1]), ("keep_drafts", 3, lambda t: t.long()),
    ("keep_drafts", 4, lambda t: t[0]), ("keep_drafts", 4, lambda t: t.t()), ("keep_drafts", 5, lambda t: t[:1]),
]


@pytest.mark.gpu
@pytest.mark.parametrize("name,i,change", WRONG)
def test_wrong_arguments_are_not_taken(cuda, name, i, change):
    args, _keep = arguments(cuda)
    args = args[name]
    held = [t for x in args for t in (x if isinstance(x, tuple) else (x,)) if isinstance(t, torch.Tensor)]
    before = [t.clone() for t in held]
    args[i] = change(args[i])
    assert getattr(paged._calls, name)(*args) is False
    torch.cuda.synchronize()
    for t, was in zip(held, before):  # nothing was done
        assert torch.equal(t.view(torch.uint8), was.view(torch.uint8))


@pytest.mark.gpu
def test_right_arguments_are_taken(cuda):
    args, _keep = arguments(cuda)
    for name, good in args.items():
        assert getattr(paged._calls, name)(*good) is True, name
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_unchecked_calls_give_what_checked_ones_give(cuda):
    gen = torch.Generator(device=cuda).manual_seed(0)
    rand = lambda *s: torch.randn(s, generator=gen, device=cuda).to(BF16)
    cache, rows = rand(2, 8, 16, 2, 64), rand(9, 2, 64)
    slots = torch.randperm(128, generator=gen, device=cuda)[:9]
    one, two = cache.clone(), cache.clone()
    paged.write_kv(rows, rows, one, slots, check=True)
    paged.write_kv(rows, rows, two, slots, check=False)
    assert torch.equal(one, two)
    tables, lengths, starts = i32([[3, 1, -1], [0, 5, 7]], cuda), i32([30, 40], cuda), i32([0, 4, 9], cuda)
    q, mask = rand(9, 6, 64), torch.full((9, 1), -1, dtype=torch.int64, device=cuda)
    for kw in (dict(), dict(tree_mask=mask), dict(max_length=40), dict(scale=0.5), dict(scale=1)):
        a = paged.tree_attention(q, cache, tables, lengths, starts, max_query=5, check=True, **kw)
        b = paged.tree_attention(q, cache, tables, lengths, starts, max_query=5, check=False, **kw)
        assert torch.equal(a, b)
    layers = [paged.LayerCaches([c]) for c in (one, two)]
    path, out = i32([[0, 3, -1], [2, 4, 6]], cuda), i32([0, 0], cuda)
    now = i32([20, 30], cuda)
    a = paged.keep_drafts(layers[0], tables, now, path, check=True)
    b = paged.keep_drafts(layers[1], tables, now, path, out=out, check=False)
    assert torch.equal(a, b) and b is out and torch.equal(one, two)
    got = []
    for check in (True, False):
        own = paged.BlockTables(12, 16, 2, 4, cuda)
        s, t = own.update(i32([20, 33], cuda), 60, check=check)
        got.append([s, t, own.tables, own.lengths, own.free, own.state])
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.gpu
def test_refusals_are_the_wrappers(cuda):
    """Unchecked calls with wrong arguments raise what checked ones do."""
    args, _keep = arguments(cuda)
    key, value, cache, slots, _ = args["write_kv"]
    with pytest.raises(TypeError):
        paged.write_kv(key.half(), value, cache, slots, check=False)
    with pytest.raises(ValueError):
        paged.write_kv(key, value, cache, slots[:4], check=False)
    q, cache, tables, lengths, starts = args["tree_attention"][:5]
    with pytest.raises(ValueError):
        paged.tree_attention(q, cache, tables, lengths, starts, max_query=3, scale=-1.0, check=False)
    with pytest.raises(TypeError):
        paged.tree_attention(q, cache, tables.long(), lengths, starts, max_query=3, check=False)
