"""The paged operators and the build where the module of the unchecked calls cannot be made: the
library is built and serves every call, with a warning."""

import subprocess
import warnings

import pytest
import torch

from kvserve_amd import _lib, build, paged


@pytest.fixture
def no_calls(monkeypatch):
    calls = _lib._NoCalls(ImportError("no such file"))
    monkeypatch.setattr(paged, "_calls", calls)
    return calls


def test_unchecked_calls_go_through_the_checks(no_calls):
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32)
    cache, rows = torch.zeros((2, 3, 4, 2, 8), dtype=torch.bfloat16), torch.zeros((3, 2, 8), dtype=torch.bfloat16)
    with pytest.warns(UserWarning, match="kvserve_amd.build"), pytest.raises(ValueError, match="CUDA"):
        paged.write_kv(rows, rows, cache, torch.zeros(3, dtype=torch.int64), check=False)
    with warnings.catch_warnings():
        warnings.simplefilter("error")  # said once
        with pytest.raises(ValueError, match="CUDA"):
            paged.write_kv(rows, rows, cache, torch.zeros(3, dtype=torch.int64), check=False)
        with pytest.raises(ValueError, match="CUDA"):
            paged.build_block_tables(i32(1), i32(1), i32(1, 2), i32(4), i32(2), 16, 5, check=False,
                                     out=paged.TablesUpdate(i32(1, 2), i32(1), i32(2), i32(5).long(), i32(2)))


@pytest.mark.parametrize("what", ["g++", "Python's headers"])
def test_the_library_is_built_without_the_module(monkeypatch, tmp_path, what):
    """What only the module needs may be missing; a module of an older library does not stay."""
    calls = tmp_path / "_calls.so"
    calls.write_bytes(b"old")
    monkeypatch.setattr(build, "CALLS", calls)
    monkeypatch.setattr(subprocess, "run", lambda *a, **k: pytest.fail("nothing to run"))
    if what == "g++":
        which = build.shutil.which
        monkeypatch.setattr(build.shutil, "which", lambda name, *a, **k: None if name == "g++" else which(name, *a, **k))
    else:
        monkeypatch.setattr(build.sysconfig, "get_paths", lambda: {"include": str(tmp_path / "nowhere")})
    with pytest.warns(UserWarning, match=what.replace("+", r"\+")):
        build._build_calls()
    assert not calls.exists()


@pytest.mark.gpu
def test_unchecked_calls_are_served(cuda, no_calls):
    cache = torch.zeros((2, 4, 16, 2, 64), dtype=torch.bfloat16, device=cuda)
    rows = torch.randn((5, 2, 64), device=cuda).to(torch.bfloat16)
    with pytest.warns(UserWarning, match="_calls.so"):
        own = paged.BlockTables(4, 16, 1, 4, cuda)
        new = torch.tensor([5], dtype=torch.int32, device=cuda)
        slots, starts = own.update(new, 5, check=False)
    paged.write_kv(rows, rows, cache, slots, check=False)
    out = paged.tree_attention(rows, cache, own.tables, own.lengths, starts, max_query=5, check=False)
    path, zero = torch.tensor([[1, 3]], dtype=torch.int32, device=cuda), torch.zeros_like(new)
    kept = paged.keep_drafts([cache], own.tables, zero, path, out=torch.empty_like(new), check=False)
    assert own.lengths.tolist() == [5] and kept.tolist() == [2] and torch.equal(out[0], rows[0])
    assert torch.equal(cache[0, 0, 0], rows[1]) and torch.equal(cache[1, 0, 1], rows[3])
