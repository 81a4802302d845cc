"""The beam-search example: what it refuses before it touches the GPU, and its steps' tables."""

import sys
from pathlib import Path

import pytest
import torch

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
import beam_search as example  # noqa: E402

from _shared_ref import consistent  # noqa: E402


@pytest.mark.parametrize("name,value", [("requests", 0), ("beams", 0), ("beams", 33), ("layers", 0), ("steps", 0),
                                        ("steps", -1), ("prompt", 1)])
def test_counts_that_leave_nothing_to_do_are_refused(name, value, capsys):
    with pytest.raises(SystemExit) as e:
        example.main([f"--{name}", str(value)])
    assert e.value.code == 2 and "at least one" in capsys.readouterr().err


@pytest.mark.gpu
def test_the_example_runs(cuda, capsys):
    example.main(["--requests", "2", "--beams", "3", "--layers", "2", "--steps", "20", "--prompt", "300"])
    assert "blocks held" in capsys.readouterr().out


@pytest.mark.gpu
def test_steps_keep_the_pool_whole(cuda):
    inst = example.BeamInstance(1, 2, 2, 64, 4, 120, 2, 3, 20, cuda)
    new = torch.zeros(6, dtype=torch.int32, device=cuda)
    new[::3] = torch.tensor([9, 5], dtype=torch.int32, device=cuda)
    inst.tables.update(new, 14)
    inst.scores[::3] = 0.0
    for i in range(10):
        best = inst.step(80)
        if i == 5:
            inst.compact()
        t = inst.tables
        consistent(t.tables.tolist(), t.lengths.tolist(), t.shares.tolist(), t.free.tolist(), t.state.tolist(), 4)
        live = best.parents >= 0
        assert bool(torch.isfinite(inst.scores[live]).all()) and int((t.lengths > 0).sum()) == int(live.sum())
    assert t.lengths.tolist() == [19] * 3 + [15] * 3
