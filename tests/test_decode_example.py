"""What the decode-instance example does before it touches the GPU."""

import sys
from pathlib import Path

import pytest

sys.path.insert(0, str(Path(__file__).resolve().parents[1] / "examples"))
import decode_instance as example  # noqa: E402


@pytest.mark.parametrize("name,value", [("requests", 0), ("layers", 0), ("steps", 0), ("steps", -1), ("prompt", 1),
                                        ("prompt", 0)])
def test_counts_that_leave_nothing_to_do_are_refused(name, value, capsys):
    with pytest.raises(SystemExit) as e:
        example.main([f"--{name}", str(value)])
    assert e.value.code == 2 and "at least one" in capsys.readouterr().err
