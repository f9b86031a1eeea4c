"""The build entry point needs the product's sources and nothing of the test tree."""
import os

import pytest

import __graft_entry__ as entry
from ginn_b200 import build as B


@pytest.mark.parametrize("makefile", [None, "", "test_host_api:\n\ttrue\n", "bench_autobatch:\n\tfalse\n"])
def test_build_does_not_depend_on_the_test_tree(tmp_path, monkeypatch, makefile):
    """No test programs at all, a Makefile without rules, one of another age, one whose rule fails."""
    if makefile is not None:
        (tmp_path / "tests" / "cpp").mkdir(parents=True)
        (tmp_path / "tests" / "cpp" / "Makefile").write_text(makefile)
    monkeypatch.setattr(entry, "ROOT", str(tmp_path))
    entry.build()
    assert os.path.exists(B.LIB)
