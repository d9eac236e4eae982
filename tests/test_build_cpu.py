"""The build of the operators' Python module (tie_b200/_ops): the library and the model do without it."""
import importlib.metadata
import os

import pytest

from tie_b200 import build


@pytest.fixture()
def elsewhere(tmp_path, monkeypatch):
    """The module's place and its compiler, away from the real one's."""
    monkeypatch.setattr(build, "OPS_PATH", str(tmp_path / "_ops.so"))
    monkeypatch.setattr(build, "OPS_STAMP", str(tmp_path / "objects" / "ops_module.torch"), raising=False)
    monkeypatch.setenv("CXX", "false")
    return tmp_path / "_ops.so"


@pytest.mark.parametrize("compiler", ["false", "/nonexistent/g++", "true"])
def test_a_module_that_does_not_build_is_left_out(elsewhere, monkeypatch, compiler):
    monkeypatch.setenv("CXX", compiler)
    with pytest.warns(RuntimeWarning, match="_ops"):
        assert build.build_ops_module() == ""
    assert not elsewhere.exists()


def test_a_module_of_another_torch_is_built_anew(elsewhere):
    elsewhere.write_text("a module")
    os.makedirs(os.path.dirname(build.OPS_STAMP))
    with open(build.OPS_STAMP, "w") as f:
        f.write(importlib.metadata.version("torch"))
    assert build.build_ops_module() == str(elsewhere)          # nothing has changed: no compiler is run
    with open(build.OPS_STAMP, "w") as f:
        f.write("2.0.0")
    with pytest.warns(RuntimeWarning):
        assert build.build_ops_module() == ""
    assert not elsewhere.exists()                              # what was built for another torch is not called
