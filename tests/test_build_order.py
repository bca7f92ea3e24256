"""What build.build() makes on hosts that lack something."""
import sys
import sysconfig

import pytest
import torch

from rlfluidcontrol_amd import build, ops


@pytest.fixture
def made(monkeypatch):
    libs = []

    def record(lib, force, verbose):
        libs.append(lib.path)
        return lib.path

    monkeypatch.setattr(build, "_build", record)
    return libs


def test_everything(made):
    assert build.build() == build.LIB and made == [build.LIB, build.OPS_LIB, build.BINDING]
    del made[:]
    assert build.build_ops() == build.OPS_LIB and made == [build.OPS_LIB, build.BINDING]


@pytest.mark.parametrize("lacks", ["torch", "the GPU's runtime", "torch's headers", "Python's headers"])
def test_without_a_torch_to_build_against(made, monkeypatch, tmp_path, lacks):
    if lacks == "torch":
        monkeypatch.setitem(sys.modules, "torch", None)
    elif lacks == "the GPU's runtime":
        monkeypatch.setattr(torch.version, "hip", None)
    elif lacks == "torch's headers":
        monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))
    else:
        monkeypatch.setattr(sysconfig, "get_paths", lambda: {"include": str(tmp_path)})
    assert build.build() == build.LIB and made == [build.LIB, build.OPS_LIB]


def test_the_environment_is_built_before_what_may_fail(monkeypatch):
    libs = []

    def fail(lib, force, verbose):
        libs.append(lib.path)
        if lib.path != build.LIB:
            raise RuntimeError("no compiler for this one")
        return lib.path

    monkeypatch.setattr(build, "_build", fail)
    with pytest.raises(RuntimeError, match="no compiler"):
        build.build()
    assert libs == [build.LIB, build.OPS_LIB]


def test_a_missing_binding_is_an_error_of_the_operators(monkeypatch):
    build.build_ops()
    monkeypatch.setattr(ops, "_gpu_module", None)
    monkeypatch.setitem(sys.modules, "rlfluidcontrol_amd._ops_torch", None)
    monkeypatch.delattr("rlfluidcontrol_amd._ops_torch", raising=False)
    with pytest.raises(ops.OpsError, match="binding"):
        ops._gpu()


def test_another_torch_makes_another_binding(monkeypatch):
    build.build_ops()

    def stale():
        flags, link = build._binding_flags()
        return build._Library(build.BINDING, build.OPS_CSRC, ["binding.cpp"], build._ops_deps, flags, build.BINDING_STAMP, link).needs_build()

    assert not stale()
    monkeypatch.setattr(torch, "__version__", torch.__version__ + ".1")
    assert stale()
