"""build.py: the C library stands by itself, whatever becomes of the Python
mirror's helper. Compilers are stood in for by a function that writes the output."""
import importlib.util
import os
import subprocess
import sys

import pytest

import omni_attn as oa


@pytest.fixture
def build(monkeypatch, tmp_path):
    spec = importlib.util.spec_from_file_location("omni_build", os.path.join(os.path.dirname(oa.__file__), "build.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    m.ran, m.fails = [], ()

    def run(cmd, **kw):
        m.ran.append(os.path.basename(cmd[0]))
        if m.ran[-1] in m.fails:
            return subprocess.CompletedProcess(cmd, 1, "", "stood in for")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("built")
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(m.subprocess, "run", run)
    m.HIPCC = "hipcc"
    m.OUT, m.TENSORS, m.BUILD = (str(tmp_path / n) for n in ("lib.so", "tensors.so", "objects"))
    return m


def test_both_are_built(build):
    assert build.build() == build.OUT and os.path.exists(build.OUT) and os.path.exists(build.TENSORS)
    assert build.ran.count("hipcc") == len(build.sources()) + 1 and build.ran.count("g++") == 1


def test_without_torch_the_library_is_built_and_the_helper_named(build, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)  # its import fails
    assert build.build() == build.OUT and os.path.exists(build.OUT)
    assert "g++" not in build.ran and not os.path.exists(build.TENSORS)
    assert "torch" in capsys.readouterr().err


def test_a_helper_that_does_not_compile_leaves_the_library(build):
    build.fails = ("g++",)
    with pytest.raises(RuntimeError, match="tensors.cpp"):
        build.build()
    assert os.path.exists(build.OUT)


def test_a_helper_of_another_torch_is_not_used(monkeypatch):
    """It reads torch's objects by the layout of the headers that it was compiled with."""
    monkeypatch.setattr(oa._torch, "__version__", "1.0.0")
    with pytest.raises(oa.OmniAttnError, match="built for torch .*, this is torch 1.0.0"):
        oa._load_tensors()
