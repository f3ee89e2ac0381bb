"""When the kernel library and the training operators' extension count as stale (ops/build.py)."""
import os
import sysconfig

import pytest
import torch

from smsgate_amd import ops
from smsgate_amd.ops import build


@pytest.fixture
def tree(tmp_path, monkeypatch):
    """A source folder with one file of each kind, all older than what was built of them."""
    for name in ("a.hip", "train_ops.hpp", "train_autograd.cpp", "build.py"):
        (tmp_path / name).write_text("")
    for name in ("lib.so", "autograd.so"):
        (tmp_path / name).write_text("")
        os.utime(tmp_path / name, (2000, 2000))
    for name in ("a.hip", "train_ops.hpp", "train_autograd.cpp", "build.py"):
        os.utime(tmp_path / name, (1000, 1000))
    monkeypatch.setattr(build, "CSRC", tmp_path)
    monkeypatch.setattr(build, "AUTOGRAD_SRC", tmp_path / "train_autograd.cpp")
    monkeypatch.setattr(build, "AUTOGRAD", tmp_path / "autograd.so")
    monkeypatch.setattr(build, "__file__", str(tmp_path / "build.py"))
    return tmp_path


def _stale(tree):
    return build.needs_build(tree / "lib.so"), build.needs_build_autograd()


def test_nothing_changed(tree):
    assert _stale(tree) == (False, False)


@pytest.mark.parametrize("name,lib,autograd", [
    ("a.hip", True, False),
    ("train_ops.hpp", True, True),  # the entries' signatures: both sides include it
    ("train_autograd.cpp", False, True),
    ("build.py", True, True),       # the flags
])
def test_a_newer_source(tree, name, lib, autograd):
    os.utime(tree / name, (3000, 3000))
    assert _stale(tree) == (lib, autograd)


@pytest.mark.parametrize("name", ["lib.so", "autograd.so"])
def test_nothing_built(tree, name):
    os.unlink(tree / name)
    assert _stale(tree) == (name == "lib.so", name == "autograd.so")


def test_another_torch_or_interpreter_has_its_own_extension():
    """It is compiled against both: another version's file is not taken for this one's."""
    assert torch.__version__ in build.AUTOGRAD.name
    assert build.AUTOGRAD.name.endswith(sysconfig.get_config_var("EXT_SUFFIX"))


def test_processes_that_build_at_once_write_apart(tmp_path, monkeypatch):
    """Ranks of one job may find the same library missing: none takes another's half-written file."""
    outs = []

    def run(cmd, check):
        outs.append(cmd[cmd.index("-o") + 1])
        with open(outs[-1], "w") as f:
            f.write("built")

    monkeypatch.setattr(build.subprocess, "run", run)
    monkeypatch.setattr(build, "LIBDIR", tmp_path)
    monkeypatch.setattr(build, "LIB", tmp_path / "lib.so")
    monkeypatch.setattr(build, "AUTOGRAD", tmp_path / "autograd.so")
    for pid in (11, 12):
        monkeypatch.setattr(build.os, "getpid", lambda: pid)
        build.build(force=True)
        build.build_autograd(force=True)
    assert len(set(outs)) == 4
    assert sorted(p.name for p in tmp_path.iterdir()) == ["autograd.so", "lib.so"]


def test_the_extension_loads():
    if not build.AUTOGRAD.exists():
        pytest.skip("not built")
    assert {"embed", "attention", "loss"} <= set(dir(ops.load_train_autograd()))
