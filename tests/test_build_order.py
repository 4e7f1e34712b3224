"""The LSTM's library needs hipcc alone: what the block operators' torch front end lacks does not keep it from being built
(the compilers are stand-ins here)."""
from __future__ import annotations

import os
import subprocess
import types

import pytest

from persistent_lstm_hip_amd import build


@pytest.fixture
def commands(tmp_path, monkeypatch):
    for name in ("LIB_PATH", "TORCH_PATH", "BENCH_PATH"):
        monkeypatch.setattr(build, name, str(tmp_path / os.path.basename(getattr(build, name))))
    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path))
    monkeypatch.setattr(build, "hipcc", lambda: "/opt/rocm/bin/hipcc")
    monkeypatch.setattr(build, "host_compiler", lambda: "/usr/bin/g++")
    seen, fail = [], []

    def run(cmd, **_):
        seen.append(cmd)
        bad = any(word in a for word in fail for a in cmd)
        if not bad:
            with open(cmd[cmd.index("-o") + 1], "w") as f:
                f.write("built")
        return types.SimpleNamespace(returncode=int(bad), stdout="Python.h: no such file" if bad else "")

    monkeypatch.setattr(subprocess, "run", run)
    return seen, fail


def _built():
    return [os.path.exists(p) for p in (build.LIB_PATH, build.BENCH_PATH, build.TORCH_PATH)]


def test_everything_is_built(commands):
    assert build.build() == build.LIB_PATH and _built() == [True, True, True]


def test_without_a_host_compiler_the_library_is_built_all_the_same(commands, monkeypatch):
    def none():
        raise RuntimeError("g++ not found: the torch front end needs a C++ compiler")

    monkeypatch.setattr(build, "host_compiler", none)
    with pytest.raises(RuntimeError, match="torch front end"):
        build.build()
    assert _built() == [True, True, False]


def test_a_failing_front_end_names_its_compiler(commands):
    commands[1].append("plh_torch.cpp")
    with pytest.raises(RuntimeError, match=r"(?s)g\+\+ failed.*Python\.h"):
        build.build()
    assert _built() == [True, True, False]


def test_a_failing_kernel_leaves_no_library(commands):
    commands[1].append("plh_scan.hip")
    with pytest.raises(RuntimeError, match="hipcc failed"):
        build.build()
    assert _built() == [False, False, False]
