"""What the build compiles, and when (no compiler runs here)."""
from __future__ import annotations

import importlib.util
import os
import types

import pytest

from batch_topk_b200 import build


@pytest.fixture
def compiled(monkeypatch, tmp_path):
    """The programs that a build would start; each leaves its output file."""
    started = []

    def run(cmd, verbose=False):
        started.append(os.path.basename(cmd[0]))
        with open(cmd[cmd.index("-o") + 1], "w"):
            pass

    monkeypatch.setattr(build, "_run", run)
    monkeypatch.setattr(build, "nvcc", lambda: "/cuda/bin/nvcc")
    monkeypatch.setattr(build, "LIB_DIR", str(tmp_path / "lib"))
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib" / "lib.so"))
    monkeypatch.setattr(build, "TENSORS", str(tmp_path / "_tensors.so"))
    monkeypatch.setattr(build, "TENSORS_STAMP", str(tmp_path / "_build" / "torch"))
    return started


def torch_at(monkeypatch, place):
    """An installed torch at `place`, or none."""
    spec = place and types.SimpleNamespace(origin=str(place / "__init__.py"))
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: spec)


def test_library_builds_where_torch_is_not_installed(monkeypatch, compiled):
    torch_at(monkeypatch, None)
    assert build.build() == build.LIB and os.path.exists(build.LIB)
    assert compiled == ["nvcc"] and not os.path.exists(build.TENSORS)


def test_module_is_built_again_for_another_torch(monkeypatch, compiled, tmp_path):
    places = []
    for version in ("1", "2"):
        place = tmp_path / version
        place.mkdir()
        (place / "version.py").write_text(f"__version__ = {version!r}\n")
        os.utime(place / "version.py", (0, 0))  # as a wheel may install it
        places.append(place)
    torch_at(monkeypatch, places[0])
    build.build()
    build.build()
    assert compiled == ["nvcc", "g++"]
    torch_at(monkeypatch, places[1])
    build.build()
    build.build()
    assert compiled == ["nvcc", "g++", "g++"]
