"""Which objects a build makes again, with the compilers' runs recorded instead
of made."""
import os
import subprocess

import pytest

from sym_b200 import build as B


@pytest.fixture
def project(tmp_path, monkeypatch):
    sources = [tmp_path / "a.cu", tmp_path / "b.cu"]
    for s in sources:
        s.write_text("")
        os.utime(s, (1, 1))
    monkeypatch.setattr(B, "CUDA_SOURCES", sources)
    monkeypatch.setattr(B, "HEADERS", [])
    monkeypatch.setattr(B, "RUNTIME_SOURCES", [])
    monkeypatch.setattr(B, "LIB_DIR", tmp_path)
    monkeypatch.setattr(B, "OBJ_DIR", tmp_path / "objects")
    monkeypatch.setattr(B, "CUDA_LIB", tmp_path / "cuda.so")
    monkeypatch.setattr(B, "RUNTIME_LIB", tmp_path / "runtime.so")
    monkeypatch.setattr(B, "_nvcc", lambda: "nvcc")
    monkeypatch.setattr(B, "_cxx", lambda: "g++")
    monkeypatch.delenv("SYM_B200_NVCC_DEFINES", raising=False)
    state = {"fail": None, "ran": []}

    def run(cmd, verbose):
        cmd = [str(c) for c in cmd]
        out = cmd[cmd.index("-o") + 1]
        if state["fail"] and out.endswith(state["fail"]):
            raise subprocess.CalledProcessError(1, cmd)
        state["ran"].append((os.path.basename(out), "-DX=1" in cmd))
        with open(out, "w") as f:
            f.write("-DX=1" if "-DX=1" in cmd else "plain")

    monkeypatch.setattr(B, "_run", run)

    def build(defines=None, fail=None):
        state["fail"], state["ran"] = fail, []
        if defines is None:
            monkeypatch.delenv("SYM_B200_NVCC_DEFINES", raising=False)
        else:
            monkeypatch.setenv("SYM_B200_NVCC_DEFINES", defines)
        B.build()
        return sorted(o for o, _ in state["ran"] if o.endswith(".o"))

    return tmp_path, sources, build


def test_objects_are_kept_while_their_sources_are_older(project):
    path, sources, build = project
    assert build() == ["a.o", "b.o"]
    assert build() == []
    os.utime(sources[1], None)
    os.utime(path / "cuda.so", (2, 2))
    os.utime(path / "objects" / "b.o", (2, 2))
    assert build() == ["b.o"]


def test_objects_of_a_build_that_failed_are_not_taken_for_another(project):
    path, sources, build = project
    build()
    os.utime(path / "cuda.so", (0, 0))
    with pytest.raises(subprocess.CalledProcessError):
        build("X=1", fail="b.o")
    os.utime(path / "cuda.so", (0, 0))
    build()
    assert [(path / "objects" / o).read_text() for o in ("a.o", "b.o")] == ["plain", "plain"]
