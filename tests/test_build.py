"""The product's build does not depend on what lies in tests/: the libraries that only tests load may fail to
build, and the sources compile against host stand-ins (tests/emu) older than themselves."""
import os
import re
import shutil
import subprocess

import pytest

from byteir_amd import build as B

CLANG = os.path.join(os.environ.get("ROCM_PATH", "/opt/rocm"), "llvm", "bin", "clang++")
EMU = os.path.join(os.path.dirname(os.path.abspath(__file__)), "emu")
needs_clang = pytest.mark.skipif(not os.path.exists(CLANG), reason="no host clang")


@needs_clang
def test_a_tests_directory_that_does_not_fit_stops_nothing(tmp_path, monkeypatch, capsys):
    done = []
    for name in ("kernels", "flash", "brt", "index_check"):
        monkeypatch.setitem(B.TARGETS, name, lambda verbose, name=name: done.append(name))
    monkeypatch.setattr(B, "ROOT", str(tmp_path))
    shutil.copytree(os.path.join(EMU, "include"), tmp_path / "tests/emu/include")
    (tmp_path / "tests/emu/wave_emu.h").write_text("#error of another age\n")
    (tmp_path / "tests/emu/lib").mkdir()
    (tmp_path / "tests/external_kernels").mkdir()
    (tmp_path / "tests/external_kernels/custom_add.hip").write_text("#error of another age\n")
    stale = [tmp_path / f for files in B.TEST_TARGETS.values() for f in files]
    for f in stale:
        f.write_text("built from other sources")
    B.build_all()
    assert done == ["kernels", "flash", "brt", "index_check"]
    assert not any(f.exists() for f in stale)
    said = capsys.readouterr().err
    assert all(f"{name} (for the tests only) does not build" in said for name in B.TEST_TARGETS)
    for name in B.TEST_TARGETS:  # asked for by name, it raises
        with pytest.raises(RuntimeError, match="build failed"):
            B.build_all(targets=[name])


def test_a_tests_directory_that_cannot_be_written_to_stops_nothing(tmp_path, monkeypatch, capsys):
    done = []
    for name in B.TARGETS:
        monkeypatch.setitem(B.TARGETS, name, lambda verbose, name=name: done.append(name))

    def refuse(path):
        raise PermissionError(path)
    monkeypatch.setattr(B, "ROOT", str(tmp_path))
    monkeypatch.setattr(B.os, "remove", refuse)
    (tmp_path / "tests/emu/lib").mkdir(parents=True)
    (tmp_path / B.TEST_TARGETS["emu"][0]).write_text("another user's")
    B.build_all()
    assert "emu (for the tests only) does not build" in capsys.readouterr().err
    assert done == [name for name in B.TARGETS if name != "emu"]


def test_a_product_library_that_does_not_build_stops_the_build(monkeypatch):
    def fail(verbose):
        raise RuntimeError("build failed")
    monkeypatch.setitem(B.TARGETS, "kernels", fail)
    with pytest.raises(RuntimeError, match="build failed"):
        B.build_all()


@needs_clang
def test_the_sources_need_no_newer_host_header(tmp_path):
    """Without what the header gained for the bounded-cache kernels, which the sources once needed of it."""
    shutil.copytree(os.path.join(EMU, "include"), tmp_path / "include")
    old = re.sub(r"(?m)^.*(\batomicAdd\b|using fa_emu::hipErrorOutOfMemory|__builtin_amdgcn_readlane).*\n", "", open(os.path.join(EMU, "wave_emu.h")).read())
    (tmp_path / "wave_emu.h").write_text(old)
    # the stand-in for <hip/hip_runtime.h> includes ../../wave_emu.h
    runs = [(f, subprocess.Popen([CLANG, "-x", "c++", "-std=c++17", "-fsyntax-only", "-DFA_EMULATE", f"-I{tmp_path / 'include'}", f"-I{B.INC}",
                                  "-Wno-unknown-attributes", f], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True))
            for f in B._glob("flash_attn", (".hip",))]
    for f, run in runs:
        out = run.communicate(timeout=300)[0]
        assert run.returncode == 0, (os.path.basename(f), out[-2000:])
