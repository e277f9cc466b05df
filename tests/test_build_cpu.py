"""What the build makes where a tool is missing, with a compiler that only writes its output file."""

from __future__ import annotations

import pytest

import build_lib


@pytest.fixture
def tree(tmp_path, monkeypatch):
    compiler = tmp_path / "hipcc"
    compiler.write_text('#!/bin/sh\nwhile [ "$1" != -o ]; do shift; done\n: > "$2"\n')
    compiler.chmod(0o755)
    monkeypatch.setattr(build_lib, "hipcc", lambda: str(compiler))
    monkeypatch.setattr(build_lib, "OBJ_DIR", tmp_path / "objects")
    monkeypatch.setattr(build_lib, "LIB", tmp_path / "libmtpk.so")
    monkeypatch.setattr(build_lib, "TORCH_LIB", tmp_path / "_mtpk_torch.so")
    return tmp_path


def test_the_library_needs_hipcc_alone(tree, monkeypatch) -> None:
    monkeypatch.setenv("PATH", str(tree))  # no g++
    with pytest.warns(UserWarning, match="_mtpk_torch.so is not built"):
        build_lib.build()
    assert (tree / "libmtpk.so").exists() and not (tree / "_mtpk_torch.so").exists()


def test_calls_that_do_not_compile_fail_the_build_after_the_library(tree, monkeypatch) -> None:
    bad = tree / "csrc"
    bad.mkdir()
    (bad / "mtpk_torch.cpp").write_text("no C++")
    monkeypatch.setattr(build_lib, "CSRC", bad)
    with pytest.raises(RuntimeError, match="mtpk_torch.cpp"):
        build_lib.build()
    assert (tree / "libmtpk.so").exists()


def test_only_what_is_missing_is_built(tree, monkeypatch) -> None:
    import __graft_entry__
    import _mtpk

    built = []
    monkeypatch.setattr(_mtpk, "LIB_PATH", tree / "libmtpk.so")
    monkeypatch.setattr(__graft_entry__, "build", lambda: built.append("both"))
    monkeypatch.setattr(build_lib, "build_torch_calls", lambda: built.append("calls"), raising=False)
    __graft_entry__._ensure_built()
    (tree / "libmtpk.so").touch()
    __graft_entry__._ensure_built()
    (tree / "_mtpk_torch.so").touch()
    __graft_entry__._ensure_built()
    assert built == ["both", "calls"]
