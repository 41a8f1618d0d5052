"""The build without what only the autograd extension needs: the library is linked all the
same, and an extension that may not fit it is taken away."""

import os
import subprocess

import pytest

from gmmxx_amd import build as builder


@pytest.fixture
def place(tmp_path, monkeypatch):
    """A build into an empty folder in which compiling and linking only leave their files."""
    monkeypatch.setattr(builder, "BUILD_DIR", str(tmp_path / "_build"))
    monkeypatch.setattr(builder, "LIB_PATH", str(tmp_path / "libgmmxx_hip.so"))
    monkeypatch.setattr(builder, "AUTOGRAD_PATH", str(tmp_path / "_autograd.so"))
    monkeypatch.setattr(builder, "_hipcc", lambda: "hipcc")
    calls = []

    def run(cmd, **kwargs):
        calls.append(cmd)
        if "autograd.cpp" in " ".join(cmd) and "broken" in calls:
            return subprocess.CompletedProcess(cmd, 1, "", "error: broken")
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(builder.subprocess, "run", run)
    return tmp_path, calls


def without(monkeypatch, what):
    if what == "torch":
        import builtins
        plain = builtins.__import__

        def refuse(name, *args, **kwargs):
            if name == "torch" or name.startswith("torch."):
                raise ImportError("no torch")
            return plain(name, *args, **kwargs)
        monkeypatch.setattr(builtins, "__import__", refuse)
    elif what == "compiler":
        monkeypatch.setattr(builder.shutil, "which", lambda name: None)
    else:
        monkeypatch.setattr(builder.sysconfig, "get_paths", lambda: {"include": "/nowhere"})


@pytest.mark.parametrize("what", ["torch", "compiler", "headers"])
def test_library_without_the_extension(place, monkeypatch, what):
    folder, calls = place
    (folder / "_autograd.so").write_text("of another library")
    without(monkeypatch, what)
    with pytest.warns(RuntimeWarning, match="_autograd"):
        path = builder.build()
    assert path == str(folder / "libgmmxx_hip.so") and os.path.exists(path)
    assert not (folder / "_autograd.so").exists()


def test_extension_that_does_not_compile(place):
    """An error, but after the library is in its place."""
    folder, calls = place
    calls.append("broken")
    with pytest.raises(RuntimeError, match="autograd.cpp"):
        builder.build()
    assert (folder / "libgmmxx_hip.so").exists()


def test_both(place):
    folder, _ = place
    assert builder.build() == str(folder / "libgmmxx_hip.so")
    assert (folder / "_autograd.so").exists()
