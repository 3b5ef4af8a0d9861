"""Calls straight from tensors (_tensors) without a GPU: what does not fit is left to the checks."""
import importlib

import pytest
import torch

COUNTS = dict(append=9, attention=10, load=5, fork=7, grow=7, compact=7, sample=9)


@pytest.fixture(scope="module")
def native(pkg):
    return importlib.import_module("artifex-assistantv5_amd._native")


@pytest.mark.parametrize("name", COUNTS)
def test_leaves_what_does_not_fit(native, name):
    f = getattr(native.direct(), name)
    t = torch.zeros(4, 4)
    for args in ((), (t,), (t,) * COUNTS[name], (None,) * COUNTS[name], (1,) * COUNTS[name],
                 ("x",) * COUNTS[name], (object(),) * COUNTS[name], (t,) * (COUNTS[name] + 1),
                 (torch.zeros(4, 4, device="meta"),) * COUNTS[name], (t.to_sparse(),) * COUNTS[name]):
        assert f(*args) is False


def test_binds_every_entry_point(native):
    assert len(native.PACKED) == len(COUNTS)
    with pytest.raises(TypeError, match="7 addresses"):
        native.direct().bind(1, 2)
    with pytest.raises(ValueError, match="null"):
        native.direct().bind(*[0] * 7)
    with pytest.raises(TypeError):
        native.direct().bind(*["x"] * 7)


def test_missing_module(native, monkeypatch, tmp_path):
    monkeypatch.setattr(native, "_tensors", None)
    monkeypatch.setattr(native, "load_library", lambda: None)
    monkeypatch.setattr(native, "LIB_PATH", str(tmp_path / "libgguf_hip.so"))
    with pytest.raises(RuntimeError, match="is not built"):
        native.direct()


def test_on_failure(native):
    for args in ((), (1,), (native.check, native.check)):
        with pytest.raises(TypeError, match="one callable"):
            native.direct().on_failure(*args)
    native.direct().on_failure(native.check)


def test_the_library_is_linked_where_the_module_cannot_be_built(pkg, monkeypatch, tmp_path):
    """A host with hipcc alone (no g++, no headers of Python's or torch's) still gets the C ABI."""
    build = importlib.import_module("artifex-assistantv5_amd.build")
    lib = tmp_path / "libgguf_hip.so"
    monkeypatch.setattr(build, "LIB", str(lib))
    monkeypatch.setattr(build, "BUILD", str(tmp_path / "_build"))
    monkeypatch.setattr(build, "hipcc", lambda: "hipcc")
    monkeypatch.setattr(build, "_compile", lambda src, verbose: str(tmp_path / src))

    def run(cmd, **kw):
        if cmd[0] == "g++":
            raise FileNotFoundError("g++")
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("linked")
        return build.subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    with pytest.raises(FileNotFoundError, match="g\\+\\+"):
        build.build()
    assert lib.read_text() == "linked"
