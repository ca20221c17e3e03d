"""The text operators' host module is theirs alone: the library loads without it, and they say what is missing."""
import subprocess
import sys

from conftest import ROOT

PROBE = """
import sys
sys.modules["siliconed_amd._text_bind"] = None  # an import of it fails, as one built for another torch does
import siliconed_amd as sq
lib = sq.abi.load()
assert lib.sq8_abi_version() == 1
assert lib.sq8_quantize_groups(None, None, 1, 0, 1, 1, None, 0, None, 0) == sq.abi.EINVAL
try:
    sq.abi.text
except ImportError as e:
    assert "build" in str(e)
else:
    raise AssertionError("no module, no refusal")
try:
    sq.abi.texts
except AttributeError:
    pass
else:
    raise AssertionError("an unknown name")
del sys.modules["siliconed_amd._text_bind"]
assert sq.abi.text.quantize_groups is sq.abi.text.quantize_groups
print("ok")
"""


def test_the_library_loads_without_the_host_module():
    r = subprocess.run([sys.executable, "-c", PROBE], cwd=ROOT, capture_output=True, text=True)
    assert r.returncode == 0 and r.stdout == "ok\n", r.stderr


def test_the_library_is_built_whatever_becomes_of_the_module(tmp_path, monkeypatch):
    import pytest
    from siliconed_amd import build

    def fails(incremental):
        raise RuntimeError("no compiler")

    monkeypatch.setattr(build, "_bind", fails)
    monkeypatch.setattr(build, "_compile", lambda item: None)
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    linked = []

    def link(cmd, **_):
        linked.append(cmd)
        open(cmd[-1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", link)
    with pytest.raises(RuntimeError, match="no compiler"):
        build.build()
    assert len(linked) == 1 and (tmp_path / "lib.so").exists()


def test_an_incremental_build_sees_another_torch(tmp_path, monkeypatch):
    import torch
    from siliconed_amd import build
    built = []

    def compiled(cmd, **_):
        built.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build, "BIND", str(tmp_path / "_text_bind.so"))
    monkeypatch.setattr(build, "OBJ", str(tmp_path))
    monkeypatch.setattr(build.subprocess, "run", compiled)
    build._bind(incremental=True)
    build._bind(incremental=True)
    assert len(built) == 1  # the second call: nothing has changed
    monkeypatch.setattr(torch, "__version__", "0.0.1+other")
    build._bind(incremental=True)
    assert len(built) == 2
    build._bind(incremental=True)
    assert len(built) == 2
    build._bind()
    assert len(built) == 3
