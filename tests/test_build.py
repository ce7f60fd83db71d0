"""The order of the build: the solver library needs neither torch nor the host extension's tools."""

import pytest

from kbench_b200 import _lib, build


def test_library_stands_without_the_host_extension(monkeypatch, capsys, tmp_path):
    done = []
    monkeypatch.setattr(build, "build_library", lambda verbose=False, force=False: done.append("library") or build.LIB)

    def fails(force=False):
        done.append("host")
        raise ImportError("No module named 'torch'")
    monkeypatch.setattr(build, "build_host", fails)
    assert build.build() == build.LIB and done == ["library", "host"]
    assert "torch" in capsys.readouterr().err


def test_extension_is_made_again_for_another_target(monkeypatch, tmp_path):
    """Another torch or Python, a newer source, or no record: what is there is neither kept nor left behind."""
    host = tmp_path / "_kb_host.so"
    monkeypatch.setattr(build, "HOST", host)
    monkeypatch.setattr(build, "REPO", tmp_path)
    monkeypatch.setenv("CXX", "false")  # the compiler that would be called: fails
    (tmp_path / "_build").mkdir()
    record = tmp_path / "_build" / "host_target.txt"
    host.write_bytes(b"")
    record.write_text(build.host_target())
    assert build.build_host() == host  # of this target and newer than its source
    record.write_text("another")
    with pytest.raises(RuntimeError):
        build.build_host()
    assert not host.exists()
    host.write_bytes(b"")
    record.unlink()
    with pytest.raises(RuntimeError):
        build.build_host()


def test_extension_of_another_target_is_not_used(monkeypatch):
    try:
        _lib.host()
    except RuntimeError:
        pytest.skip("_kb_host.so not built")
    monkeypatch.setattr(_lib, "_host", None)
    monkeypatch.setattr(build, "host_target", lambda: "another")
    with pytest.raises(RuntimeError, match="another"):
        _lib.host()
