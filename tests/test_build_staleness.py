"""The build is repeated when what it was made from changes: a source, or the torch that torch_calls.so is compiled against."""
import os

from dace_onnx_b200 import build


def files(tmp_path, monkeypatch):
    for name in ("LIB_PATH", "CALLS_PATH", "STAMP_PATH"):
        p = tmp_path / name
        p.write_text(build._torch_stamp() if name == "STAMP_PATH" else "")
        os.utime(p, (2 ** 33, 2 ** 33))   # newer than every source
        monkeypatch.setattr(build, name, str(p))


def test_up_to_date(tmp_path, monkeypatch):
    files(tmp_path, monkeypatch)
    assert not build._stale()


def test_another_torch(tmp_path, monkeypatch):
    files(tmp_path, monkeypatch)
    from importlib import metadata
    monkeypatch.setattr(metadata, "version", lambda name: "0.0")
    assert build._stale()


def test_missing_files_and_newer_sources(tmp_path, monkeypatch):
    for name in ("LIB_PATH", "CALLS_PATH", "STAMP_PATH"):
        files(tmp_path, monkeypatch)
        os.remove(getattr(build, name))
        assert build._stale()
    files(tmp_path, monkeypatch)
    os.utime(build.CALLS_PATH, (1, 1))
    assert build._stale()
