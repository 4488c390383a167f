"""Flags that every HIP source of the library is compiled with.  No GPU work."""
import os

from facedetection_amd import _build


def test_packed_float32_arithmetic_is_off_in_every_source(monkeypatch, tmp_path):
    commands = []
    monkeypatch.setattr(_build.subprocess, "check_call", commands.append)
    monkeypatch.setattr(_build, "OBJ", str(tmp_path))
    _build.build(force=True, verbose=False)
    compiled = [c for c in commands if "-c" in c]
    assert len(compiled) == len(_build.SOURCES)
    for c in compiled:
        at = c.index("-packed-fp32-ops")
        assert c[at - 3:at] == ["-Xclang", "-target-feature", "-Xclang"]


def test_objects_of_other_flags_are_stale(monkeypatch, tmp_path):
    """Objects newer than every source and older than the file with the flags are compiled again."""
    commands = []
    monkeypatch.setattr(_build.subprocess, "check_call", commands.append)
    monkeypatch.setattr(_build, "OBJ", str(tmp_path))
    monkeypatch.setattr(_build, "_newer", lambda a, b: os.path.basename(a) == "_build.py")
    _build.build(force=False, verbose=False)
    assert len([c for c in commands if "-c" in c]) == len(_build.SOURCES)
