"""Flags that every HIP source of the library is compiled with.  No GPU work."""
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
