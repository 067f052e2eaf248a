"""The native build: when an object is compiled again."""
import os

import pytest

from oap_mllib_amd import build


@pytest.fixture
def unit(tmp_path, monkeypatch):
    """One host unit with a header, compiled."""
    csrc, out = tmp_path / "csrc", tmp_path / "out"
    csrc.mkdir()
    out.mkdir()
    monkeypatch.setattr(build, "CSRC", csrc)
    monkeypatch.setattr(build, "BUILD", out)
    (csrc / "number.h").write_text("constexpr int kNumber = 7;\n")
    src = csrc / "number.cpp"
    src.write_text('#include "number.h"\nint number() { return kNumber; }\n')
    assert build._stale(src, False)
    build._compile(src, False)
    return src


def test_an_object_is_kept_while_nothing_changed(unit):
    assert not build._stale(unit, False)


def test_another_command_makes_an_object_stale(unit, monkeypatch):
    assert build._stale(unit, True)  # (debug)
    monkeypatch.setattr(build, "_common_flags", lambda debug: ["-O3", "-std=c++17", "-DOTHER"])
    assert build._stale(unit, False)
    build._compile(unit, False)
    assert not build._stale(unit, False)
    build._obj(unit).with_suffix(".cmd").unlink()  # (an object of unknown flags)
    assert build._stale(unit, False)


def test_device_flags_are_part_of_the_command(tmp_path, monkeypatch):
    monkeypatch.setattr(build, "CSRC", tmp_path)
    monkeypatch.setattr(build, "BUILD", tmp_path)
    src = tmp_path / "k.hip"
    src.write_text("")
    build._obj(src).write_text("")
    build._obj(src).with_suffix(".d").write_text(f"k.o: {src}\n")
    build._obj(src).with_suffix(".cmd").write_text("\n".join(build._command(src, False)))
    os.utime(src, (1, 1))
    assert not build._stale(src, False)
    monkeypatch.setattr(build, "NO_PACKED_FP32", [])
    assert build._stale(src, False)


def test_a_newer_header_or_source_makes_an_object_stale(unit):
    later = build._obj(unit).stat().st_mtime + 5
    os.utime(unit.parent / "number.h", (later, later))
    assert build._stale(unit, False)


def test_a_failed_compile_leaves_the_object_stale(unit):
    text = unit.read_text()
    unit.write_text(text + "#error no\n")
    with pytest.raises(RuntimeError):
        build._compile(unit, False)
    unit.write_text(text)
    os.utime(unit, (1, 1))
    assert build._stale(unit, False)
